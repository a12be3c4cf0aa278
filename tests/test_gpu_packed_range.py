"""Packed attention where magnitudes differ: large scores, tokens far above their neighbours, values of
zero beside small ones, keys that hardly any row attends to, and what the row kernels take.

Against float64 with the bounds of test_gpu_packed.py (u = 2^-24, an operation counted at 2u), with two
differences: a score's error counts the products that are not zero, and a row's probabilities are off by
what the scores of the keys that it attends to are off by: a key of probability below 2^-100 takes no part,
and a row whose largest score stands out by more than 200 and both scores' errors is that key's alone,
p = 1, whatever the scores' rounding.

The kernels hold an operand to 2^-23 of it, which the counts above cover, or to 2^-33 of the largest magnitude
of its token and head, as the header says: 64 tokens are scaled so that their largest lies in [2^14, 2^15),
where half a step of the second fp16 term, at least 2^-25, is at most 2^-39 of it; and tokens that differ by more
than 2^6 are scaled each by itself. What that leaves of a value alone (a probability of 1 and a value of 1e-6
beside ones of 4) is part of the bound."""
import math

import numpy as np
import pytest

from test_gpu_packed import U2, _Call, _check

pytestmark = pytest.mark.gpu

NAMES = ("out", "dq", "dk", "dv")


def _held(x):
    """The largest magnitude of each row."""
    return abs(x).max(1, keepdims=True)


def _ref(call, settled=False):
    """{name: (value, bound)} of the call's out, dq, dk, dv. settled: for each row and head whether its
    largest score stands out; the other rows must have no gradient."""
    H, Hk, dh, T = call.H, call.Hk, call.dh, call.T
    q, k, v = (p[:T].astype(np.float64) for p in call.parts(call.x))
    g = call.g[:T, call.pad:].astype(np.float64)
    a, G, at = 1 / math.sqrt(dh), H // Hk, 0
    res = {n: (np.zeros(x.shape), np.zeros(x.shape)) for n, x in zip(NAMES, (q, q, k, v))}
    alone = np.zeros((T, H), bool)
    for n in call.lengths:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        mask = np.tril(np.ones((n, n), bool))
        for h in range(H):
            c, ck = slice(h * dh, h * dh + dh), slice(h // G * dh, h // G * dh + dh)
            Q, K, V, O = q[rows, c], k[rows, ck], v[rows, ck], g[rows, c]
            s = np.where(mask, Q @ K.T * a, -np.inf)
            terms = min((Q != 0).sum(1).max(), (K != 0).sum(1).max())
            e = U2 * (terms + 8) * a * np.where(mask, abs(Q) @ abs(K).T, 0)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            f = 2 * np.where(p > 2.0 ** -100, e, 0).max(1, keepdims=True) + U2 * (n + 8)
            top = s.argmax(1)
            lead = s.max(1) - e[np.arange(n), top]
            rest = s + e
            rest[np.arange(n), top] = -np.inf
            one = lead - rest.max(1) > 200
            alone[rows, h] = one
            f[one] = 0
            out = p @ V
            out_err = (p * f) @ abs(V) + U2 * (n + 8) * (p @ abs(V)) + 2.0 ** -33 * (p @ _held(V))
            r = O @ V.T
            D = (O * out).sum(1, keepdims=True)
            D_err = (abs(O) * out_err).sum(1, keepdims=True) + U2 * (dh + 8) * (abs(O) * abs(out)).sum(1, keepdims=True)
            ds = p * (r - D)
            ds_err = p * (f * abs(r - D) + U2 * (dh + 8) * (abs(O) @ abs(V).T) + D_err)
            for name, s_, x, err in (("out", c, out, out_err),
                                     ("dq", c, a * (ds @ K), a * (ds_err + U2 * (n + 8) * abs(ds)) @ abs(K)),
                                     ("dk", ck, a * (ds.T @ Q), a * (ds_err + U2 * (n * G + 8) * abs(ds)).T @ abs(Q)),
                                     ("dv", ck, p.T @ O, (p * (f + U2 * (n * G + 8))).T @ abs(O) + 2.0 ** -33 * (p.T @ _held(O)))):
                res[name][0][rows, s_] += x
                res[name][1][rows, s_] += err
    return (res, alone) if settled else res


def _run(call):
    call.upload()
    out = call.forward()[:call.T]
    d = call.backward(call.c.empty(call.x.shape))
    return dict(zip(NAMES, (out, *(p[:call.T] for p in call.parts(d)))))


def _within(got, ref, what, rows=slice(None)):
    """Every value within its bound."""
    x, err = (r[rows] for r in ref)
    d = abs(got[rows].astype(np.float64) - x)
    bad = ~(d <= err + 1e-37)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside their bounds, by up to " \
                          f"{np.nanmax(d / (err + 1e-300)):.2g}"


@pytest.mark.parametrize("dh", [64, 40, 128])
@pytest.mark.parametrize("size", [20, 300, 3e3, 1e5, 1e10, 1e14])
def test_large_scores_forward(hip_ctx, size, dh):
    """q and k times `size`: scores of 400 to 1e28. A row whose largest score stands out has that key's
    value, and a token that sees only itself its own."""
    call = _Call(hip_ctx, [1] * 40 + [2, 64, 65, 150], 4, 2, dh, np.random.default_rng(int(math.log2(size)) + dh))
    call.x[:, :call.wq + call.wk] *= np.float32(size)
    ref, alone = _ref(call, settled=True)
    assert alone[:40].all() and alone.mean() > (0.3 if size < 100 else 0.9)
    call.upload()
    out = call.forward().reshape(call.T, call.H, dh)
    x, err = (r.reshape(out.shape)[alone] for r in ref["out"])
    _within(out[alone], (x, err), "out")


@pytest.mark.parametrize("dh", [64, 40, 128])
@pytest.mark.parametrize("size", [20, 300, 3e3, 1e5, 1e10, 1e14])
def test_large_scores_backward(hip_ctx, size, dh):
    """The same rows' gradients: the output's gradient goes to the one key's value, and nothing but the
    rounding of r - D to queries and keys."""
    call = _Call(hip_ctx, [1] * 40 + [2, 64, 65, 150], 4, 2, dh, np.random.default_rng(int(math.log2(size)) + dh))
    call.x[:, :call.wq + call.wk] *= np.float32(size)
    alone = _ref(call, settled=True)[1]
    call.g *= np.repeat(alone, dh, axis=1)
    ref, got = _ref(call), _run(call)
    for name in ("dq", "dk", "dv"):
        x, err = ref[name]
        # a settled row's other probabilities are below e^-200, whatever float64 has of them
        _within(got[name], (x, err), name)


def test_large_scores_of_many_sequences_backward(hip_ctx):
    """20 thousand tokens that see only themselves, at every size of score: dv is the output's gradient."""
    rng, n, H, dh = np.random.default_rng(12), 20000, 2, 64
    call = _Call(hip_ctx, [1] * n, H, H, dh, rng)
    call.x[:, :2 * H * dh] *= (10.0 ** rng.uniform(-2, 14, (n, 1))).astype(np.float32)
    got = _run(call)
    x, v, g = call.x, call.parts(call.x)[2], call.g
    assert np.abs(got["out"] - v).max() <= 9 * U2 * np.abs(v).max()
    assert np.abs(got["dv"] - g).max() <= 9 * U2 * np.abs(g).max()
    # r - D: both sums of dh products of v and the gradient
    bound = 2 * U2 * (dh + 8) * (np.abs(g) * np.abs(v)).reshape(n, H, dh).sum(2) / math.sqrt(dh)
    for name, other in (("dq", x[:, H * dh:2 * H * dh]), ("dk", x[:, :H * dh])):
        assert (np.abs(got[name]).reshape(n, H, dh) <= bound[:, :, None] * np.abs(other).reshape(n, H, dh)).all(), name


@pytest.mark.parametrize("lengths", [[65], [200], [140] * 30])
@pytest.mark.parametrize("size", [1e-3, 1e-6, 1e-12])
def test_values_of_zero_beside_small_ones(hip_ctx, size, lengths):
    """A sequence of small values whose last token's is zero, alone in its tile of 64."""
    call = _Call(hip_ctx, lengths, 16, 4, 64, np.random.default_rng(21))
    v = call.parts(call.x)[2]
    v *= np.float32(size)
    ends = np.cumsum(lengths)
    v[ends - 1] = 0
    got, ref = _run(call), _ref(call)
    for name in NAMES:
        _check(got[name], ref[name], name)


@pytest.mark.parametrize("lengths", [[256], [900]])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e9, 1e15])
def test_a_value_far_above_the_others(hip_ctx, size, lengths):
    """A value that the rows behind it have no probability for: their gradients keep their accuracy."""
    call = _Call(hip_ctx, lengths, 4, 2, 64, np.random.default_rng(9))
    q, k, v = call.parts(call.x)
    q[:] = abs(q)
    k[100], v[100] = -200, size
    call.g[100] = 0  # its own row attends to keys before it with a value among them that only it has
    got, ref = _run(call), _ref(call)
    for name in NAMES:
        _check(got[name], ref[name], name)


@pytest.mark.parametrize("gap", [15, 30, 60])
@pytest.mark.parametrize("lengths", [[200], [140] * 30])
def test_keys_with_hardly_any_probability(hip_ctx, gap, lengths):
    """A key with 2^-gap of the others' probability in every row, its value 2^gap times theirs: half of the
    output, and of the sums in dq; and what it gets of the gradients, 2^-gap of theirs, to the same relative
    accuracy, less what a score's own roundings (its scale's, its own, the difference's: half a step of gap
    each) leave of its probability."""
    norm = 2e-6 + 3 * gap * math.log(2) * U2 / 2
    call = _Call(hip_ctx, lengths, 16, 4, 64, np.random.default_rng(gap))
    q, k, v = call.parts(call.x)
    q[:], k[:] = 0, 0
    # one product a score: q k / 8, in base 2
    q[:, ::64] = 8
    k[:, ::64] = np.random.default_rng(3).uniform(-1, 1, (call.T, 4))
    starts = np.cumsum(lengths) - lengths
    k[starts + 70, ::64] = -np.float32(gap * math.log(2))
    v[starts + 70] *= np.float32(2.0 ** gap)
    got, ref = _run(call), _ref(call)
    for name in NAMES:
        _check(got[name], ref[name], name, norm)
        if name in ("dk", "dv"):
            rows = starts + 70
            _check(got[name][rows], tuple(r[rows] for r in ref[name]), f"{name} of those keys", norm)


def _all_but(call, ref, got, rows, what):
    """Every row of the outputs but the named ones."""
    keep = np.ones(call.T, bool)
    keep[rows] = False
    for name in NAMES:
        _check(got[name][keep], tuple(r[keep] for r in ref[name]), f"{what}: {name}")


@pytest.mark.parametrize("lengths", [[64], [500], [150] * 30])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 1e12, 1e14])
def test_later_tokens_far_above(hip_ctx, size, lengths):
    """A last query, key and value far above the others', which no earlier row attends to: the earlier rows
    and what they pass on are as accurate as without it."""
    call = _Call(hip_ctx, lengths, 16, 4, 64, np.random.default_rng(22))
    last = np.cumsum(lengths) - 1
    for x in call.parts(call.x):
        x[last] *= np.float32(size)
    call.g[last] = 0  # what its own row passes on has another scale
    _all_but(call, _ref(call), _run(call), last, "last")


@pytest.mark.parametrize("lengths", [[64], [500], [150] * 30])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e8, 1e12])
def test_early_tokens_far_above(hip_ctx, size, lengths):
    """A first output's gradient far above the others', which reaches the first key and value only; and a
    second token whose key no later row attends to (their scores for it are far below) and whose value is
    as far above the others'."""
    call = _Call(hip_ctx, lengths, 16, 4, 64, np.random.default_rng(23))
    q, k, v = call.parts(call.x)
    first = np.cumsum(lengths) - lengths
    call.g[first] *= np.float32(size)
    q[:] = abs(q)
    k[first + 1] = -abs(k[first + 1]) * np.float32(size) - 100
    v[first + 1] *= np.float32(size)
    call.g[first + 1] = 0
    _all_but(call, _ref(call), _run(call), np.concatenate([first, first + 1]), "first")


@pytest.mark.parametrize("part", ["q", "k", "v", "g"])
@pytest.mark.parametrize("power", [-100, -75, -30, -13, 13, 30, 59, 75])
def test_tokens_of_every_size(hip_ctx, power, part):
    """One operand's tokens spread over 2^|power|, the scores kept ordinary by the others. (Queries and keys of
    2^75 are the row kernels'.)"""
    call = _Call(hip_ctx, [64, 300, 33], 4, 2, 40, np.random.default_rng(power + 200))
    rng = np.random.default_rng(5)
    x = dict(zip("qkv", call.parts(call.x)), g=call.g)
    spread = (2.0 ** (power * rng.random((call.T, 1)))).astype(np.float32)
    x[part][:] *= spread
    if part in "qk":
        # so that the largest meets ordinary scores
        x["k" if part == "q" else "q"][:] *= np.float32(2.0 ** min(0, -power))
    got, ref = _run(call), _ref(call)
    for name in NAMES:
        _within(got[name], ref[name], name)


@pytest.mark.parametrize("lengths", [[90, 200], [140] * 30])
def test_small_gradients(hip_ctx, lengths):
    """Gradients of 2^-105, well inside fp32's normal range as their results are."""
    call = _Call(hip_ctx, lengths, 16, 4, 64, np.random.default_rng(24))
    call.g *= np.float32(2.0 ** -105)
    got, ref = _run(call), _ref(call)
    for name in NAMES:
        _check(got[name], ref[name], name)


@pytest.mark.parametrize("dh", [24, 128])
def test_a_row_whose_first_scores_are_minus_infinity(hip_ctx, dh):
    """The first 64 keys score -inf (an infinite column, or products past fp32): the rows behind attend to
    the others alone, the rows before have no softmax."""
    for kind in ("infinite", "past fp32"):
        call = _Call(hip_ctx, [200], 2, 1, dh, np.random.default_rng(31))
        q, k, v = call.parts(call.x)
        q[:, 0], q[:, dh] = abs(q[:, 0]) + 1, abs(q[:, dh]) + 1
        k[:, 0] = 0
        k[:70, 0] = -np.inf
        if kind == "past fp32":
            q[:, 0] = q[:, dh] = 2e19
            k[:70, 0] = -3e19
        call.g[:70] = 0
        got = _run(call)
        # the same with the first 70 tokens' keys far below instead
        call.x = call.x.copy()
        q, k, v = call.parts(call.x)
        q[:, 0] = q[:, dh] = 1
        k[:70, 0] = -1e4
        ref = _ref(call)
        assert np.isnan(got["out"][:70]).all(), kind
        _check(got["out"][70:], tuple(r[70:] for r in ref["out"]), f"{kind}: out")
        if kind == "infinite":
            continue  # its dq has 0 times infinity in it
        for name in ("dq", "dk", "dv"):
            # dk's first column has the queries' 2e19 in it
            cols = slice(1, None) if name == "dk" else slice(None)
            _check(got[name][70:, cols], tuple(r[70:, cols] for r in ref[name]), f"{kind}: {name}")


@pytest.mark.parametrize("lengths,H,Hk", [([200, 65], 4, 2), ([140] * 30, 16, 4), ([129] * 150, 12, 4), ([33], 3, 1)])
def test_the_row_kernels(hip_ctx, lengths, H, Hk):
    """Finite values past what the tiles take, with ordinary results, so that whole sequences go to the row
    kernels: in blocks of 64 and of 128 rows, a group's heads apart and together, written and added."""
    call = _Call(hip_ctx, lengths, H, Hk, 32, np.random.default_rng(len(lengths)), pad=1)
    q, k, v = call.parts(call.x)
    q *= np.float32(2.0 ** 55)
    k *= np.float32(2.0 ** -55)
    ref = _ref(call)
    call.upload()
    T = call.T
    _check(call.forward()[:T], ref["out"], "out")
    prev = np.random.default_rng(1).standard_normal(call.x.shape).astype(np.float32)
    # as large as what is added to it
    for p, s in zip(call.parts(prev), (2.0 ** -55, 2.0 ** 55, 1)):
        p *= np.float32(s)
    for acc in (0, 1):
        got = call.backward(hip_ctx.to_device(prev), acc=acc)
        for name, part, old in zip(NAMES[1:], call.parts(got), call.parts(prev)):
            x, err = ref[name]
            if acc:
                x, err = x + old[:T], err + U2 * abs(x + old[:T])
            _check(part[:T], (x, err), f"{name}, {acc}")


# blocks of 64 and of 128 rows; a group's heads apart and together
BLOCKS = [([300, 33], 4, 2), ([150] * 30, 16, 4), ([260] * 50, 16, 4)]


@pytest.mark.parametrize("lengths,H,Hk", BLOCKS)
@pytest.mark.parametrize("dh", [8, 32, 72, 128])
def test_large_scores_of_every_head_size(hip_ctx, dh, lengths, H, Hk):
    """Scores of about 1e9 in every form of the kernels, forward and backward."""
    call = _Call(hip_ctx, lengths, H, Hk, dh, np.random.default_rng(dh), pad=1)
    call.x[:, :call.pad + call.wq + call.wk] *= np.float32(3e4)
    alone = _ref(call, settled=True)[1]
    assert alone.mean() > 0.9
    call.g[:, call.pad:] *= np.repeat(alone, dh, axis=1)
    ref, got = _ref(call), _run(call)
    keep = np.repeat(alone, dh, axis=1)
    x, err = (r[keep] for r in ref["out"])
    _within(got["out"][keep], (x, err), "out")
    for name in NAMES[1:]:
        _within(got[name], ref[name], name)


@pytest.mark.parametrize("lengths,H,Hk", BLOCKS)
@pytest.mark.parametrize("dh", [8, 32, 72, 128])
def test_mixed_tiles_of_every_head_size(hip_ctx, dh, lengths, H, Hk):
    """Last tokens of 1e6 times the others', first gradients as large, and tokens in between of 1e-4, in every
    form of the kernels."""
    call = _Call(hip_ctx, lengths, H, Hk, dh, np.random.default_rng(dh + 1), pad=1)
    ends = np.cumsum(lengths)
    last, first = ends - 1, ends - np.array(lengths)
    for x in call.parts(call.x):
        x[last] *= np.float32(1e6)
        x[first + 20] *= np.float32(1e-4)
    call.g[last] = 0
    call.g[first] *= np.float32(1e6)
    _all_but(call, _ref(call), _run(call), np.concatenate([first, last]), "mixed")


@pytest.mark.parametrize("part,low,high", [("q", -110, 40), ("k", -110, 40), ("v", -75, 75), ("g", -75, 75), ("v", -110, 0)])
def test_tokens_of_more_than_the_tiles_range(hip_ctx, part, low, high):
    """One operand's tokens spread over 2^150, which the row kernels take, and over 2^110, which the tiles do."""
    call = _Call(hip_ctx, [64, 150, 33], 4, 2, 40, np.random.default_rng(77))
    x = dict(zip("qkv", call.parts(call.x)), g=call.g)
    size = np.random.default_rng(6).uniform(low, high, (call.T, 1))
    size[::7], size[1::7] = low, high  # both in every tile
    x[part][:] *= (2.0 ** size).astype(np.float32)
    if part in "qk":
        x["k" if part == "q" else "q"][:] *= np.float32(2.0 ** -high)
    got, ref = _run(call), _ref(call)
    for name in NAMES:
        _within(got[name], ref[name], name)
