"""Causal attention over packed sequences against float64.

Tolerances.  Let u = 2^-24 be half a step of fp32, and count an operation at 2u, which covers sums
that are cut off instead of rounded.  A score of n products is off by at most e_ij = 2u (dh + 8)
sum |q k| / sqrt(dh) (dh + 8: its products, their sum, the scale, the reference's subtraction and
the exponential's own step), so a probability by the factor 1 + f_i with f_i = 2 max_j e_ij + 2u (L
+ 8), the second part from the row sum over L tokens.  From there each bound adds up the terms'
magnitudes (`_ref`).  These bounds are of the worst case, where every rounding has one sign, and
far above what is met; so the 2-norm of each error is held to 2e-6 of the result's besides, twice
what fp32 sums of a few hundred terms come to."""
import ctypes
import math

import numpy as np
import pytest

import numrs_amd as nr
from conftest import assert_bits, rand
from numrs_amd import _lib as L
from numrs_amd import nn

pytestmark = pytest.mark.gpu

U2 = 2.0 ** -23


def _ref(q, k, v, g, lengths, H, Hk):
    """out, dq, dk, dv in float64 and the bounds of their errors, rows and heads as in q and k."""
    dh, G = q.shape[1] // H, H // Hk
    a = 1 / math.sqrt(dh)
    res = {n: (np.zeros(x.shape), np.zeros(x.shape)) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    at = 0
    for n in lengths:
        rows = slice(at, at + n)
        at += n
        mask = np.tril(np.ones((n, n), bool))
        for h in range(H):
            c, ck = slice(h * dh, h * dh + dh), slice(h // G * dh, h // G * dh + dh)
            Q, K, V, O = (x[rows, s].astype(np.float64) for x, s in ((q, c), (k, ck), (v, ck), (g, c)))
            s = np.where(mask, Q @ K.T * a, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True)) if n else s
            p /= p.sum(1, keepdims=True) if n else 1
            e = U2 * (dh + 8) * a * np.where(mask, abs(Q) @ abs(K).T, 0)
            f = (2 * e.max(1, keepdims=True) if n else 0) + U2 * (n + 8)
            out = p @ V
            out_err = (p * f) @ abs(V) + U2 * (n + 8) * (p @ abs(V))
            r = O @ V.T
            D = (O * out).sum(1, keepdims=True)
            D_err = (abs(O) * out_err).sum(1, keepdims=True) + U2 * (dh + 8) * (abs(O) * abs(out)).sum(1, keepdims=True)
            ds = p * (r - D)
            ds_err = p * (f * abs(r - D) + U2 * (dh + 8) * (abs(O) @ abs(V).T) + D_err)
            for name, s_, x, err in (("out", c, out, out_err),
                                     ("dq", c, a * (ds @ K), a * (ds_err + U2 * (n + 8) * abs(ds)) @ abs(K)),
                                     ("dk", ck, a * (ds.T @ Q), a * (ds_err + U2 * (n * G + 8) * abs(ds)).T @ abs(Q)),
                                     ("dv", ck, p.T @ O, (p * (f + U2 * (n * G + 8))).T @ abs(O))):
                res[name][0][rows, s_] += x
                res[name][1][rows, s_] += err
    return res


def _check(got, ref, what, norm=2e-6):
    x, err = ref
    d = abs(got.astype(np.float64) - x)
    bad = ~(d <= err + 1e-37)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside their bounds, by up to " \
                          f"{(d / (err + 1e-300)).max():.2g}"
    # A token that sees only itself has p = 1 and r = D, so its dq and dk are 0 and what is computed is
    # the rounding of r - D alone: no share of the result, and inside the bounds above.
    if np.linalg.norm(x) > np.linalg.norm(err):
        rel = np.linalg.norm(d) / max(np.linalg.norm(x), 1e-300)
        assert rel <= norm, f"{what}: 2-norm error {rel:.2g}"


class _Call:
    """One packed call on column blocks of a projection, with `pad` more columns before them, and
    `extra` rows behind the last sequence."""

    def __init__(self, c, lengths, H, Hk, dh, rng, pad=0, extra=0):
        self.c, self.lengths, self.H, self.Hk, self.dh = c, lengths, H, Hk, dh
        self.T, self.pad, self.wq, self.wk = sum(lengths), pad, H * dh, Hk * dh
        self.rows, self.ld = self.T + extra, pad + self.wq + 2 * self.wk
        self.x = rand(rng, (self.rows, self.ld))
        self.g = rand(rng, (self.rows, self.wq + pad))
        self.seqs = nr.PackedSequences(lengths, ctx=c)

    def parts(self, x):
        p = self.pad
        return (x[:, p:p + self.wq], x[:, p + self.wq:p + self.wq + self.wk], x[:, p + self.wq + self.wk:])

    def upload(self):
        c, at = self.c, lambda a, o: a.ptr + 4 * o
        self.xd, self.gd = c.to_device(self.x), c.to_device(self.g)
        self.out = c.to_device(np.full(self.g.shape, 7, np.float32))
        self.stats = c.empty((max(self.rows, 1), self.H, 2))
        self.ptrs = [at(self.xd, o) for o in (self.pad, self.pad + self.wq, self.pad + self.wq + self.wk)]
        return self

    def forward(self, stats=True):
        q, k, v = self.ptrs
        self.c._check(L.load().numrs_hip_attention_packed_forward(
            self.c.handle, self.seqs.handle, q, self.ld, k, v, self.ld, self.out.ptr + 4 * self.pad,
            self.wq + self.pad, self.stats.ptr if stats else None, self.H, self.Hk, self.dh))
        return self.out.numpy()[:, self.pad:]

    def backward(self, d, keep=(1, 1, 1), acc=0):
        """d: the gradients' array, laid out as x."""
        q, k, v = self.ptrs
        to = [d.ptr + 4 * o if w else None
              for w, o in zip(keep, (self.pad, self.pad + self.wq, self.pad + self.wq + self.wk))]
        self.c._check(L.load().numrs_hip_attention_packed_backward(
            self.c.handle, self.seqs.handle, q, self.ld, k, v, self.ld, self.out.ptr + 4 * self.pad,
            self.gd.ptr + 4 * self.pad, self.wq + self.pad, self.stats.ptr, *to, self.H, self.Hk, self.dh, acc))
        return d.numpy()

    def ref(self):
        T = self.T
        return _ref(*(p[:T] for p in self.parts(self.x)), self.g[:T, self.pad:], self.lengths, self.H, self.Hk)


# One token, empty sequences, one short of and past 32, 64, 128 and 256, heads of every padded size,
# groups of 1 to 16, many sequences of which few are long.
SHAPES = [([1], 1, 1, 8), ([3, 0, 5, 0], 2, 1, 16), ([64], 8, 8, 64), ([65, 63, 1, 33], 4, 2, 40),
          ([127, 129], 6, 3, 80), ([300, 1, 257], 8, 2, 128), ([513], 5, 1, 96), ([200, 31], 4, 4, 72),
          ([777], 3, 1, 64), ([255, 256], 2, 2, 32), ([1, 2, 3, 4, 5, 6, 7] * 5, 16, 1, 24),
          ([640], 16, 4, 64), ([400, 1, 1, 90], 2, 1, 104), ([1100, 60], 4, 2, 128),
          # enough blocks of 128 rows for two a CU, of each padded size; and enough blocks of key rows
          # that a workgroup takes all heads of a group
          ([140] * 20, 16, 4, 64), ([260] * 8, 24, 8, 128), ([131] * 18, 16, 16, 96), ([100, 300] * 9, 16, 8, 32),
          ([5, 33] * 150, 16, 4, 24)]


@pytest.mark.parametrize("lengths,H,Hk,dh", SHAPES)
def test_forward_backward(hip_ctx, lengths, H, Hk, dh):
    print(f"[gpu] packed {lengths} H={H} Hk={Hk} dh={dh}", flush=True)
    rng = np.random.default_rng(sum(lengths) * 31 + dh)
    # odd offsets and strides: no row lies on 16 bytes; rows behind the last sequence stay
    call = _Call(hip_ctx, lengths, H, Hk, dh, rng, pad=dh % 3 + 1, extra=3).upload()
    T, pad, ref = call.T, call.pad, call.ref()
    out = call.forward()
    _check(out[:T], ref["out"], "out")
    assert (out[T:] == 7).all() and (call.out.numpy()[:, :pad] == 7).all()
    prev = rand(rng, call.x.shape)
    for what, keep, acc in (("all", (1, 1, 1), 0), ("added", (1, 1, 1), 1), ("dq", (1, 0, 0), 0),
                            ("dk", (0, 1, 0), 1), ("dv", (0, 0, 1), 0)):
        got = call.backward(hip_ctx.to_device(prev), keep, acc)
        assert_bits(got[:, :pad], prev[:, :pad], f"{what}: columns beside")
        assert_bits(got[T:], prev[T:], f"{what}: rows behind")
        for name, part, old, w in zip(("dq", "dk", "dv"), call.parts(got), call.parts(prev), keep):
            if not w:
                assert_bits(part, old, f"{what}: {name} touched")
                continue
            x, err = ref[name]
            if acc:
                x, err = x + old[:T], err + U2 * abs(x + old[:T])
            _check(part[:T], (x, err), f"{what}: {name}")


def test_forward_without_statistics_gives_the_same(hip_ctx):
    call = _Call(hip_ctx, [70, 200], 4, 2, 64, np.random.default_rng(1)).upload()
    a = call.forward()
    assert_bits(call.forward(stats=False), a)


def test_rows_past_32_bits(hip_ctx):
    """Rows 2^30 + 8 elements apart: the fourth lies past 2^31 elements and 2^33 bytes."""
    c, rng, lib, H, Hk, dh, n, ld = hip_ctx, np.random.default_rng(17), L.load(), 2, 1, 32, 4, 2**30 + 8
    near = _Call(c, [n], H, Hk, dh, rng).upload()
    out, d = near.forward(), near.backward(c.empty(near.x.shape))
    w, wq = near.ld, near.wq
    far = [c.empty(((n - 1) * ld + w,)) for _ in range(2)]  # q, k, v, out, dout; dq, dk, dv
    x, dx = far[0].ptr, far[1].ptr
    for i in range(n):
        far[0].view(i * ld, (w,)).upload(near.x[i])
    o = c.empty(((n - 1) * ld + 2 * wq,))
    for i in range(n):
        o.view(i * ld + wq, (wq,)).upload(near.g[i])
    stats = c.empty((n, H, 2))
    c._check(lib.numrs_hip_attention_packed_forward(c.handle, near.seqs.handle, x, ld, x + 4 * wq, x + 4 * (wq + dh),
                                                    ld, o.ptr, ld, stats.ptr, H, Hk, dh))
    c._check(lib.numrs_hip_attention_packed_backward(
        c.handle, near.seqs.handle, x, ld, x + 4 * wq, x + 4 * (wq + dh), ld, o.ptr, o.ptr + 4 * wq, ld, stats.ptr,
        dx, dx + 4 * wq, dx + 4 * (wq + dh), H, Hk, dh, 0))
    for i in range(n):
        assert_bits(o.view(i * ld, (wq,)).numpy(), out[i])
        assert_bits(far[1].view(i * ld, (w,)).numpy(), d[i])


def test_the_same_call_gives_the_same_bits(hip_ctx):
    call = _Call(hip_ctx, [300, 17, 520], 8, 2, 64, np.random.default_rng(2)).upload()
    d = hip_ctx.empty(call.x.shape)
    first = call.forward(), call.backward(d)
    for _ in range(3):
        assert_bits(call.forward(), first[0])
        assert_bits(call.backward(d), first[1])


@pytest.mark.parametrize("dh", [64, 128])
def test_values_that_no_row_attends_to(hip_ctx, dh):
    """NaN and infinities in a later token and in another sequence: earlier rows and other
    sequences come out to the bit as without them; rows that attend to them have what fp32
    arithmetic makes of them."""
    rng = np.random.default_rng(dh)
    lengths, H, Hk = [200, 150], 4, 2
    call = _Call(hip_ctx, lengths, H, Hk, dh, rng)
    clean = _Call(hip_ctx, lengths, H, Hk, dh, rng)
    clean.x, clean.g = call.x.copy(), call.g.copy()
    at = 77  # in the first sequence
    q, k, v = call.parts(call.x)
    k[at, 0], v[at, dh + 1] = np.nan, np.inf   # kv head 0's key, kv head 1's value
    call.upload(), clean.upload()
    a, b = call.forward(), clean.forward()
    assert np.array_equal(a[200:], b[200:])
    # the same values up to rounding: the rows' tiles may be computed another way
    assert np.abs(a[:at] - b[:at]).max() <= 1e-5
    assert np.isnan(a[at:200, :2 * dh]).all()          # query heads 0 and 1
    assert np.isposinf(a[at:200, 2 * dh + 1]).all() and np.isposinf(a[at:200, 3 * dh + 1]).all()
    rest = np.ones(4 * dh, bool)
    rest[:2 * dh] = rest[2 * dh + 1] = rest[3 * dh + 1] = False
    assert np.abs(a[at:200, rest] - b[at:200, rest]).max() <= 1e-5
    d, e = (x.backward(hip_ctx.empty(x.x.shape)) for x in (call, clean))
    assert np.array_equal(d[200:], e[200:])
    dq, eq = call.parts(d)[0], call.parts(e)[0]
    assert np.abs(dq[:at] - eq[:at]).max() <= 1e-4
    assert np.isnan(dq[at:200, :2 * dh]).all()
    # a non-finite output gradient at one row reaches the keys up to it and no later ones
    call = _Call(hip_ctx, lengths, H, Hk, dh, rng)
    call.x, call.g = clean.x.copy(), clean.g.copy()
    call.g[at, 5] = np.inf
    call.upload()
    call.forward()
    d = call.backward(hip_ctx.empty(call.x.shape))
    assert np.array_equal(d[200:], e[200:])
    for x, y in zip(call.parts(d)[1:], clean.parts(e)[1:]):
        assert np.abs(x[at + 1:200] - y[at + 1:200]).max() <= 1e-4
        assert not np.isfinite(x[:at + 1, :dh]).all()
    assert np.abs(call.parts(d)[0][:at] - clean.parts(e)[0][:at]).max() <= 1e-4


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
def test_values_that_no_row_attends_to_among_many(hip_ctx, dh):
    """The same where there are two blocks of 128 rows and more for each CU: a sequence of ordinary values
    among others gives the same bits whatever those hold, earlier rows the same values."""
    # 3 blocks each; of 90 also enough key rows that a workgroup takes all heads of a group
    lengths, H, Hk = [300] * (90 if dh == 32 else 15), 12, 4
    call, clean = (_Call(hip_ctx, lengths, H, Hk, dh, np.random.default_rng(dh)) for _ in range(2))
    bad = 300 * 7 + 150
    q, k, v = call.parts(call.x)
    k[bad, 0], v[bad, dh + 1] = np.nan, np.inf
    call.g[bad, 2 * (H // Hk) * dh] = np.inf  # kv head 2's first query head
    q[bad, -1] = 1e20  # the last query head: finite, and past what the tiles take
    call.upload(), clean.upload()
    a, b = call.forward(), clean.forward()
    d, e = (x.backward(hip_ctx.empty(x.x.shape)) for x in (call, clean))
    inside = slice(300 * 7, 300 * 8)
    for x, y in ((a, b), (d, e)):
        others = np.ones(len(x), bool)
        others[inside] = False
        assert_bits(x[others], y[others])
    assert np.abs(a[300 * 7:bad] - b[300 * 7:bad]).max() <= 1e-5
    assert np.isnan(a[bad:300 * 8, :(H // Hk) * dh]).all()
    dq, dk, dv = call.parts(d)
    eq, ek, ev = clean.parts(e)
    assert np.abs(dq[300 * 7:bad] - eq[300 * 7:bad]).max() <= 1e-4
    for x, y in ((dk, ek), (dv, ev)):
        x, y = x[inside], y[inside]
        assert np.isnan(x[:151, :dh]).any() and not np.isfinite(x[:151, 2 * dh:3 * dh]).all()
        # kv head 2's keys behind the row, which no such gradient reaches
        assert np.abs(x[151:, 2 * dh:3 * dh] - y[151:, 2 * dh:3 * dh]).max() <= 1e-4


@pytest.mark.parametrize("sq,sk,sv,sg", [(1e-18, 1e18, 1, 1), (1e15, 1e-15, 1e-30, 1e20), (1, 1, 1e30, 1e-30),
                                         (1, 1, 1e-37, 1), (1e-3, 1e-3, 1e-3, 1e-3), (0, 1, 1, 1), (1, 1, 0, 0)])
def test_magnitudes(hip_ctx, sq, sk, sv, sg):
    """Operands of very large and small magnitude whose results are ordinary fp32 values."""
    call = _Call(hip_ctx, [130, 66], 4, 2, 64, np.random.default_rng(8))
    for x, s in zip(call.parts(call.x), (sq, sk, sv)):
        x *= np.float32(s)
    call.g *= np.float32(sg)
    call.upload()
    ref = call.ref()
    _check(call.forward(), ref["out"], "out")
    d = call.backward(hip_ctx.empty(call.x.shape))
    for name, part in zip(("dq", "dk", "dv"), call.parts(d)):
        if sv == 1e-37 and name != "dv":
            continue  # below fp32's normal range
        _check(part, ref[name], name)


def test_one_token_far_above_the_others(hip_ctx):
    """A key and a value 1e4 times the others': the rows that do not see them, and those whose
    probability for it is nearly 0, keep their accuracy."""
    call = _Call(hip_ctx, [256], 2, 1, 64, np.random.default_rng(9))
    q, k, v = call.parts(call.x)
    q[:] = abs(q)
    k[100] = -1e4
    v[100] = 1e4
    call.upload()
    ref = call.ref()
    _check(call.forward(), ref["out"], "out")


def test_a_recorded_step_replays(hip_ctx):
    """Forward and backward in a graph, replayed on new data with eager calls in between."""
    c, rng = hip_ctx, np.random.default_rng(3)
    call = _Call(c, [190, 3, 65], 4, 2, 64, rng).upload()
    d = c.empty(call.x.shape)
    q, k, v = call.ptrs

    def step():
        lib, s, wq = L.load(), call.seqs.handle, call.wq
        c._check(lib.numrs_hip_attention_packed_forward(c.handle, s, q, call.ld, k, v, call.ld, call.out.ptr,
                                                        wq, call.stats.ptr, 4, 2, 64))
        c._check(lib.numrs_hip_attention_packed_backward(
            c.handle, s, q, call.ld, k, v, call.ld, call.out.ptr, call.gd.ptr, wq, call.stats.ptr, d.ptr,
            d.ptr + 4 * wq, d.ptr + 4 * (wq + call.wk), 4, 2, 64, 0))

    step()
    graph, second = nr.StepGraph(c, step), nr.StepGraph(c, step)
    other = _Call(c, [300, 40], 4, 2, 64, rng).upload()
    for i in range(4):
        x = rand(rng, call.x.shape)
        call.xd.upload(x)
        step()
        want = call.out.numpy(), d.numpy()
        d.fill(0)
        other.forward(), other.backward(c.empty(other.x.shape))
        (graph if i % 2 else second).replay()
        assert_bits(call.out.numpy(), want[0])
        assert_bits(d.numpy(), want[1])
    graph.close(), second.close()


def test_a_graph_keeps_its_sequences(hip_ctx):
    """A recorded step is replayed after the handle is gone and others have taken its memory."""
    c, rng = hip_ctx, np.random.default_rng(13)
    call = _Call(c, [190, 3, 65], 4, 2, 64, rng).upload()
    q, k, v = call.ptrs
    d = c.empty(call.x.shape)
    cache = nr.KVCache(20, 16, 2, 64, "int8", ctx=c)
    table = c.to_device(np.arange(60, dtype=np.int32).reshape(3, 20) % 20)
    ends = c.to_device(np.array([190, 3, 65], np.int32))
    ko, vo = c.empty((258, 128)), c.empty((258, 128))

    def step():
        lib, s, wq = L.load(), call.seqs.handle, call.wq
        c._check(lib.numrs_hip_attention_packed_forward(c.handle, s, q, call.ld, k, v, call.ld, call.out.ptr,
                                                        wq, call.stats.ptr, 4, 2, 64))
        c._check(lib.numrs_hip_attention_packed_backward(
            c.handle, s, q, call.ld, k, v, call.ld, call.out.ptr, call.gd.ptr, wq, call.stats.ptr, d.ptr,
            d.ptr + 4 * wq, d.ptr + 4 * (wq + call.wk), 4, 2, 64, 0))
        p = ctypes.byref(cache.pages)
        c._check(lib.numrs_hip_kv_cache_read(c.handle, p, s, ko.ptr, vo.ptr, 128, table.ptr, 20, ends.ptr))

    for a in (cache.k, cache.v):
        a.upload(rng.integers(1, 256, a.shape, dtype=np.uint8))
    cache.k_scale.fill(0.5), cache.v_scale.fill(0.25)
    step()
    want = [a.numpy() for a in (call.out, d, ko, vo)]
    graph = nr.StepGraph(c, step)
    call.seqs.close()
    # as many lists of the same size, of sequences that would lead elsewhere
    others = [nr.PackedSequences([3, 65, 190], ctx=c) for _ in range(4)]
    for a in (call.out, d, ko, vo):
        a.fill(0)
    for _ in range(2):
        graph.replay()
        for a, w in zip((call.out, d, ko, vo), want):
            assert_bits(a.numpy(), w)
    graph.close()
    assert all(len(o) == 3 for o in others)


def test_two_contexts_and_a_stream_each():
    """Two contexts (a stream each) at once give what each gives alone."""
    rng = np.random.default_rng(4)
    with nr.Context(0) as a, nr.Context(0) as b:
        calls = [_Call(c, [500, 77], 8, 2, 64, rng).upload() for c in (a, b)]
        ds = [c.c.empty(c.x.shape) for c in calls]
        want = [(c.forward(), c.backward(d)) for c, d in zip(calls, ds)]
        lib = L.load()
        for _ in range(3):
            for c in calls:  # queued on both streams before either is read
                q, k, v = c.ptrs
                assert lib.numrs_hip_attention_packed_forward(c.c.handle, c.seqs.handle, q, c.ld, k, v, c.ld,
                                                              c.out.ptr, c.wq, c.stats.ptr, 8, 2, 64) == 0
            for c, d, (out, dx) in zip(calls, ds, want):
                assert_bits(c.backward(d), dx)
                assert_bits(c.out.numpy(), out)
        with pytest.raises(nr.HipError, match="another context"):
            calls[0].seqs, calls[1].seqs = calls[1].seqs, calls[0].seqs
            calls[0].forward()
        del calls, ds, c, d


def test_refusals(hip_ctx):
    c, lib = hip_ctx, L.load()
    call = _Call(c, [8], 4, 2, 16, np.random.default_rng(0)).upload()
    q, k, v = call.ptrs
    h, s, ld, out = c.handle, call.seqs.handle, call.ld, call.out.ptr
    fwd = lib.numrs_hip_attention_packed_forward
    good = [h, s, q, ld, k, v, ld, out, 64, None, 4, 2, 16]
    assert fwd(*good) == 0
    for i, value, code in ((1, None, L.E_INVALID), (2, None, L.E_INVALID), (4, None, L.E_INVALID),
                           (5, None, L.E_INVALID), (7, None, L.E_INVALID), (3, 63, L.E_SHAPE),
                           (6, 31, L.E_SHAPE), (8, 63, L.E_SHAPE), (3, 2**31, L.E_SHAPE), (10, 3, L.E_SHAPE),
                           (10, 0, L.E_SHAPE), (11, 0, L.E_SHAPE), (11, 3, L.E_SHAPE), (12, 12, L.E_SHAPE),
                           (12, 136, L.E_SHAPE), (12, 0, L.E_SHAPE)):
        bad = list(good)
        bad[i] = value
        assert fwd(*bad) == code, i
        assert lib.numrs_hip_last_error(h)
    bwd = lib.numrs_hip_attention_packed_backward
    good = [h, s, q, ld, k, v, ld, out, call.gd.ptr, 64, call.stats.ptr, call.xd.ptr, None, None, 4, 2, 16, 0]
    for i in (1, 2, 4, 5, 7, 8, 10):
        bad = list(good)
        bad[i] = None
        assert bwd(*bad) == L.E_INVALID, i
    # more work than a launch can have: refused before anything is read
    long = nr.PackedSequences([64 * 64 + 1], ctx=c)
    assert fwd(h, long.handle, q, 524280, k, v, 524280, out, 524280, None, 65535, 65535, 8) == L.E_SHAPE
    assert b"too many" in lib.numrs_hip_last_error(h)
    out_h = ctypes.c_void_p()
    for lengths, n, code in (([-1], 1, L.E_SHAPE), ([2**30, 1], 2, L.E_SHAPE), ([1], -1, L.E_INVALID),
                             ([1], 2**24, L.E_INVALID)):
        a = (ctypes.c_int64 * len(lengths))(*lengths)
        assert lib.numrs_hip_seqs_create(h, a, n, ctypes.byref(out_h)) == code
        assert out_h.value is None
    assert lib.numrs_hip_seqs_create(h, None, 1, ctypes.byref(out_h)) == L.E_INVALID
    assert lib.numrs_hip_seqs_create(h, None, 0, None) == L.E_INVALID
    empty = nr.PackedSequences([0, 0], ctx=c)
    assert empty.total == 0 and len(empty) == 2
    assert fwd(h, empty.handle, None, 64, None, None, 32, None, 64, None, 4, 2, 16) == 0
    assert lib.numrs_hip_graph_begin(h) == 0
    try:
        a = (ctypes.c_int64 * 1)(4)
        assert lib.numrs_hip_seqs_create(h, a, 1, ctypes.byref(out_h)) == L.E_INVALID
    finally:
        assert lib.numrs_hip_graph_abort(h) == 0


# ---------------------------------------------------------------------------
# The tensor engine and the module
# ---------------------------------------------------------------------------


@pytest.fixture()
def engine(hip_ctx):
    before = nr.default_context()
    nr.set_default_context(hip_ctx)
    yield hip_ctx
    nr.set_default_context(before)


def test_tensor_gradients(engine):
    """Column blocks of one tensor and three tensors, against float64; a second backward adds."""
    rng, lengths, H, Hk, dh = np.random.default_rng(5), [90, 1, 33], 4, 2, 24
    call = _Call(engine, lengths, H, Hk, dh, rng)
    ref = call.ref()
    g = nr.Tensor.new(call.g)

    def check(grads, times):
        for name, got in zip(("dq", "dk", "dv"), grads):
            x, err = ref[name]
            _check(got, (times * x, times * (err + U2 * abs(x))), name)

    x = nr.Tensor.new(call.x, True)
    y = x.attention_packed_qkv(call.seqs, H, Hk)
    _check(y.values(), ref["out"], "out")
    loss = y.mul(g).sum()
    loss.backward()
    check(call.parts(x.gradient()), 1)
    loss.backward()
    # every cell adds: the product's holds 2, y's 1 + 2 = 3 and x's 1 + 3 = 4 times the gradient
    check(call.parts(x.gradient()), 4)
    parts = [nr.Tensor.new(np.ascontiguousarray(p), True) for p in call.parts(call.x)]
    y = parts[0].attention_packed(parts[1], parts[2], call.seqs, H, Hk)
    y.mul(g).sum().backward()
    check([p.gradient() for p in parts], 1)
    with nr.no_grad():
        assert not x.attention_packed_qkv(call.seqs, H, Hk).requires_grad


def test_shared_tensors_and_mixed_gradients(engine):
    """One tensor as q, k and v, as k and v, and operands without or with earlier gradients."""
    rng, lengths, H, dh = np.random.default_rng(6), [70, 20], 2, 32
    seqs, T, w = nr.PackedSequences(lengths, ctx=engine), 90, H * dh
    a, b, g = (rand(rng, (T, w)) for _ in range(3))

    def run(make):
        t = make()
        (t[0].attention_packed(t[1], t[2], seqs, H, H).mul(nr.Tensor.new(g))).sum().backward()
        return t

    r = _ref(a, a, a, g, lengths, H, H)
    t = run(lambda: [nr.Tensor.new(a, True)] * 3)
    _check(t[0].gradient(), tuple(r["dq"][i] + r["dk"][i] + r["dv"][i] for i in (0, 1)), "q = k = v", 4e-6)
    r = _ref(a, b, b, g, lengths, H, H)
    x = nr.Tensor.new(b, True)
    t = run(lambda: [nr.Tensor.new(a, True), x, x])
    _check(t[0].gradient(), r["dq"], "dq")
    _check(x.gradient(), tuple(r["dk"][i] + r["dv"][i] for i in (0, 1)), "k = v", 4e-6)
    r = _ref(a, b, a, g, lengths, H, H)
    v = nr.Tensor.new(a, True)
    v.mul(nr.Tensor.new(g)).sum().backward()
    k = nr.Tensor.new(b)
    t = run(lambda: [nr.Tensor.new(a, True), k, v])
    assert k.gradient() is None
    _check(t[0].gradient(), r["dq"], "dq")
    _check(v.gradient(), (r["dv"][0] + g, r["dv"][1] + U2 * abs(r["dv"][0] + g)), "v")


def test_gradients_against_differences(engine):
    """Central differences of sum(out * g) in float64 along random directions of q, k and v."""
    rng, lengths, H, Hk, dh = np.random.default_rng(7), [40, 9], 4, 1, 16
    call = _Call(engine, lengths, H, Hk, dh, rng)
    x = nr.Tensor.new(call.x, True)
    x.attention_packed_qkv(call.seqs, H, Hk).mul(nr.Tensor.new(call.g)).sum().backward()
    got = x.gradient().astype(np.float64)

    def value(x):
        parts = call.parts(x)
        return (_ref(*parts, call.g, lengths, H, Hk)["out"][0] * call.g).sum()

    for part in range(3):
        for _ in range(3):
            d = np.zeros(call.x.shape)
            view = call.parts(d)[part]
            view[:] = rng.standard_normal(view.shape)
            h = 1e-5
            slope = (value(call.x + h * d) - value(call.x - h * d)) / (2 * h)
            # differences: h^2 / 6 of the third derivative, below 1e-7; the gradient: 2e-6 of its norm
            assert abs(slope - (got * d).sum()) <= 1e-5 * np.linalg.norm(got) * np.linalg.norm(d) ** 0.5 + 1e-5


def test_tensor_refusals(engine):
    seqs = nr.PackedSequences([4], ctx=engine)
    t = lambda *s: nr.Tensor.new(np.zeros(s, np.float32))  # noqa: E731
    for call in (lambda: t(5, 64).attention_packed_qkv(seqs, 2, 1),
                 lambda: t(4, 65).attention_packed_qkv(seqs, 2, 1),
                 lambda: t(4, 64).attention_packed_qkv(seqs, 0, 1),
                 lambda: t(4, 20).attention_packed_qkv(seqs, 2, 1),  # heads of 5
                 lambda: t(4, 64).attention_packed_qkv(seqs, 3, 2),
                 lambda: t(4, 32).attention_packed(t(4, 16), t(4, 32), seqs, 2, 1),
                 lambda: t(4, 32).attention_packed(t(3, 16), t(3, 16), seqs, 2, 1),
                 lambda: t(4, 2, 16).attention_packed(t(4, 16), t(4, 16), seqs, 2, 1)):
        with pytest.raises(nr.HipError):
            call()
    empty = nr.PackedSequences([0], ctx=engine)
    assert t(0, 64).attention_packed_qkv(empty, 2, 1).shape() == (0, 32)


def test_module_is_causal_and_trains(engine):
    """forward_packed of one sequence is what it is beside another, up to a token changed later;
    its parameters' gradients come from the same nodes."""
    rng, d, H, Hk = np.random.default_rng(11), 48, 4, 2
    w = [rand(rng, s, 0.2) for s in ((64, d), (32, d), (32, d), (d, 64))]
    attn = nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk)
    x = rand(rng, (30, d))
    one, two = nr.PackedSequences([20, 10]), nr.PackedSequences([20])
    y = attn.forward_packed(nr.Tensor.new(x), one).values()
    alone = attn.forward_packed(nr.Tensor.new(x[:20]), two).values()
    assert np.abs(y[:20] - alone).max() <= 1e-5
    z = x.copy()
    z[12] += 1
    y2 = attn.forward_packed(nr.Tensor.new(z), one, residual=nr.Tensor.new(np.zeros_like(x))).values()
    assert np.abs(y[:12] - y2[:12]).max() <= 1e-5 and np.abs(y[12:20] - y2[12:20]).max() > 1e-3
    attn.forward_packed(nr.Tensor.new(x), one).sum().backward()
    # the output projection's bias sees a one from every row; all gradients are there
    assert np.abs(attn.o.bias.gradient() - 30).max() <= 1e-4
    assert all(p.gradient() is not None and np.isfinite(p.gradient()).all() for p in attn.parameters())
    assert np.abs(attn.qkv.weight.gradient()).max() > 0
    with pytest.raises(ValueError):
        nn.CausalSelfAttention(*w, heads=4, kv_heads=3)


@pytest.mark.parametrize("lengths", [[70, 3, 129], [140] * 40])
def test_a_recorded_training_step(engine, lengths):
    """Steps of the module and SGD as a graph's replays equal eager ones to the bit, while an eager forward
    of the same parameters is still to be swept, and after the sequences' handle is closed."""
    from numrs_amd import optim
    rng, d, H, Hk = np.random.default_rng(18), 32, 16, 4
    w = [rand(rng, s, 0.2) for s in ((16 * H, d), (16 * Hk, d), (16 * Hk, d), (d, 16 * H))]
    x, t = nr.Tensor.new(rand(rng, (sum(lengths), d))), nr.Tensor.new(rand(rng, (sum(lengths), d)))
    seqs = nr.PackedSequences(lengths)

    def make():
        attn = nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk)
        sgd = optim.SGD.simple(attn.parameters(), 0.1)

        def step():
            loss = attn.forward_packed(x, seqs).mse_loss(t)
            loss.backward()
            sgd.step()
            sgd.zero_grad()
            return loss
        return attn, step

    (a, eager), (b, recorded) = make(), make()
    assert eager().item() == recorded().item()
    alive = b.forward_packed(x, seqs).sum()
    graph = nr.StepGraph(engine, recorded)
    want = [eager().item() for _ in range(4)]
    seqs.close()
    filler = [nr.PackedSequences(lengths[::-1]) for _ in range(3)]
    for i, loss in enumerate(want):
        graph.replay()
        assert graph.outputs.item() == loss, i
        if i == 1:  # the sweep adds to gradients that the next replay's step would take
            alive.backward()
            for p in b.parameters():
                p.zero_grad()
    for p, q in zip(a.parameters(), b.parameters()):
        assert_bits(q.values(), p.values())
    graph.close()
    del filler
