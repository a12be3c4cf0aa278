"""Attention of new tokens over a paged cache against float64.  A score is a product of two fp16 pairs (2^-22
of the terms' magnitudes) summed in fp32, a result a sum of such products over the tokens, so the bounds are
those of attention over the cache a token at a time: e = 2^-23 (dh + 8) max |q| . |k| / sqrt(dh) for a score,
(2 e + 2 . 2^-23 (tokens + 8)) p . |v| for a result.  Besides, a weight p f of a token (f its values' factor)
is split in two fp16 terms relative to the largest of 64: that one is in [2^14, 2^15) and fp16's smallest step
2^-24, so that a weight is off by up to 2^-25, 2^-39 of the largest.  A value's terms are at most twice the
largest token's over its factor, so this moves a result by 2^-38 max(p |v|) a token at most: what counts in a
column where the tokens of any weight have zeros."""
import ctypes
import math

import numpy as np
import pytest

import numrs_amd as nr
from conftest import assert_bits, rand
from numrs_amd import _lib as L
from test_gpu_kvcache import U2, _Paged, _stands_for

pytestmark = pytest.mark.gpu


class _Chunk:
    """Sequences of new and cached tokens, all in the cache, and the new ones' queries."""

    def __init__(self, c, new, context, page, H, Hk, dh, format, rng, **kw):
        self.c, self.new, self.H, self.Hk, self.dh, self.format = c, new, H, Hk, dh, format
        self.total = [a + b for a, b in zip(new, context)]
        self.s = _Paged(c, self.total, page, Hk, dh, format, rng, **kw)
        T, self.T = sum(self.total), sum(new)
        self.k, self.v = rand(rng, (T, Hk * dh)), rand(rng, (T, Hk * dh))
        self.q = rand(rng, (self.T, H * dh))
        self.seqs = nr.PackedSequences(new, ctx=c)
        self.table, self.ends = self.s.td, self.s.ends
        self.most = self.s.table.shape[1]

    def write(self):
        c = self.c
        self.s.cache.write(self.s.seqs, c.to_device(self.k), c.to_device(self.v), self.s.td, self.s.ends)
        return self

    def run(self):
        """The result [T, H, dh], rows at strides of their own and what lies beside them untouched."""
        c, w = self.c, self.H * self.dh
        qd = c.to_device(np.pad(self.q, ((0, 1), (1, 4)), constant_values=np.nan))
        out = c.to_device(np.full((self.T + 1, w + 3), 7, np.float32))
        c._check(L.load().numrs_hip_attention_paged_chunk(
            c.handle, ctypes.byref(self.s.cache.pages), self.seqs.handle, qd.ptr + 4, w + 5, self.H, self.table.ptr,
            self.most, self.ends.ptr, out.ptr + 8, w + 3))
        got = out.numpy()
        assert (got[:, :2] == 7).all() and (got[:, 2 + w:] == 7).all() and (got[self.T] == 7).all()
        return got[:self.T, 2:2 + w].reshape(self.T, self.H, self.dh)

    def stands(self):
        """Each sequence's keys and values [n, Hk, dh] as the cache has them."""
        k, v = (_stands_for(x.reshape(-1, self.Hk, self.dh), self.format) for x in (self.k, self.v))
        at = np.concatenate([[0], np.cumsum(self.total)])
        return [(k[a:b], v[a:b]) for a, b in zip(at, at[1:])]

    def reference(self, only=None):
        """Results and bounds [T, H, dh]; of the sequences in `only`, if given."""
        out, err = np.zeros((2, self.T, self.H, self.dh))
        at = 0
        for i, ((k, v), n) in enumerate(zip(self.stands(), self.new)):
            if n and (only is None or i in only):
                seen = np.arange(len(k)) <= np.arange(len(k) - n, len(k))[:, None]
                out[at:at + n], err[at:at + n] = _rows(self.q[at:at + n].reshape(n, self.H, self.dh), k, v, seen)
            at += n
        return out, err

    def check(self, got, only=None):
        ref, err = self.reference(only)
        at = np.concatenate([[0], np.cumsum(self.new)])
        for i in range(len(self.new)) if only is None else only:
            part = slice(at[i], at[i + 1])
            _check(got[part], ref[part], err[part], f"sequence {i}")


def _rows(q, k, v, seen):
    """Rows q [n, H, dh] over the tokens k, v [m, Hk, dh] that `seen` [n, m] gives them."""
    n, H, dh = q.shape
    out, err = np.zeros((2, n, H, dh))
    group = H // k.shape[1]
    some = seen.any(1)
    for h in range(H):
        Q, K, V = (x.astype(np.float64) for x in (q[:, h], k[:, h // group], v[:, h // group]))
        s = np.where(seen, Q @ K.T / math.sqrt(dh), -np.inf)
        p = np.exp(s - s.max(1, keepdims=True, initial=-1e300))
        p /= np.maximum(p.sum(1, keepdims=True), 1e-300)
        e = U2 * (dh + 8) * np.where(seen, abs(Q) @ abs(K).T, 0).max(1, keepdims=True) / math.sqrt(dh)
        out[:, h] = np.where(some[:, None], p @ V, 0)
        err[:, h] = (2 * e + 2 * U2 * (seen.sum(1, keepdims=True) + 8)) * (p @ abs(V))
        err[:, h] += 2.0 ** -38 * seen.sum(1, keepdims=True) * (p * abs(V).max(1)).max(1, keepdims=True)
    return out, err


def _check(got, ref, err, what):
    d = abs(got - ref)
    assert (d <= err).all(), f"{what}: outside its bound by {(d / (err + 1e-300)).max():.2g}"
    rel = np.linalg.norm(d) / max(np.linalg.norm(ref), 1e-300)
    assert rel <= 2e-6, f"{what}: 2-norm error {rel:.2g}"


# One row to many, groups of 1 to 40 heads (rows of a token cut by a block's border), contexts of none, ends
# inside, at and past a page and a stage of tokens, empty sequences between, one long, many short.
SHAPES = [
    ([1], [0], 16, 1, 1, 8),
    ([2, 0, 3, 1], [0, 5, 15, 16], 16, 4, 2, 40),
    ([7], [333], 16, 8, 8, 64),
    ([64, 65, 63, 1], [64, 0, 1, 127], 64, 6, 3, 64),
    ([300], [1000], 64, 16, 2, 128),
    ([129, 40], [511, 0], 128, 10, 2, 80),
    ([5] * 40, [70] * 40, 32, 8, 4, 64),
    ([16], [20000], 256, 8, 1, 128),
    ([33, 100], [300, 40], 16, 17, 1, 24),
    ([9, 5, 77], [3000, 0, 400], 64, 40, 1, 64),
    ([31], [255], 16, 64, 2, 96),
    ([700, 1, 1, 90, 0, 13], [2048, 4097, 3, 0, 77, 640], 1024, 12, 3, 72),
    ([257, 513], [0, 31], 16, 1, 1, 128),
    ([1, 1, 1, 1], [5000, 1, 64, 63], 16, 4, 4, 32),
]


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_chunk(hip_ctx, i, format):
    new, context, page, H, Hk, dh = SHAPES[i]
    print(f"[gpu] chunk {new[:6]} after {context[:6]} page={page} H={H} Hk={Hk} dh={dh} {format}", flush=True)
    t = _Chunk(hip_ctx, new, context, page, H, Hk, dh, format, np.random.default_rng(i)).write()
    got = t.run()
    t.check(got)
    assert_bits(t.run(), got, "the same call again")


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_many_sequences(hip_ctx, format):
    """1300 sequences, most with a few new tokens, some without, some long."""
    rng = np.random.default_rng(21)
    new, context = rng.integers(0, 6, 1300).tolist(), rng.integers(0, 60, 1300).tolist()
    new[0], new[511], new[512], new[1100], new[1299] = 0, 130, 0, 2, 65
    context[511], context[1100] = 700, 2500
    t = _Chunk(hip_ctx, new, context, 16, 8, 2, 64, format, rng).write()
    got = t.run()
    t.check(got)
    assert_bits(t.run(), got)


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_bad_tables(hip_ctx, format, n):
    """Ends past the table, before the new tokens or negative, pages that the cache lacks, one page in two
    tables: each row sees what there is of the tokens up to itself, or is zeros."""
    c, rng, H, Hk, dh, page = hip_ctx, np.random.default_rng(22 + n), 6, 2, 32, 16
    t = _Chunk(c, [n] * 6, [336 - n] * 6, page, H, Hk, dh, format, rng, wider=0).write()
    table, cols = t.s.table.copy(), 21
    table[0, 2], table[1, 0], table[1, 20] = -3, t.s.pages, 2**31 - 1
    table[2, 1] = table[3, 0]
    table[4] = -1
    ends = np.array([336, 300, 336 + 1000, n - 1, 336, -7], np.int32)
    t.table, t.ends = c.to_device(table), c.to_device(ends)
    got = t.run().reshape(6, n, H, dh)
    kv = t.stands()
    where = {p: (i, j) for i in range(6) for j, p in enumerate(t.s.table[i])}
    for i in range(6):
        there = np.zeros(cols * page, bool)
        k, v = np.zeros((2, cols * page, Hk, dh), np.float32)
        for j, p in enumerate(table[i]):
            if p in where:
                a, b = where[p]
                there[j * page:(j + 1) * page] = True
                k[j * page:(j + 1) * page], v[j * page:(j + 1) * page] = (x[b * page:(b + 1) * page] for x in kv[a])
        at = int(ends[i]) - n + np.arange(n)
        seen = there & (np.arange(cols * page) <= at[:, None])
        ref, err = _rows(t.q.reshape(6, n, H, dh)[i], k, v, seen)
        assert (got[i][~seen.any(1)] == 0).all()
        _check(got[i], ref, err, f"sequence {i}")
    assert (got[4:] == 0).all()


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("n", [3, 150])
def test_values_that_are_not_finite(hip_ctx, format, n):
    """What is not finite reaches its own head and sequence, and there the rows that see it (the others have
    what they had, up to their bounds); infinite keys and values do what fp32 arithmetic does with them."""
    c, rng, H, Hk, dh = hip_ctx, np.random.default_rng(23), 4, 2, 64
    t = _Chunk(c, [n, n, n, n], [200, 70, 0, 333], 16, H, Hk, dh, format, rng).write()
    clean, bound = t.run().reshape(4, n, Hk, 2, dh), t.reference()[1].reshape(4, n, Hk, 2, dh)
    at = np.concatenate([[0], np.cumsum(t.total)])
    k, v, q = t.k.copy(), t.v.copy(), t.q.copy()
    t.k[50, 3] = np.nan                            # sequence 0, head 0: every row
    seen = n // 2                                  # of sequence 1, the rows that see it
    t.v[at[1] + 70 + seen, dh + 5] = np.inf        # head 1
    t.v[at[2] + n - 1, 7] = np.nan                 # sequence 2, head 0: the last row's own token
    t.k[at[3] + 10, dh:2 * dh] = -np.inf * np.sign(t.q[3 * n, 2 * dh:3 * dh])  # head 1: a score of -inf for its row 0
    t.write()
    got = t.run().reshape(4, n, Hk, 2, dh)
    assert np.isnan(got[0, :, 0]).all()
    assert_bits(got[0, :, 1], clean[0, :, 1])
    assert_bits(got[1, :, 0], clean[1, :, 0])
    same = lambda i, rows, h: (abs(got[i, rows, h] - clean[i, rows, h]) <= 2 * bound[i, rows, h]).all()  # noqa: E731
    assert same(1, slice(seen), 1)
    rest = np.arange(dh) != 5
    if format == "f32":
        assert np.isposinf(got[1, seen:, 1, :, 5]).all()
        _check(got[1, seen:, 1][..., rest], clean[1, seen:, 1][..., rest], 1e-5 + 0 * clean[1, seen:, 1][..., rest], "beside")
    else:
        assert np.isnan(got[1, seen:, 1]).all()  # such a row reads back as NaN
    assert_bits(got[2, :, 1], clean[2, :, 1])
    assert same(2, slice(n - 1), 0)
    assert np.isnan(got[2, n - 1, 0, :, 7]).all()
    if format == "f32":
        others = np.arange(dh) != 7
        assert np.isfinite(got[2, n - 1, 0][:, others]).all()
        # the first row without that key
        (K, V), Q = t.stands()[3], q[3 * n].reshape(H, dh)
        live = np.arange(len(K)) <= 333
        live[10] = False
        K = np.where(np.isfinite(K), K, 0)
        ref, err = _rows(Q[None], K, V, live[None])
        _check(got[3, 0].reshape(1, H, dh)[:, 2], ref[:, 2], err[:, 2], "a score of -inf")
    assert_bits(got[3, :, 0], clean[3, :, 0])
    # a query that is not finite: its own row
    t.k, t.v = k, v
    t.write()
    t.q[0, 1], t.q[2 * n + 1, dh + 3] = np.nan, np.inf
    got = t.run().reshape(4 * n, H, dh)
    clean = clean.reshape(4 * n, H, dh)
    bad = np.zeros((4 * n, H), bool)
    bad[0, 0] = bad[2 * n + 1, 1] = True
    assert np.isnan(got[bad]).all()
    assert (abs(got - clean) <= 2 * bound.reshape(4 * n, H, dh))[~bad].all()


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("sq,sk,sv", [(30, 30, 1), (1e-20, 1e20, 1e30), (1, 1, 1e-36), (0, 1, 1), (1e10, 1e-10, 1),
                                      (1e-30, 1e-30, 1e37), (1e15, 1e15, 1)])
def test_magnitudes(hip_ctx, sq, sk, sv, format):
    """Scores far apart (a softmax that is one token's), tiny and huge values."""
    rng = np.random.default_rng(24)
    t = _Chunk(hip_ctx, [100], [500], 64, 4, 1, 64, format, rng)
    t.q, t.k, t.v = t.q * np.float32(sq), t.k * np.float32(sk), t.v * np.float32(sv)
    got = t.write().run()
    ref, err = t.reference()
    d = abs(got - ref)
    assert (d <= err + 1e-44).all(), (d / (err + 1e-300)).max()


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("n", [2, 90])
@pytest.mark.parametrize("gap", [0, 13, 20, 30, 60, 500])
def test_a_token_far_above_the_others(hip_ctx, gap, n, format):
    """A token with 2^-gap of the others' probability and a value 2^min(gap, 60) times theirs; of 500, none of it."""
    c, H, Hk, dh, rng = hip_ctx, 8, 2, 64, np.random.default_rng(gap + n)
    t = _Chunk(c, [n], [1000], 16, H, Hk, dh, format, rng)
    m = n + 1000
    t.q[:], t.k[:] = 0, 0
    t.q[:, ::dh] = 8
    # a row of one value has the code 127 for it: the cache holds it to a rounding
    t.k[:, ::dh] = rng.uniform(-1, 1, (m, Hk)).astype(np.float32)
    t.k[7, ::dh] = -np.float32(gap * math.log(2))
    t.v[7] *= np.float32(2.0 ** min(gap, 60))
    got = t.write().run()
    (K, V), = t.stands()
    for h in range(H):
        x, y = K[:, h // (H // Hk), 0].astype(np.float64), V[:, h // (H // Hk)].astype(np.float64)
        for r in (0, n - 1):
            s = x[:m - n + r + 1]
            p = np.exp(s - s.max())
            p /= p.sum()
            # a score is one product here: ten operations' roundings
            f = 2 * U2 * 10 * abs(s[p > 2.0 ** -100]).max() + U2 * (len(s) + 8)
            ref, err = p @ y[:len(s)], f * (p @ abs(y[:len(s)]))
            d = abs(got[r, h] - ref)
            assert (d <= err).all(), f"row {r}, head {h}: off by {(d / err).max():.2g} of the bound"
            norm = 2e-6 + 3 * min(gap, 60) * math.log(2) * U2 / 2
            assert np.linalg.norm(d) <= norm * np.linalg.norm(ref), f"row {r}, head {h}: {np.linalg.norm(d):.2g}"


@pytest.mark.parametrize("gap", [20, 60, 100])
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_tokens_of_very_different_size(hip_ctx, which, gap):
    """Neighbouring tokens' keys, values or queries 2^gap apart: none costs another its bits."""
    rng = np.random.default_rng(25 + gap)
    t = _Chunk(hip_ctx, [70], [400], 16, 4, 2, 64, "f32", rng)
    x = getattr(t, which)
    x *= np.ldexp(np.float32(1), -(rng.integers(0, 2, len(x)) * gap)).astype(np.float32)[:, None]
    t.check(t.write().run())


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_scores_near_the_lowest(hip_ctx, format):
    """Equal scores of -3.5e32: the mean of the values, as for any other score."""
    rng, n, m, dh = np.random.default_rng(26), 50, 300, 8
    t = _Chunk(hip_ctx, [n], [m - n], 16, 1, 1, dh, format, rng)
    t.k[:], t.q[:] = 0, 0
    t.k[:, 3], t.q[:, 3] = -1e16, 1e17
    got = t.write().run()[:, 0]
    (_, v), = t.stands()
    v = v[:, 0].astype(np.float64)
    for r in range(n):
        y = v[:m - n + r + 1]
        assert (abs(got[r] - y.mean(0)) <= 2 * U2 * (len(y) + 8) * abs(y).mean(0)).all(), r


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_rows_of_one_are_the_decoding_steps(hip_ctx, format):
    """A token for each sequence: what attention a token at a time gives, to its bounds."""
    c, rng, H, Hk, dh, n = hip_ctx, np.random.default_rng(27), 8, 2, 64, 9
    t = _Chunk(c, [1] * n, rng.integers(0, 900, n).tolist(), 16, H, Hk, dh, format, rng).write()
    got, out, qd = t.run(), c.empty((n, H * dh)), c.to_device(t.q)
    c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(t.s.cache.pages), qd.ptr, H * dh, H, t.table.ptr,
                                                t.most, t.ends.ptr, n, out.ptr, H * dh))
    _, err = t.reference()
    assert (abs(got - out.numpy().reshape(n, H, dh)) <= 2 * err).all()


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_pages_past_32_bits(hip_ctx, format):
    """A cache of 2.2e9 values: pages whose elements, and bytes, lie past 2^31 and 2^32."""
    c, rng, page, Hk, dh, H = hip_ctx, np.random.default_rng(28), 1024, 2, 128, 6
    pages = 2 ** 31 // (page * Hk * dh) + 10
    t = _Chunk(c, [300, 2, 40], [2200, 2047, 1060], page, H, Hk, dh, format, rng)
    t.s.cache = nr.KVCache(pages, page, Hk, dh, format, ctx=c)
    table = np.array([[pages - 1, pages // 2, 3], [pages // 4, pages - 2, pages // 2 + 1], [0, pages - 9, 1]], np.int32)
    t.s.td = t.table = c.to_device(table)
    t.s.pages, t.most = pages, 3
    t.check(t.write().run())


def test_recorded_and_replayed(hip_ctx):
    """Two recorded graphs and eager calls of other sizes take turns; ends and tables change between the
    replays, and the sequences' handle is gone."""
    c, rng = hip_ctx, np.random.default_rng(29)
    t = _Chunk(c, [40, 1, 130], [300, 700, 0], 16, 8, 2, 64, "f32", rng).write()
    other = _Chunk(c, [3, 90], [2000, 10], 16, 4, 2, 128, "int8", rng).write()
    w = 8 * 64
    qd, out = c.to_device(t.q), c.empty((t.T, w))
    step = lambda: c._check(L.load().numrs_hip_attention_paged_chunk(  # noqa: E731
        c.handle, ctypes.byref(t.s.cache.pages), t.seqs.handle, qd.ptr, w, 8, t.table.ptr, t.most, t.ends.ptr, out.ptr, w))
    step()
    graphs, wants = [nr.StepGraph(c, step) for _ in range(2)], []
    ends = [np.array(e, np.int32) for e in ([340, 701, 130], [100, 1, 130], [339, 350, 60], [341, 0, 131])]
    for e in ends:
        t.ends.upload(e)
        step()
        wants.append(out.numpy())
    t.seqs.close()
    filler = [nr.PackedSequences([1, 130, 40], ctx=c) for _ in range(3)]
    for i, (e, want) in enumerate(zip(ends, wants)):
        t.ends.upload(e)
        out.fill(0)
        other.run()
        graphs[i % 2].replay()
        assert_bits(out.numpy(), want)
    for g in graphs:
        g.close()
    del filler


def test_two_contexts_at_once():
    rng = np.random.default_rng(30)
    with nr.Context(0) as a, nr.Context(0) as b:
        calls = [_Chunk(c, [200, 7], [500, 3000], 16, 8, 2, 64, "f32", rng).write() for c in (a, b)]
        want = [t.run() for t in calls]
        w = 8 * 64
        qs, outs = [t.c.to_device(t.q) for t in calls], [t.c.empty((t.T, w)) for t in calls]
        for _ in range(3):
            for t, q, out in zip(calls, qs, outs):  # queued on both streams before either is read
                t.c._check(L.load().numrs_hip_attention_paged_chunk(
                    t.c.handle, ctypes.byref(t.s.cache.pages), t.seqs.handle, q.ptr, w, 8, t.table.ptr, t.most, t.ends.ptr,
                    out.ptr, w))
            for out, x in zip(outs, want):
                assert_bits(out.numpy().reshape(x.shape), x)
        with pytest.raises(nr.HipError, match="another context"):
            calls[0].seqs = calls[1].seqs
            calls[0].run()
        del calls, qs, outs, t, q, out


def test_refusals(hip_ctx):
    c, lib, rng = hip_ctx, L.load(), np.random.default_rng(31)
    t = _Chunk(c, [5, 3], [2, 0], 16, 4, 2, 16, "int8", rng).write()
    h, cp, fn = c.handle, ctypes.byref(t.s.cache.pages), lib.numrs_hip_attention_paged_chunk
    q, out = c.to_device(t.q), c.empty((8, 64))
    good = [h, cp, t.seqs.handle, q.ptr, 64, 4, t.table.ptr, t.most, t.ends.ptr, out.ptr, 64]
    assert fn(*good) == 0
    for i, value, code in ((1, None, L.E_INVALID), (2, None, L.E_INVALID), (3, None, L.E_INVALID), (4, 63, L.E_SHAPE),
                           (4, 2**31, L.E_SHAPE), (5, 3, L.E_SHAPE), (5, 0, L.E_SHAPE), (5, 65536, L.E_SHAPE),
                           (6, None, L.E_INVALID), (7, 0, L.E_SHAPE), (8, None, L.E_INVALID), (9, None, L.E_INVALID),
                           (10, 63, L.E_SHAPE)):
        bad = list(good)
        bad[i] = value
        assert fn(*bad) == code, i
        assert lib.numrs_hip_last_error(h)
    assert fn(None, *good[1:]) == L.E_INVALID
    bad = nr.KVPages.from_buffer_copy(t.s.cache.pages)
    bad.page_size = 24
    assert fn(h, ctypes.byref(bad), *good[2:]) == L.E_SHAPE
    empty = nr.PackedSequences([0, 0], ctx=c)
    assert fn(h, cp, empty.handle, None, 64, 4, t.table.ptr, t.most, t.ends.ptr, None, 64) == 0
    none = nr.PackedSequences([], ctx=c)
    assert fn(h, cp, none.handle, None, 64, 4, None, 1, None, None, 64) == 0
    x = nr.Tensor.new(t.q, True, ctx=c)
    with pytest.raises(nr.HipError, match="no backward"):
        x.attention_paged_chunk(t.s.cache, t.seqs, 4, t.table, t.ends)
    x = nr.Tensor.new(t.q, ctx=c)
    assert_bits(x.attention_paged_chunk(t.s.cache, t.seqs, 4, t.table, t.ends).values().reshape(8, 4, 16), t.run())
    with pytest.raises(nr.HipError):
        x.attention_paged_chunk(t.s.cache, empty, 4, t.table, t.ends)
    with pytest.raises(ValueError):
        x.attention_paged_chunk(t.s.cache, t.seqs, 4, t.ends, t.table)
    with nr.Context(0) as other, pytest.raises(ValueError, match="one context"):
        nr.Tensor.new(t.q, ctx=other).attention_paged_chunk(t.s.cache, t.seqs, 4, t.table, t.ends)


# From 2048 rows of a kv head on a sequence the cached tokens are laid out for the matrix cores first (fp32): fewer and
# more of them, every head size's layout, sequences of one and of none between, tables too wide for that.
MANY = [
    ([1100], [500], 16, 1, 1, 8, 0),
    ([200, 300], [0, 700], 64, 14, 2, 40, 3),
    ([260], [3000], 16, 8, 2, 64, 0),
    ([400], [64], 32, 12, 4, 96, 1),
    ([1030], [63], 1024, 1, 1, 32, 0),
    ([512, 1, 0, 700], [2, 900, 7, 0], 16, 12, 3, 128, 0),
    ([300], [400], 1024, 4, 1, 128, 1100),
    ([2100], [500], 16, 1, 1, 8, 0),
    ([300, 340], [0, 700], 64, 14, 2, 40, 3),
    ([700], [64], 32, 12, 4, 96, 1),
    ([2050], [63], 1024, 1, 1, 32, 0),
    ([520], [400], 1024, 4, 1, 128, 1100),
]


@pytest.mark.parametrize("i", range(len(MANY)))
def test_many_rows(hip_ctx, i):
    new, context, page, H, Hk, dh, wider = MANY[i]
    t = _Chunk(hip_ctx, new, context, page, H, Hk, dh, "f32", np.random.default_rng(40 + i), wider=wider).write()
    got = t.run()
    t.check(got)
    assert_bits(t.run(), got, "the same call again")


@pytest.mark.parametrize("n", [300, 600])
@pytest.mark.parametrize("gap", [20, 60, 100])
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_many_rows_of_very_different_size(hip_ctx, which, gap, n):
    rng = np.random.default_rng(50 + gap)
    t = _Chunk(hip_ctx, [n], [200], 16, 8, 2, 64, "f32", rng)
    x = getattr(t, which)
    x *= np.ldexp(np.float32(1), -(rng.integers(0, 2, len(x)) * gap)).astype(np.float32)[:, None]
    t.check(t.write().run())


@pytest.mark.parametrize("H", [16, 32])
def test_many_rows_with_what_is_not_finite(hip_ctx, H):
    """A key, a query and a value that are not finite, a page that is missing, ends below the new tokens."""
    c, rng, n, Hk, dh, page = hip_ctx, np.random.default_rng(60), 150, 2, 32, 16
    t = _Chunk(c, [n] * 5, [106] * 5, page, H, Hk, dh, "f32", rng).write()
    clean, bound = t.reference()
    clean, bound = clean.reshape(5, n, Hk, H // Hk, dh), bound.reshape(5, n, Hk, H // Hk, dh)
    t.k[40, 3] = np.nan                   # sequence 0, head 0: every row
    t.v[256 + 106 + 70, dh + 5] = np.inf  # sequence 1, head 1: the rows from 70 on, column 5
    t.write()
    t.q[2 * n + 9, 4] = np.nan            # sequence 2, row 9, the first query head
    table, ends = t.s.table.copy(), np.array([256, 256, 256, 256, n - 1], np.int32)
    table[3, 2] = -1
    t.table, t.ends = c.to_device(table), c.to_device(ends)
    got = t.run().reshape(5, n, Hk, H // Hk, dh)
    assert np.isnan(got[0, :, 0]).all()
    _check(got[0, :, 1], clean[0, :, 1], bound[0, :, 1], "beside a key that is NaN")
    assert np.isposinf(got[1, 70:, 1, :, 5]).all()
    rest = np.arange(dh) != 5
    _check(got[1, 70:, 1][..., rest], clean[1, 70:, 1][..., rest], bound[1, 70:, 1][..., rest], "beside an infinite value")
    _check(got[1, :70, 1], clean[1, :70, 1], bound[1, :70, 1], "before an infinite value")
    _check(got[1, :, 0], clean[1, :, 0], bound[1, :, 0], "another head")
    assert np.isnan(got[2, 9, 0, 0]).all()
    others = np.ones((n, Hk, H // Hk), bool)
    others[9, 0, 0] = False
    _check(got[2][others], clean[2][others], bound[2][others], "beside a query that is NaN")
    (k, v), q = t.stands()[3], t.q.reshape(5, n, H, dh)
    at = np.arange(256)
    seen = (at <= 106 + np.arange(n)[:, None]) & (at // page != 2)
    ref, err = _rows(q[3], k, v, seen)
    _check(got[3].reshape(n, H, dh), ref, err, "a page that is missing")
    k, v = t.stands()[4]
    ref, err = _rows(q[4], k, v, at <= np.arange(-1, n - 1)[:, None])
    assert (got[4, 0] == 0).all()
    _check(got[4].reshape(n, H, dh), ref, err, "an end below the new tokens")


@pytest.mark.parametrize("H", [16, 32])
def test_many_rows_recorded_and_replayed(hip_ctx, H):
    """What was laid out for one replay is not what the next reads: keys, values and ends change between them."""
    c, rng = hip_ctx, np.random.default_rng(61)
    t = _Chunk(c, [300, 2], [200, 50], 16, H, 2, 64, "f32", rng).write()
    w = H * 64
    qd, out = c.to_device(t.q), c.empty((t.T, w))
    step = lambda: c._check(L.load().numrs_hip_attention_paged_chunk(  # noqa: E731
        c.handle, ctypes.byref(t.s.cache.pages), t.seqs.handle, qd.ptr, w, H, t.table.ptr, t.most, t.ends.ptr, out.ptr, w))
    step()
    graph = nr.StepGraph(c, step)
    for e in ([500, 52], [300, 52], [470, 10], [500, 2]):
        t.k, t.v = rand(rng, t.k.shape), rand(rng, t.v.shape)
        t.write()
        t.ends.upload(np.array(e, np.int32))
        graph.replay()
        first = out.numpy()
        out.fill(0)
        step()
        assert_bits(out.numpy(), first)
        if e == [500, 52]:
            t.check(first.reshape(t.T, H, 64))
    graph.close()


@pytest.mark.parametrize("n", [16, 33])
def test_many_rows_of_many_sequences(hip_ctx, n):
    """600 sequences of a few tokens and 64 heads on one key head: more of them than a workgroup has threads."""
    rng = np.random.default_rng(62)
    t = _Chunk(hip_ctx, [n] * 600, rng.integers(0, 50, 600).tolist(), 16, 64, 1, 8, "f32", rng).write()
    got = t.run()
    t.check(got, only=[0, 1, 255, 511, 512, 513, 598, 599])
    assert np.isfinite(got).all()


def test_refusals_of_sizes_and_places(hip_ctx):
    """Results over their inputs, tables and groups past what is counted in 32 bits."""
    c, lib, rng = hip_ctx, L.load(), np.random.default_rng(63)
    t = _Chunk(c, [5, 3], [2, 0], 16, 4, 2, 16, "f32", rng).write()
    h, cp, fn = c.handle, ctypes.byref(t.s.cache.pages), lib.numrs_hip_attention_paged_chunk
    q, out = c.to_device(t.q), c.empty((8, 64))
    args = lambda dst, most=t.most: [h, cp, t.seqs.handle, q.ptr, 64, 4, t.table.ptr, most, t.ends.ptr, dst, 64]  # noqa: E731
    assert fn(*args(out.ptr)) == 0
    assert fn(*args(q.ptr)) == L.E_INVALID and fn(*args(q.ptr + 63 * 4)) == L.E_INVALID
    assert fn(*args(q.ptr - 63 * 4)) == L.E_INVALID
    assert fn(*args(out.ptr, 2 ** 27)) == L.E_SHAPE
    one = nr.KVCache(4, 16, 1, 8, "f32", ctx=c)
    long = nr.PackedSequences([40000], ctx=c)
    assert fn(h, ctypes.byref(one.pages), long.handle, q.ptr, 65535 * 8, 65535, t.table.ptr, 1, t.ends.ptr, out.ptr,
              65535 * 8) == L.E_SHAPE
    x, app = c.to_device(rand(rng, (8, 192))), lib.numrs_hip_kv_cache_append
    args = lambda dst: [h, cp, t.seqs.handle, x.ptr, 192, None, None, 1e-6, None, dst, 192, 4, t.table.ptr, t.most,  # noqa: E731
                        t.ends.ptr]
    assert app(*args(x.ptr)) == L.E_INVALID and app(*args(x.ptr + 127 * 4)) == L.E_INVALID
    assert app(*args(x.ptr + 128 * 4)) == 0  # beside the projection, in the same rows


# Where a bad token and the one that takes all of the softmax lie: in one stage, in stages of a block that nobody
# cuts, in up to 32 parts, in more, among images, and in the decoding steps.
FAR = [
    ([2], [50], 4, 2),
    ([2] * 64, [638] * 64, 8, 8),
    ([2], [1280], 2, 1),
    ([3, 2], [700, 1300], 8, 2),
    ([2], [3840], 2, 1),
    ([2100], [1000], 1, 1),
    ([1], [50], 4, 2),
    ([1], [1280], 2, 1),
]


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("bad_first", [True, False])
@pytest.mark.parametrize("i", range(len(FAR)))
def test_what_is_not_finite_far_below_the_softmax(hip_ctx, i, bad_first, format):
    """A NaN and an infinite value on tokens whose scores lie 200 below another's: their probabilities are 0 in
    fp32, and 0 times either is NaN, whichever way the tokens are dealt and joined."""
    new, context, H, Hk = FAR[i]
    dh, rng = 64, np.random.default_rng(70 + i)
    t = _Chunk(hip_ctx, new, context, 64, H, Hk, dh, format, rng)
    t.q[:] = 0
    t.q[:, ::dh] = 8  # over sqrt(64): a score is a key's first column
    t.k[:, ::dh] = 0
    first, last = 5, context[0] - 3
    low, high = (first, last) if bad_first else (last, first)
    t.k[high, ::dh] = 200
    t.v[low, 3], t.v[low + 1, 4] = np.nan, np.inf  # of the first sequence and head
    got, n = t.write().run(), new[0]
    t.v[low, 3] = t.v[low + 1, 4] = 0
    ref, err = t.reference()
    bad = np.zeros(got.shape, bool)
    bad[:n, :H // Hk, slice(3, 5) if format == "f32" else slice(None)] = True
    assert np.isnan(got[bad]).all(), f"{np.isfinite(got[bad]).sum()} of {bad.sum()} are finite"
    assert (abs(got - ref) <= err)[~bad].all()


def test_results_in_their_inputs_rows(hip_ctx):
    """A result one or several rows into its input, at the same stride or another, is refused; column blocks side by
    side in the same rows are not."""
    c, lib, rng = hip_ctx, L.load(), np.random.default_rng(80)
    t = _Chunk(c, [5, 3], [2, 0], 16, 4, 2, 16, "f32", rng).write()
    h, cp = c.handle, ctypes.byref(t.s.cache.pages)
    big = c.to_device(rand(rng, (40, 200)))
    q = big.ptr + 4 * 16 * 200
    chunk = lambda at, ld: lib.numrs_hip_attention_paged_chunk(  # noqa: E731
        h, cp, t.seqs.handle, q, 200, 4, t.table.ptr, t.most, t.ends.ptr, q + 4 * at, ld)
    for at in (0, 200, 7 * 200, -200, -7 * 200, 3 * 200 + 63, -3 * 200 - 63, 200 - 63):
        assert chunk(at, 200) == L.E_INVALID, at
    for at, ld in ((-64, 70), (0, 400), (-7 * 100, 100)):
        assert chunk(at, ld) == L.E_INVALID, (at, ld)
    assert b"overlaps" in lib.numrs_hip_last_error(h)
    before = big.numpy()
    for at in (64, 200 - 64, -64, 8 * 200 - 10):
        assert chunk(at, 200) == 0, at
    assert chunk(100, 400) == 0
    assert_bits(big.numpy()[16:24, :64], before[16:24, :64])
    app = lambda at, ld: lib.numrs_hip_kv_cache_append(  # noqa: E731
        h, cp, t.seqs.handle, q, 200, None, None, 1e-6, None, q + 4 * at, ld, 4, t.table.ptr, t.most, t.ends.ptr)
    for at, ld in ((200, 200), (-200, 200), (5 * 200 + 127, 200), (-6 * 200 - 63, 200), (0, 64), (-64, 300)):
        assert app(at, ld) == L.E_INVALID, (at, ld)
    for at in (128, -64, -72):
        assert app(at, 200) == 0, at


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dh", [32, 64, 128])
@pytest.mark.parametrize("new,H,Hk", [([2] * 64, 8, 8), ([66] * 64, 32, 8), ([520], 4, 1)])
def test_a_beginning_of_zeros(hip_ctx, new, H, Hk, dh, which):
    """128 tokens of zeros, then keys (or values) from 8 to 16 and 2^7 times those over queries of 2^-7: each is a
    product of two terms at a power of two of its own, so that all sums are the same ones and results have the same
    bits (of the values, 2^7 times).  In plain fp32, token by token, the larger ones' would differ."""
    rng = np.random.default_rng(81)
    t = _Chunk(hip_ctx, new, [640 - new[0]] * len(new), 64, H, Hk, dh, "f32", rng)
    x = getattr(t, which)
    x *= 8
    x[:, ::dh] = rng.uniform(8, 15, (len(x), Hk))  # a token's largest
    x.reshape(len(new), 640, -1)[:, :128] = 0
    t.q /= 8
    first = t.write().run()
    t.check(first, only=[0, len(new) - 1])
    x *= np.float32(128)
    if which == "k":
        t.q /= 128
        assert_bits(t.write().run(), first)
    else:
        assert_bits(t.write().run(), first * np.float32(128))


@pytest.mark.parametrize("n", [2, 300, 600])
@pytest.mark.parametrize("gap", [0, 8, 9])
def test_values_far_below_their_tokens_largest(hip_ctx, gap, n):
    """A row whose softmax is its own token's gives that token's value, the token 2^-gap of those before it: to 2^-22 of
    itself or 2^-30 of the token's largest, to 2^-39 of that for the weight, and to the 2^-23 of each of four roundings
    (the weight, the product's sum, the sum over stages, 1 / l and what it multiplies)."""
    H, Hk, dh, rng = 8, 2, 64, np.random.default_rng(82)
    t = _Chunk(hip_ctx, [n], [200], 16, H, Hk, dh, "f32", rng)
    m = n + 200
    t.k[:], t.q[:] = 0, 0
    t.k[:, ::dh] = 256 * np.arange(m)[:, None] / 8  # each 200 and more above the one before
    t.q[:, ::dh] = 64
    t.v *= np.ldexp(np.float32(1), -rng.integers(0, 30, t.v.shape)).astype(np.float32)
    t.v[:, 1::dh] = 1.5
    t.v[200:] *= np.float32(2.0 ** -gap)
    got = t.write().run()
    v = np.repeat(t.v[200:].reshape(n, Hk, dh), H // Hk, axis=1).astype(np.float64)
    top = abs(v).max(-1, keepdims=True)
    err = np.maximum(2.0 ** -22 * abs(v), 2.0 ** -30 * top) + 2.0 ** -39 * top + 5 * U2 * abs(v)
    assert (abs(got - v) <= err).all(), (abs(got - v) / err).max()
