"""The paged key-value cache and attention over it against numpy: codes and scales to the bit (the
format rounds in fp32, as numpy's float32 does), attention against float64 with the bounds of
test_gpu_packed.py."""
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


def _quantise(x):
    """Codes and scales of x [..., d]."""
    with np.errstate(all="ignore"):
        scale = np.abs(x).max(-1) / np.float32(127)
        scale = np.where(np.isfinite(x).all(-1), scale, np.float32(np.nan)).astype(np.float32)
        safe = np.where(scale > 0, scale, np.float32(1))
        q = np.clip(np.rint(x / safe[..., None]), -127, 127)
        q = np.where((scale > 0)[..., None], q, 0)
    return (q + 128).astype(np.uint8), scale


def _stands_for(x, format):
    if format == "f32":
        return x
    codes, scale = _quantise(x)
    return (codes.astype(np.float32) - np.float32(128)) * scale[..., None]


class _Paged:
    """A cache with sequences of `lengths` tokens on scattered pages, some of the cache's pages left
    to no one."""

    def __init__(self, c, lengths, page, Hk, dh, format, rng, spare=2, wider=1):
        self.c, self.lengths, self.page, self.Hk, self.dh = c, list(lengths), page, Hk, dh
        need = [-(-n // page) for n in lengths]
        self.pages = max(sum(need) + spare, 1)
        order = rng.permutation(self.pages)
        self.table = np.full((len(need), max(need + [0]) + wider), -1, np.int32)
        for i, n in enumerate(need):
            self.table[i, :n], order = order[:n], order[n:]
        self.free = order
        self.cache = nr.KVCache(self.pages, page, Hk, dh, format, ctx=c)
        # what no one has written must not matter
        if format == "f32":
            for a in (self.cache.k, self.cache.v):
                a.fill(float("nan"))
        else:
            for a in (self.cache.k, self.cache.v):
                a.upload(np.full(a.shape, 77, np.uint8))
            for a in (self.cache.k_scale, self.cache.v_scale):
                a.fill(float("nan"))
        self.td, self.ends = c.to_device(self.table), c.to_device(np.array(lengths, np.int32))
        self.seqs = nr.PackedSequences(lengths, ctx=c)

    def raw(self):
        return [a.numpy() for a in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale)
                if a is not None]


SHAPES = [([1], 16, 1, 8), ([5, 0, 33, 16], 16, 2, 40), ([64, 65, 63], 64, 3, 64), ([300, 17], 32, 2, 128),
          ([200, 1], 256, 1, 96), ([7] * 9, 16, 8, 24), ([129], 128, 5, 72)]


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("lengths,page,Hk,dh", SHAPES)
def test_write_and_read(hip_ctx, lengths, page, Hk, dh, format):
    print(f"[gpu] cache {lengths} page={page} Hk={Hk} dh={dh} {format}", flush=True)
    rng = np.random.default_rng(sum(lengths) + dh)
    s, c = _Paged(hip_ctx, lengths, page, Hk, dh, format, rng), hip_ctx
    before = s.raw()
    T, w = sum(lengths), Hk * dh
    # column blocks of a wider array, off 16 bytes
    x = rand(rng, (T + 2, 2 * w + 3)) * 10.0 ** rng.integers(-3, 4, (T + 2, 1)).astype(np.float32)
    xd = c.to_device(x)
    fn = L.load().numrs_hip_kv_cache_write
    c._check(fn(c.handle, ctypes.byref(s.cache.pages), s.seqs.handle, xd.ptr + 4, xd.ptr + 4 * (1 + w),
                2 * w + 3, s.td.ptr, s.table.shape[1], s.ends.ptr))
    k, v = (x[:T, a:a + w].reshape(T, Hk, dh) for a in (1, 1 + w))
    # the whole cache: rows where the table says, everything else as it was
    want, at = [a.copy() for a in before], 0
    for i, n in enumerate(lengths):
        for r in range(n):
            p, slot = s.table[i, r // page], r % page
            if format == "f32":
                want[0][p, :, slot], want[1][p, :, slot] = k[at], v[at]
            else:
                want[0][p, :, slot], want[2][p, :, slot] = _quantise(k[at])
                codes, want[3][p, :, slot] = _quantise(v[at])
                flat = want[1].reshape(s.pages, Hk, page // 4, dh, 4)
                flat[p, :, slot // 4, :, slot % 4] = codes
            at += 1
    for got, ref, name in zip(s.raw(), want, ("keys", "values", "key scales", "value scales")):
        assert np.array_equal(got, ref, equal_nan=got.dtype == np.float32), name
    rk, rv = s.cache.read(s.seqs, s.td, s.ends)
    assert_bits(rk.numpy(), _stands_for(k, format).reshape(T, w), "k")
    assert_bits(rv.numpy(), _stands_for(v, format).reshape(T, w), "v")


def test_quantised_borders(hip_ctx):
    """Rows of zeros, of one value, of subnormals and of fp32's largest, halves between two codes,
    and rows that are not finite."""
    rng = np.random.default_rng(1)
    s = _Paged(hip_ctx, [12], 16, 1, 16, "int8", rng)
    x = np.zeros((12, 16), np.float32)
    x[1, 3] = -5
    x[2] = 127
    x[3] = np.arange(16) - 7.5 + 0.0
    x[3, 0] = 127  # scale 1: halves, to even
    x[4] = 1e-45
    x[5] = rng.standard_normal(16) * 1e-43
    x[6] = np.float32(3.4028235e38)
    x[6, ::2] *= -1
    x[7, 2] = np.inf
    x[8, 9] = np.nan
    x[9] = -0.0
    x[10] = rng.standard_normal(16) * 1e38
    x[11, 5] = np.float32(1.1754944e-38)
    d = hip_ctx.to_device(x)
    s.cache.write(s.seqs, d, d, s.td, s.ends)
    k, v = (a.numpy() for a in s.cache.read(s.seqs, s.td, s.ends))
    codes, scale = _quantise(x)
    want = (codes.astype(np.float32) - 128) * scale[:, None]
    for got in (k, v):
        assert np.isnan(got[7:9]).all()
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_positions_and_pages_outside(hip_ctx, format):
    """Pages that the cache lacks, positions before the first and past the table: nothing is
    written there, and reads are zeros."""
    c, rng, page, Hk, dh = hip_ctx, np.random.default_rng(2), 16, 2, 24
    s = _Paged(c, [40, 40, 40, 40], page, Hk, dh, format, rng, wider=0)
    table = s.table.copy()
    table[0, 1], table[1, 0], table[2, 2] = -1, s.pages, 2**31 - 1
    td = c.to_device(table)
    ends = np.array([40, 45, 30, 2**31 - 1], np.int32)  # 45: to 44; 30: from -10; the last: all past
    ed = c.to_device(ends)
    x = rand(rng, (160, Hk * dh))
    xd, before = c.to_device(x), s.raw()
    s.cache.write(s.seqs, xd, xd, td, ed)
    ok = np.zeros((4, 40), bool)
    for i in range(4):
        for r in range(40):
            pos = int(ends[i]) - 40 + r
            ok[i, r] = 0 <= pos < 48 and 0 <= table[i, pos // 16] < s.pages
    # 0: a page of 16 missing; 1: positions 5..44 less 0..15; 2: -10..29, page 2 is not reached; 3: none
    assert ok.sum(1).tolist() == [24, 29, 30, 0]
    k, v = (a.numpy().reshape(4, 40, Hk, dh) for a in s.cache.read(s.seqs, td, ed))
    want = np.where(ok[..., None, None], _stands_for(x.reshape(4, 40, Hk, dh), format), 0)
    assert_bits(k, want, "k")
    assert_bits(v, want, "v")
    after = s.raw()
    changed = {p for p in range(s.pages) if not np.array_equal(before[0][p], after[0][p], equal_nan=format == "f32")}
    pos = lambda i, r: int(ends[i]) - 40 + r  # noqa: E731
    assert changed == {table[i, pos(i, r) // 16] for i in range(4) for r in range(40) if ok[i, r]}


def _attention(q, k, v, Hk):
    """One row over tokens k, v [n, Hk, dh]: result and the bound of its error."""
    H, dh = q.shape
    out, err = np.zeros((H, dh)), np.zeros((H, dh))
    for h in range(H if len(k) else 0):
        K, V, Q = (x.astype(np.float64) for x in (k[:, h // (H // Hk)], v[:, h // (H // Hk)], q[h]))
        s = K @ Q / math.sqrt(dh)
        p = np.exp(s - s.max())
        p /= p.sum()
        e = U2 * (dh + 8) * (abs(K) @ abs(Q)).max() / math.sqrt(dh)
        out[h] = p @ V
        err[h] = (2 * e + 2 * U2 * (len(k) + 8)) * (p @ abs(V))
    return out, err


def _check(got, ref, err, what):
    d = abs(got - ref)
    assert (d <= err).all(), f"{what}: outside its bound by {(d / (err + 1e-300)).max():.2g}"
    rel = np.linalg.norm(d) / max(np.linalg.norm(ref), 1e-300)
    assert rel <= 2e-6, f"{what}: 2-norm error {rel:.2g}"


# Groups of 1 to 40 query heads, lengths of 0 and 1, ends inside, at and past a page, one of many
# pages, many rows of few.
PAGED = [([1], 16, 1, 1, 8), ([0, 1, 15, 16, 17], 16, 4, 2, 40), ([333], 16, 8, 8, 64),
         ([1000, 3, 0, 250], 64, 16, 2, 128), ([129, 511], 128, 10, 2, 80), ([70] * 40, 32, 8, 4, 64),
         ([20000], 256, 8, 1, 128), ([300, 40], 16, 17, 1, 24), ([9000, 5, 77], 64, 40, 1, 64),
         ([255], 16, 64, 2, 96), ([2048, 4097], 1024, 12, 3, 72)]


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("lengths,page,H,Hk,dh", PAGED)
def test_attention_paged(hip_ctx, lengths, page, H, Hk, dh, format):
    print(f"[gpu] paged {lengths[:6]} page={page} H={H} Hk={Hk} dh={dh} {format}", flush=True)
    c, rng = hip_ctx, np.random.default_rng(sum(lengths) + H)
    s, n, T, w = _Paged(c, lengths, page, Hk, dh, format, rng), len(lengths), sum(lengths), Hk * dh
    k, v = rand(rng, (T, w)), rand(rng, (T, w))
    s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
    q = rand(rng, (n + 1, H * dh + 5))
    qd, out = c.to_device(q), c.to_device(np.full((n + 1, H * dh + 3), 7, np.float32))
    call = lambda: c._check(L.load().numrs_hip_attention_paged(  # noqa: E731
        c.handle, ctypes.byref(s.cache.pages), qd.ptr + 4, H * dh + 5, H, s.td.ptr, s.table.shape[1],
        s.ends.ptr, n, out.ptr + 8, H * dh + 3))
    call()
    got = out.numpy()
    assert (got[:, :2] == 7).all() and (got[:, 2 + H * dh:] == 7).all() and (got[n] == 7).all()
    k, v = (_stands_for(x.reshape(T, Hk, dh), format) for x in (k, v))
    at = 0
    for i, m in enumerate(lengths):
        ref, err = _attention(q[i, 1:1 + H * dh].reshape(H, dh), k[at:at + m], v[at:at + m], Hk)
        if m == 0:
            assert (got[i, 2:2 + H * dh] == 0).all()
        else:
            _check(got[i, 2:2 + H * dh].reshape(H, dh), ref, err, f"row {i}")
        at += m
    call()
    assert_bits(out.numpy(), got, "the same call again")


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_attention_over_bad_tables(hip_ctx, format):
    """Lengths past the table or negative, pages that the cache lacks, one page in two tables."""
    c, rng, page, H, Hk, dh = hip_ctx, np.random.default_rng(3), 16, 6, 2, 32
    lengths = [64, 64, 64, 64, 64]
    s = _Paged(c, lengths, page, Hk, dh, format, rng, wider=0)
    T = sum(lengths)
    k, v = rand(rng, (T, Hk * dh)), rand(rng, (T, Hk * dh))
    s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
    k, v = (_stands_for(x.reshape(5, 64, Hk, dh), format) for x in (k, v))
    table = s.table.copy()
    table[0, 2], table[1, 0] = -3, s.pages
    table[2, 1] = table[3, 0]
    table[4] = -1
    use = np.array([64, 50, 1000, -7, 64], np.int32)
    q = rand(rng, (5, H * dh))
    out = c.empty((5, H * dh))
    td, ud, qd = c.to_device(table), c.to_device(use), c.to_device(q)
    c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(s.cache.pages), qd.ptr, H * dh, H, td.ptr,
                                                4, ud.ptr, 5, out.ptr, H * dh))
    got = out.numpy().reshape(5, H, dh)
    sees = [(0, list(range(32)) + list(range(48, 64))), (1, range(16, 50)), (2, range(64))]
    for i, rows in sees:
        K, V = k[i, list(rows)].copy(), v[i, list(rows)].copy()
        if i == 2:
            K[16:32], V[16:32] = k[3, :16], v[3, :16]
        _check(got[i], *_attention(q[i].reshape(H, dh), K, V, Hk), f"row {i}")
    assert (got[3:] == 0).all()


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_special_values(hip_ctx, format):
    """A NaN key or value reaches its own sequence and head only; infinite keys and values do what
    fp32 arithmetic does with them."""
    c, rng, H, Hk, dh, lengths = hip_ctx, np.random.default_rng(4), 4, 2, 64, [100, 90, 80]
    s = _Paged(c, lengths, 16, Hk, dh, format, rng)
    T = sum(lengths)
    k, v, q = rand(rng, (T, Hk * dh)), rand(rng, (T, Hk * dh)), rand(rng, (3, H * dh))
    qd, out = c.to_device(q), c.empty((3, H * dh))

    def run(k, v):
        s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
        c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(s.cache.pages), qd.ptr, H * dh, H,
                                                    s.td.ptr, s.table.shape[1], s.ends.ptr, 3, out.ptr, H * dh))
        return out.numpy().reshape(3, Hk, 2, dh)

    clean = run(k, v)
    k2, v2 = k.copy(), v.copy()
    k2[50, 3] = np.nan        # sequence 0, head 0
    v2[120, dh + 5] = np.inf  # sequence 1, head 1
    got = run(k2, v2)
    assert np.isnan(got[0, 0]).all()
    if format == "f32":
        assert np.isposinf(got[1, 1, :, 5]).all()
        rest = np.arange(dh) != 5
        assert_bits(got[1, 1][:, rest], clean[1, 1][:, rest])
    else:
        assert np.isnan(got[1, 1]).all()  # the row reads back as NaN
    for i, h in ((0, 1), (1, 0), (2, 0), (2, 1)):
        assert_bits(got[i, h], clean[i, h])


def test_large_magnitudes(hip_ctx):
    """Scores far apart (a softmax that is one token's), tiny and huge values."""
    c, rng, H, Hk, dh, n = hip_ctx, np.random.default_rng(5), 4, 1, 64, 500
    for sq, sk, sv in ((30, 30, 1), (1e-20, 1e20, 1e30), (1, 1, 1e-36), (0, 1, 1), (1e10, 1e-10, 1)):
        for format in ("f32", "int8"):
            s = _Paged(c, [n], 64, Hk, dh, format, rng)
            k, v = rand(rng, (n, dh)) * np.float32(sk), rand(rng, (n, dh)) * np.float32(sv)
            q = rand(rng, (1, H * dh)) * np.float32(sq)
            s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
            out, qd = c.empty((1, H * dh)), c.to_device(q)
            c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(s.cache.pages), qd.ptr, H * dh, H,
                                                        s.td.ptr, s.table.shape[1], s.ends.ptr, 1, out.ptr, H * dh))
            k, v = (_stands_for(x.reshape(n, 1, dh), format) for x in (k, v))
            ref, err = _attention(q.reshape(H, dh), k, v, Hk)
            d = abs(out.numpy().reshape(H, dh) - ref)
            assert (d <= err + 1e-44).all(), (sq, sk, sv, format, (d / (err + 1e-300)).max())


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_scores_near_the_lowest(hip_ctx, format):
    """Equal scores of -3.5e32: the mean of the values, as for any other score."""
    c, rng, n, dh = hip_ctx, np.random.default_rng(14), 300, 8
    s = _Paged(c, [n], 16, 1, dh, format, rng)
    k, v = np.zeros((n, dh), np.float32), rand(rng, (n, dh))
    k[:, 3] = -1e16
    q = np.zeros((1, dh), np.float32)
    q[0, 3] = 1e17
    s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
    out, qd = c.empty((1, dh)), c.to_device(q)
    c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(s.cache.pages), qd.ptr, dh, 1, s.td.ptr,
                                                s.table.shape[1], s.ends.ptr, 1, out.ptr, dh))
    v = _stands_for(v.reshape(n, 1, dh), format)[:, 0].astype(np.float64)
    assert (abs(out.numpy()[0] - v.mean(0)) <= 2 * U2 * (n + 8) * abs(v).mean(0)).all()


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_more_sequences_than_a_workgroup_looks_at_once(hip_ctx, format):
    """1300 sequences, most short, some empty, one long behind the first thousand: also the same twice."""
    c, rng, page, H, Hk, dh = hip_ctx, np.random.default_rng(15), 16, 8, 2, 64
    lengths = rng.integers(0, 40, 1300).tolist()
    lengths[0], lengths[511], lengths[512], lengths[1100], lengths[1299] = 0, 130, 0, 2500, 65
    s, n, T, w = _Paged(c, lengths, page, Hk, dh, format, rng), 1300, sum(lengths), Hk * dh
    k, v, q = rand(rng, (T, w)), rand(rng, (T, w)), rand(rng, (n, H * dh))
    s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
    out, qd = c.empty((n, H * dh)), c.to_device(q)
    call = lambda: c._check(L.load().numrs_hip_attention_paged(  # noqa: E731
        c.handle, ctypes.byref(s.cache.pages), qd.ptr, H * dh, H, s.td.ptr, s.table.shape[1], s.ends.ptr, n,
        out.ptr, H * dh))
    call()
    got = out.numpy()
    k, v = (_stands_for(x.reshape(T, Hk, dh), format) for x in (k, v))
    at = np.concatenate([[0], np.cumsum(lengths)])
    for i in range(n):
        ref, err = _attention(q[i].reshape(H, dh), k[at[i]:at[i + 1]], v[at[i]:at[i + 1]], Hk)
        if lengths[i] == 0:
            assert (got[i] == 0).all(), i
        else:
            _check(got[i].reshape(H, dh), ref, err, f"row {i}")
    call()
    assert_bits(out.numpy(), got)


def test_refusals(hip_ctx):
    c, lib, rng = hip_ctx, L.load(), np.random.default_rng(6)
    s = _Paged(c, [5, 3], 16, 2, 16, "int8", rng)
    x = c.to_device(rand(rng, (8, 32)))
    h, cp = c.handle, ctypes.byref(s.cache.pages)
    for fn in (lib.numrs_hip_kv_cache_write, lib.numrs_hip_kv_cache_read):
        good = [h, cp, s.seqs.handle, x.ptr, x.ptr, 32, s.td.ptr, 2, s.ends.ptr]
        assert fn(*good) == 0
        for i, value, code in ((1, None, L.E_INVALID), (2, None, L.E_INVALID), (3, None, L.E_INVALID),
                               (4, None, L.E_INVALID), (5, 31, L.E_SHAPE), (6, None, L.E_INVALID),
                               (7, 0, L.E_SHAPE), (8, None, L.E_INVALID)):
            bad = list(good)
            bad[i] = value
            assert fn(*bad) == code, i
            assert lib.numrs_hip_last_error(h)
    wide = nr.KVPages.from_buffer_copy(s.cache.pages)
    wide.kv_heads, wide.head_dim, wide.pages = 65535, 8, 1
    long = nr.PackedSequences([64 * 256 + 1], ctx=c)  # more work than a launch can have
    assert lib.numrs_hip_kv_cache_write(h, ctypes.byref(wide), long.handle, x.ptr, x.ptr, 524280, s.td.ptr, 2,
                                        s.ends.ptr) == L.E_SHAPE
    assert b"too many" in lib.numrs_hip_last_error(h)
    fn = lib.numrs_hip_attention_paged
    good = [h, cp, x.ptr, 64, 4, s.td.ptr, 2, s.ends.ptr, 2, x.ptr + 512, 64]
    for i, value, code in ((1, None, L.E_INVALID), (2, None, L.E_INVALID), (3, 63, L.E_SHAPE), (4, 3, L.E_SHAPE),
                           (4, 0, L.E_SHAPE), (5, None, L.E_INVALID), (6, 0, L.E_SHAPE), (7, None, L.E_INVALID),
                           (8, -1, L.E_INVALID), (9, None, L.E_INVALID), (10, 63, L.E_SHAPE)):
        bad = list(good)
        bad[i] = value
        assert fn(*bad) == code, i
    bad = nr.KVPages.from_buffer_copy(s.cache.pages)
    bad.page_size = 24
    assert fn(h, ctypes.byref(bad), *good[2:]) == L.E_SHAPE
    assert fn(h, cp, None, 64, 4, None, 2, None, 0, None, 64) == 0  # no rows
    with pytest.raises(ValueError):
        nr.KVCache(1, 16, 1, 16, "bf16", ctx=c)
    with pytest.raises(ValueError):
        s.cache.write(s.seqs, x, x, s.ends, s.td)
    with pytest.raises(ValueError):
        s.cache.write(s.seqs, x, c.empty((8, 16)), s.td, s.ends)
    with pytest.raises(ValueError):
        s.cache.write(s.seqs, x, x, c.to_device(rand(rng, (2, 2))), s.ends)
    t = nr.Tensor.new(rand(rng, (2, 64)), True, ctx=c)
    with pytest.raises(nr.HipError, match="no backward"):
        t.attention_paged(s.cache, 4, s.td, s.ends)
    with pytest.raises(nr.HipError):
        nr.Tensor.new(rand(rng, (2, 60)), ctx=c).attention_paged(s.cache, 4, s.td, s.ends)
    with nr.Context(0) as other, pytest.raises(ValueError, match="one context"):
        nr.Tensor.new(rand(rng, (2, 64)), ctx=other).attention_paged(s.cache, 4, s.td, s.ends)


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_more_tokens_than_the_caches_hold(hip_ctx, format):
    """600 sequences of up to 4096 tokens on the same pages, 1.2 GB and more read by one call."""
    c, rng, page, H, Hk, dh, n = hip_ctx, np.random.default_rng(19), 64, 4, 2, 128, 600
    s = _Paged(c, [4096], page, Hk, dh, format, rng, wider=0)
    k, v = rand(rng, (4096, Hk * dh)), rand(rng, (4096, Hk * dh))
    s.cache.write(s.seqs, c.to_device(k), c.to_device(v), s.td, s.ends)
    k, v = (_stands_for(x.reshape(4096, Hk, dh), format) for x in (k, v))
    lengths = rng.integers(3900, 4097, n).astype(np.int32)
    lengths[17], lengths[18] = 1, 0
    q, out = rand(rng, (n, H * dh)), c.empty((n, H * dh))
    td, ends, qd = c.to_device(np.repeat(s.table, n, 0)), c.to_device(lengths), c.to_device(q)
    c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(s.cache.pages), qd.ptr, H * dh, H, td.ptr,
                                                s.table.shape[1], ends.ptr, n, out.ptr, H * dh))
    got = out.numpy().reshape(n, H, dh)
    assert (got[18] == 0).all()
    for i in [0, 16, 17, 19, 300, 598, 599]:
        m = lengths[i]
        _check(got[i], *_attention(q[i].reshape(H, dh), k[:m], v[:m], Hk), f"row {i}")
    # the others against float64 without the bound's arithmetic: the same 2-norm
    K, V, Q = k.astype(np.float64), v.astype(np.float64), q.reshape(n, H, dh).astype(np.float64)
    for h in range(H):
        sc = Q[:, h] @ K[:, h // 2].T / math.sqrt(dh)
        sc[np.arange(4096)[None] >= lengths[:, None]] = -np.inf
        p = np.exp(sc - sc.max(1, keepdims=True, where=np.isfinite(sc), initial=-1e30))
        ref = p @ V[:, h // 2] / np.maximum(p.sum(1, keepdims=True), 1e-300)
        err = np.linalg.norm(got[:, h] - ref, axis=1) / np.maximum(np.linalg.norm(ref, axis=1), 1e-300)
        assert np.delete(err, 18).max() <= 2e-6


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_pages_past_32_bits(hip_ctx, format):
    """A cache of 2.2e9 values: pages whose elements, and bytes, lie past 2^31 and 2^32."""
    c, rng, page, Hk, dh, H = hip_ctx, np.random.default_rng(16), 1024, 2, 128, 6
    pages = 2 ** 31 // (page * Hk * dh) + 10
    cache = nr.KVCache(pages, page, Hk, dh, format, ctx=c)
    # around 2^31 and 2^32 bytes of fp32 and around 2^31 values, and the last
    table = np.array([[pages - 1, pages // 2, 3], [pages // 4, pages - 2, pages // 2 + 1], [0, pages - 9, 1]], np.int32)
    lengths = [2500, 2049, 1100]
    td, ends, seqs = c.to_device(table), c.to_device(np.array(lengths, np.int32)), nr.PackedSequences(lengths, ctx=c)
    T = sum(lengths)
    k, v, q = rand(rng, (T, Hk * dh)), rand(rng, (T, Hk * dh)), rand(rng, (3, H * dh))
    cache.write(seqs, c.to_device(k), c.to_device(v), td, ends)
    k, v = (_stands_for(x.reshape(T, Hk, dh), format) for x in (k, v))
    got = [a.numpy().reshape(T, Hk, dh) for a in cache.read(seqs, td, ends)]
    assert_bits(got[0], k)
    assert_bits(got[1], v)
    out, qd = c.empty((3, H * dh)), c.to_device(q)
    c._check(L.load().numrs_hip_attention_paged(c.handle, ctypes.byref(cache.pages), qd.ptr, H * dh, H, td.ptr, 3,
                                                ends.ptr, 3, out.ptr, H * dh))
    got, at = out.numpy().reshape(3, H, dh), np.concatenate([[0], np.cumsum(lengths)])
    for i in range(3):
        _check(got[i], *_attention(q[i].reshape(H, dh), k[at[i]:at[i + 1]], v[at[i]:at[i + 1]], Hk), f"row {i}")


# ---------------------------------------------------------------------------
# A conversation: prompts, then a token at a time
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_prompt_and_steps(hip_ctx, format):
    """A module's prompts and then its tokens one by one, eager and as a replayed graph: with an
    fp32 cache each step is the packed forward's row of the whole sequence; with an 8-bit one it is
    the attention over what the cache stands for."""
    before = nr.default_context()
    nr.set_default_context(hip_ctx)
    try:
        c, rng, d, H, Hk, dh = hip_ctx, np.random.default_rng(12), 64, 4, 2, 32
        w = [rand(rng, s, 0.2) for s in ((H * dh, d), (Hk * dh, d), (Hk * dh, d), (d, H * dh))]
        attn = nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk)
        lens, steps, page = [17, 1, 48, 30], 20, 16
        whole = [n + steps for n in lens]
        s = _Paged(c, whole, page, Hk, dh, format, rng)
        x = [rand(rng, (n, d)) for n in whole]
        ends = np.array(lens, np.int32)
        ed = c.to_device(ends)
        prompts, ones = nr.PackedSequences(lens), nr.PackedSequences([1] * 4)
        full = attn.forward_packed(nr.Tensor.new(np.concatenate(x)), nr.PackedSequences(whole)).values()
        full = np.split(full, np.cumsum(whole)[:-1])
        with nr.no_grad():
            y = attn.prefill(nr.Tensor.new(np.concatenate([a[:n] for a, n in zip(x, lens)])), prompts,
                             s.cache, s.td, ed).values()
            y = np.split(y, np.cumsum(lens)[:-1])
            for i, n in enumerate(lens):
                assert np.abs(y[i] - full[i][:n]).max() <= 1e-5
            x1 = nr.Tensor.new(np.zeros((4, d), np.float32))
            xd = nr.DeviceArray(c, x1.device_ptrs()[0], (4, d), owned=False, base=x1)
            step = lambda: attn.decode(x1, ones, s.cache, s.td, ed)  # noqa: E731
            graph = None
            for t in range(steps):
                ends = ends + 1
                ed.upload(ends)
                xd.upload(np.stack([a[n + t] for a, n in zip(x, lens)]))
                if t == 5:
                    graph = nr.StepGraph(c, step)
                if graph:
                    graph.replay()
                    got = graph.outputs.values()
                else:
                    got = step().values()
                if format == "f32":
                    want = np.stack([full[i][n + t] for i, n in enumerate(lens)])
                    # two orders of the same fp32 sums over values of order 1
                    assert np.abs(got - want).max() <= 1e-5, t
                else:
                    qkv = attn.qkv(x1).values()
                    now = nr.PackedSequences(ends.tolist())
                    k, v = (a.numpy().reshape(-1, Hk, dh) for a in s.cache.read(now, s.td, ed))
                    at = np.concatenate([[0], np.cumsum(ends)])
                    a = np.stack([_attention(qkv[i, :H * dh].reshape(H, dh), k[at[i]:at[i + 1]], v[at[i]:at[i + 1]],
                                             Hk)[0].reshape(-1) for i in range(4)])
                    assert np.abs(got - a @ w[3].T.astype(np.float64)).max() <= 1e-5, t
            graph.close()
    finally:
        nr.set_default_context(before)
