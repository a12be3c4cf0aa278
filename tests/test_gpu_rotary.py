"""Query and key heads normed and rotated, forward and backward and on the way into a paged cache,
against numpy in 80 bits.  The kernels work in 64 bits and round once, so a result is within half a step
of fp32 of the formula's, and besides within what 64 bits leave of an angle (two roundings of the
frequency in circles, one of the product) and of the sums."""
import ctypes

import numpy as np
import pytest

import numrs_amd as nr
from conftest import assert_bits, rand
from numrs_amd import _lib as L
from numrs_amd import nn
from test_gpu_chunk import _rows
from test_gpu_kvcache import _Paged, _quantise

pytestmark = pytest.mark.gpu

LD = np.longdouble
HALF, U64 = 2.0 ** -24, 2.0 ** -53
EPS = 1e-6


def _turn(x, pos, rot, back=False):
    """x [T, heads, dh] in 80 bits, turned, and the size of what 64 bits leave of it."""
    y, off = x.copy(), np.zeros(x.shape, LD)
    n = rot.dims
    angle = LD(1) * np.asarray(pos, LD)[:, None] * rot.freqs.astype(LD)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    if back:
        s = -s
    i = np.arange(n // 2)
    a, b = (i, n // 2 + i) if rot.layout == "halves" else (2 * i, 2 * i + 1)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    err = (4 * abs(angle)[:, None] + 16) * U64 * (abs(x[..., a]) + abs(x[..., b]))
    off[..., a], off[..., b] = err, err
    return y, off


def _norm(x, w, eps=EPS):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + LD(np.float32(eps)))
    return x * r, r


class _Case:
    def __init__(self, lengths, H, Hk, dh, rng, dims=None, layout="halves", base=10000.0, norm="qk", starts=None):
        self.lengths, self.H, self.Hk, self.dh = lengths, H, Hk, dh
        self.T, self.W = sum(lengths), (H + 2 * Hk) * dh
        self.rot = nr.Rotary(dh, dims, base, layout) if dims != 0 else None
        self.starts = starts or [0] * len(lengths)
        self.pos = np.concatenate([np.arange(s, s + n) for n, s in zip(lengths, self.starts)] + [np.zeros(0, int)])
        self.x = rand(rng, (self.T, self.W))
        self.wq = rand(rng, dh, 0.3) + np.float32(1) if "q" in norm else None
        self.wk = rand(rng, dh, 0.3) + np.float32(1) if "k" in norm else None

    def heads(self, x):
        return x.reshape(self.T, -1, self.dh)

    def forward(self):
        """The result [T, W] in 80 bits and its bound."""
        x = self.heads(self.x).astype(LD)
        y, off = x.copy(), np.zeros(x.shape, LD)
        for part, w in ((slice(0, self.H), self.wq), (slice(self.H, self.H + self.Hk), self.wk)):
            z = x[:, part]
            if w is not None:
                z = _norm(z, w)[0] * w.astype(LD)
            e = 32 * U64 * abs(z)
            if self.rot is not None:
                y[:, part], more = _turn(z, self.pos, self.rot)
                off[:, part] = e.max(-1, keepdims=True) + more
            else:
                y[:, part], off[:, part] = z, e
        return y.reshape(self.T, self.W), (off + HALF * abs(y) + 2.0 ** -149).reshape(self.T, self.W)

    def backward(self, dy):
        """dx, dwq, dwk and their bounds."""
        x, g = self.heads(self.x).astype(LD), self.heads(dy).astype(LD)
        dx, off, dw = g.copy(), np.zeros(g.shape, LD), []
        for part, w in ((slice(0, self.H), self.wq), (slice(self.H, self.H + self.Hk), self.wk)):
            z, e = g[:, part], np.zeros(g[:, part].shape, LD)
            if self.rot is not None:
                z, e = _turn(z, self.pos, self.rot, back=True)
            if w is not None:
                xh, r = _norm(x[:, part], w)
                terms = z * xh
                sure = (abs(terms) * 64 * U64 + e * abs(xh)).sum((0, 1)) + self.T * U64 * abs(terms).sum((0, 1))
                dw.append((terms.sum((0, 1)), sure))
                gw = z * w.astype(LD)
                dot = (gw * xh).mean(-1, keepdims=True)
                size = abs(gw).max(-1, keepdims=True) * (1 + abs(xh) * abs(xh).max(-1, keepdims=True))
                z, e = r * (gw - xh * dot), r * (64 * U64 * size + 4 * e.max(-1, keepdims=True) * (1 + abs(xh) ** 2) * abs(w).max())
            else:
                dw.append(None)
            dx[:, part], off[:, part] = z, e
        return (dx.reshape(self.T, self.W), (off + HALF * abs(dx) + 2.0 ** -149).reshape(self.T, self.W)), dw


def _close(got, ref, err, what):
    d = abs(got.astype(LD) - ref)
    assert (d <= err).all(), f"{what}: off by {float((d / err).max()):.3g} of the bound"


def _d(c, a):
    return c.to_device(a) if a is not None else None


def _p(a):
    return a.ptr if a is not None else None


# One lane a head to sixteen, heads that fill their lanes and not, parts of a head turned, tiles of one
# token, rows of 64 and more, one weight of the two, no rotation, far positions.
CASES = [
    dict(lengths=[1], H=1, Hk=1, dh=8),
    dict(lengths=[3, 0, 65, 64, 1], H=6, Hk=2, dh=16, layout="pairs"),
    dict(lengths=[70], H=3, Hk=3, dh=24, dims=16, norm=""),
    dict(lengths=[33, 129], H=4, Hk=1, dh=40, dims=8, norm="q"),
    dict(lengths=[200, 5], H=8, Hk=2, dh=64, norm="", layout="pairs"),
    dict(lengths=[17] * 9, H=10, Hk=2, dh=80, dims=40),
    dict(lengths=[260], H=2, Hk=2, dh=96, dims=0),
    dict(lengths=[130, 61], H=16, Hk=4, dh=128, base=1e6),
    dict(lengths=[64, 2], H=5, Hk=5, dh=120, dims=64, layout="pairs", norm="k"),
    dict(lengths=[40, 9], H=4, Hk=2, dh=64, starts=[2**31 - 41, 10**6], norm="qk"),
    dict(lengths=[12, 5], H=4, Hk=4, dh=128, starts=[131000, -3], layout="pairs"),
    dict(lengths=[2500, 1111], H=8, Hk=1, dh=128),
]


@pytest.mark.parametrize("i", range(len(CASES)))
def test_forward_backward(hip_ctx, i):
    print(f"[gpu] rotary {CASES[i]}", flush=True)
    c, rng, lib = hip_ctx, np.random.default_rng(i), L.load()
    t = _Case(rng=rng, **CASES[i])
    T, W, H, Hk, dh = t.T, t.W, t.H, t.Hk, t.dh
    seqs = nr.PackedSequences(t.lengths, ctx=c)
    ends = _d(c, np.array([n + s for n, s in zip(t.lengths, t.starts)], np.int64).astype(np.int32)) if any(t.starts) else None
    # strides of their own, off 16 bytes
    lx, ly, lg, ld = W + 3, W + 5, W + 1, W + 2
    pad = lambda a, ld: np.pad(a, ((0, 1), (1, ld - W - 1)), constant_values=9)  # noqa: E731
    dy = rand(rng, (T, W), 0.1)
    xd, gd = c.to_device(pad(t.x, lx)), c.to_device(pad(dy, lg))
    y, dx = c.to_device(np.full((T + 1, ly), 7, np.float32)), c.to_device(np.full((T + 1, ld), 7, np.float32))
    wq, wk = _d(c, t.wq), _d(c, t.wk)
    rot = ctypes.byref(t.rot.spec) if t.rot is not None else None
    c._check(lib.numrs_hip_qk_rotary_forward(c.handle, seqs.handle, _p(ends), xd.ptr + 4, lx, _p(wq), _p(wk), EPS, rot,
                                             y.ptr + 4, ly, H, Hk, dh))
    got = y.numpy()
    assert (got[:, 0] == 7).all() and (got[:, W + 1:] == 7).all() and (got[T] == 7).all()
    ref, err = t.forward()
    _close(got[:T, 1:W + 1], ref, err, "y")
    assert_bits(got[:T, 1 + (H + Hk) * dh:W + 1], t.x[:, (H + Hk) * dh:], "values")
    dwq, dwk = (c.to_device(np.full(dh, 5, np.float32)) if w is not None else None for w in (wq, wk))
    back = lambda acc, to, p, q: c._check(lib.numrs_hip_qk_rotary_backward(  # noqa: E731
        c.handle, seqs.handle, _p(ends), xd.ptr + 4, lx, _p(wq), _p(wk), EPS, rot, gd.ptr + 4, lg, to, ld, _p(p), _p(q),
        H, Hk, dh, acc))
    back(0, dx.ptr + 4, dwq, dwk)
    got = dx.numpy()
    assert (got[:, 0] == 7).all() and (got[:, W + 1:] == 7).all() and (got[T] == 7).all()
    (ref, err), dw = t.backward(dy)
    _close(got[:T, 1:W + 1], ref, err, "dx")
    first = [w.numpy() if w is not None else None for w in (dwq, dwk)]
    for w, r, name in zip(first, dw, ("dwq", "dwk")):
        if r is not None:
            _close(w, r[0], r[1] + HALF * abs(r[0]), name)
    # added to what is there, to the bit of one fp32 sum (the weights' in 64 bits first); and without dx
    back(7, dx.ptr + 4, dwq, dwk)
    assert_bits(dx.numpy()[:T, 1:W + 1], got[:T, 1:W + 1] + got[:T, 1:W + 1], "dx added")
    for w, a, r in zip((dwq, dwk), first, dw):
        if r is not None:
            _close(w.numpy(), r[0] + a, r[1] + HALF * abs(r[0] + a), "dw added")
    if wq is not None or wk is not None:
        again = [c.empty((dh,)) if w is not None else None for w in (wq, wk)]
        back(0, None, *again)
        for w, a in zip(again, first):
            if w is not None:
                assert_bits(w.numpy(), a, "without dx")
    # in place
    z = c.to_device(pad(t.x, lx))
    c._check(lib.numrs_hip_qk_rotary_forward(c.handle, seqs.handle, _p(ends), z.ptr + 4, lx, _p(wq), _p(wk), EPS, rot,
                                             z.ptr + 4, lx, H, Hk, dh))
    assert_bits(z.numpy()[:T, 1:W + 1], y.numpy()[:T, 1:W + 1], "in place")
    c._check(lib.numrs_hip_qk_rotary_backward(c.handle, seqs.handle, _p(ends), xd.ptr + 4, lx, _p(wq), _p(wk), EPS, rot,
                                              gd.ptr + 4, lg, gd.ptr + 4, lg, None, None, H, Hk, dh, 0))
    assert_bits(gd.numpy()[:T, 1:W + 1], got[:T, 1:W + 1], "gradient in place")


def test_sizes_and_values_that_are_not_finite(hip_ctx):
    """Rows of zeros, of tiny and of huge values; a NaN or an infinity stays in its head, and without a
    norm in its pair."""
    c, rng, lib = hip_ctx, np.random.default_rng(30), L.load()
    t = _Case([9], 2, 1, 16, rng, layout="pairs")
    sizes = np.array([0, 1e-45, 1e-30, 1e-19, 1, 1e19, 1e30, 3e37, 1], np.float32)
    t.x *= sizes[:, None]
    seqs, xd, y = nr.PackedSequences([9], ctx=c), c.to_device(t.x), c.empty(t.x.shape)
    wq, wk, rot = _d(c, t.wq), _d(c, t.wk), ctypes.byref(t.rot.spec)
    run = lambda a, b: c._check(lib.numrs_hip_qk_rotary_forward(  # noqa: E731
        c.handle, seqs.handle, None, xd.ptr, t.W, a, b, EPS, rot, y.ptr, t.W, 2, 1, 16))
    run(wq.ptr, wk.ptr)
    _close(y.numpy(), *t.forward(), "normed")
    clean = y.numpy()
    x = t.x.copy()
    x[4, 3], x[5, 17], x[6, 2 * 16 + 8] = np.nan, np.inf, -np.inf
    xd.upload(x)
    run(wq.ptr, wk.ptr)
    got = y.numpy().reshape(9, 4, 16)
    assert np.isnan(got[4, 0]).all()
    bad = np.zeros((9, 4), bool)
    bad[4, 0] = bad[5, 1] = bad[6, 2] = True
    # an infinite head's root mean square is infinite: the others of it are 0, the pair NaN
    assert np.isnan(got[5, 1, :2]).all() and (got[5, 1, 2:] == 0).all()
    assert np.isnan(got[6, 2, 8:10]).all() and (np.delete(got[6, 2], [8, 9]) == 0).all()
    assert_bits(got[~bad], clean.reshape(9, 4, 16)[~bad])
    run(None, None)
    t.wq = t.wk = None
    ref, err = t.forward()
    got, want = y.numpy(), ~np.isfinite(x)
    pair = want | want.reshape(9, -1, 2)[..., ::-1].reshape(9, -1)
    assert not np.isfinite(got[pair]).any()
    d = abs(got.astype(LD) - ref)
    assert (d[~pair] <= err[~pair]).all()


def test_one_array_as_both_weights(hip_ctx):
    c, rng, lib = hip_ctx, np.random.default_rng(31), L.load()
    t = _Case([150, 7], 4, 2, 32, rng)
    t.wk = t.wq
    dy = rand(rng, t.x.shape)
    (_, _), dw = t.backward(dy)
    seqs, xd, gd, w, g = nr.PackedSequences(t.lengths, ctx=c), c.to_device(t.x), c.to_device(dy), c.to_device(t.wq), c.empty((32,))
    for start in (0.0, 3.0):
        g.fill(start)
        c._check(lib.numrs_hip_qk_rotary_backward(
            c.handle, seqs.handle, None, xd.ptr, t.W, w.ptr, w.ptr, EPS, ctypes.byref(t.rot.spec), gd.ptr, t.W, None, t.W,
            g.ptr, g.ptr, 4, 2, 32, L.ACC_K_WEIGHT | (L.ACC_Q_WEIGHT if start else 0)))
        both = dw[0][0] + dw[1][0] + start
        _close(g.numpy(), both, dw[0][1] + dw[1][1] + 2 * HALF * (abs(both) + abs(dw[0][0] + start)), "both")


@pytest.mark.parametrize("i", [1, 3, 5, 7, 8])
@pytest.mark.parametrize("format", ["f32", "int8"])
def test_append(hip_ctx, i, format):
    """New tokens at places inside and across pages: the same bits as the rotation and the write in turn,
    nothing else of the cache touched, and close to the formula by themselves."""
    print(f"[gpu] append {CASES[i]} {format}", flush=True)
    c, rng, lib = hip_ctx, np.random.default_rng(40 + i), L.load()
    case = dict(CASES[i])
    case["starts"] = [int(a) for a in rng.integers(0, 90, len(case["lengths"]))]
    t = _Case(rng=rng, **case)
    T, W, H, Hk, dh, page = t.T, t.W, t.H, t.Hk, t.dh, 16
    total = [n + s for n, s in zip(t.lengths, t.starts)]
    s = _Paged(c, total, page, Hk, dh, format, rng)
    seqs, ends = nr.PackedSequences(t.lengths, ctx=c), s.ends
    xd, wq, wk = c.to_device(np.pad(t.x, ((0, 0), (1, 2)))), _d(c, t.wq), _d(c, t.wk)
    rot, ld = ctypes.byref(t.rot.spec), W + 3
    y = c.empty((T, W))
    c._check(lib.numrs_hip_qk_rotary_forward(c.handle, seqs.handle, ends.ptr, xd.ptr + 4, ld, _p(wq), _p(wk), EPS, rot,
                                             y.ptr, W, H, Hk, dh))
    before = s.raw()
    s.cache.write_qkv(seqs, y, H, s.td, ends)
    want = s.raw()
    for a, b in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), before):
        a.upload(b)
    q = c.to_device(np.full((T + 1, H * dh + 3), 7, np.float32))
    call = lambda qp: c._check(lib.numrs_hip_kv_cache_append(  # noqa: E731
        c.handle, ctypes.byref(s.cache.pages), seqs.handle, xd.ptr + 4, ld, _p(wq), _p(wk), EPS, rot, qp, H * dh + 3, H,
        s.td.ptr, s.table.shape[1], ends.ptr))
    call(q.ptr + 8)
    for got, ref, name in zip(s.raw(), want, ("keys", "values", "key scales", "value scales")):
        assert np.array_equal(got, ref, equal_nan=got.dtype == np.float32), name
    got, rot_y = q.numpy(), y.numpy()
    assert (got[:, :2] == 7).all() and (got[:, 2 + H * dh:] == 7).all() and (got[T] == 7).all()
    assert_bits(got[:T, 2:2 + H * dh], rot_y[:, :H * dh], "q")
    ref, err = t.forward()
    _close(rot_y, ref, err, "y")
    if format == "int8":  # the scale of the rounded row, as the format has it
        k = rot_y[:, H * dh:(H + Hk) * dh].reshape(T, Hk, dh)
        codes, scale = _quantise(k)
        back = s.cache.read(seqs, s.td, ends)[0].numpy().reshape(T, Hk, dh)
        assert_bits(back, (codes.astype(np.float32) - 128) * scale[..., None])
    # keys and values only
    for a, b in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), before):
        a.upload(b)
    call(None)
    for got, ref in zip(s.raw(), want):
        assert np.array_equal(got, ref, equal_nan=got.dtype == np.float32)


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_append_outside(hip_ctx, format):
    """Positions before the first, past the table and on pages that the cache lacks are not written; the
    queries are there all the same, at their positions."""
    c, rng, H, Hk, dh, page = hip_ctx, np.random.default_rng(50), 4, 2, 24, 16
    s = _Paged(c, [40] * 4, page, Hk, dh, format, rng, wider=0)
    table = s.table.copy()
    table[0, 1], table[1, 0], table[2, 2] = -1, s.pages, 2**31 - 1
    ends = np.array([40, 45, 30, 2**31 - 1], np.int64)
    t = _Case([40] * 4, H, Hk, dh, rng, dims=16, starts=[int(e) - 40 for e in ends])
    td, ed, xd = c.to_device(table), c.to_device(ends.astype(np.int32)), c.to_device(t.x)
    q, before = c.empty((160, H * dh)), s.raw()
    wq, wk = _d(c, t.wq), _d(c, t.wk)
    c._check(L.load().numrs_hip_kv_cache_append(
        c.handle, ctypes.byref(s.cache.pages), s.seqs.handle, xd.ptr, t.W, wq.ptr, wk.ptr, EPS, ctypes.byref(t.rot.spec),
        q.ptr, H * dh, H, td.ptr, 3, ed.ptr))
    ref, err = t.forward()
    _close(q.numpy(), ref[:, :H * dh], err[:, :H * dh], "q")
    ok = np.array([[0 <= e - 40 + r < 48 and 0 <= table[i, (e - 40 + r) // 16] < s.pages for r in range(40)]
                   for i, e in enumerate(ends)])
    assert ok.sum(1).tolist() == [24, 29, 30, 0]
    k = s.cache.read(s.seqs, td, ed)[0].numpy().reshape(4, 40, -1)
    assert (k[~ok] == 0).all() and (abs(k[ok]).max(-1) > 0).all()
    changed = {p for p in range(s.pages) if not np.array_equal(before[0][p], s.raw()[0][p], equal_nan=format == "f32")}
    assert changed == {table[i, (e - 40 + r) // 16] for i, e in enumerate(ends) for r in range(40) if ok[i, r]}


def test_recorded_and_replayed(hip_ctx):
    """Forward, backward and append in a graph, whose sequences and rotation are gone by its replays."""
    c, rng, lib = hip_ctx, np.random.default_rng(60), L.load()
    t = _Case([70, 3, 130], 4, 2, 64, rng)
    T, W, H, Hk, dh = t.T, t.W, t.H, t.Hk, t.dh
    seqs, s = nr.PackedSequences(t.lengths, ctx=c), _Paged(c, t.lengths, 16, Hk, dh, "int8", rng)
    xd, gd, wq, wk = c.to_device(t.x), c.to_device(rand(rng, (T, W))), _d(c, t.wq), _d(c, t.wk)
    y, dx, q, dwq, dwk = c.empty((T, W)), c.empty((T, W)), c.empty((T, H * dh)), c.empty((dh,)), c.empty((dh,))
    rot = nr.Rotary(dh)

    def step():
        r = ctypes.byref(rot.spec)
        c._check(lib.numrs_hip_qk_rotary_forward(c.handle, seqs.handle, None, xd.ptr, W, wq.ptr, wk.ptr, EPS, r, y.ptr, W,
                                                 H, Hk, dh))
        c._check(lib.numrs_hip_qk_rotary_backward(c.handle, seqs.handle, None, xd.ptr, W, wq.ptr, wk.ptr, EPS, r, gd.ptr,
                                                  W, dx.ptr, W, dwq.ptr, dwk.ptr, H, Hk, dh, 0))
        c._check(lib.numrs_hip_kv_cache_append(c.handle, ctypes.byref(s.cache.pages), seqs.handle, xd.ptr, W, wq.ptr,
                                               wk.ptr, EPS, r, q.ptr, H * dh, H, s.td.ptr, s.table.shape[1], s.ends.ptr))

    outs = [y, dx, q, dwq, dwk, s.cache.k_scale]
    step()
    graph, wants = nr.StepGraph(c, step), []
    xs = [rand(rng, (T, W)) for _ in range(3)]
    for x in xs:
        xd.upload(x)
        step()
        wants.append([a.numpy() for a in outs])
    seqs.close()
    rot.freqs[:] = 0.5
    del rot
    filler = [nr.PackedSequences([130, 70, 3], ctx=c) for _ in range(3)]
    for x, want in zip(xs, wants):
        xd.upload(x)
        for a in outs:
            a.fill(float("nan"))  # as the scales of slots without a token are
        graph.replay()
        for a, w in zip(outs, want):
            assert_bits(a.numpy(), w)
    graph.close()
    del filler


def test_refusals(hip_ctx):
    c, lib, rng = hip_ctx, L.load(), np.random.default_rng(70)
    seqs, x, y, w = nr.PackedSequences([8], ctx=c), c.to_device(rand(rng, (8, 128))), c.empty((8, 128)), c.to_device(np.ones(16, np.float32))
    rot = nr.Rotary(16)
    r, h = ctypes.byref(rot.spec), c.handle
    fwd = lib.numrs_hip_qk_rotary_forward
    good = [h, seqs.handle, None, x.ptr, 128, w.ptr, w.ptr, EPS, r, y.ptr, 128, 4, 2, 16]
    assert fwd(*good) == 0
    wide = nr.Rotary(24)
    for i, value, code in ((1, None, L.E_INVALID), (3, None, L.E_INVALID), (4, 127, L.E_SHAPE), (4, 2**31, L.E_SHAPE),
                           (7, -1.0, L.E_INVALID), (7, float("nan"), L.E_INVALID), (8, ctypes.byref(wide.spec), L.E_SHAPE),
                           (9, None, L.E_INVALID), (10, 127, L.E_SHAPE), (11, 3, L.E_SHAPE), (11, 0, L.E_SHAPE),
                           (12, 0, L.E_SHAPE), (13, 12, L.E_SHAPE), (13, 136, L.E_SHAPE)):
        bad = list(good)
        bad[i] = value
        assert fwd(*bad) == code, i
        assert lib.numrs_hip_last_error(h)
    assert fwd(*good[:9], x.ptr, 130, 4, 2, 16) == L.E_SHAPE  # in place with another stride
    bwd = lib.numrs_hip_qk_rotary_backward
    good = [h, seqs.handle, None, x.ptr, 128, w.ptr, w.ptr, EPS, r, x.ptr, 128, y.ptr, 128, None, None, 4, 2, 16, 0]
    assert bwd(*good) == 0
    for i, value, code in ((3, None, L.E_INVALID), (9, None, L.E_INVALID), (10, 127, L.E_SHAPE), (12, 127, L.E_SHAPE)):
        bad = list(good)
        bad[i] = value
        assert bwd(*bad) == code, i
    for add in ({5: None, 13: w.ptr}, {6: None, 14: w.ptr}, {11: x.ptr, 18: L.ACC_X}, {11: x.ptr, 12: 130}):
        bad = list(good)
        for i, value in add.items():
            bad[i] = value
        assert bwd(*bad) == L.E_INVALID, add
    bad = list(good)
    bad[3], bad[5], bad[6] = None, None, None  # without norms x is not needed
    assert bwd(*bad) == 0
    empty, z = nr.PackedSequences([0], ctx=c), c.to_device(np.full(16, 4, np.float32))
    assert fwd(h, empty.handle, None, None, 128, None, None, EPS, None, None, 128, 4, 2, 16) == 0
    assert bwd(h, empty.handle, None, None, 128, w.ptr, w.ptr, EPS, r, None, 128, None, 128, z.ptr, None, 4, 2, 16,
               L.ACC_Q_WEIGHT) == 0 and (z.numpy() == 4).all()
    assert bwd(h, empty.handle, None, None, 128, w.ptr, w.ptr, EPS, r, None, 128, None, 128, z.ptr, None, 4, 2, 16, 0) == 0
    assert (z.numpy() == 0).all()
    s = _Paged(c, [8], 16, 2, 16, "f32", rng)
    app, cp = lib.numrs_hip_kv_cache_append, ctypes.byref(s.cache.pages)
    good = [h, cp, seqs.handle, x.ptr, 128, w.ptr, w.ptr, EPS, r, y.ptr, 64, 4, s.td.ptr, s.table.shape[1], s.ends.ptr]
    assert app(*good) == 0
    for i, value, code in ((1, None, L.E_INVALID), (2, None, L.E_INVALID), (3, None, L.E_INVALID), (4, 127, L.E_SHAPE),
                           (7, -1.0, L.E_INVALID), (8, ctypes.byref(wide.spec), L.E_SHAPE), (10, 63, L.E_SHAPE),
                           (11, 3, L.E_SHAPE), (12, None, L.E_INVALID), (13, 0, L.E_SHAPE), (14, None, L.E_INVALID)):
        bad = list(good)
        bad[i] = value
        assert app(*bad) == code, i
    t = nr.Tensor.new(rand(rng, (8, 128)), ctx=c)
    for bad in (dict(heads=3), dict(heads=4, q_weight=nr.Tensor.new(np.ones(8), ctx=c)), dict(heads=4, rotary=wide)):
        with pytest.raises(nr.HipError):
            t.qk_rotary(seqs, bad.pop("heads"), 2, **bad)
    with pytest.raises(nr.HipError):
        t.qk_rotary(empty, 4, 2)
    before = s.raw()
    for x1, kw in ((nr.Tensor.new(rand(rng, (8, 128)), True, ctx=c), {}),
                   (t, dict(q_weight=nr.Tensor.new(np.ones(16), True, ctx=c)))):
        with pytest.raises(nr.HipError, match="no backward"):
            x1.kv_cache_append(s.cache, seqs, 4, s.td, s.ends, rot, **kw)
    with pytest.raises(nr.HipError):
        t.kv_cache_append(s.cache, seqs, 3, s.td, s.ends, rot)
    for a, b in zip(s.raw(), before):
        assert_bits(a, b)
    with nr.Context(0) as other:
        o = nr.PackedSequences([8], ctx=other)
        assert fwd(h, o.handle, *[None, x.ptr, 128, None, None, EPS, None, y.ptr, 128, 4, 2, 16]) == L.E_INVALID
        with pytest.raises(ValueError, match="one context"):
            t.qk_rotary(seqs, 4, 2, rot, q_weight=nr.Tensor.new(np.ones(16), ctx=other))
        o.close()


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
    """Through the tape, the rotation changed after the forward; a second sweep adds; one tensor as both
    weights; a projection that wants no gradient."""
    rng = np.random.default_rng(80)
    t = _Case([20, 1, 77], 4, 2, 32, rng, dims=24)
    seqs, g = nr.PackedSequences(t.lengths), rand(rng, (t.T, t.W))
    x, wq, wk = nr.Tensor.new(t.x, True), nr.Tensor.new(t.wq, True), nr.Tensor.new(t.wk, True)
    up = nr.Tensor.new(g)
    (dx, ex), dw = t.backward(g)
    rot = nr.Rotary(32, 24)
    y = x.qk_rotary(seqs, 4, 2, rot, wq, wk)
    rot.freqs[:] = 1
    _close(y.values(), *t.forward(), "y")
    y.mul(up).sum().backward()
    _close(x.gradient(), dx, ex, "dx")
    for w, (r, e) in zip((wq, wk), dw):
        _close(w.gradient(), r, e + HALF * abs(r), "dw")
    x.qk_rotary(seqs, 4, 2, nr.Rotary(32, 24), wq, wk).mul(up).sum().backward()
    _close(x.gradient(), 2 * dx, 2 * ex + 2 * HALF * abs(dx), "dx twice")
    _close(wq.gradient(), 2 * dw[0][0], 2 * dw[0][1] + 4 * HALF * abs(dw[0][0]), "dw twice")
    t.wk = t.wq
    _, dw = t.backward(g)
    w, plain = nr.Tensor.new(t.wq, True), nr.Tensor.new(t.x)
    plain.qk_rotary(seqs, 4, 2, nr.Rotary(32, 24), w, w).mul(up).sum().backward()
    both = dw[0][0] + dw[1][0]
    _close(w.gradient(), both, dw[0][1] + dw[1][1] + 2 * HALF * (abs(both) + abs(dw[0][0])), "one weight")
    assert plain.gradient() is None


def test_gradients_against_differences(engine):
    rng = np.random.default_rng(81)
    t = _Case([5, 3], 2, 1, 16, rng, layout="pairs")
    g = rand(rng, (t.T, t.W))
    f = lambda: float((t.forward()[0] * g).sum())  # noqa: E731
    seqs = nr.PackedSequences(t.lengths)
    x, wq, wk = nr.Tensor.new(t.x, True), nr.Tensor.new(t.wq, True), nr.Tensor.new(t.wk, True)
    x.qk_rotary(seqs, 2, 1, t.rot, wq, wk).mul(nr.Tensor.new(g)).sum().backward()
    for a, tensor, count in ((t.x, x, 20), (t.wq, wq, 8), (t.wk, wk, 8)):
        got, flat = tensor.gradient().ravel(), a.reshape(-1)
        for i in rng.choice(flat.size, count, replace=False):
            was, h = flat[i], np.float32(2.0 ** -9)
            flat[i] = was + h
            up, top = f(), flat[i]
            flat[i] = was - h
            down, bottom = f(), flat[i]
            flat[i] = was
            # central difference: the third derivative's h^2 / 6, of terms of order 10
            assert abs((up - down) / (float(top) - float(bottom)) - got[i]) <= 3e-4, i


@pytest.mark.parametrize("format", ["f32", "int8"])
@pytest.mark.parametrize("norm", [False, True])
def test_a_decoder_with_positions(engine, format, norm):
    """A module's prompts in one call and in pieces, then single tokens, steps replayed from a graph too: with
    an fp32 cache every row is the packed forward's of the whole sequence, with an 8-bit one the attention
    over what the cache stands for."""
    c, rng, d, H, Hk, dh = engine, np.random.default_rng(82), 64, 4, 2, 32
    w = [rand(rng, s, 0.2) for s in ((H * dh, d), (Hk * dh, d), (Hk * dh, d), (d, H * dh))]
    norms = {"q_norm": 1 + rand(rng, dh, 0.2), "k_norm": 1 + rand(rng, dh, 0.2)} if norm else {}
    attn = nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk, rotary=nr.Rotary(dh, base=1000.0), **norms)
    assert len(attn.parameters()) == (6 if norm else 4)
    whole, page = [60, 25, 90], 16
    x = [rand(rng, (n, d)) for n in whole]
    full = attn.forward_packed(nr.Tensor.new(np.concatenate(x)), nr.PackedSequences(whole)).values()
    full = np.split(full, np.cumsum(whole)[:-1])
    plain = nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk)
    alone = plain.forward_packed(nr.Tensor.new(x[0]), nr.PackedSequences([60])).values()
    assert np.abs(alone - full[0]).max() > 1e-2  # positions count
    s = _Paged(c, whole, page, Hk, dh, format, rng)
    done, ed = np.zeros(3, np.int32), c.to_device(np.zeros(3, np.int32))

    def take(new):
        seqs = nr.PackedSequences(new)
        a = nr.Tensor.new(np.concatenate([x[i][done[i]:done[i] + n] for i, n in enumerate(new)]))
        done[:] += np.array(new, np.int32)
        ed.upload(done)
        return seqs, a

    def check(y, new, a=None):
        """Two orders of the same fp32 sums over values of order 1 to 10."""
        parts = np.split(y, np.cumsum(new)[:-1])
        if format == "f32" or a is None:
            for i, (part, n) in enumerate(zip(parts, new)):
                assert np.abs(part - full[i][done[i] - n:done[i]]).max(initial=0) <= 1e-5, (i, n)
            return
        qkv, now = attn.qkv(a).values(), nr.PackedSequences(done.tolist())
        k, v = (z.numpy().reshape(-1, Hk, dh) for z in s.cache.read(now, s.td, ed))
        at, row = np.concatenate([[0], np.cumsum(done)]), 0
        for i, n in enumerate(new):
            q = qkv[row:row + n, :H * dh].reshape(n, H, dh).astype(LD)
            row += n
            if norm:
                q = _norm(q, None)[0] * norms["q_norm"].astype(LD)
            q = _turn(q, np.arange(done[i] - n, done[i]), attn.rotary)[0].astype(np.float64)
            seen = np.arange(done[i]) <= np.arange(done[i] - n, done[i])[:, None]
            ref = _rows(q, k[at[i]:at[i + 1]], v[at[i]:at[i + 1]], seen)[0].reshape(n, H * dh) @ w[3].T.astype(np.float64)
            assert np.abs(parts[i] - ref).max(initial=0) <= 1e-5, (i, n)

    with nr.no_grad():
        new = [10, 1, 33]
        seqs, a = take(new)
        check(attn.prefill(a, seqs, s.cache, s.td, ed).values(), new)
        for new in ([17, 5, 1], [0, 1, 40], [1, 1, 1]):
            seqs, a = take(new)
            check(attn.extend(a, seqs, s.cache, s.td, ed).values(), new, a)
        ones = nr.PackedSequences([1] * 3)
        x1 = nr.Tensor.new(np.zeros((3, d), np.float32))
        xd = nr.DeviceArray(c, x1.device_ptrs()[0], (3, d), owned=False, base=x1)
        step = lambda: attn.decode(x1, ones, s.cache, s.td, ed)  # noqa: E731
        graph = None
        for t in range(10):
            _, a = take([1] * 3)
            xd.upload(a.values())
            if t == 4:
                graph = nr.StepGraph(c, step)
            if graph is None:
                y = step().values()
            else:
                graph.replay()
                y = graph.outputs.values()
            check(y, [1] * 3, a)
        graph.close()
    with pytest.raises(nr.HipError, match="no backward"):
        attn.extend(nr.Tensor.new(x[0][:3]), nr.PackedSequences([1] * 3), s.cache, s.td, ed)
    with pytest.raises(ValueError):
        nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk, rotary=nr.Rotary(64))
    with pytest.raises(ValueError):
        nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk, q_norm=np.ones(16))


def test_a_recorded_training_step(engine):
    """Steps of the module with norms and positions as replays equal eager ones to the bit, while an eager
    forward of the same parameters is still to be swept and after the handles are gone."""
    from numrs_amd import optim
    rng, d, H, Hk, lengths = np.random.default_rng(83), 32, 4, 2, [70, 3, 129]
    w = [rand(rng, s, 0.2) for s in ((16 * H, d), (16 * Hk, d), (16 * Hk, d), (d, 16 * H))]
    x, t = nr.Tensor.new(rand(rng, (sum(lengths), d))), nr.Tensor.new(rand(rng, (sum(lengths), d)))
    seqs = nr.PackedSequences(lengths)

    def make():
        attn = nn.CausalSelfAttention(*w, heads=H, kv_heads=Hk, rotary=nr.Rotary(16), q_norm=np.ones(16), k_norm=np.ones(16))
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
    b.rotary.freqs[:] = 0
    filler = [nr.PackedSequences(lengths[::-1]) for _ in range(3)]
    for i, loss in enumerate(want):
        graph.replay()
        assert graph.outputs.item() == loss, i
        if i == 1:
            alive.backward()
            for p in b.parameters():
                p.zero_grad()
    for p, q in zip(a.parameters(), b.parameters()):
        assert_bits(q.values(), p.values())
    assert abs(a.q_norm.values() - 1).max() > 0
    graph.close()
    del filler


def test_calls_past_the_caches(hip_ctx):
    """Calls of more than 256 MB, whose rows go past the caches, against calls of their sequences one by one: the same
    bits; the weights' gradients, sums of four rounded ones, within half a step of each."""
    c, lib, H, Hk, dh, n = hip_ctx, L.load(), 20, 4, 128, 2500
    W = (H + 2 * Hk) * dh
    rng = np.random.default_rng(80)
    x, dy = rand(rng, (4 * n, W)), rand(rng, (4 * n, W))
    rot = nr.Rotary(dh, layout="pairs")
    xd, gd, y, dx = c.to_device(x), c.to_device(dy), c.empty(x.shape), c.empty(x.shape)
    wq, wk, r = c.to_device(rand(rng, dh)), c.to_device(rand(rng, dh)), ctypes.byref(rot.spec)

    def both(seqs, ends, at, to, back, dq, dk):
        at *= W * 4
        c._check(lib.numrs_hip_qk_rotary_forward(c.handle, seqs.handle, ends, xd.ptr + at, W, wq.ptr, wk.ptr, EPS, r,
                                                 to.ptr, W, H, Hk, dh))
        c._check(lib.numrs_hip_qk_rotary_backward(c.handle, seqs.handle, ends, xd.ptr + at, W, wq.ptr, wk.ptr, EPS, r,
                                                  gd.ptr + at, W, back.ptr, W, dq.ptr, dk.ptr, H, Hk, dh, 0))

    dq, dk, one_y, one_dx = c.empty((dh,)), c.empty((dh,)), c.empty((n, W)), c.empty((n, W))
    both(nr.PackedSequences([n] * 4, ctx=c), None, 0, y, dx, dq, dk)
    whole, got_y, got_dx = [dq.numpy(), dk.numpy()], y.numpy(), dx.numpy()
    parts, one = [], nr.PackedSequences([n], ctx=c)
    for i in range(4):
        both(one, None, i * n, one_y, one_dx, dq, dk)
        parts.append([dq.numpy().astype(np.float64), dk.numpy().astype(np.float64)])
        assert_bits(one_y.numpy(), got_y[i * n:(i + 1) * n], "y")
        assert_bits(one_dx.numpy(), got_dx[i * n:(i + 1) * n], "dx")
    for k in range(2):
        p = np.array([q[k] for q in parts])
        # what 64-bit sums leave of terms that cancel: a head's normed values are below sqrt(dh), gradients below 8
        size = 4 * n * (H if k == 0 else Hk) * dh ** 0.5 * 8
        bound = HALF * (abs(p).sum(0) + abs(p.sum(0))) + 64 * U64 * size * 4 * n
        assert (abs(whole[k] - p.sum(0)) <= bound).all()
    # the same call again, and both in place
    both(nr.PackedSequences([n] * 4, ctx=c), None, 0, y, dx, dq, dk)
    assert_bits(dq.numpy(), whole[0])
    assert_bits(dk.numpy(), whole[1])
    all4 = nr.PackedSequences([n] * 4, ctx=c)
    c._check(lib.numrs_hip_qk_rotary_backward(c.handle, all4.handle, None, xd.ptr, W, wq.ptr, wk.ptr, EPS, r, gd.ptr, W,
                                              gd.ptr, W, None, None, H, Hk, dh, 0))
    assert_bits(gd.numpy(), got_dx, "gradient in place")
    c._check(lib.numrs_hip_qk_rotary_forward(c.handle, all4.handle, None, xd.ptr, W, wq.ptr, wk.ptr, EPS, r, xd.ptr, W,
                                             H, Hk, dh))
    assert_bits(xd.numpy(), got_y, "in place")


@pytest.mark.parametrize("format", ["f32", "int8"])
def test_append_past_the_caches(hip_ctx, format):
    """An append of more than 128 MB of keys and values, against appends of its sequences one by one."""
    c, lib, H, Hk, dh, n, page = hip_ctx, L.load(), 20, 20, 128, 1700, 64
    rng = np.random.default_rng(81)
    t = _Case([n] * 4, H, Hk, dh, rng, starts=[0, 5, 64, 130])
    total = [n + s for s in t.starts]
    s = _Paged(c, total, page, Hk, dh, format, rng)
    xd, wq, wk, q = c.to_device(t.x), _d(c, t.wq), _d(c, t.wk), c.empty((4 * n, H * dh))
    before = s.raw()

    def call(seqs, row, i):
        c._check(lib.numrs_hip_kv_cache_append(
            c.handle, ctypes.byref(s.cache.pages), seqs.handle, xd.ptr + row * t.W * 4, t.W, wq.ptr, wk.ptr, EPS,
            ctypes.byref(t.rot.spec), q.ptr + row * H * dh * 4, H * dh, H, s.td.ptr + i * s.table.shape[1] * 4,
            s.table.shape[1], s.ends.ptr + i * 4))

    call(nr.PackedSequences([n] * 4, ctx=c), 0, 0)
    want, queries = s.raw(), q.numpy()
    for a, b in zip((s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale), before):
        a.upload(b)
    q.fill(0)
    one = nr.PackedSequences([n], ctx=c)
    for i in range(4):
        call(one, i * n, i)
    for got, ref in zip(s.raw(), want):
        assert np.array_equal(got, ref, equal_nan=got.dtype == np.float32)
    assert_bits(q.numpy(), queries, "q")


def test_results_in_their_inputs_rows(hip_ctx):
    """Results over their inputs are refused but where the header allows them, those with the bits of a call of
    separate arrays."""
    c, lib, rng = hip_ctx, L.load(), np.random.default_rng(90)
    t = _Case([150, 7, 64], 4, 2, 16, rng)
    seqs, w, W = nr.PackedSequences(t.lengths, ctx=c), c.to_device(t.wq), t.W
    T, h, r, ld = t.T, c.handle, ctypes.byref(t.rot.spec), 2 * t.W + 16
    big = c.to_device(rand(rng, (3 * T, ld)))
    x = big.ptr + 4 * T * ld
    fwd = lambda to, ld_y: lib.numrs_hip_qk_rotary_forward(  # noqa: E731
        h, seqs.handle, None, x, ld, w.ptr, w.ptr, EPS, r, to, ld_y, 4, 2, 16)
    for at, ld_y in ((1, ld), (ld, ld), (-ld, ld), (5 * ld + W - 1, ld), (-5 * ld - W + 1, ld), (1, W), (-W, ld - 1)):
        assert fwd(x + 4 * at, ld_y) == L.E_INVALID, (at, ld_y)
    assert fwd(x + 4 * W, ld) == 0 and fwd(x - 4 * W, ld) == 0
    bwd = lambda gy, ld_g, to, ld_dx, wq=w.ptr, wk=w.ptr, dq=None, dk=None: lib.numrs_hip_qk_rotary_backward(  # noqa: E731
        h, seqs.handle, None, x, ld, wq, wk, EPS, r, gy, ld_g, to, ld_dx, dq, dk, 4, 2, 16, 0)
    g, dx = c.to_device(rand(rng, (3 * T, ld), 0.1)), c.empty((T, W))
    gy = g.ptr + 4 * T * ld
    for at in (1, ld, -ld, 5 * ld + 95, -5 * ld - W + 1):
        assert bwd(gy, ld, gy + 4 * at, ld) == L.E_INVALID, at  # over dy
        assert bwd(gy, ld, x + 4 * at, ld) == L.E_INVALID, at   # over x
    assert bwd(gy, ld, x, ld - 1) == L.E_INVALID and bwd(gy, ld, gy + 4, ld - 1) == L.E_INVALID
    # only what is read of x counts: the normed heads, its columns 0 to 63 or 64 to 95
    assert bwd(gy, ld, x + 4 * 64, ld, wk=None) == 0 and bwd(gy, ld, x + 4 * 63, ld, wk=None) == L.E_INVALID
    assert bwd(gy, ld, x + 4 * 96, ld, wq=None) == 0 and bwd(gy, ld, x + 4 * 95, ld, wq=None) == L.E_INVALID
    assert bwd(gy, ld, x + 4 * 5 * ld, ld, wq=None, wk=None) == 0
    two = c.empty((24,))
    assert bwd(gy, ld, dx.ptr, W, dq=two.ptr, dk=two.ptr + 4 * 8) == L.E_INVALID
    assert bwd(gy, ld, dx.ptr, W) == 0
    assert bwd(gy, ld, x, ld) == 0  # the gradient in x's place
    assert_bits(big.numpy()[T:2 * T, :W], dx.numpy())
