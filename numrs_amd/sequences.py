"""Packed batches and the paged key-value cache (no counterpart in numrs, whose
attention-free ops take one shape).

    seqs = PackedSequences([17, 256, 3])            # rows 0..16, 17..272, 273..275
    out = qkv.attention_packed_qkv(seqs, heads, kv_heads)      # causal, with backward

    cache = KVCache(pages, page_size, kv_heads, head_dim, "int8")
    cache.write_qkv(seqs, qkv, heads, table, lengths)           # a prompt's keys and values
    cache.write_qkv(ones, qkv1, heads, table, lengths)          # one more token each
    out = qkv1.attention_paged(cache, heads, table, lengths)    # its attention

`table` [n, max_pages] and `lengths` [n] are int32 device arrays that the
program keeps and advances: which pages of the cache each sequence owns, and
how many tokens it has there, the ones being written included.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib as L
from ._lib import KVPages
from .autograd import Tensor, default_context
from .device import Context, DeviceArray

FORMATS = {"f32": L.KV_F32, "int8": L.KV_INT8}


class PackedSequences:
    """The lengths of a packed batch (numrs_hip_seqs), made once and used by any
    number of calls."""

    def __init__(self, lengths, ctx: Context | None = None):
        self.ctx = ctx or default_context()
        self.lengths = tuple(int(n) for n in lengths)
        n = (ctypes.c_int64 * max(len(self.lengths), 1))(*self.lengths)
        h = ctypes.c_void_p()
        self.handle = None
        self.ctx._check(L.load().numrs_hip_seqs_create(self.ctx.handle, n, len(self.lengths),
                                                       ctypes.byref(h)))
        self.handle = h.value

    @property
    def total(self) -> int:
        return sum(self.lengths)

    def __len__(self) -> int:
        return len(self.lengths)

    def close(self) -> None:
        if self.handle:
            L.load().numrs_hip_seqs_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _rows(x, what: str):
    """(device pointer, shape, context) of a 2-D Tensor or float32 DeviceArray."""
    if isinstance(x, Tensor):
        ptr, shape, ctx = x.device_ptrs()[0], x.shape(), x.ctx
    else:
        if x.dtype != np.float32:
            raise ValueError(f"{what} must be float32")
        ptr, shape, ctx = x.ptr, x.shape, x.ctx
    if len(shape) != 2:
        raise ValueError(f"{what} must be [tokens, columns]")
    return ptr, shape, ctx


class KVCache:
    """Pages of keys and values on the device, float32 ("f32") or 8-bit codes
    with a scale for each token and head ("int8"); include/numrs_hip.h has the
    layout.  Which sequence owns which page is the program's business."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 format: str = "f32", ctx: Context | None = None):
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}")
        if min(pages, page_size, kv_heads, head_dim) < 1:
            raise ValueError("a cache's sizes must be positive")
        self.ctx = ctx or default_context()
        self.format, shape = format, (pages, kv_heads, page_size, head_dim)
        kind = np.float32 if format == "f32" else np.uint8
        self.k, self.v = self.ctx.empty(shape, kind), self.ctx.empty(shape, kind)
        self.k_scale = self.v_scale = None
        if format == "int8":
            self.k_scale, self.v_scale = self.ctx.empty(shape[:3]), self.ctx.empty(shape[:3])
        ptr = lambda a: a.ptr if a is not None else None  # noqa: E731
        self.pages = KVPages(self.k.ptr, self.v.ptr, ptr(self.k_scale), ptr(self.v_scale), pages,
                             page_size, kv_heads, head_dim, FORMATS[format])

    @property
    def width(self) -> int:
        """Columns of a row of keys or values: kv_heads * head_dim."""
        return self.pages.kv_heads * self.pages.head_dim

    def table_width(self, table: DeviceArray, lengths: DeviceArray, n: int) -> int:
        """The table's columns, after a look at the shapes of both arrays."""
        if len(table.shape) != 2 or table.dtype != np.int32 or table.shape[0] != n:
            raise ValueError(f"the table must be int32 [{n}, pages of a sequence]")
        if lengths.size != n or lengths.dtype != np.int32:
            raise ValueError(f"the lengths must be int32 [{n}]")
        if table.ctx is not self.ctx or lengths.ctx is not self.ctx:
            raise ValueError("table, lengths and cache must belong to one context")
        return table.shape[1]

    def _call(self, fn, seqs, k_ptr, v_ptr, ld, table, ends):
        most = self.table_width(table, ends, len(seqs))
        self.ctx._check(fn(self.ctx.handle, ctypes.byref(self.pages), seqs.handle, k_ptr, v_ptr, ld,
                           table.ptr, most, ends.ptr))

    def _check_rows(self, shape, ctx, seqs, columns, what):
        if shape[0] < seqs.total or shape[1] != columns:
            raise ValueError(f"{what} must be [{seqs.total}, {columns}], not {list(shape)}")
        if ctx is not self.ctx or seqs.ctx is not self.ctx:
            raise ValueError(f"{what}, sequences and cache must belong to one context")

    def write(self, seqs: PackedSequences, k, v, table: DeviceArray, ends: DeviceArray) -> None:
        """Writes packed rows k, v [tokens, kv_heads * head_dim]; sequence i's rows
        become its positions ends[i] - length .. ends[i] - 1."""
        (kp, ks, kc), (vp, vs, vc) = _rows(k, "k"), _rows(v, "v")
        self._check_rows(ks, kc, seqs, self.width, "k")
        self._check_rows(vs, vc, seqs, self.width, "v")
        self._call(L.load().numrs_hip_kv_cache_write, seqs, kp, vp, self.width, table, ends)

    def write_qkv(self, seqs: PackedSequences, qkv, heads: int, table: DeviceArray,
                  ends: DeviceArray) -> None:
        """The same from a projection [tokens, (heads + 2 kv_heads) * head_dim]
        whose column blocks are q, k and v."""
        p, shape, ctx = _rows(qkv, "qkv")
        wq = heads * self.pages.head_dim
        self._check_rows(shape, ctx, seqs, wq + 2 * self.width, "qkv")
        self._call(L.load().numrs_hip_kv_cache_write, seqs, p + 4 * wq, p + 4 * (wq + self.width),
                   shape[1], table, ends)

    def read(self, seqs: PackedSequences, table: DeviceArray, ends: DeviceArray
             ) -> tuple[DeviceArray, DeviceArray]:
        """The packed rows at those positions, as float32 arrays k, v."""
        k, v = (self.ctx.empty((seqs.total, self.width)) for _ in range(2))
        self._check_rows(k.shape, k.ctx, seqs, self.width, "k")
        self._call(L.load().numrs_hip_kv_cache_read, seqs, k.ptr, v.ptr, self.width, table, ends)
        return k, v


__all__ = ["PackedSequences", "KVCache", "KVPages"]
