// Where a token of a paged key-value cache lies, and the checks of a cache's description: plain
// integer arithmetic, the same on the host and in the kernels.
#pragma once

#include <stdint.h>

#include "numrs_hip.h"

#ifdef __HIPCC__
#define NRS_HD __host__ __device__ __forceinline__
#else
#define NRS_HD inline
#endif

namespace paging {

// The page that holds position `pos` of the sequence whose pages `row` lists, or -1: a position
// before the first or past the listed pages, or a page that the cache does not have.  Every
// access to a cache goes through here, so no table and no length can lead outside it.
// (In two steps, so that a kernel can wait for an entry later than it asks for it.)
NRS_HD int32_t entry_of(const int32_t *row, int64_t max_pages, int shift, int64_t pos) {
  return pos < 0 || pos >> shift >= max_pages ? -1 : row[pos >> shift];
}
NRS_HD int page_in(int32_t entry, int64_t pages) { return entry >= 0 && entry < pages ? entry : -1; }
NRS_HD int page_of(const int32_t *row, int64_t max_pages, int shift, int64_t pages, int64_t pos) {
  return page_in(entry_of(row, max_pages, shift, pos), pages);
}

// Element offset of slot 0 of a page and head; rows of keys (and of fp32 values) follow at dh
// elements each.
NRS_HD int64_t page_base(int64_t page, int64_t kv_heads, int64_t head, int shift, int64_t dh) {
  return ((page * kv_heads + head) << shift) * dh;
}

// Offset, within a page and head, of the 8-bit code of value d of a slot: four neighbouring
// slots' codes of a d lie together, so that one 4-byte load has a column of four tokens.
NRS_HD int64_t value_code(int64_t slot, int64_t d, int64_t dh) {
  return ((slot >> 2) * dh + d) * 4 + (slot & 3);
}

// Tokens of a sequence that attention reads: its length within what its pages can hold.
NRS_HD int64_t held(int64_t len, int64_t max_pages, int shift) {
  const int64_t most = max_pages << shift;
  return len < 0 ? 0 : len < most ? len : most;
}

NRS_HD int log2_of(int64_t page_size) {
  int s = 0;
  while ((int64_t{1} << s) < page_size) ++s;
  return s;
}

inline bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// What is wrong with a cache's description, or null; *code is the error to return.
inline const char *refuse_cache(const numrs_hip_kv_cache *c, int *code) {
  *code = NUMRS_HIP_E_INVALID;
  if (c == nullptr) return "null cache";
  if (c->format != NUMRS_HIP_KV_F32 && c->format != NUMRS_HIP_KV_INT8) return "unknown cache format";
  if (c->k == nullptr || c->v == nullptr) return "null pages";
  const bool q = c->format == NUMRS_HIP_KV_INT8;
  if (q && (c->k_scale == nullptr || c->v_scale == nullptr)) return "an 8-bit cache needs scales";
  if (!on16(c->k) || !on16(c->v) || (q && (!on16(c->k_scale) || !on16(c->v_scale))))
    return "the pages and scales must lie on 16 bytes";
  *code = NUMRS_HIP_E_SHAPE;
  if (c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)) != 0)
    return "the page size must be a power of two in 16..65536";
  if (c->kv_heads < 1 || c->kv_heads > 65535) return "kv_heads must be in 1..65535";
  if (c->head_dim < 8 || c->head_dim > 128 || c->head_dim % 8 != 0)
    return "head_dim must be a multiple of 8 in 8..128";
  if (c->pages < 1 || c->pages >= int64_t{1} << 31) return "the cache must have 1 to 2^31 - 1 pages";
  if (c->pages > (int64_t{1} << 46) / (c->page_size * c->kv_heads * c->head_dim))
    return "the cache must hold at most 2^46 values";
  return nullptr;
}

// The same for a table of n sequences.
inline const char *refuse_table(const void *table, int64_t max_pages, const void *lengths, int64_t n,
                                int *code) {
  *code = NUMRS_HIP_E_INVALID;
  if (n < 0) return "negative number of sequences";
  if (n > 0 && (table == nullptr || lengths == nullptr)) return "null table or lengths";
  *code = NUMRS_HIP_E_SHAPE;
  if (n >= int64_t{1} << 24) return "at most 2^24 - 1 sequences";
  if (max_pages < 1 || max_pages >= int64_t{1} << 31) return "a table must have 1 to 2^31 - 1 columns";
  return nullptr;
}

// What is wrong with a call's heads and row strides, or null.
inline const char *refuse_heads(int64_t heads, int64_t kv_heads, int64_t dh) {
  if (heads < 1 || kv_heads < 1 || heads > 65535 || heads % kv_heads != 0)
    return "heads must be a multiple of kv_heads, both in 1..65535";
  if (dh < 8 || dh > 128 || dh % 8 != 0) return "the head size must be a multiple of 8 in 8..128";
  return nullptr;
}

inline bool bad_stride(int64_t ld, int64_t width) { return ld < width || ld >= int64_t{1} << 31; }

// More workgroups of 256 threads than a launch, of at most 2^32 - 1 threads, can have.
inline bool bad_grid(int64_t groups) { return groups >= int64_t{1} << 24; }

// Rows of an array that a call reads or writes: `width` floats each from `at` on, ld floats apart, ld >= width.
struct Rows {
  const float *at;
  int64_t width, ld;
};
// Whether any of the first `rows` rows of a meets any of b.  Column blocks side by side in the same rows do not.
inline bool rows_meet(const Rows &a, const Rows &b, int64_t rows) {
  typedef __int128 wide;  // (bytes of 2^30 rows, 2^31 floats apart, and an address)
  if (rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  const wide f = sizeof(float), na = a.width * f, nb = b.width * f, la = a.ld * f, lb = b.ld * f;
  const wide from = (wide) reinterpret_cast<uintptr_t>(b.at) - (wide) reinterpret_cast<uintptr_t>(a.at);  // a to b
  if (from >= (rows - 1) * la + na || from + (rows - 1) * lb + nb <= 0) return false;
  if (la == lb) {
    // b's row j lies from + (j - i) la beyond a's row i: the least such distance above -nb that two rows have
    const wide x = -nb - from, below = x >= 0 ? x / la : -((la - 1 - x) / la);  // x / la rounded down
    const wide d = below + 1 < -(wide)(rows - 1) ? -(wide)(rows - 1) : below + 1;
    return d < rows && from + d * la < na;
  }
  wide x = 0, y = from;  // the rows of both in their order
  for (int64_t i = 0, j = 0; i < rows && j < rows;) {
    if (x + na <= y)
      ++i, x += la;
    else if (y + nb <= x)
      ++j, y += lb;
    else
      return true;
  }
  return false;
}

// Lengths of a packed batch: their sum, or -1 if one is negative or they pass 2^30 tokens.
inline int64_t packed_total(const int64_t *lengths, int64_t n) {
  int64_t total = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (lengths[i] < 0 || lengths[i] > int64_t{1} << 30) return -1;
    total += lengths[i];
    if (total > int64_t{1} << 30) return -1;
  }
  return total;
}

}  // namespace paging
