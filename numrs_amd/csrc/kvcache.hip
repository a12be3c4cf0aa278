// A paged key-value cache in fp32 or 8-bit codes, written, read back and attended to (no reference
// op).  paging.h says where a token lies; every position goes through paging::page_of.
#include <algorithm>
#include <cmath>

#include "packed.h"
#include "paged_split.h"
#include "rotary.h"

namespace {

using namespace numrs_hip;

constexpr float kLog2e = 1.44269504088896341f;

using paged::Cache;

struct RowArgs {
  Cache c;
  const SeqTile *tiles;
  const int32_t *ends;
  const float *k, *v;  // written from
  float *ko, *vo;      // read into
  int64_t ld;
};

// The rows of a batch go by groups of four positions, 4 q .. + 3: four slots of one page, whose 8-bit
// values lie together.  A thread has four columns of a group: four 16-byte loads of keys and of values
// in flight, and 16 bytes of codes to store or load at once.
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

struct Group {
  int64_t pos;   // its first position
  int64_t base;  // element offset of its first slot in its page and head
  int page;      // -1: the cache has no place for it
  int row[4];    // the packed rows within the sequence, -1 for a position that is none of the tile's
};

// Calls f(group, d) for this thread's groups of tile t and head g, for its columns d .. + 3; lanes of a
// wave that share a group's rows are 2^lanes neighbours, d >= dh for those past the head.
//
// A workgroup has one tile and one head.  Bound by memory: 28 thousand tokens of 8 heads of 128 in 8 bits,
// 290 MB each way, are written in 57 us (5.1 TB/s) and read in 44 (6.5 TB/s); 452 tokens of 8 heads of 64
// in fp32 take 4 us each, latency.  Slot by slot, without groups, both took 249 us in place of 132; with all
// heads of its tokens in a workgroup 141.
template <class F>
__device__ __forceinline__ void for_groups(const Cache &c, const SeqTile &t, int g, const int32_t *ends, int lanes, F &&f) {
  const int rows = min(t.len - t.t0, kTile), d = 4 * (threadIdx.x & ((1 << lanes) - 1));
  const int64_t start = (int64_t)ends[t.seq] - t.len, p0 = start + t.t0;
  const int64_t q0 = p0 >> 2, q1 = (p0 + rows - 1) >> 2;
  for (int64_t q = q0 + (threadIdx.x >> lanes); q <= q1; q += 256 >> lanes) {
    Group x;
    x.pos = 4 * q;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = 4 * q + r - start;
      x.row[r] = row >= t.t0 && row < t.t0 + rows ? (int)row : -1;
    }
    x.page = paging::page_of(c.table + (int64_t)t.seq * c.max_pages, c.max_pages, c.shift, c.pages, 4 * q);
    x.base = paging::page_base(max(x.page, 0), c.kv_heads, g, c.shift, 1) + (int)((4 * q) & ((1 << c.shift) - 1));
    f(x, d);
  }
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}

// The largest of 2^lanes neighbours of each of N values, for `lanes` up to 5: lanes 1 and 2 apart by
// quads, then the other four of eight and the other eight of sixteen by mirrors (what they hold is
// their group's already), then the other row of a pair.
template <int N>
__device__ __forceinline__ void max_of(unsigned (&v)[N], int lanes) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (lanes > 0) v[i] = dpp_max<0xB1>(v[i]);
    if (lanes > 1) v[i] = dpp_max<0x4E>(v[i]);
    if (lanes > 2) v[i] = dpp_max<0x141>(v[i]);
    if (lanes > 3) v[i] = dpp_max<0x140>(v[i]);
    if (lanes > 4) {
      const auto r = __builtin_amdgcn_permlane16_swap(v[i], v[i], false, false);
      v[i] = max((unsigned)r[0], (unsigned)r[1]);
    }
  }
}

// Codes of four values of a row of that scale: x / scale is rounded to fp32, then to a whole number.
// x times the reciprocal is within 2 of its last places (2^-16 at 127) of the quotient and rounds to
// the same number unless it lies that near the middle between two: then, in a wave where any does, the
// quotient is formed.  A row of zeros, or whose scale is NaN, has the codes 128.
__device__ __forceinline__ unsigned codes_of(f4 x, float scale) {
  // Added to 1.5 2^23, a number below 2^22 is rounded to a whole one, whose low bits end the sum's.
  constexpr float kWhole = 12582912.f;
  const float inv = __builtin_amdgcn_rcpf(scale);
  unsigned b[4];
  float off = 0.f;
  bool odd = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float z = x[j] * inv, s = z + kWhole;
    b[j] = __builtin_bit_cast(unsigned, s);
    off = fmaxf(off, fabsf(z - (s - kWhole)));
  }
  // (an inverse that is infinite makes z infinite or NaN)
  odd = scale > 0.f && !(off < 0.4999f && inv < INFINITY);
  if (__any(odd)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float s = fminf(fmaxf(rintf(x[j] / scale), -127.f), 127.f) + kWhole;
      b[j] = __builtin_bit_cast(unsigned, s);
    }
  }
  const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return scale > 0.f ? (lo | hi) ^ 0x80808080u : 0x80808080u;
}

// The scale of a row from its largest magnitude's bits: NaN is above infinity, infinity above every
// number, and such a row's scale is NaN.
__device__ __forceinline__ float scale_of(unsigned top) {
  return top < 0x7f800000u ? __builtin_bit_cast(float, top) / 127.0f : NAN;
}
__device__ __forceinline__ unsigned top_of(f4 x) {
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y = x[j];  // (a bit cast of the vector's element itself takes the first element's bits)
    top = max(top, __builtin_bit_cast(unsigned, y) & 0x7fffffffu);
  }
  return top;
}

// A 4 x 4 block of bytes, rows to columns.
__device__ __forceinline__ u4 transposed(u4 x) {
  const unsigned a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
  const unsigned c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
  return u4{__builtin_amdgcn_perm(c, a, 0x05040100u), __builtin_amdgcn_perm(c, a, 0x07060302u),
            __builtin_amdgcn_perm(d, b, 0x05040100u), __builtin_amdgcn_perm(d, b, 0x07060302u)};
}

// A group's scales, and its codes of four columns: keys' at pk, a row dh apart, values' 16 bytes at pv.  Slots
// that are not the batch's are left alone; `whole`: all four are.
__device__ __forceinline__ void put_scales(const Cache &c, const Group &x, bool whole, f4 ks, f4 vs) {
  if (whole) {
    *reinterpret_cast<f4 *>(c.ks + x.base) = ks, *reinterpret_cast<f4 *>(c.vs + x.base) = vs;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (x.row[r] >= 0) c.ks[x.base + r] = ks[r], c.vs[x.base + r] = vs[r];
  }
}
__device__ __forceinline__ void put_codes(const Group &x, bool whole, uint8_t *pk, uint8_t *pv, int dh, u4 kc, u4 vc) {
  if (whole) *reinterpret_cast<u4 *>(pv) = transposed(vc);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (x.row[r] < 0) continue;
    *reinterpret_cast<unsigned *>(pk + r * dh) = kc[r];
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 4; ++j) pv[4 * j + r] = (uint8_t)(vc[r] >> (8 * j));
    }
  }
}

// PAST: the rows go past the caches (see rows_past).
template <bool INT8, bool PAST>
__global__ void __launch_bounds__(256) write_rows(RowArgs a, int lanes) {
  const SeqTile t = a.tiles[blockIdx.x / a.c.kv_heads];
  const int g = blockIdx.x % a.c.kv_heads, dh = a.c.dh;
  for_groups(a.c, t, g, a.ends, lanes, [&](const Group &x, int d) {
    f4 k[4], v[4];
    const bool in = d < dh;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      k[r] = v[r] = f4{};
      if (!in || x.row[r] < 0) continue;
      const int64_t at = (int64_t)(t.row0 + x.row[r]) * a.ld + (int64_t)g * dh + d;
      k[r] = paged::load<f4u, PAST>(reinterpret_cast<const char *>(a.k + at));
      v[r] = paged::load<f4u, PAST>(reinterpret_cast<const char *>(a.v + at));
    }
    if constexpr (!INT8) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (!in || x.row[r] < 0 || x.page < 0) continue;
        const int64_t at = (x.base + r) * dh + d;
        *reinterpret_cast<f4 *>(static_cast<float *>(a.c.k) + at) = k[r];
        *reinterpret_cast<f4 *>(static_cast<float *>(a.c.v) + at) = v[r];
      }
    } else {
      u4 kc, vc;
      f4 ks, vs;
      unsigned top[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) top[r] = top_of(k[r]), top[4 + r] = top_of(v[r]);
      max_of(top, lanes);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ks[r] = scale_of(top[r]), vs[r] = scale_of(top[4 + r]);
        kc[r] = codes_of(k[r], ks[r]), vc[r] = codes_of(v[r], vs[r]);
      }
      if (x.page < 0) return;
      const bool whole = (x.row[0] | x.row[1] | x.row[2] | x.row[3]) >= 0;
      if (d == 0) put_scales(a.c, x, whole, ks, vs);
      if (!in) return;
      uint8_t *pk = static_cast<uint8_t *>(a.c.k) + x.base * dh + d, *pv = static_cast<uint8_t *>(a.c.v) + x.base * dh + 4 * d;
      put_codes(x, whole, pk, pv, dh, kc, vc);
    }
  });
}

template <bool INT8, bool PAST>
__global__ void __launch_bounds__(256) read_rows(RowArgs a, int lanes) {
  const SeqTile t = a.tiles[blockIdx.x / a.c.kv_heads];
  const int g = blockIdx.x % a.c.kv_heads, dh = a.c.dh;
  for_groups(a.c, t, g, a.ends, lanes, [&](const Group &x, int d) {
    if (d >= dh) return;
    f4 k[4] = {}, v[4] = {};
    if (x.page >= 0) {
      if constexpr (!INT8) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t at = (x.base + r) * dh + d;
          k[r] = *reinterpret_cast<const f4 *>(static_cast<const float *>(a.c.k) + at);
          v[r] = *reinterpret_cast<const f4 *>(static_cast<const float *>(a.c.v) + at);
        }
      } else {
        const uint8_t *pk = static_cast<const uint8_t *>(a.c.k) + x.base * dh + d;
        u4 kc;
#pragma unroll
        for (int r = 0; r < 4; ++r) kc[r] = *reinterpret_cast<const unsigned *>(pk + r * dh);
        const u4 vc = transposed(*reinterpret_cast<const u4 *>(static_cast<const uint8_t *>(a.c.v) + x.base * dh + 4 * d));
        const f4 ks = *reinterpret_cast<const f4 *>(a.c.ks + x.base), vs = *reinterpret_cast<const f4 *>(a.c.vs + x.base);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            k[r][j] = (float)((int)(kc[r] >> (8 * j) & 255) - 128) * ks[r];
            v[r][j] = (float)((int)(vc[r] >> (8 * j) & 255) - 128) * vs[r];
          }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (x.row[r] < 0) continue;
      const int64_t at = (int64_t)(t.row0 + x.row[r]) * a.ld + (int64_t)g * dh + d;
      f4u *ko = reinterpret_cast<f4u *>(a.ko + at), *vo = reinterpret_cast<f4u *>(a.vo + at);
      if constexpr (PAST)
        __builtin_nontemporal_store(f4u(k[r]), ko), __builtin_nontemporal_store(f4u(v[r]), vo);
      else
        *ko = k[r], *vo = v[r];
    }
  });
}

// Neighbours that share a row, four columns each: the power of two that covers a head.
int row_lanes(int dh) { return paging::log2_of((dh + 3) / 4); }

struct AppendArgs {
  RowArgs c;            // where the keys and values go; k and v are not used
  rotary::RowArgs row;  // the projection, and the queries' rows
  unsigned keys;        // workgroups of keys and values, before those of queries
  int parts;            // of a tile, for the queries
};

// Keys, normed and rotated, and values on their way into the cache: a workgroup a tile and kv head, a thread four
// positions and eight columns.  After them a workgroup a tile's part and some of the query heads.  A projection of 460 MB
// into fp32 pages 195 us (4.7 TB/s, the memory's); a token for each of 40 sequences into 8 bits 8.3 us, a chain of loads and
// arithmetic.  Rows of a group that are not there are skipped whole: their instructions, fetched for nothing, took 1 us
// of a step and 14 of the large call.
template <bool INT8, bool PAST>
__global__ void __launch_bounds__(256) append_rows(AppendArgs b) {
  if (blockIdx.x >= b.keys) {
    const unsigned n = b.row.slots > 0 ? (b.row.slots + b.row.per - 1) / b.row.per : 1, i = blockIdx.x - b.keys;
    const int h0 = i % n * b.row.per;
    rotary::rotate_part<PAST>(b.row, b.row.tiles[i / n / b.parts], i / n % b.parts, h0, min(h0 + b.row.per, b.row.slots));
    return;
  }
  const RowArgs &a = b.c;
  const rotary::RowArgs &ra = b.row;
  const SeqTile t = a.tiles[blockIdx.x / a.c.kv_heads];
  const int g = blockIdx.x % a.c.kv_heads, dh = a.c.dh;
  const bool nb = ra.turn.pairs;
  // What no row decides is asked for before the rows' pages are looked up.
  const int i = threadIdx.x & ((1 << ra.lanes) - 1);
  const rotary::Item it = rotary::item_of(i, dh, ra.turn);
  const rotary::Steps steps = rotary::steps_of(ra.turn, i, it);
  rotary::Weight w;
  w.load(ra.wk, it, nb);
  for_groups(a.c, t, g, a.ends, ra.lanes, [&](const Group &x, int) {
    f4 k0[4], k1[4], v0[4], v1[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      k0[r] = k1[r] = v0[r] = v1[r] = f4{};
      if (!it.in || x.row[r] < 0) continue;
      const char *k = reinterpret_cast<const char *>(ra.x + (int64_t)(t.row0 + x.row[r]) * ra.ld_x + (int64_t)(ra.heads + g) * dh);
      const char *v = k + (int64_t)a.c.kv_heads * dh * 4;
      k0[r] = paged::load<f4u, PAST>(k + 4 * it.d0), k1[r] = paged::load<f4u, PAST>(k + 4 * it.d1);
      v0[r] = paged::load<f4u, PAST>(v + 32 * i), v1[r] = paged::load<f4u, PAST>(v + 32 * i + 16);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (x.row[r] < 0) continue;  // (a step has one row of four: the others' code is not even fetched)
      double y[8];
      rotary::pairs_of(k0[r], k1[r], nb, y);
      if (ra.wk != nullptr) {
        const double s = rotary::inverse_rms(y, ra.lanes, ra.inv_dh, ra.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = y[j] * s * w.w[j];
      }
      rotary::turn<false>(y, rotary::units_of(steps, it, x.pos + r), it.turned);
      rotary::columns_of(y, nb, k0[r], k1[r]);
    }
    if constexpr (!INT8) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (!it.in || x.row[r] < 0 || x.page < 0) continue;
        float *k = static_cast<float *>(a.c.k) + (x.base + r) * dh, *v = static_cast<float *>(a.c.v) + (x.base + r) * dh;
        *reinterpret_cast<f4 *>(k + it.d0) = k0[r], *reinterpret_cast<f4 *>(k + it.d1) = k1[r];
        *reinterpret_cast<f4 *>(v + 8 * i) = v0[r], *reinterpret_cast<f4 *>(v + 8 * i + 4) = v1[r];
      }
    } else {
      u4 kc0{}, kc1{}, vc0{}, vc1{};
      f4 ks{}, vs{};
      unsigned top[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // (a lane past the head has zeros, or NaN where the norm of zeros is)
        top[r] = it.in ? max(top_of(k0[r]), top_of(k1[r])) : 0, top[4 + r] = max(top_of(v0[r]), top_of(v1[r]));
      }
      max_of(top, ra.lanes);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (x.row[r] < 0) continue;
        ks[r] = scale_of(top[r]), vs[r] = scale_of(top[4 + r]);
        kc0[r] = codes_of(k0[r], ks[r]), kc1[r] = codes_of(k1[r], ks[r]);
        vc0[r] = codes_of(v0[r], vs[r]), vc1[r] = codes_of(v1[r], vs[r]);
      }
      if (x.page < 0) return;
      const bool whole = (x.row[0] | x.row[1] | x.row[2] | x.row[3]) >= 0;
      if (i == 0) put_scales(a.c, x, whole, ks, vs);
      if (!it.in) return;
      uint8_t *pk = static_cast<uint8_t *>(a.c.k) + x.base * dh, *pv = static_cast<uint8_t *>(a.c.v) + x.base * dh + 32 * i;
      put_codes(x, whole, pk + it.d0, pv, dh, kc0, vc0);
      put_codes(x, whole, pk + it.d1, pv + 16, dh, kc1, vc1);
    }
  });
}

// Whether a batch's rows go past the caches: where keys and values are more than half of the last cache's 256 MB,
// so that they would take the place of what the next kernel reads.  On MI355X, through them against past, us:
// 8 heads of 128, writes of rows just made | and attention over them | reads back | and attention over those, in
// fp32: 16 MB 7.1, 7.4 | 59.6, 60.8 | 6.5, 5.2 | 48.7, 49.6; 64 MB 20, 22 | 182, 190 | 22, 22 | 137, 147; 128 MB
// 35, 42 | 363, 366 | 41, 40 | 266, 272; 256 MB 110, 75 | 777, 765 | 97, 79 | 539, 534; in 8 bits: 64 MB 15, 18 |
// 165, 174 | 14, 15 | 131, 136; 256 MB 69, 63 | 735, 716 | 73, 54 | 523, 513.  (Codes go through them throughout:
// past, 11 us more at 230 MB of rows.)
bool rows_past(const Seqs &s, const numrs_hip_kv_cache &c) {
  return s.total * 2 * c.kv_heads * c.head_dim * (int64_t)sizeof(float) > int64_t{128} << 20;
}

// Calls f(std::bool_constant<8 bits>, std::bool_constant<past>).
template <class F>
void with_kind(bool int8, bool past, F &&f) {
  if (int8)
    past ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
  else
    past ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

Cache device_cache(const numrs_hip_kv_cache &c, const int32_t *table, int64_t max_pages) {
  return {c.k, c.v, c.k_scale, c.v_scale, c.pages, max_pages, table, paging::log2_of(c.page_size),
          (int)c.kv_heads, (int)c.head_dim};
}

// The checks that the calls on a cache share.
int check_cache(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache, const int32_t *table,
                int64_t max_pages, const int32_t *lengths, int64_t n, const char *what) {
  if (ctx->destroyed) return fail(ctx, NUMRS_HIP_E_INVALID, "context already destroyed");
  int code = 0;
  if (const char *why = paging::refuse_cache(cache, &code)) return fail(ctx, code, "%s: %s", what, why);
  if (const char *why = paging::refuse_table(table, max_pages, lengths, n, &code))
    return fail(ctx, code, "%s: %s", what, why);
  return NUMRS_HIP_OK;
}

int check_rows(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache, const numrs_hip_seqs *seqs,
               const void *k, const void *v, int64_t ld, const int32_t *table, int64_t max_pages,
               const int32_t *ends, const char *what) {
  if (seqs == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: null sequences", what);
  const Seqs &s = *seqs->s;
  if (s.ctx != ctx)
    return fail(ctx, NUMRS_HIP_E_INVALID, "%s: the sequences belong to another context", what);
  if (int rc = check_cache(ctx, cache, table, max_pages, ends, s.n, what)) return rc;
  if (s.total > 0 && (k == nullptr || v == nullptr))
    return fail(ctx, NUMRS_HIP_E_INVALID, "%s: null pointer", what);
  if (paging::bad_stride(ld, cache->kv_heads * cache->head_dim))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: the row stride is below a row's width or above 2^31 - 1",
                what);
  if (paging::bad_grid(s.tiles * cache->kv_heads))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many tokens times heads", what);
  return NUMRS_HIP_OK;
}

}  // namespace

namespace numrs_hip {

int paged_steps(numrs_hip_ctx *ctx, const numrs_hip_kv_cache &cache, const float *q, int64_t ld_q, int64_t heads,
                const int32_t *table, int64_t max_pages, const int32_t *lengths, int64_t n, const SeqTile *list,
                float *out, int64_t ld_out) {
  const int hk = (int)cache.kv_heads, dh = (int)cache.head_dim, group = (int)heads / hk;
  const int blocks = (group + 15) / 16;
  // A workgroup of eight waves a CU, which the registers allow, each with an even share of the tokens;
  // a kv head has as many at most as two levels of joins add.  Against two of four waves, with all loads
  // through the caches, us: 333 tokens of 8 heads of 64 in fp32 11.6, 11; 34 thousand tokens of 40 sequences
  // in 8 bits 39, 52; 131072 tokens of one head of 128 41, 50; 640 thousand tokens of 96 sequences, 5.2 GB, 868,
  // 882 (784 past the caches as now).  Shares of 2 to 16 units
  // at least, which leave fewer parts to join, were slower throughout.
  const int shares = std::min(std::max(1, (ctx->num_cus + hk * blocks - 1) / (hk * blocks)),
                              paged::kJoin * paged::kJoin);
  const int64_t wgs = (int64_t)shares * hk * blocks;
  TempBlock parts(ctx);
  const int dp = (dh + 31) / 32 * 32;
  if (int rc = parts.alloc((size_t)(2 * wgs * (32 + 16 * dp)) * sizeof(float))) return rc;
  unsigned *arrivals = nullptr;
  if (int rc = arrival_counters(ctx, (size_t)(3 * wgs), &arrivals)) return rc;
  const paged::SplitArgs a{device_cache(cache, table, max_pages), q, lengths, out, parts.f(), arrivals, ld_q,
                           ld_out, (int)n, (int)heads, blocks, shares,
                           kLog2e / std::sqrt((float)dh), list};
  auto launch = [&](auto padded) {
    constexpr int DP = decltype(padded)::value;
    auto kind = [&](auto int8, auto listed) {
      paged::split_rows<decltype(int8)::value, DP, decltype(listed)::value>
          <<<(unsigned)wgs, 64 * paged::kWaves, 0, ctx->stream>>>(a);
    };
    with_kind(cache.format == NUMRS_HIP_KV_INT8, list != nullptr, kind);
  };
  switch (dp) {
    case 32: launch(std::integral_constant<int, 32>{}); break;
    case 64: launch(std::integral_constant<int, 64>{}); break;
    case 96: launch(std::integral_constant<int, 96>{}); break;
    default: launch(std::integral_constant<int, 128>{});
  }
  return check_launch(ctx, "split_rows");
}

}  // namespace numrs_hip

extern "C" {

int numrs_hip_kv_cache_write(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache,
                             const numrs_hip_seqs *seqs, const float *k, const float *v,
                             int64_t ld, const int32_t *table, int64_t max_pages,
                             const int32_t *ends) {
  NRS_CHECK_CTX(ctx);
  if (int rc = check_rows(ctx, cache, seqs, k, v, ld, table, max_pages, ends, "kv_cache_write"))
    return rc;
  const Seqs &s = *seqs->s;
  if (s.total == 0) return NUMRS_HIP_OK;
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  const RowArgs a{device_cache(*cache, table, max_pages), s.in_order, ends, k, v, nullptr, nullptr, ld};
  const unsigned grid = (unsigned)(s.tiles * cache->kv_heads);
  with_kind(cache->format == NUMRS_HIP_KV_INT8, rows_past(s, *cache), [&](auto int8, auto past) {
    write_rows<decltype(int8)::value, decltype(past)::value>
        <<<grid, 256, 0, ctx->stream>>>(a, row_lanes((int)cache->head_dim));
  });
  return check_launch(ctx, "write_rows");
}

int numrs_hip_kv_cache_read(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache,
                            const numrs_hip_seqs *seqs, float *k, float *v, int64_t ld,
                            const int32_t *table, int64_t max_pages, const int32_t *ends) {
  NRS_CHECK_CTX(ctx);
  if (int rc = check_rows(ctx, cache, seqs, k, v, ld, table, max_pages, ends, "kv_cache_read"))
    return rc;
  const Seqs &s = *seqs->s;
  if (s.total == 0) return NUMRS_HIP_OK;
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  const RowArgs a{device_cache(*cache, table, max_pages), s.in_order, ends, nullptr, nullptr, k, v, ld};
  const unsigned grid = (unsigned)(s.tiles * cache->kv_heads);
  with_kind(cache->format == NUMRS_HIP_KV_INT8, rows_past(s, *cache), [&](auto int8, auto past) {
    read_rows<decltype(int8)::value, decltype(past)::value>
        <<<grid, 256, 0, ctx->stream>>>(a, row_lanes((int)cache->head_dim));
  });
  return check_launch(ctx, "read_rows");
}

int numrs_hip_kv_cache_append(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache,
                              const numrs_hip_seqs *seqs, const float *qkv, int64_t ld,
                              const float *q_weight, const float *k_weight, float eps,
                              const numrs_hip_rotary *rotary, float *q, int64_t ld_q, int64_t heads,
                              const int32_t *table, int64_t max_pages, const int32_t *ends) {
  NRS_CHECK_CTX(ctx);
  const char *what = "kv_cache_append";
  if (int rc = check_rows(ctx, cache, seqs, qkv, qkv, ld, table, max_pages, ends, what)) return rc;
  const int64_t hk = cache->kv_heads, dh = cache->head_dim;
  if (const char *why = paging::refuse_heads(heads, hk, dh)) return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: %s", what, why);
  if (paging::bad_stride(ld, (heads + 2 * hk) * dh) || (q != nullptr && paging::bad_stride(ld_q, heads * dh)))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: a row stride is below its row's width or above 2^31 - 1", what);
  int code = 0;
  if (const char *why = rotary::refuse_rotary(rotary, dh, &code)) return fail(ctx, code, "%s: %s", what, why);
  if (const char *why = rotary::refuse_eps(eps)) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: %s", what, why);
  const Seqs &s = *seqs->s;
  const int lanes = rotary::lanes_of(dh), parts = rotary::parts_of(lanes);
  if (paging::bad_grid(s.tiles * (hk + 2 * parts)))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many tokens times heads", what);
  if (s.total == 0) return NUMRS_HIP_OK;
  if (q != nullptr && paging::rows_meet({qkv, (heads + 2 * hk) * dh, ld}, {q, heads * dh, ld_q}, s.total))
    return fail(ctx, NUMRS_HIP_E_INVALID, "%s: the queries' result overlaps the projection", what);
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  AppendArgs b{{device_cache(*cache, table, max_pages), s.in_order, ends, nullptr, nullptr, nullptr, nullptr, ld},
               {s.in_order, ends, qkv, q_weight, k_weight, q, ld, ld_q, (int)heads, (int)hk, q != nullptr ? (int)heads : 0,
                1, (int)dh, lanes, eps, 1.0 / (double)dh, rotary::turn_of(rotary)},
               (unsigned)(s.tiles * hk), parts};
  unsigned grid = b.keys;
  if (q != nullptr) {
    b.row.per = rotary::heads_each(ctx, s.tiles * parts, b.row.slots);
    grid += (unsigned)(s.tiles * parts) * ((b.row.slots + b.row.per - 1) / b.row.per);
  }
  with_kind(cache->format == NUMRS_HIP_KV_INT8, rows_past(s, *cache), [&](auto int8, auto past) {
    append_rows<decltype(int8)::value, decltype(past)::value><<<grid, 256, 0, ctx->stream>>>(b);
  });
  return check_launch(ctx, "append_rows");
}

int numrs_hip_attention_paged(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache, const float *q,
                              int64_t ld_q, int64_t heads, const int32_t *table,
                              int64_t max_pages, const int32_t *lengths, int64_t n, float *out,
                              int64_t ld_out) {
  NRS_CHECK_CTX(ctx);
  if (int rc = check_cache(ctx, cache, table, max_pages, lengths, n, "attention_paged")) return rc;
  if (const char *why = paging::refuse_heads(heads, cache->kv_heads, cache->head_dim))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "attention_paged: %s", why);
  if (paging::bad_stride(ld_q, heads * cache->head_dim) ||
      paging::bad_stride(ld_out, heads * cache->head_dim))
    return fail(ctx, NUMRS_HIP_E_SHAPE,
                "attention_paged: a row stride is below its row's width or above 2^31 - 1");
  if (n * heads >= int64_t{1} << 31)
    return fail(ctx, NUMRS_HIP_E_SHAPE, "attention_paged: too many rows times heads");
  if (n == 0) return NUMRS_HIP_OK;
  if (q == nullptr || out == nullptr)
    return fail(ctx, NUMRS_HIP_E_INVALID, "attention_paged: null pointer");
  DeviceScope dev(ctx);
  return paged_steps(ctx, *cache, q, ld_q, heads, table, max_pages, lengths, n, nullptr, out, ld_out);
}

}  // extern "C"
