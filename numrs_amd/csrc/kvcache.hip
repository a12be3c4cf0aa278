// A paged key-value cache in fp32 or 8-bit codes, written, read back and attended to (no reference
// op).  paging.h says where a token lies; every position goes through paging::page_of.
#include <algorithm>
#include <cmath>

#include "packed.h"
#include "paged_split.h"

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

// The slot of a packed row: element offset of its page and head, and its place there; page < 0
// where it has none.
struct Slot {
  int64_t base;
  int at, page;
};
__device__ __forceinline__ Slot slot_of(const Cache &c, int seq, int64_t pos, int g) {
  const int page = paging::page_of(c.table + seq * c.max_pages, c.max_pages, c.shift, c.pages, pos);
  if (page < 0) return {0, 0, -1};
  return {paging::page_base(page, c.kv_heads, g, c.shift, c.dh), (int)(pos & ((1 << c.shift) - 1)), page};
}

__device__ __forceinline__ float quantised_scale(float top) { return top / 127.0f; }

// The code of x in a row of that scale: x / scale is rounded to fp32, then to a whole number.
__device__ __forceinline__ uint8_t code_of(float x, float scale) {
  if (!(scale > 0.f)) return 128;
  return (uint8_t)((int)fminf(fmaxf(rintf(x / scale), -127.f), 127.f) + 128);
}

// One wave: a row of keys or values.
template <bool INT8>
__device__ void write_row(const Cache &c, const float *x, const Slot &s, bool values) {
  const int lane = threadIdx.x & 63;
  const float x0 = lane < c.dh ? x[lane] : 0.f, x1 = lane + 64 < c.dh ? x[lane + 64] : 0.f;
  void *p = values ? c.v : c.k;
  if constexpr (!INT8) {
    float *o = static_cast<float *>(p) + s.base + (int64_t)s.at * c.dh;
    if (lane < c.dh) o[lane] = x0;
    if (lane + 64 < c.dh) o[lane + 64] = x1;
  } else {
    const bool finite = __builtin_isfinite(x0) && __builtin_isfinite(x1);
    const float top = wave_max(fmaxf(fabsf(x0), fabsf(x1)));
    const float scale = __all(finite) ? quantised_scale(top) : NAN;
    uint8_t *o = static_cast<uint8_t *>(p) + s.base;
    const int64_t row = (int64_t)s.at * c.dh;
    if (lane < c.dh) o[values ? paging::value_code(s.at, lane, c.dh) : row + lane] = code_of(x0, scale);
    if (lane + 64 < c.dh)
      o[values ? paging::value_code(s.at, lane + 64, c.dh) : row + lane + 64] = code_of(x1, scale);
    if (lane == 0) (values ? c.vs : c.ks)[s.base / c.dh + s.at] = scale;
  }
}

template <bool INT8>
__global__ void __launch_bounds__(256) write_rows(RowArgs a) {
  const SeqTile t = a.tiles[blockIdx.x / a.c.kv_heads];
  const int g = blockIdx.x % a.c.kv_heads, end = min(t.len, t.t0 + kTile);
  for (int r = t.t0 + (threadIdx.x >> 6); r < end; r += 4) {
    const Slot s = slot_of(a.c, t.seq, (int64_t)a.ends[t.seq] - t.len + r, g);
    if (s.page < 0) continue;
    const int64_t at = (int64_t)(t.row0 + r) * a.ld + (int64_t)g * a.c.dh;
    write_row<INT8>(a.c, a.k + at, s, false);
    write_row<INT8>(a.c, a.v + at, s, true);
  }
}

template <bool INT8>
__device__ __forceinline__ float read_one(const Cache &c, const Slot &s, int d, bool values) {
  if (s.page < 0) return 0.f;
  const void *p = values ? c.v : c.k;
  if constexpr (!INT8) return static_cast<const float *>(p)[s.base + (int64_t)s.at * c.dh + d];
  const uint8_t *o = static_cast<const uint8_t *>(p) + s.base;
  const float scale = (values ? c.vs : c.ks)[s.base / c.dh + s.at];
  const int code = o[values ? paging::value_code(s.at, d, c.dh) : (int64_t)s.at * c.dh + d];
  return (float)(code - 128) * scale;
}

template <bool INT8>
__global__ void __launch_bounds__(256) read_rows(RowArgs a) {
  const SeqTile t = a.tiles[blockIdx.x / a.c.kv_heads];
  const int g = blockIdx.x % a.c.kv_heads, end = min(t.len, t.t0 + kTile), lane = threadIdx.x & 63;
  for (int r = t.t0 + (threadIdx.x >> 6); r < end; r += 4) {
    const Slot s = slot_of(a.c, t.seq, (int64_t)a.ends[t.seq] - t.len + r, g);
    const int64_t at = (int64_t)(t.row0 + r) * a.ld + (int64_t)g * a.c.dh;
    for (int d = lane; d < a.c.dh; d += 64) {
      a.ko[at + d] = read_one<INT8>(a.c, s, d, false);
      a.vo[at + d] = read_one<INT8>(a.c, s, d, true);
    }
  }
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
  if (s.tiles * cache->kv_heads >= int64_t{1} << 31)
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many tokens times heads", what);
  return NUMRS_HIP_OK;
}

}  // namespace

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
  DeviceScope dev(ctx);
  const RowArgs a{device_cache(*cache, table, max_pages), s.in_order, ends, k, v, nullptr, nullptr, ld};
  const unsigned grid = (unsigned)(s.tiles * cache->kv_heads);
  if (cache->format == NUMRS_HIP_KV_F32)
    write_rows<false><<<grid, 256, 0, ctx->stream>>>(a);
  else
    write_rows<true><<<grid, 256, 0, ctx->stream>>>(a);
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
  DeviceScope dev(ctx);
  const RowArgs a{device_cache(*cache, table, max_pages), s.in_order, ends, nullptr, nullptr, k, v, ld};
  const unsigned grid = (unsigned)(s.tiles * cache->kv_heads);
  if (cache->format == NUMRS_HIP_KV_F32)
    read_rows<false><<<grid, 256, 0, ctx->stream>>>(a);
  else
    read_rows<true><<<grid, 256, 0, ctx->stream>>>(a);
  return check_launch(ctx, "read_rows");
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
  const int hk = (int)cache->kv_heads, dh = (int)cache->head_dim, group = (int)heads / hk;
  const int blocks = (group + 15) / 16;
  // A workgroup of eight waves a CU, which the registers allow, each with an even share of the tokens;
  // a kv head has as many at most as two levels of joins add.
  const int shares = std::min(std::max(1, (ctx->num_cus + hk * blocks - 1) / (hk * blocks)),
                              paged::kJoin * paged::kJoin);
  const int64_t wgs = (int64_t)shares * hk * blocks;
  TempBlock parts(ctx);
  const int dp = (dh + 31) / 32 * 32;
  if (int rc = parts.alloc((size_t)(2 * wgs * (32 + 16 * dp)) * sizeof(float))) return rc;
  unsigned *arrivals = nullptr;
  if (int rc = arrival_counters(ctx, (size_t)(3 * wgs), &arrivals)) return rc;
  const paged::SplitArgs a{device_cache(*cache, table, max_pages), q, lengths, out, parts.f(), arrivals, ld_q,
                           ld_out, (int)n, (int)heads, blocks, shares,
                           kLog2e / std::sqrt((float)dh)};
  auto launch = [&](auto padded) {
    constexpr int DP = decltype(padded)::value;
    if (cache->format == NUMRS_HIP_KV_F32)
      paged::split_rows<false, DP><<<(unsigned)wgs, 64 * paged::kWaves, 0, ctx->stream>>>(a);
    else
      paged::split_rows<true, DP><<<(unsigned)wgs, 64 * paged::kWaves, 0, ctx->stream>>>(a);
  };
  switch (dp) {
    case 32: launch(std::integral_constant<int, 32>{}); break;
    case 64: launch(std::integral_constant<int, 64>{}); break;
    case 96: launch(std::integral_constant<int, 96>{}); break;
    default: launch(std::integral_constant<int, 128>{});
  }
  return check_launch(ctx, "split_rows");
}

}  // extern "C"
