// Attention of new tokens over a paged key-value cache (no reference op): token r of a sequence with n new
// tokens, at position p = ends - n + r, attends to the cached tokens 0 .. p,
//   out = sum_j softmax_j(q . k_j / sqrt(dh)) v_j,   j <= p.
#include <algorithm>
#include <cmath>

#include "packed.h"
#include "paged_split.h"

namespace {

using namespace numrs_hip;
using paged::Cache;

struct ChunkArgs {
  Cache c;
  const SeqTile *tiles;
  const int32_t *ends;
  const float *q;
  float *out;
  int64_t ld_q, ld_out;
  int heads;
  bool int8;
  float alpha;  // log2(e) / sqrt(dh)
};

// Value d of a cached key or value.
__device__ __forceinline__ float key_at(const ChunkArgs &a, int64_t row, int d) {
  if (!a.int8) return static_cast<const float *>(a.c.k)[row * a.c.dh + d];
  return (float)((int)static_cast<const uint8_t *>(a.c.k)[row * a.c.dh + d] - 128) * a.c.ks[row];
}
__device__ __forceinline__ float value_at(const ChunkArgs &a, int64_t row, int d) {
  if (!a.int8) return static_cast<const float *>(a.c.v)[row * a.c.dh + d];
  const int64_t at = (row & ~int64_t{3}) * a.c.dh + 4 * d + (row & 3);
  return (float)((int)static_cast<const uint8_t *>(a.c.v)[at] - 128) * a.c.vs[row];
}

// A wave a row: 64 tokens at a time, one a lane for the scores, a column a lane for the result.
__global__ void __launch_bounds__(64) chunk_rows(ChunkArgs a) {
  __shared__ float x[128];
  const SeqTile t = a.tiles[blockIdx.x / a.heads];
  const int h = blockIdx.x % a.heads, lane = threadIdx.x, dh = a.c.dh, g = h / (a.heads / a.c.kv_heads);
  const int64_t len = paging::held(a.ends[t.seq], a.c.max_pages, a.c.shift);
  const int32_t *pages = a.c.table + (int64_t)t.seq * a.c.max_pages;
  for (int r = t.t0; r < min(t.len, t.t0 + kTile); ++r) {
    const int64_t row = t.row0 + r, end = min(len, (int64_t)a.ends[t.seq] - t.len + r + 1);
    __syncthreads();
    for (int d = lane; d < dh; d += 64) x[d] = a.q[row * a.ld_q + (int64_t)h * dh + d];
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    double o0 = 0.0, o1 = 0.0;  // sums of values before the division: they may pass fp32's range
    bool seen = false;
    for (int64_t j0 = 0; j0 < end; j0 += 64) {
      const int64_t j = j0 + lane;
      const int page = j < end ? paging::page_of(pages, a.c.max_pages, a.c.shift, a.c.pages, j) : -1;
      const int64_t at = paging::page_base(max(page, 0), a.c.kv_heads, g, a.c.shift, 1) + (j & ((1 << a.c.shift) - 1));
      float s = -INFINITY;
      if (page >= 0) {
        s = 0.f;
        for (int d = 0; d < dh; ++d) s = fmaf(x[d], key_at(a, at, d), s);
        s *= a.alpha;
      }
      seen |= __any(page >= 0);
      const float top = fmaxf(m, wave_max(s));
      const float p = page < 0 || s == -INFINITY ? 0.f : exp2f(s - top), c = m == -INFINITY ? 0.f : exp2f(m - top);
      m = top;
      l = l * c + wave_sum(p);
      o0 *= c, o1 *= c;
      for (int e = 0; e < 64; ++e) {
        const int pe = __shfl(page, e);
        if (pe < 0) continue;
        const float w = __shfl(p, e);
        const int64_t ae = paging::page_base(pe, a.c.kv_heads, g, a.c.shift, 1) + ((j0 + e) & ((1 << a.c.shift) - 1));
        if (lane < dh) o0 = fma((double)w, (double)value_at(a, ae, lane), o0);
        if (lane + 64 < dh) o1 = fma((double)w, (double)value_at(a, ae, lane + 64), o1);
      }
    }
    float *o = a.out + row * a.ld_out + (int64_t)h * dh;
    if (lane < dh) o[lane] = seen ? (float)(o0 / l) : 0.f;
    if (lane + 64 < dh) o[lane + 64] = seen ? (float)(o1 / l) : 0.f;
  }
}

}  // namespace

extern "C" int numrs_hip_attention_paged_chunk(numrs_hip_ctx *ctx, const numrs_hip_kv_cache *cache,
                                               const numrs_hip_seqs *seqs, const float *q, int64_t ld_q,
                                               int64_t heads, const int32_t *table, int64_t max_pages,
                                               const int32_t *ends, float *out, int64_t ld_out) {
  NRS_CHECK_CTX(ctx);
  const char *what = "attention_paged_chunk";
  if (ctx->destroyed) return fail(ctx, NUMRS_HIP_E_INVALID, "context already destroyed");
  if (seqs == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: null sequences", what);
  const Seqs &s = *seqs->s;
  if (s.ctx != ctx) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: the sequences belong to another context", what);
  int code = 0;
  if (const char *why = paging::refuse_cache(cache, &code)) return fail(ctx, code, "%s: %s", what, why);
  if (const char *why = paging::refuse_table(table, max_pages, ends, s.n, &code)) return fail(ctx, code, "%s: %s", what, why);
  const int64_t hk = cache->kv_heads, dh = cache->head_dim;
  if (const char *why = paging::refuse_heads(heads, hk, dh)) return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: %s", what, why);
  if (paging::bad_stride(ld_q, heads * dh) || paging::bad_stride(ld_out, heads * dh))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: a row stride is below its row's width or above 2^31 - 1", what);
  if (paging::bad_grid(s.tiles * heads)) return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many tokens times heads", what);
  if (s.total == 0) return NUMRS_HIP_OK;
  if (q == nullptr || out == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: null pointer", what);
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  const ChunkArgs a{{cache->k, cache->v, cache->k_scale, cache->v_scale, cache->pages, max_pages, table,
                     paging::log2_of(cache->page_size), (int)hk, (int)dh},
                    s.in_order, ends, q, out, ld_q, ld_out, (int)heads, cache->format == NUMRS_HIP_KV_INT8,
                    1.44269504088896341f / std::sqrt((float)dh)};
  chunk_rows<<<(unsigned)(s.tiles * heads), 64, 0, ctx->stream>>>(a);
  return check_launch(ctx, "chunk_rows");
}
