// Attention of new tokens over a paged key-value cache (no reference op): token r of a sequence with n new
// tokens, at position p = ends - n + r, attends to the cached tokens 0 .. p,
//   out = sum_j softmax_j(q . k_j / sqrt(dh)) v_j,   j <= p.
#include <algorithm>
#include <cmath>

#include "chunk_tiles.h"

namespace {

using namespace numrs_hip;

constexpr float kLog2e = 1.44269504088896341f;

// From kManyRows query rows of a kv head on a sequence (the batch's mean), over caches in fp32, stages are made images
// first, which costs a pass over the cached tokens and saves every block of 256 rows its own splitting.  On MI355X, without against with,
// us, 32 heads of 128 in groups of 4 over 8192 tokens: 256 rows 70, 84; 512 rows 95, 105; 1024 rows 145, 149; 2048
// rows 260, 242; of four sequences in groups of 8: 1024 rows over 8192 147, 146; 2048 over 2048 101, 97; 4096 over none
// 65, 63; 16384 over 0 to 16384 1546, 1352; heads of 64 over 2048: 1024 rows 67, 71; 2048 rows 110, 110.  The images
// have room for all that the table's width can hold, since only the device knows what it does; past kMostImages they
// are not made, and a table that is wider than its sequences need can lose them so (two sequences of 2048 rows and 8 kv
// heads of 128: from 65536 tokens on).
constexpr int64_t kManyRows = 2048, kMostImages = int64_t{1} << 30;
// Up to so many rows blocks have 128 in two sets of waves, beyond 256 in one, which reads the tokens half as often.
// 256 against 128, us: 128 rows over 131072 tokens 70, 71; 32 heads of 128 over 8192, fp32 and 8 bits: 32 rows 44, 44
// and 34, 33; 128 rows 50, 51 and 39, 41; 256 rows 68, 66 and 51, 52; 512 rows 95, 97 and 68, 75; eight sequences
// over 500, heads of 64: 64 rows 24, 24; 128 rows 27, 28; 256 rows 35, 32; 512 rows 46, 47.
constexpr int64_t kFewRows = 256;

template <bool INT8, int DP, int Z, bool PACKED>
int walk(numrs_hip_ctx *ctx, chunk::Args a) {
  constexpr int ROWS = 256 / Z;
  const unsigned wgs = (unsigned)ctx->num_cus;
  TempBlock parts(ctx);
  const size_t image = (size_t)(2 * wgs) * chunk::kPart<DP, ROWS> * sizeof(float);
  if (int rc = parts.alloc(image + wgs * sizeof(chunk::Cut))) return rc;
  a.parts = parts.f();
  a.cuts = reinterpret_cast<chunk::Cut *>(static_cast<char *>(parts.p) + image);
  chunk::walk_blocks<INT8, DP, Z, PACKED><<<wgs, chunk::kThreads, 0, ctx->stream>>>(a);
  if (int rc = check_launch(ctx, "walk_blocks")) return rc;
  chunk::join_parts<DP, ROWS><<<4 * wgs, 256, 0, ctx->stream>>>(a, (int)wgs);
  return check_launch(ctx, "join_parts");
}

template <bool INT8, int DP, int Z>
int run(numrs_hip_ctx *ctx, const Seqs &s, chunk::Args a) {
  if constexpr (!INT8 && Z == 1) {
    const int64_t rows = (s.total - s.singles) * a.group;
    const int64_t stages = ((a.c.max_pages << a.c.shift) + chunk::kStage - 1) / chunk::kStage;
    const int64_t images = s.severals * a.c.kv_heads * stages, bytes = images * chunk::kImage<DP>;
    if (rows >= s.severals * kManyRows && bytes <= kMostImages) {
      TempBlock block(ctx);
      if (int rc = block.alloc((size_t)bytes)) return rc;
      a.images = static_cast<char *>(block.p);
      a.most_stages = (int)stages;
      chunk::pack_stages<DP><<<(unsigned)images, chunk::kThreads, 0, ctx->stream>>>(a);
      if (int rc = check_launch(ctx, "pack_stages")) return rc;
      return walk<INT8, DP, Z, true>(ctx, a);
    }
  }
  return walk<INT8, DP, Z, false>(ctx, a);
}

template <bool INT8, int Z>
int run_dp(numrs_hip_ctx *ctx, const Seqs &s, const chunk::Args &a) {
  switch ((a.c.dh + 31) / 32) {
    case 1: return run<INT8, 32, Z>(ctx, s, a);
    case 2: return run<INT8, 64, Z>(ctx, s, a);
    case 3: return run<INT8, 96, Z>(ctx, s, a);
    default: return run<INT8, 128, Z>(ctx, s, a);
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
  // rows and tokens are counted in 32 bits, in blocks and stages
  if (s.longest * (heads / hk) > INT32_MAX - 1024)
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many new tokens times heads of a group in one sequence", what);
  if (max_pages > (INT32_MAX - 1024) / cache->page_size)
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: a table's row has pages for 2^31 tokens or more", what);
  if (s.total == 0) return NUMRS_HIP_OK;
  if (q == nullptr || out == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: null pointer", what);
  if (paging::rows_meet({q, heads * dh, ld_q}, {out, heads * dh, ld_out}, s.total))
    return fail(ctx, NUMRS_HIP_E_INVALID, "%s: the result overlaps the queries", what);
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  // Sequences of one row go the way of the decoding steps, made for few rows and many tokens: 24 of them, of 1 to 5000
  // tokens, beside five pieces of prompts, 8 heads of 128 in 8 bits: 20 us less than as blocks of rows.
  if (s.singles > 0)
    if (int rc = paged_steps(ctx, *cache, q, ld_q, heads, table, max_pages, ends, s.singles, s.single, out, ld_out))
      return rc;
  if (s.severals == 0) return NUMRS_HIP_OK;
  chunk::Args a{{cache->k, cache->v, cache->k_scale, cache->v_scale, cache->pages, max_pages, table,
                 paging::log2_of(cache->page_size), (int)hk, (int)dh},
                s.several, ends, q, out, nullptr, nullptr, 0, nullptr, ld_q, ld_out, (int)s.severals,
                (int)(heads / hk), 0.f, 0};
  a.mant = std::frexp(kLog2e / std::sqrt((float)dh), &a.exp);
  const bool few = s.longest * a.group <= kFewRows;
  if (cache->format == NUMRS_HIP_KV_INT8) return few ? run_dp<true, 2>(ctx, s, a) : run_dp<true, 1>(ctx, s, a);
  return few ? run_dp<false, 2>(ctx, s, a) : run_dp<false, 1>(ctx, s, a);
}
