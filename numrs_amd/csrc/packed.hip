// Causal attention with grouped heads over packed sequences (no reference op), without an S x S
// buffer: the forward keeps a running softmax reference m and sum l for each row,
//   p_ij = exp(s_ij - m_i) / l_i,  s_ij = q_i . k_j / sqrt(dh),  j <= i of the same sequence,
// and the backward forms p again from them.
//
// packed_tiles.h has the kernels that ordinary values take.  The row kernels here are the plain fp32 form,
// a wave a row, for blocks that meet a value which those cannot take: not finite, from 2^50 (queries and keys)
// or 2^80 (values and the output's gradient) on, or of 64 tokens that differ by more than 2^140.  They read every
// key a row at a time, some 150 times slower (8192 tokens, 16 heads of 128, a value at their start infinite:
// 134 ms against 0.8; rows that are NaN throughout end at the first such score), and are there so that such a
// value does to the rows that attend to it what fp32 arithmetic does, and nothing to the others.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "packed_tiles.h"
#include "paging.h"

namespace {

using namespace numrs_hip;

constexpr float kLog2e = 1.44269504088896341f;

struct FwdArgs {
  const SeqTile *tiles;
  const float *q, *k, *v;
  float *out, *stats;
  int64_t ld_q, ld_kv, ld_out;
  int heads, kv_heads, dh;
  float alpha;  // log2(e) / sqrt(dh)
};

__device__ __forceinline__ float lane_of(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// Dot product of a row in LDS and one in memory.
__device__ __forceinline__ float dot_row(const float *x, const float *y, int dh) {
  float s = 0.f;
  for (int d = 0; d < dh; d += 8) {
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaf(x[d + e], y[d + e], a);
    s += a;
  }
  return s;
}

// One wave: query row r of head h, in plain fp32, 64 keys at a time (a key a lane for the scores,
// a column a lane for the output).  x: the wave's dh floats of LDS.
__device__ void row_forward(const FwdArgs &a, const SeqTile &t, int r, int h, float *x) {
  const int lane = threadIdx.x & 63, g = h / (a.heads / a.kv_heads);
  const int64_t row = t.row0 + r;
  for (int d = lane; d < a.dh; d += 64) x[d] = a.q[row * a.ld_q + (int64_t)h * a.dh + d];
  __builtin_amdgcn_wave_barrier();
  const float *k = a.k + t.row0 * a.ld_kv + (int64_t)g * a.dh, *v = a.v + t.row0 * a.ld_kv + (int64_t)g * a.dh;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 <= r; j0 += 64) {
    const int j = j0 + lane, n = min(64, r + 1 - j0);
    const float s = lane < n ? dot_row(x, k + j * a.ld_kv, a.dh) * a.alpha : -INFINITY;
    const float top = fmaxf(m, wave_max(s));
    // Scores of -inf so far count nothing beside a finite one that may follow. A row that has no other has no
    // softmax: l stays 0 and the result NaN, as the formula has it.
    const float p = lane >= n || s == -INFINITY ? 0.f : exp2f(s - top), c = m == -INFINITY ? 0.f : exp2f(m - top);
    m = top;
    l = l * c + wave_sum(p);
    if (l != l) break;  // a score is NaN or infinite: so is the row, whatever follows
    float t0 = 0.f, t1 = 0.f;  // the block's sum apart, so that a long sum's rounding stays small
    for (int e = 0; e < n; ++e) {
      const float w = lane_of(p, e);
      const float *y = v + (j0 + e) * a.ld_kv;
      if (lane < a.dh) t0 = fmaf(w, y[lane], t0);
      if (lane + 64 < a.dh) t1 = fmaf(w, y[lane + 64], t1);
    }
    o0 = fmaf(o0, c, t0), o1 = fmaf(o1, c, t1);
  }
  float *o = a.out + row * a.ld_out + (int64_t)h * a.dh;
  if (lane < a.dh) o[lane] = o0 / l;
  if (lane + 64 < a.dh) o[lane + 64] = o1 / l;
  if (a.stats != nullptr && lane == 0) {
    float *st = a.stats + (row * a.heads + h) * 2;
    st[0] = m, st[1] = l;
  }
}

constexpr int kRows = 4;  // waves of a workgroup

// A block of query rows of one head.
template <int DP, int Z>
__global__ void __launch_bounds__(256, 2) forward_block(FwdArgs a, tiles::ForwardArgs f) {
  __shared__ __attribute__((aligned(16))) char lds[tiles::Walk<DP, Z>::kForward];
  const SeqTile t = a.tiles[blockIdx.x / a.heads];
  const int h = blockIdx.x % a.heads;
  if (tiles::forward_tile<DP, Z>(f, t, h, lds)) return;
  const int w = threadIdx.x >> 6, end = min(t.len, t.t0 + 128 / Z);
  for (int r = t.t0 + w; r < end; r += kRows) row_forward(a, t, r, h, reinterpret_cast<float *>(lds) + 128 * w);
}

struct BwdArgs {
  const SeqTile *tiles;
  const float *q, *k, *v, *out, *dout, *stats;
  int64_t ld_q, ld_kv, ld_out;
};

// A score less the row's largest. Where the tiles had the row in the forward, whose sums run in another order, it
// is off by some 2^-23 of the score, and may come out above 0, which at large scores would be any power of
// two. NaN stays.
__device__ __forceinline__ float at_most_0(float x) { return x > 0.f ? 0.f : x; }

__device__ __forceinline__ void put(float *p, float v, int accumulate) { *p = accumulate ? *p + v : v; }

// One wave: dq of query row r and head h, in plain fp32.  x: two rows of LDS.
__device__ void row_dq(const BwdArgs &b, const tiles::BackwardArgs &a, const SeqTile &t, int r, int h, float *x) {
  const int lane = threadIdx.x & 63, g = h / (a.heads / a.kv_heads);
  const int64_t row = t.row0 + r, at = row * b.ld_out + (int64_t)h * a.dh;
  float dot = 0.f;
  for (int d = lane; d < a.dh; d += 64) {
    x[d] = b.q[row * b.ld_q + (int64_t)h * a.dh + d];
    x[128 + d] = b.dout[at + d];
    dot = fmaf(x[128 + d], b.out[at + d], dot);
  }
  const float D = wave_sum(dot);
  __builtin_amdgcn_wave_barrier();
  const float *k = b.k + t.row0 * b.ld_kv + (int64_t)g * a.dh, *v = b.v + t.row0 * b.ld_kv + (int64_t)g * a.dh;
  const float *st = b.stats + (row * a.heads + h) * 2;
  const float m = st[0], l = st[1];
  float o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 <= r; j0 += 64) {
    const int j = j0 + lane, n = min(64, r + 1 - j0);
    float ds = 0.f;
    if (lane < n) {
      const float p = exp2f(at_most_0(dot_row(x, k + j * b.ld_kv, a.dh) * a.alpha - m)) / l;
      ds = p * (dot_row(x + 128, v + j * b.ld_kv, a.dh) - D);
    }
    float t0 = 0.f, t1 = 0.f;
    for (int e = 0; e < n; ++e) {
      const float w = lane_of(ds, e);
      const float *y = k + (j0 + e) * b.ld_kv;
      if (lane < a.dh) t0 = fmaf(w, y[lane], t0);
      if (lane + 64 < a.dh) t1 = fmaf(w, y[lane + 64], t1);
    }
    o0 += t0, o1 += t1;
    if (l != l) break;
  }
  float *o = a.dq + row * a.ld_q + (int64_t)h * a.dh;
  if (lane < a.dh) put(o + lane, o0 * a.scale, a.accumulate);
  if (lane + 64 < a.dh) put(o + lane + 64, o1 * a.scale, a.accumulate);
}

// One wave: dk and dv of key row r, over a.each query heads from h0 in order.
__device__ void row_dkv(const BwdArgs &b, const tiles::BackwardArgs &a, const SeqTile &t, int r, int h0, float *x) {
  const int lane = threadIdx.x & 63, group = a.heads / a.kv_heads, g = h0 / group;
  const int64_t row = t.row0 + r, at = row * b.ld_kv + (int64_t)g * a.dh;
  for (int d = lane; d < a.dh; d += 64) x[d] = b.k[at + d], x[128 + d] = b.v[at + d];
  __builtin_amdgcn_wave_barrier();
  float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
  for (int h = h0; h < h0 + a.each; ++h) {
    const float *q = b.q + (int64_t)h * a.dh, *go = b.dout + (int64_t)h * a.dh, *out = b.out + (int64_t)h * a.dh;
    for (int i0 = r; i0 < t.len; i0 += 64) {
      const int n = min(64, t.len - i0);
      float p = 0.f, ds = 0.f;
      if (lane < n) {
        const int64_t i = t.row0 + i0 + lane;
        const float *st = b.stats + (i * a.heads + h) * 2;
        p = exp2f(at_most_0(dot_row(x, q + i * b.ld_q, a.dh) * a.alpha - st[0])) / st[1];
        ds = p * (dot_row(x + 128, go + i * b.ld_out, a.dh) - dot_row(out + i * b.ld_out, go + i * b.ld_out, a.dh));
      }
      float tk0 = 0.f, tk1 = 0.f, tv0 = 0.f, tv1 = 0.f;
      for (int e = 0; e < n; ++e) {
        const int64_t i = t.row0 + i0 + e;
        const float w = lane_of(p, e), u = lane_of(ds, e);
        if (lane < a.dh) {
          tv0 = fmaf(w, go[i * b.ld_out + lane], tv0);
          tk0 = fmaf(u, q[i * b.ld_q + lane], tk0);
        }
        if (lane + 64 < a.dh) {
          tv1 = fmaf(w, go[i * b.ld_out + lane + 64], tv1);
          tk1 = fmaf(u, q[i * b.ld_q + lane + 64], tk1);
        }
      }
      k0 += tk0, k1 += tk1, v0 += tv0, v1 += tv1;
      if (__any(p != p)) {  // (and ds with it) a row of NaN: so are all of these
        h = h0 + a.each;
        break;
      }
    }
  }
  const int64_t part = ((int64_t)h0 * a.total + row) * a.dh;
  const int64_t ck = a.each < group ? part : row * a.ld_k + (int64_t)g * a.dh;
  const int64_t cv = a.each < group ? part : row * a.ld_v + (int64_t)g * a.dh;
  if (a.dk != nullptr) {
    if (lane < a.dh) put(a.dk + ck + lane, k0 * a.scale, a.acc_kv);
    if (lane + 64 < a.dh) put(a.dk + ck + lane + 64, k1 * a.scale, a.acc_kv);
  }
  if (a.dv != nullptr) {
    if (lane < a.dh) put(a.dv + cv + lane, v0, a.acc_kv);
    if (lane + 64 < a.dh) put(a.dv + cv + lane + 64, v1, a.acc_kv);
  }
}

// The backward's blocks in one launch, so that each kind's last workgroups run beside the other's (37 us for 16
// x 256 tokens, 8 heads of 64, 97 for 2736 tokens, 10 heads of 80; with earlier splits 35 against 18 + 23 apart,
// and 93 against 46 + 57):
// first `keys` workgroups with a block of key rows of one kv head, or one query head's part of it, then a
// block of query rows of one head each.
template <int DP, int Z>
__global__ void __launch_bounds__(256, DP <= 64 ? 2 : 1)
    backward_block(BwdArgs b, tiles::BackwardArgs a, const SeqTile *key_tiles, unsigned keys) {
  __shared__ __attribute__((aligned(16))) char lds[tiles::Walk<DP, Z>::kBack];
  const int w = threadIdx.x >> 6;
  float *row = reinterpret_cast<float *>(lds) + 256 * w;
  if (blockIdx.x < keys) {
    const int slots = a.heads / a.each;
    const SeqTile t = key_tiles[blockIdx.x / slots];
    const int h0 = blockIdx.x % slots * a.each;
    if (tiles::dkv_tile<DP, Z>(a, t, h0, lds)) return;
    for (int r = t.t0 + w; r < min(t.len, t.t0 + 128 / Z); r += kRows) row_dkv(b, a, t, r, h0, row);
  } else {
    const unsigned i = blockIdx.x - keys;
    const SeqTile t = b.tiles[i / a.heads];
    const int h = i % a.heads;
    if (tiles::dq_tile<DP, Z>(a, t, h, lds)) return;
    for (int r = t.t0 + w; r < min(t.len, t.t0 + 128 / Z); r += kRows) row_dq(b, a, t, r, h, row);
  }
}

// Adds the parts of a group's query heads in order, four values a thread: part [heads, total, dh]; dk's and
// dv's by the grid's second index.  Bound by memory: 2 x 8192 tokens, 16 heads of 128 on 4 in 38 us, 4.4 TB/s.
struct Join {
  const float *part[2];
  float *out[2];
};
__global__ void __launch_bounds__(256)
    join_heads(Join j, int64_t ld, int64_t total, int heads, int kv_heads, int dh, int accumulate) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = dh / 4, group = heads / kv_heads;
  if (i >= total * kv_heads * per) return;
  const int64_t row = i / (kv_heads * per);
  const int g = (int)(i / per % kv_heads), d = (int)(i % per) * 4;
  const float *part = j.part[blockIdx.y];
  tiles::f4 s{};
  for (int h = g * group; h < (g + 1) * group; ++h)
    s += *reinterpret_cast<const tiles::f4 *>(part + ((int64_t)h * total + row) * dh + d);
  tiles::f4u *o = reinterpret_cast<tiles::f4u *>(j.out[blockIdx.y] + row * ld + (int64_t)g * dh + d);
  if (accumulate) s += tiles::f4(*o);
  *o = s;
}

// The arguments that the forward and the backward share.
int check_packed(numrs_hip_ctx *ctx, const Seqs &s, int64_t ld_q, int64_t ld_kv, int64_t ld_out,
                 PackedHeads h, const char *what) {
  if (ctx->destroyed) return fail(ctx, NUMRS_HIP_E_INVALID, "context already destroyed");
  if (s.ctx != ctx)
    return fail(ctx, NUMRS_HIP_E_INVALID, "%s: the sequences belong to another context", what);
  if (const char *why = paging::refuse_heads(h.heads, h.kv_heads, h.dh))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: %s", what, why);
  if (paging::bad_stride(ld_q, h.heads * h.dh) || paging::bad_stride(ld_kv, h.kv_heads * h.dh) ||
      paging::bad_stride(ld_out, h.heads * h.dh))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: a row stride is below its row's width or above 2^31 - 1",
                what);
  if (paging::bad_grid(s.tiles * 2 * (h.heads + h.kv_heads)))  // the backward's largest
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many tokens times heads", what);
  return NUMRS_HIP_OK;
}

// Magnitudes from which a tile's products might pass fp32's range: a score of two such operands
// stays below 2^107, a sum of 2^20 such values times 2^22 below 2^123.
constexpr float kMostScore = 0x1p50f, kMostValue = 0x1p80f;

// Whether the kernels take blocks of 64 rows whose keys two sets of waves share, in place of 128: where
// there are fewer than two of the latter for each CU, and the longest walk decides.  Forward | forward and
// backward on MI355X, 64 rows against 128, us: 256 blocks (16 x 256 tokens, 8 heads of 64) 20, 21 | 68.6,
// 65.2; 260 (2736 tokens, 10 heads of 80) 40, 52 | 146, 160; 752 (5023 tokens, 16 heads of 64) 51, 53 | 224,
// 215; 1024 (2 x 4096 tokens, 16 heads of 128) 571, 421 | 2430, 2136.  The backward alone, 256 blocks of 8 heads
// of 64: 49, 44 for 16 x 256 tokens, but 77, 91 for 4 x 1024 and 124, 156 for 2 x 2048.
bool few_blocks(numrs_hip_ctx *ctx, const Seqs &s, int heads) { return s.blocks * heads < 2 * ctx->num_cus; }

int padded(int dh) { return (dh + 31) / 32 * 32; }

template <class F>
int with_dp(int dh, F &&f) {
  switch (padded(dh)) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 96: return f(std::integral_constant<int, 96>{});
    default: return f(std::integral_constant<int, 128>{});
  }
}

// Memory for one operand's fragments and exponents.
struct Packed {
  TempBlock block;
  char *rows = nullptr;
  int *exps = nullptr, *each = nullptr;
  explicit Packed(numrs_hip_ctx *ctx) : block(ctx) {}
  int alloc(const Seqs &s, int heads, int dh) {
    const size_t n = (size_t)s.tiles * heads, image = n * kTile * padded(dh) * 4;
    if (int rc = block.alloc(image + n * (kTile + 1) * sizeof(int))) return rc;
    rows = static_cast<char *>(block.p);
    each = reinterpret_cast<int *>(rows + image);
    exps = each + n * kTile;
    return NUMRS_HIP_OK;
  }
  tiles::Source source(const float *x, int64_t ld, int heads, float most, float by = 1.f) const {
    return {x, ld, rows, exps, each, most, by, heads, nullptr, nullptr, nullptr};
  }
};

}  // namespace

namespace numrs_hip {

int packed_forward(numrs_hip_ctx *ctx, const Seqs &s, const float *q, int64_t ld_q, const float *k,
                   const float *v, int64_t ld_kv, float *out, int64_t ld_out, float *stats,
                   PackedHeads h) {
  if (int rc = check_packed(ctx, s, ld_q, ld_kv, ld_out, h, "attention_packed")) return rc;
  if (s.total == 0) return NUMRS_HIP_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr)
    return fail(ctx, NUMRS_HIP_E_INVALID, "attention_packed: null pointer");
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  Packed pk(ctx), pv(ctx);
  const int H = (int)h.heads, Hk = (int)h.kv_heads, dh = (int)h.dh;
  if (int rc = pk.alloc(s, Hk, dh)) return rc;
  if (int rc = pv.alloc(s, Hk, dh)) return rc;
  const tiles::PackArgs p{s.in_order,
                          {pk.source(k, ld_kv, Hk, kMostScore), pv.source(v, ld_kv, Hk, kMostValue), {}, {}},
                          2 * Hk, dh};
  const float alpha = kLog2e / std::sqrt((float)dh);
  const FwdArgs a{s.by_work, q, k, v, out, stats, ld_q, ld_kv, ld_out, H, Hk, dh, alpha};
  const bool few = few_blocks(ctx, s, H);
  tiles::ForwardArgs f{q, pk.rows, pv.rows, pk.exps, pv.exps, pk.each, pv.each, out, stats,
                       ld_q, ld_out, H, Hk, dh, 0.f, 0, kMostScore};
  f.mant = std::frexp(alpha, &f.exp);
  return with_dp(dh, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    tiles::pack<DP><<<(unsigned)(s.tiles * p.slots), 256, 0, ctx->stream>>>(p);
    if (int rc = check_launch(ctx, "pack")) return rc;
    FwdArgs b = a;
    if (few) {
      b.tiles = s.few_by_work;
      forward_block<DP, 2><<<(unsigned)(s.tiles * H), 256, 0, ctx->stream>>>(b, f);
    } else {
      forward_block<DP, 1><<<(unsigned)(s.blocks * H), 256, 0, ctx->stream>>>(b, f);
    }
    return check_launch(ctx, "forward_block");
  });
}

int packed_backward(numrs_hip_ctx *ctx, const Seqs &s, const float *q, int64_t ld_q, const float *k,
                    const float *v, int64_t ld_kv, const float *out, const float *dout,
                    int64_t ld_out, const float *stats, float *dq, float *dk, float *dv,
                    PackedHeads h, int accumulate) {
  if (int rc = check_packed(ctx, s, ld_q, ld_kv, ld_out, h, "attention_packed_backward")) return rc;
  if (s.total == 0 || (dq == nullptr && dk == nullptr && dv == nullptr)) return NUMRS_HIP_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || dout == nullptr ||
      stats == nullptr)
    return fail(ctx, NUMRS_HIP_E_INVALID, "attention_packed_backward: null pointer");
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  const int H = (int)h.heads, Hk = (int)h.kv_heads, dh = (int)h.dh, group = H / Hk;
  const bool keys = dk != nullptr || dv != nullptr;
  // The query heads of a group go to workgroups of their own, whose parts are added afterwards, unless the
  // kv heads' blocks of key rows alone are two for each CU.  Forward and backward on MI355X, heads apart
  // against together, us: 64 blocks (16 x 256 tokens, 8 heads on 2, of 64) 67, 70; 256 (2 x 4096, 16 on 4,
  // of 128) 2126, 2230; 512 (16 x 1024, 16 on 4, of 64) 717, 659; 1024 (32 x 1024, of 128) 3137, 2830.
  const int each = group > 1 && s.blocks * Hk >= 2 * ctx->num_cus ? group : 1;
  Packed pq(ctx), pk(ctx), pv(ctx), pg(ctx);
  TempBlock rowstat(ctx), parts(ctx);
  // The key rows walk over the queries and the output's gradient, the query rows over keys and values
  // (whose factors both need).
  if (int rc = pk.alloc(s, Hk, dh)) return rc;
  if (int rc = pv.alloc(s, Hk, dh)) return rc;
  if (keys) {
    if (int rc = pq.alloc(s, H, dh)) return rc;
    if (int rc = pg.alloc(s, H, dh)) return rc;
    if (int rc = rowstat.alloc((size_t)s.tiles * H * kTile * 2 * sizeof(float))) return rc;
  }
  const size_t part = (size_t)s.total * H * dh * sizeof(float);
  if (keys && each < group)
    if (int rc = parts.alloc(((dk != nullptr) + (dv != nullptr)) * part)) return rc;
  const float alpha = kLog2e / std::sqrt((float)dh), scale = 1.0f / std::sqrt((float)dh);
  int exp;
  const float mant = std::frexp(alpha, &exp), scale_q = (float)((double)scale / mant);
  tiles::PackArgs p{s.in_order,
                    {pk.source(k, ld_kv, Hk, kMostScore), pv.source(v, ld_kv, Hk, kMostValue),
                     pq.source(q, ld_q, H, kMostScore, mant), pg.source(dout, ld_out, H, kMostValue)},
                    2 * Hk + (keys ? 2 * H : 0), dh};
  p.src[3].out = out, p.src[3].stats = stats, p.src[3].rowstat = rowstat.f();
  const bool few = few_blocks(ctx, s, H);
  BwdArgs b{few ? s.few_by_work : s.by_work, q, k, v, out, dout, stats, ld_q, ld_kv, ld_out};
  tiles::BackwardArgs a{q, k, v, out, dout, stats, ld_q, ld_kv, ld_out, pq.rows, pk.rows, pv.rows, pg.rows,
                        pq.exps, pk.exps, pv.exps, pg.exps, pq.each, pk.each, pv.each, pg.each, rowstat.f(), dq, dk,
                        dv, ld_q, ld_kv, ld_kv, s.total, H, Hk, dh, accumulate, accumulate, each, alpha, scale,
                        mant, exp, scale_q, kMostScore, kMostValue};
  return with_dp(dh, [&](auto dp) {
    constexpr int DP = decltype(dp)::value;
    tiles::pack<DP><<<(unsigned)(s.tiles * p.slots), 256, 0, ctx->stream>>>(p);
    if (int rc = check_launch(ctx, "pack")) return rc;
    Join j{};
    int joins = 0;
    if (keys && each < group) {
      float *at = parts.f();
      for (float **p : {&a.dk, &a.dv})
        if (*p != nullptr) j.out[joins] = *p, j.part[joins++] = *p = at, at += part / sizeof(float);
    }
    a.acc_kv = joins > 0 ? 0 : accumulate;
    const int64_t n = few ? s.tiles : s.blocks;
    const unsigned nk = keys ? (unsigned)(n * (H / each)) : 0, nq = dq != nullptr ? (unsigned)(n * H) : 0;
    if (few)
      backward_block<DP, 2><<<nk + nq, 256, 0, ctx->stream>>>(b, a, s.few_by_rest, nk);
    else
      backward_block<DP, 1><<<nk + nq, 256, 0, ctx->stream>>>(b, a, s.by_rest, nk);
    if (int rc = check_launch(ctx, "backward_block")) return rc;
    if (joins == 0) return (int)NUMRS_HIP_OK;
    join_heads<<<dim3(grid_for(s.total * Hk * (dh / 4), 256), joins), 256, 0, ctx->stream>>>(
        j, ld_kv, s.total, H, Hk, dh, accumulate);
    return check_launch(ctx, "join_heads");
  });
}

}  // namespace numrs_hip

extern "C" {

int numrs_hip_seqs_create(numrs_hip_ctx *ctx, const int64_t *lengths, int64_t n,
                          numrs_hip_seqs **out) {
  NRS_CHECK_CTX(ctx);
  if (out == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "numrs_hip_seqs_create: null out pointer");
  *out = nullptr;
  if (ctx->destroyed) return fail(ctx, NUMRS_HIP_E_INVALID, "context already destroyed");
  if (n < 0 || n >= int64_t{1} << 24 || (n > 0 && lengths == nullptr))
    return fail(ctx, NUMRS_HIP_E_INVALID, "numrs_hip_seqs_create: 0 to 2^24 - 1 lengths are needed");
  if (ctx->capturing)
    return fail(ctx, NUMRS_HIP_E_INVALID,
                "numrs_hip_seqs_create is not allowed while a graph is being recorded");
  const int64_t total = paging::packed_total(lengths, n);
  if (total < 0)
    return fail(ctx, NUMRS_HIP_E_SHAPE,
                "numrs_hip_seqs_create: lengths must be at least 0 and sum to at most 2^30");
  DeviceScope dev(ctx);
  try {
    auto s = std::make_shared<Seqs>();
    s->ctx = ctx, s->n = n, s->total = total;
    std::vector<SeqTile> tiles;
    int64_t row = 0;
    for (int64_t i = 0; i < n; ++i) {
      const int first = (int)tiles.size();
      for (int64_t t = 0; t < lengths[i]; t += kTile)
        tiles.push_back({(int)row, (int)lengths[i], (int)t, first, (int)i, {0, 0, 0}});
      row += lengths[i];
    }
    s->tiles = (int64_t)tiles.size();
    // Blocks of 128 rows, those with the most keys before them first: the last workgroups to start
    // are the shortest.
    std::vector<SeqTile> blocks;
    for (const SeqTile &t : tiles)
      if (t.t0 % 128 == 0) blocks.push_back(t);
    s->blocks = (int64_t)blocks.size();
    std::vector<SeqTile> lists = tiles;
    auto add = [&](std::vector<SeqTile> &list, bool rest) {
      std::stable_sort(list.begin(), list.end(), [=](const SeqTile &a, const SeqTile &b) {
        return rest ? a.len - a.t0 > b.len - b.t0 : a.t0 > b.t0;
      });
      lists.insert(lists.end(), list.begin(), list.end());
    };
    add(blocks, false), add(blocks, true), add(tiles, false), add(tiles, true);
    for (const SeqTile &t : tiles)
      if (t.t0 == 0 && t.len > 1) lists.push_back(t), ++s->severals, s->longest = std::max<int64_t>(s->longest, t.len);
    for (const SeqTile &t : tiles)
      if (t.len == 1) lists.push_back(t), ++s->singles;
    auto h = std::make_unique<numrs_hip_seqs>();
    if (!lists.empty()) {
      void *p = nullptr;
      const size_t bytes = lists.size() * sizeof(SeqTile);
      if (int rc = block_alloc(ctx, bytes, &p)) return rc;
      s->in_order = static_cast<SeqTile *>(p), s->bytes = bytes;
      s->by_work = s->in_order + s->tiles, s->by_rest = s->by_work + s->blocks;
      s->few_by_work = s->by_rest + s->blocks, s->few_by_rest = s->few_by_work + s->tiles;
      s->several = s->few_by_rest + s->tiles, s->single = s->several + s->severals;
      if (int rc = numrs_hip_upload(ctx, p, lists.data(), bytes)) return rc;
    }
    h->s = std::move(s);
    *out = h.release();
  } catch (const std::bad_alloc &) {
    return fail(ctx, NUMRS_HIP_E_NOMEM, "numrs_hip_seqs_create: out of host memory");
  }
  return NUMRS_HIP_OK;
}

int numrs_hip_seqs_destroy(numrs_hip_seqs *seqs) {
  delete seqs;
  return NUMRS_HIP_OK;
}

int64_t numrs_hip_seqs_total(const numrs_hip_seqs *seqs) {
  return seqs == nullptr ? -1 : seqs->s->total;
}

int numrs_hip_attention_packed_forward(numrs_hip_ctx *ctx, const numrs_hip_seqs *seqs,
                                       const float *q, int64_t ld_q, const float *k,
                                       const float *v, int64_t ld_kv, float *out, int64_t ld_out,
                                       float *stats, int64_t heads, int64_t kv_heads, int64_t dh) {
  NRS_CHECK_CTX(ctx);
  if (seqs == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "attention_packed: null sequences");
  return packed_forward(ctx, *seqs->s, q, ld_q, k, v, ld_kv, out, ld_out, stats,
                        {heads, kv_heads, dh});
}

int numrs_hip_attention_packed_backward(numrs_hip_ctx *ctx, const numrs_hip_seqs *seqs,
                                        const float *q, int64_t ld_q, const float *k,
                                        const float *v, int64_t ld_kv, const float *out,
                                        const float *dout, int64_t ld_out, const float *stats,
                                        float *dq, float *dk, float *dv, int64_t heads,
                                        int64_t kv_heads, int64_t dh, int accumulate) {
  NRS_CHECK_CTX(ctx);
  if (seqs == nullptr)
    return fail(ctx, NUMRS_HIP_E_INVALID, "attention_packed_backward: null sequences");
  return packed_backward(ctx, *seqs->s, q, ld_q, k, v, ld_kv, out, dout, ld_out, stats, dq, dk, dv,
                         {heads, kv_heads, dh}, accumulate);
}

}  // extern "C"
