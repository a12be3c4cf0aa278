// Norm and rotation of a packed projection's query and key heads, and their gradients (no reference op).
// rotary.h has the arithmetic.
//
// Both directions are bound by memory: each value is read once and written once, and the angles, the same for
// all heads of a token, are formed once for a token and a workgroup's heads.  On MI355X: 62 MB of ragged prompts in
// 12.4 us (5.0 TB/s); 16384 tokens of 16 + 8 + 8 heads of 128 with norms forward 105 to 108 us (5.0 to 5.1 TB/s, past
// the caches), backward 137 to 143 (which reads the normed heads again: 738 MB, 5.2 to 5.4 TB/s), the weights' sums 9
// to 10; 4096 tokens of 24 heads of 64 forward 10, backward 14, sums 8; 64 tokens 3.5, latency.
#include <algorithm>

#include "rotary.h"
#include "paging.h"

namespace {

using namespace numrs_hip;
using namespace rotary;

template <bool PAST>
__global__ void __launch_bounds__(256) rotate_rows(RowArgs a, int parts) {
  const int h0 = blockIdx.y * a.per;
  rotate_part<PAST>(a, a.tiles[blockIdx.x / parts], blockIdx.x % parts, h0, min(h0 + a.per, a.slots));
}

struct BackArgs {
  RowArgs r;  // x and the weights; y: the gradient of x
  const float *dy;
  int64_t ld_dy;
  double *sums;  // [workgroups][2][dh]: of the weights' gradients, or null
  int accumulate;
};

// With g = R^T dy and xh = x / sqrt(mean(x^2) + eps):
//   dw = sum g xh,   dx = (g w - xh mean(g w xh)) / sqrt(mean(x^2) + eps).
template <bool PAST>
__global__ void __launch_bounds__(256) rotate_rows_back(BackArgs b, int parts) {
  __shared__ double sum[256][8];
  const RowArgs &a = b.r;
  const SeqTile t = a.tiles[blockIdx.x / parts];
  const int i = threadIdx.x & ((1 << a.lanes) - 1), r = token_of(t, blockIdx.x % parts, a.lanes);
  const int h0 = blockIdx.y * a.per, h1 = min(h0 + a.per, a.slots);
  const Item it = item_of(i, a.dh, a.turn);
  const int64_t row = t.row0 + max(r, 0), start = a.ends != nullptr ? (int64_t)a.ends[t.seq] - t.len : 0;
  const float *px = a.x + row * a.ld_x, *pg = b.dy + row * b.ld_dy;
  float *py = a.y + row * a.ld_y;
  const bool nb = a.turn.pairs, live = r >= 0;
  const Units u = units_of(steps_of(a.turn, i, it), it, start + r);
  double acc[8] = {};
  Weight w;
  int kind = -1;
  // The sums of the kind just done, over the workgroup's tokens in order.
  auto flush = [&](int k) {
    if (b.sums == nullptr || k < 0 || k > 1) return;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[threadIdx.x][j] = live ? acc[j] : 0.0, acc[j] = 0.0;
    __syncthreads();
    double *to = b.sums + ((int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 + k) * a.dh;
    for (int e = threadIdx.x; e < 8 << a.lanes; e += 256) {
      const int lane = e >> 3, j = e & 7;
      const Item x = item_of(lane, a.dh, a.turn);
      if (!x.in) continue;
      double s = 0.0;
      for (int from = lane; from < 256; from += 1 << a.lanes) s += sum[from][j];
      // pair j & 3's first or second member
      const int at = nb ? 2 * (j & 3) + (j >> 2) : j;
      to[at < 4 ? x.d0 + at : x.d1 + at - 4] = s;
    }
  };
  if (b.sums != nullptr) {  // of a kind that the workgroup has no head of
    double *to = b.sums + (int64_t)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * a.dh;
    for (int e = threadIdx.x; e < 2 * a.dh; e += 256) {
      const bool some = e < a.dh ? h0 < a.heads : h1 > a.heads && h0 < a.heads + a.kv_heads;
      if (!some) to[e] = 0.0;
    }
  }
  for (int h = h0; h < h1; ++h) {
    const int now = h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;
    const float *pw = now == 0 ? a.wq : now == 1 ? a.wk : nullptr;
    if (now != kind) {
      flush(kind);
      kind = now;
      w.load(pw, it, nb);
    }
    if (!live) continue;
    f4 g0{}, g1{}, x0{}, x1{};
    if (it.in) {
      const float *p = pg + (int64_t)h * a.dh;
      g0 = get4<PAST>(p + it.d0), g1 = get4<PAST>(p + it.d1);
      if (pw != nullptr) {
        p = px + (int64_t)h * a.dh;
        x0 = get4<PAST>(p + it.d0), x1 = get4<PAST>(p + it.d1);
      }
    }
    if (now < 2) {
      double g[8];
      pairs_of(g0, g1, nb, g);
      turn<true>(g, u, it.turned);
      if (pw != nullptr) {
        double x[8], dot = 0.0;
        pairs_of(x0, x1, nb, x);
        const double s = inverse_rms(x, a.lanes, a.inv_dh, a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] *= s;
          acc[j] = fma(g[j], x[j], acc[j]);
          g[j] *= w.w[j];
          dot = fma(g[j], x[j], dot);
        }
        dot = row_sum(dot, a.lanes) * a.inv_dh;
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = fma(-x[j], dot, g[j]) * s;
      }
      columns_of(g, nb, g0, g1);
    }
    if (it.in && a.y != nullptr) {
      float *p = py + (int64_t)h * a.dh;
      if (b.accumulate) g0 += f4(*reinterpret_cast<f4u *>(p + it.d0)), g1 += f4(*reinterpret_cast<f4u *>(p + it.d1));
      put4<PAST>(p + it.d0, g0), put4<PAST>(p + it.d1, g1);
    }
  }
  flush(kind);
}

// The workgroups' sums [n][2][dh] added in order: a thread a column, a workgroup every gridDim.x-th of them, whose
// results the last workgroup to finish adds.  A column's query and key parts belong to one thread then, so that one
// array may be both gradients.  (16 workgroups with every column of eight: 29 us for 2048 sums of 256 columns.)
__global__ void __launch_bounds__(256)
    add_sums(const double *sums, int n, int dh, double *partial, unsigned *arrivals, float *dq, float *dk, int acc_q, int acc_k) {
  __shared__ int last;
  const int d = threadIdx.x, cols = 2 * dh;
  constexpr int kAhead = 8;
  if (d < cols) {
    double s = 0.0;
    for (int i = blockIdx.x; i < n; i += kAhead * gridDim.x) {
      double x[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) x[k] = i + k * (int)gridDim.x < n ? sums[(int64_t)(i + k * (int)gridDim.x) * cols + d] : 0.0;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) s += x[k];
    }
    __hip_atomic_store(partial + blockIdx.x * cols + d, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (d == 0) {
    last = __hip_atomic_fetch_add(arrivals, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == gridDim.x;
    if (last) __hip_atomic_store(arrivals, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last || d >= dh) return;
  double q = 0.0, k = 0.0;
  for (int i = 0; i < (int)gridDim.x; i += kAhead) {
    double x[kAhead], y[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const double *p = partial + min(i + j, (int)gridDim.x - 1) * cols + d;
      x[j] = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      y[j] = __hip_atomic_load(p + dh, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i + j < (int)gridDim.x) q += x[j], k += y[j];
  }
  if (dq != nullptr) dq[d] = (float)(acc_q ? dq[d] + q : q);
  if (dk != nullptr) dk[d] = (float)(acc_k ? dk[d] + k : k);
}

// Whether rows go past the caches: where a call reads and writes more than the last cache's 256 MB.  On MI355X, through
// against past, us: forward of 64 MB 25.1, 24.6; 128 MB 42, 54; 256 MB 108, 107; 512 MB 207, 195; forward and backward of
// 32 MB 45, 43; 48 MB 57, 57; 96 MB 97, 98; 256 MB 271, 260.
bool rows_past(const Seqs &s, const RowArgs &a, int arrays) {
  return s.total * (a.heads + 2 * a.kv_heads) * a.dh * (int64_t)sizeof(float) * arrays > int64_t{256} << 20;
}

int check_rows(numrs_hip_ctx *ctx, const numrs_hip_seqs *seqs, int64_t ld_a, int64_t ld_b, int64_t ld_c,
               const numrs_hip_rotary *rot, float eps, int64_t heads, int64_t kv_heads, int64_t dh, const char *what) {
  if (seqs == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: null sequences", what);
  if (ctx->destroyed) return fail(ctx, NUMRS_HIP_E_INVALID, "context already destroyed");
  if (seqs->s->ctx != ctx)
    return fail(ctx, NUMRS_HIP_E_INVALID, "%s: the sequences belong to another context", what);
  if (const char *why = paging::refuse_heads(heads, kv_heads, dh)) return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: %s", what, why);
  int code = 0;
  if (const char *why = refuse_rotary(rot, dh, &code)) return fail(ctx, code, "%s: %s", what, why);
  if (const char *why = refuse_eps(eps)) return fail(ctx, NUMRS_HIP_E_INVALID, "%s: %s", what, why);
  const int64_t width = (heads + 2 * kv_heads) * dh;
  if (paging::bad_stride(ld_a, width) || paging::bad_stride(ld_b, width) || paging::bad_stride(ld_c, width))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: a row stride is below its row's width or above 2^31 - 1", what);
  if (paging::bad_grid(seqs->s->tiles * parts_of(lanes_of(dh)) * 2))
    return fail(ctx, NUMRS_HIP_E_SHAPE, "%s: too many tokens", what);
  return NUMRS_HIP_OK;
}

RowArgs row_args(const Seqs &s, const int32_t *ends, const float *x, int64_t ld_x, const float *wq, const float *wk,
                 float eps, const numrs_hip_rotary *rot, float *y, int64_t ld_y, int64_t heads, int64_t kv_heads,
                 int64_t dh, int64_t slots) {
  RowArgs a{s.in_order, ends, x, wq, wk, y, ld_x, ld_y, (int)heads, (int)kv_heads, (int)slots, 0, (int)dh,
            lanes_of(dh), eps, 1.0 / (double)dh, turn_of(rot)};
  a.per = heads_each(s.ctx, s.tiles * parts_of(a.lanes), a.slots);
  return a;
}

}  // namespace

extern "C" {

int numrs_hip_qk_rotary_forward(numrs_hip_ctx *ctx, const numrs_hip_seqs *seqs, const int32_t *ends,
                                const float *x, int64_t ld_x, const float *q_weight,
                                const float *k_weight, float eps, const numrs_hip_rotary *rotary,
                                float *y, int64_t ld_y, int64_t heads, int64_t kv_heads, int64_t dh) {
  NRS_CHECK_CTX(ctx);
  if (int rc = check_rows(ctx, seqs, ld_x, ld_y, ld_y, rotary, eps, heads, kv_heads, dh, "qk_rotary")) return rc;
  const Seqs &s = *seqs->s;
  if (s.total == 0) return NUMRS_HIP_OK;
  if (x == nullptr || y == nullptr) return fail(ctx, NUMRS_HIP_E_INVALID, "qk_rotary: null pointer");
  if (x == y && ld_x != ld_y)
    return fail(ctx, NUMRS_HIP_E_SHAPE, "qk_rotary: in place, both row strides must be the same");
  const int64_t width = (heads + 2 * kv_heads) * dh;
  if (x != y && paging::rows_meet({x, width, ld_x}, {y, width, ld_y}, s.total))
    return fail(ctx, NUMRS_HIP_E_INVALID, "qk_rotary: the result overlaps the projection");
  if (int rc = s.keep()) return rc;
  DeviceScope dev(ctx);
  // in place the values are there already
  const RowArgs a = row_args(s, ends, x, ld_x, q_weight, k_weight, eps, rotary, y, ld_y, heads, kv_heads, dh,
                             heads + (x == y ? 1 : 2) * kv_heads);
  const int parts = parts_of(a.lanes);
  const dim3 grid((unsigned)(s.tiles * parts), (a.slots + a.per - 1) / a.per);
  if (rows_past(s, a, 2))
    rotate_rows<true><<<grid, 256, 0, ctx->stream>>>(a, parts);
  else
    rotate_rows<false><<<grid, 256, 0, ctx->stream>>>(a, parts);
  return check_launch(ctx, "rotate_rows");
}

int numrs_hip_qk_rotary_backward(numrs_hip_ctx *ctx, const numrs_hip_seqs *seqs, const int32_t *ends,
                                 const float *x, int64_t ld_x, const float *q_weight,
                                 const float *k_weight, float eps, const numrs_hip_rotary *rotary,
                                 const float *dy, int64_t ld_dy, float *dx, int64_t ld_dx,
                                 float *dq_weight, float *dk_weight, int64_t heads, int64_t kv_heads,
                                 int64_t dh, int accumulate) {
  NRS_CHECK_CTX(ctx);
  if (int rc = check_rows(ctx, seqs, ld_x, ld_dy, ld_dx, rotary, eps, heads, kv_heads, dh, "qk_rotary_backward"))
    return rc;
  const Seqs &s = *seqs->s;
  if ((dq_weight != nullptr && q_weight == nullptr) || (dk_weight != nullptr && k_weight == nullptr))
    return fail(ctx, NUMRS_HIP_E_INVALID, "qk_rotary_backward: a gradient of a weight that is not there");
  const int acc_q = accumulate & NUMRS_HIP_ACC_Q_WEIGHT, acc_k = accumulate & NUMRS_HIP_ACC_K_WEIGHT;
  const bool weights = dq_weight != nullptr || dk_weight != nullptr;
  DeviceScope dev(ctx);
  if (s.total == 0) {
    if (dq_weight != nullptr && !acc_q)
      if (int rc = numrs_hip_fill(ctx, dq_weight, dh, 0.f)) return rc;
    if (dk_weight != nullptr && !acc_k && !(dk_weight == dq_weight && acc_q))
      if (int rc = numrs_hip_fill(ctx, dk_weight, dh, 0.f)) return rc;
    return NUMRS_HIP_OK;
  }
  if (dx == nullptr && !weights) return NUMRS_HIP_OK;
  if (dy == nullptr || (x == nullptr && (q_weight != nullptr || k_weight != nullptr)))
    return fail(ctx, NUMRS_HIP_E_INVALID, "qk_rotary_backward: null pointer");
  const bool acc = (accumulate & NUMRS_HIP_ACC_X) != 0;
  if (dx == dy && (acc || ld_dx != ld_dy))
    return fail(ctx, NUMRS_HIP_E_INVALID,
                "qk_rotary_backward: in place, the row strides must be the same and nothing is added");
  if (dx != nullptr) {
    // (each value of x is read by the thread that writes its gradient, before it does: dx may be x too)
    const int64_t width = (heads + 2 * kv_heads) * dh, from = q_weight != nullptr ? 0 : heads * dh,
                  to = k_weight != nullptr ? (heads + kv_heads) * dh : q_weight != nullptr ? heads * dh : from;
    if ((dx != dy && paging::rows_meet({dy, width, ld_dy}, {dx, width, ld_dx}, s.total)) ||
        ((dx != x || ld_dx != ld_x) && paging::rows_meet({x + from, to - from, ld_x}, {dx, width, ld_dx}, s.total)))
      return fail(ctx, NUMRS_HIP_E_INVALID, "qk_rotary_backward: dx overlaps what it is formed from");
  }
  if (dq_weight != dk_weight && dq_weight != nullptr && dk_weight != nullptr &&
      paging::rows_meet({dq_weight, dh, dh}, {dk_weight, dh, dh}, 1))
    return fail(ctx, NUMRS_HIP_E_INVALID, "qk_rotary_backward: the weights' gradients overlap");
  if (int rc = s.keep()) return rc;
  BackArgs b{row_args(s, ends, x, ld_x, q_weight, k_weight, eps, rotary, dx, ld_dx, heads, kv_heads, dh,
                      heads + (dx == dy || dx == nullptr ? 1 : 2) * kv_heads),
             dy, ld_dy, nullptr, acc};
  const int parts = parts_of(b.r.lanes);
  const dim3 grid((unsigned)(s.tiles * parts), (b.r.slots + b.r.per - 1) / b.r.per);
  const int64_t groups = (int64_t)grid.x * grid.y;
  TempBlock sums(ctx);
  if (weights) {
    if (int rc = sums.alloc((size_t)(groups * 2 * dh) * sizeof(double))) return rc;
    b.sums = static_cast<double *>(sums.p);
  }
  if (rows_past(s, b.r, 3))
    rotate_rows_back<true><<<grid, 256, 0, ctx->stream>>>(b, parts);
  else
    rotate_rows_back<false><<<grid, 256, 0, ctx->stream>>>(b, parts);
  if (int rc = check_launch(ctx, "rotate_rows_back")) return rc;
  if (!weights) return NUMRS_HIP_OK;
  const unsigned adders = (unsigned)std::min<int64_t>(64, (groups + 7) / 8);
  TempBlock partial(ctx);
  if (int rc = partial.alloc((size_t)(adders * 2 * dh) * sizeof(double))) return rc;
  unsigned *arrivals = nullptr;
  if (int rc = arrival_counters(ctx, 1, &arrivals)) return rc;
  add_sums<<<adders, 256, 0, ctx->stream>>>(b.sums, (int)groups, (int)dh, static_cast<double *>(partial.p), arrivals,
                                            dq_weight, dk_weight, acc_q, acc_k);
  return check_launch(ctx, "add_sums");
}

}  // extern "C"
