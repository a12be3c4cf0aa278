// Queries and keys made ready for attention: each head normed, then rotated by its token's position.
//   y = R(pos) (x / sqrt(mean(x^2) + eps) * w)
// The first part is the checks of a rotation's description, plain arithmetic that needs no GPU.
#pragma once

#include <cmath>
#include <cstdint>

#include "numrs_hip.h"

namespace rotary {

constexpr int kMostAngles = 64;  // of a head of 128

// A rotation as the kernels have it, by value in their arguments: no memory of the device that a
// recorded graph or a tape would have to keep.
struct Turn {
  double turns[kMostAngles];  // of a whole circle, a position
  int dims, pairs;            // columns that turn; neighbours (else the halves' columns) together
};

// What is wrong with a rotation for heads of dh, or null; null stands for no rotation.
inline const char *refuse_rotary(const numrs_hip_rotary *r, int64_t dh, int *code) {
  *code = NUMRS_HIP_E_INVALID;
  if (r == nullptr) return nullptr;
  if (r->layout != NUMRS_HIP_ROTARY_HALVES && r->layout != NUMRS_HIP_ROTARY_PAIRS) return "unknown rotary layout";
  *code = NUMRS_HIP_E_SHAPE;
  if (r->dims < 0 || r->dims > dh || r->dims % 8 != 0)
    return "the rotated columns must be a multiple of 8 within the head size";
  *code = NUMRS_HIP_E_INVALID;
  if (r->dims > 0 && r->freqs == nullptr) return "null frequencies";
  for (int64_t i = 0; i < r->dims / 2; ++i)
    if (!(std::fabs(r->freqs[i]) <= 1e6)) return "a frequency must be finite and at most 10^6 radians a position";
  return nullptr;
}

inline const char *refuse_eps(float eps) {
  return eps >= 0.f && eps < INFINITY ? nullptr : "the norm's eps must be finite and not negative";
}

inline Turn turn_of(const numrs_hip_rotary *r) {
  Turn t{};
  if (r == nullptr) return t;
  t.dims = (int)r->dims, t.pairs = r->layout == NUMRS_HIP_ROTARY_PAIRS;
  for (int i = 0; i < t.dims / 2; ++i) t.turns[i] = r->freqs[i] / 6.283185307179586476925;
  return t;
}

// log2 of the lanes that share a row of a head, eight columns each.
inline int lanes_of(int64_t dh) {
  int s = 0;
  while ((8 << s) < dh) ++s;
  return s;
}

}  // namespace rotary

#ifdef __HIPCC__

#include "packed.h"

// Everything between the load and the store is in 64 bits, which cost the same as 32 on this card's vector
// units and far less here than the memory does: a result is the formula's, rounded once, and so the same bits
// in every kernel that forms it (an 8-bit cache's codes have borders that a last bit would move).
namespace rotary {

using numrs_hip::kTile;
using numrs_hip::SeqTile;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// A lane's eight columns of a head: two pieces of four, at d0 and d1.  Column pairs that turn together
// are in one lane, so that a rotation needs no exchange.
struct Item {
  int d0, d1;
  bool in, turned;
};
__device__ __forceinline__ Item item_of(int i, int dh, const Turn &t) {
  Item x;
  x.in = 8 * i < dh, x.turned = 8 * i < t.dims;
  const bool halves = x.turned && !t.pairs;
  x.d0 = halves ? 4 * i : 8 * i;
  x.d1 = halves ? t.dims / 2 + 4 * i : 8 * i + 4;
  return x;
}

// The eight values as the first (0 to 3) and second (4 to 7) members of four pairs.
__device__ __forceinline__ void pairs_of(f4 lo, f4 hi, bool neighbours, double (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f4 from = j < 2 ? lo : hi;
    v[j] = neighbours ? from[2 * (j & 1)] : lo[j];
    v[4 + j] = neighbours ? from[2 * (j & 1) + 1] : hi[j];
  }
}
__device__ __forceinline__ void columns_of(const double (&v)[8], bool neighbours, f4 &lo, f4 &hi) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)v[j];
  lo = neighbours ? f4{x[0], x[4], x[1], x[5]} : f4{x[0], x[1], x[2], x[3]};
  hi = neighbours ? f4{x[2], x[6], x[3], x[7]} : f4{x[4], x[5], x[6], x[7]};
}

// Cosine and sine of pos * turns whole circles, to the last bits of 64 that the product leaves: the circles
// drop out exactly, then the quarters, and the rest, within an eighth of a circle, goes into the two power
// series (terms from x^17 / 17! and x^18 / 18! on are below 2^-54).
__device__ __forceinline__ void unit_of(double turns, int64_t pos, double &c, double &s) {
  double t = (double)pos * turns;
  t -= rint(t);
  const double quarter = rint(4.0 * t);
  const double x = fma(4.0, t, -quarter) * 1.57079632679489661923, z = x * x;
  double a = -1.0 / 1307674368000.0, b = 1.0 / 20922789888000.0;
  a = fma(a, z, 1.0 / 6227020800.0), b = fma(b, z, -1.0 / 87178291200.0);
  a = fma(a, z, -1.0 / 39916800.0), b = fma(b, z, 1.0 / 479001600.0);
  a = fma(a, z, 1.0 / 362880.0), b = fma(b, z, -1.0 / 3628800.0);
  a = fma(a, z, -1.0 / 5040.0), b = fma(b, z, 1.0 / 40320.0);
  a = fma(a, z, 1.0 / 120.0), b = fma(b, z, -1.0 / 720.0);
  a = fma(a, z, -1.0 / 6.0), b = fma(b, z, 1.0 / 24.0);
  a = fma(a * z, x, x), b = fma(fma(b, z, -0.5), z, 1.0);
  const int q = (int)quarter;  // -2 to 2
  const double m = q & 1 ? a : b, n = q & 1 ? b : a;
  c = (q + 1) & 2 ? -m : m;
  s = q & 2 ? -n : n;
}

// Circles a position, of a lane's four pairs.
struct Steps {
  double turns[4];
};
__device__ __forceinline__ Steps steps_of(const Turn &t, int i, const Item &x) {
  Steps s{};
  if (x.turned) {
#pragma unroll
    for (int j = 0; j < 4; ++j) s.turns[j] = t.turns[4 * i + j];
  }
  return s;
}
struct Units {
  double c[4], s[4];
};
__device__ __forceinline__ Units units_of(const Steps &t, const Item &x, int64_t pos) {
  Units u{};
  if (x.turned) {
#pragma unroll
    for (int j = 0; j < 4; ++j) unit_of(t.turns[j], pos, u.c[j], u.s[j]);
  }
  return u;
}

// The pairs turned; BACK: the other way.
template <bool BACK>
__device__ __forceinline__ void turn(double (&v)[8], const Units &u, bool turned) {
  if (!turned) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double a = v[j], b = v[4 + j], s = BACK ? -u.s[j] : u.s[j];
    v[j] = fma(a, u.c[j], -(b * s));
    v[4 + j] = fma(a, s, b * u.c[j]);
  }
}

template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// The sum over 2^lanes neighbours, up to 16: lanes 1 and 2 apart by quads, the other four of eight and the
// other eight of sixteen by mirrors (what they hold is their group's already).
__device__ __forceinline__ double row_sum(double v, int lanes) {
  if (lanes > 0) v += dpp<0xB1>(v);
  if (lanes > 1) v += dpp<0x4E>(v);
  if (lanes > 2) v += dpp<0x141>(v);
  if (lanes > 3) v += dpp<0x140>(v);
  return v;
}

// 1 / sqrt(x): the card's estimate and two steps of Newton's.
__device__ __forceinline__ double inverse_root(double x) {
  double y = __builtin_amdgcn_rsq(x);
  if (x > 0.0 && x < INFINITY) {
#pragma unroll
    for (int k = 0; k < 2; ++k) y = fma(y * 0.5, fma(-(x * y), y, 1.0), y);
  }
  return y;
}

// 1 / sqrt(mean of the head's squares + eps).
__device__ __forceinline__ double inverse_rms(const double (&v)[8], int lanes, double inv_dh, float eps) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fma(v[j], v[j], s);
  return inverse_root(fma(row_sum(s, lanes), inv_dh, (double)eps));
}

// A head's weight as it is used: in pairs' order.
struct Weight {
  double w[8];
  __device__ __forceinline__ void load(const float *p, const Item &x, bool neighbours) {
    f4 lo{}, hi{};
    if (p != nullptr && x.in) lo = *reinterpret_cast<const f4u *>(p + x.d0), hi = *reinterpret_cast<const f4u *>(p + x.d1);
    pairs_of(lo, hi, neighbours, w);
  }
};

struct RowArgs {
  const SeqTile *tiles;
  const int32_t *ends;  // null: a position is the row's place in its sequence
  const float *x, *wq, *wk;
  float *y;
  int64_t ld_x, ld_y;
  int heads, kv_heads, slots, per, dh, lanes;  // slots: heads of all kinds that go to y; per: of a workgroup
  float eps;
  double inv_dh;
  Turn turn;
};

// The token of a thread in part `part` of a tile, -1 past it.
__device__ __forceinline__ int token_of(const SeqTile &t, int part, int lanes) {
  const int r = t.t0 + part * (256 >> lanes) + (int)(threadIdx.x >> lanes);
  return r < min(t.len, t.t0 + kTile) ? r : -1;
}

// Rows past the caches, or through them.
template <bool PAST>
__device__ __forceinline__ f4 get4(const float *p) {
  if constexpr (PAST) return __builtin_nontemporal_load(reinterpret_cast<const f4u *>(p));
  return *reinterpret_cast<const f4u *>(p);
}
template <bool PAST>
__device__ __forceinline__ void put4(float *p, f4 v) {
  if constexpr (PAST)
    __builtin_nontemporal_store(f4u(v), reinterpret_cast<f4u *>(p));
  else
    *reinterpret_cast<f4u *>(p) = v;
}

// A part of a tile's tokens, some of its heads: the angles are formed once for all of them.
template <bool PAST>
__device__ __forceinline__ void rotate_part(const RowArgs &a, const SeqTile &t, int part, int h0, int h1) {
  const int i = threadIdx.x & ((1 << a.lanes) - 1), r = token_of(t, part, a.lanes);
  const Item it = item_of(i, a.dh, a.turn);
  if (r < 0) return;  // (all lanes of a row together)
  const int64_t row = t.row0 + r, start = a.ends != nullptr ? (int64_t)a.ends[t.seq] - t.len : 0;
  const float *px = a.x + row * a.ld_x;
  float *py = a.y + row * a.ld_y;
  const bool nb = a.turn.pairs;
  auto ask = [&](int h, f4 &lo, f4 &hi) {
    lo = f4{}, hi = f4{};
    if (it.in && h < h1) {
      const float *p = px + (int64_t)h * a.dh;
      lo = get4<PAST>(p + it.d0), hi = get4<PAST>(p + it.d1);
    }
  };
  f4 lo, hi;
  ask(h0, lo, hi);
  const Units u = units_of(steps_of(a.turn, i, it), it, start + r);
  Weight w;
  int kind = -1;
  for (int h = h0; h < h1; ++h) {
    const f4 x0 = lo, x1 = hi;
    ask(h + 1, lo, hi);
    f4 y0 = x0, y1 = x1;
    const int now = h < a.heads ? 0 : h < a.heads + a.kv_heads ? 1 : 2;
    if (now < 2) {
      const float *pw = now == 0 ? a.wq : a.wk;
      if (now != kind) w.load(pw, it, nb), kind = now;
      double v[8];
      pairs_of(x0, x1, nb, v);
      if (pw != nullptr) {
        const double s = inverse_rms(v, a.lanes, a.inv_dh, a.eps);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * s * w.w[j];
      }
      turn<false>(v, u, it.turned);
      columns_of(v, nb, y0, y1);
    }
    if (it.in) {
      float *p = py + (int64_t)h * a.dh;
      put4<PAST>(p + it.d0, y0), put4<PAST>(p + it.d1, y1);
    }
  }
}

// Parts of a tile, and how many heads a workgroup takes so that there are eight workgroups a CU.  2, 4, 8 and 16 of them, us:
// 62 MB of ragged prompts 13.9, 13.1, 12.6, 15.5 (angles are formed again for each part of the heads); 4096 tokens of 24 heads
// of 64 10.9, 10.2, 10.0, 12.8; 16384 tokens of 32 heads of 128 103, 103, 103, 106.
inline int parts_of(int lanes) { return kTile / (256 >> lanes) > 0 ? kTile / (256 >> lanes) : 1; }
inline int heads_each(const numrs_hip_ctx *ctx, int64_t parts, int slots) {
  const int64_t want = 8 * (int64_t)ctx->num_cus, split = (want + parts - 1) / parts;
  return split >= slots ? 1 : (int)((slots + split - 1) / split);
}

}  // namespace rotary

#endif  // __HIPCC__
