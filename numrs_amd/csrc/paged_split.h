// One query row a sequence over a paged key-value cache.
//
// What bounds it is reading the cache once: 4 dh floats' worth of work a byte at most, so all query
// heads of a kv head (up to 16 a workgroup) share a read as the columns of 16-wide matrix products:
//   S^T = K Q^T    (rows: 16 tokens, columns: heads),  p = 2^(s - m),  O^T += V^T P^T.
// Every operand of the cache is in the lane that needs it as it is loaded, 8 or 16 bytes a lane, so
// nothing of it passes through LDS: the products' sums may run over the columns of a head, or the
// tokens, in any order that both operands share, and
//   fp32    lane (g, c) of a K block has token c, columns 16 t + 4 g .. + 3; of a V block tokens 4 g
//           .. + 3, columns 4 c .. + 3: v_mfma_f32_16x16x4_f32, plain fp32;
//   8 bits  a K block's lane has token c, columns 32 t + 8 g .. + 7, a V block's the codes of tokens
//           4 g .. + 3 of columns 4 c .. + 3, which lie together: fp16 holds a code exactly, so the
//           queries, and the probabilities times the values' scales, split in two fp16 terms (with
//           a power of two that keeps them in range), are the products' only rounding:
//           v_mfma_f32_16x16x32_f16.
// S^T's result rows, tokens 4 g .. + 3 of a block, are the second product's operand in place.
//
// The tokens of all sequences, in units of 64, are dealt evenly to the workgroups of a kv head,
// whatever the lengths (which only the device knows): a workgroup's share is a stretch of units over
// one or several sequences.  A sequence cut by stretches leaves parts (m, l, O), and the workgroup
// that finishes last of up to 16 adds theirs in order, the last of those groups the groups': no
// workgroup waits, and the order of the sums does not depend on who is last.
#pragma once

#include "packed_tiles.h"
#include "paging.h"

namespace paged {

using tiles::f2;
using tiles::f4;
using tiles::f4u;
using tiles::h2;
using tiles::h8;
using tiles::Terms;
using tiles::u4;

typedef unsigned u2 __attribute__((ext_vector_type(2)));

struct Cache {
  void *k, *v;
  float *ks, *vs;
  int64_t pages, max_pages;
  const int32_t *table;
  int shift, kv_heads, dh;
};

struct SplitArgs {
  Cache c;
  const float *q;
  const int32_t *lengths;
  float *out, *parts;
  unsigned *arrivals;  // [3 * workgroups], zero between launches
  int64_t ld_q, ld_out;
  int n, heads, blocks, shares;  // blocks: of 16 query heads in a group; shares: workgroups of a kv head's block
  float alpha;                   // log2(e) / sqrt(dh)
};

constexpr int kUnit = 64;       // tokens
constexpr int kJoin = 16;       // parts that one workgroup adds
constexpr float kNever = -1e30f;  // a softmax reference before any score

// Floats of a part: references and sums of 16 heads, then their outputs.
template <int DP>
constexpr int kPart = 32 + 16 * DP;

// The four bytes of w as fp16 code - 128: 1024 + byte is 0x6400 | byte, then less 1152.
__device__ __forceinline__ void halves(unsigned w, unsigned &lo, unsigned &hi) {
  const h2 off = {(_Float16)1152.f, (_Float16)1152.f};
  lo = __builtin_bit_cast(unsigned, h2(__builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off));
  hi = __builtin_bit_cast(unsigned, h2(__builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off));
}

__device__ __forceinline__ float max4(f4 x) { return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])); }

// A wave's running softmax of 16 heads over some tokens: lane (g, c) has head c; O of columns 64 u +
// 16 g + 4 r + e in o[u][e][r].
template <bool INT8, int DP>
struct State {
  static constexpr int NU = (DP + 63) / 64, NT = INT8 ? DP / 32 : DP / 16;
  static constexpr int NB = INT8 ? 4 : 2;  // blocks of 16 tokens a step
  float m, l;
  f4 o[NU][4];
  bool seen;
  // the head's queries: fp32 a lane's four columns of each 16; else two terms and what their factor
  // leaves of alpha
  f4 q[INT8 ? 1 : NT];
  Terms qt[INT8 ? NT : 1];
  float fq;

  __device__ __forceinline__ void begin(const SplitArgs &a, int i, int head, bool live) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const float *p = a.q + i * a.ld_q + (int64_t)head * a.c.dh;
    m = kNever, l = 0.f, seen = false;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[u][e] = f4{};
    if constexpr (!INT8) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int d = 16 * t + 4 * g;
        q[t] = live && d < a.c.dh ? f4(*reinterpret_cast<const f4u *>(p + d)) : f4{};
      }
      fq = a.alpha;
    } else {
      float x[NT][8], big = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int d = 32 * t + 8 * g;
        const bool in = live && d < a.c.dh;
        const f4 lo = in ? f4(*reinterpret_cast<const f4u *>(p + d)) : f4{};
        const f4 hi = in ? f4(*reinterpret_cast<const f4u *>(p + d + 4)) : f4{};
#pragma unroll
        for (int j = 0; j < 4; ++j) x[t][j] = lo[j], x[t][4 + j] = hi[j];
#pragma unroll
        for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[t][j]));
      }
      big = rows4(big, [](float y, float z) { return fmaxf(y, z); });
      const int e = big > 0.f && big < INFINITY ? min(12 - __builtin_amdgcn_frexp_expf(big), 120) : 0;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[t][j] = __builtin_amdgcn_ldexpf(x[t][j], e);
        qt[t] = tiles::split8(x[t]);
      }
      fq = __builtin_amdgcn_ldexpf(a.alpha, -e);
    }
  }

  // Tokens pos .. + 16 NB - 1 of kv head `kv`, those before `end`; pages: of each block, -1 for one
  // that the cache does not have.
  __device__ __forceinline__ void step(const SplitArgs &a, int kv, int64_t pos, int64_t end, const int (&pages)[NB]) {
    const Cache &c = a.c;
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const int slot = (int)(pos & ((1 << c.shift) - 1));
    f4 s[NB];
    bool full = true;
    if constexpr (!INT8) {
      f4 k[NB][NT], v[NB][4][NU];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int at = (slot + 16 * b) & ((1 << c.shift) - 1);
        const int64_t base = paging::page_base(max(pages[b], 0), c.kv_heads, kv, c.shift, c.dh) + (int64_t)at * c.dh;
        const float *p = static_cast<const float *>(c.k) + base + (int64_t)col * c.dh + 4 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          k[b][t] = 16 * t + 4 * g < c.dh ? *reinterpret_cast<const f4 *>(p + 16 * t) : f4{};
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int at = (slot + 16 * b) & ((1 << c.shift) - 1);
        const int64_t base = paging::page_base(max(pages[b], 0), c.kv_heads, kv, c.shift, c.dh) + (int64_t)at * c.dh;
        const float *p = static_cast<const float *>(c.v) + base + (int64_t)(4 * g) * c.dh + 4 * col;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int u = 0; u < NU; ++u)
            v[b][r][u] = 64 * u + 4 * col < c.dh ? *reinterpret_cast<const f4 *>(p + r * c.dh + 64 * u) : f4{};
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        s[b] = f4{};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[b][t][e], q[t][e], s[b], 0, 0, 0);
      }
      probabilities(pos, end, pages, s, nullptr, full);
      if (!full) {  // what lies in slots of no token must not reach the sums
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pages[b] < 0 || pos + 16 * b + 4 * g + r >= end) {
#pragma unroll
              for (int u = 0; u < NU; ++u) v[b][r][u] = f4{};
            }
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f4 t{};
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) t = __builtin_amdgcn_mfma_f32_16x16x4f32(v[b][r][u][e], s[b][r], t, 0, 0, 0);
          o[u][e] += t;
        }
    } else {
      u2 k[NB][NT];
      u4 v[NB][NU];
      f4 ks[NB], vs[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int at = (slot + 16 * b) & ((1 << c.shift) - 1);
        const int64_t head = paging::page_base(max(pages[b], 0), c.kv_heads, kv, c.shift, 1) + at;
        const uint8_t *p = static_cast<const uint8_t *>(c.k) + (head + col) * c.dh + 8 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          k[b][t] = 32 * t + 8 * g < c.dh ? *reinterpret_cast<const u2 *>(p + 32 * t) : u2{};
        ks[b] = *reinterpret_cast<const f4 *>(c.ks + head + 4 * g);
        vs[b] = *reinterpret_cast<const f4 *>(c.vs + head + 4 * g);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int at = (slot + 16 * b) & ((1 << c.shift) - 1);
        const int64_t head = paging::page_base(max(pages[b], 0), c.kv_heads, kv, c.shift, 1) + at;
        // slot group at / 4 + g, columns 4 col .. + 3
        const uint8_t *p = static_cast<const uint8_t *>(c.v) + (head + 4 * g) * c.dh + 16 * col;
#pragma unroll
        for (int u = 0; u < NU; ++u)
          v[b][u] = 64 * u + 4 * col < c.dh ? *reinterpret_cast<const u4 *>(p + 256 * u) : u4{};
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        s[b] = f4{};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          u4 w;
          unsigned x, y;
          halves(k[b][t][0], x, y), w[0] = x, w[1] = y;
          halves(k[b][t][1], x, y), w[2] = x, w[3] = y;
          const h8 kh = __builtin_bit_cast(h8, w);
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qt[t].m, s[b], 0, 0, 0);
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qt[t].h, s[b], 0, 0, 0);
        }
      }
      probabilities(pos, end, pages, s, ks, full);
      if (!full) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pages[b] < 0 || pos + 16 * b + 4 * g + r >= end) vs[b][r] = 0.f;
      }
      float big = max4(vs[0]);
#pragma unroll
      for (int b = 1; b < NB; ++b) big = fmaxf(big, max4(vs[b]));
      big = rows4(big, [](float x, float y) { return fmaxf(x, y); });
      const int ev = big > 0.f ? max(__builtin_amdgcn_frexp_expf(big), -110) : 0;
      const float up = __builtin_amdgcn_ldexpf(1.f, 7 - ev), back = __builtin_amdgcn_ldexpf(1.f, ev - 7);
      Terms w[NB / 2];
#pragma unroll
      for (int b = 0; b < NB; b += 2) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = s[b][r] * (vs[b][r] * up), x[4 + r] = s[b + 1][r] * (vs[b + 1][r] * up);
        w[b / 2] = tiles::split8(x);
      }
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f4 t{};
#pragma unroll
          for (int b = 0; b < NB; b += 2) {
            u4 y;
            unsigned lo, hi;
            halves(v[b][u][e], lo, hi), y[0] = lo, y[1] = hi;
            halves(v[b + 1][u][e], lo, hi), y[2] = lo, y[3] = hi;
            const h8 vh = __builtin_bit_cast(h8, y);
            t = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, w[b / 2].m, t, 0, 0, 0);
            t = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, w[b / 2].h, t, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) o[u][e][r] = fmaf(t[r], back, o[u][e][r]);
        }
    }
  }

  // Scores to probabilities in place; the reference moves where one passes it by 2^8.
  __device__ __forceinline__ void probabilities(int64_t pos, int64_t end, const int (&pages)[NB], f4 (&s)[NB],
                                                const f4 *ks, bool &full) {
    const int g = (threadIdx.x & 63) >> 4;
    full = pos + 16 * NB <= end;
    bool any = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      full &= pages[b] >= 0;
      any |= pages[b] >= 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) s[b][r] *= ks != nullptr ? ks[b][r] * fq : fq;
    }
    seen |= any;
    if (!full) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (pages[b] < 0 || pos + 16 * b + 4 * g + r >= end) s[b][r] = -INFINITY;
    }
    float most = max4(s[0]);
#pragma unroll
    for (int b = 1; b < NB; ++b) most = fmaxf(most, max4(s[b]));
    if (__any(most > m + 8.f)) {
      const float now = fmaxf(m, rows4(most, [](float x, float y) { return fmaxf(x, y); }));
      const float r = __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= r;
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[u][e] *= r;
    }
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - m);
      sum += (s[b][0] + s[b][1]) + (s[b][2] + s[b][3]);
    }
    l += sum;
  }
};

// The workgroup of a kv head's block of query heads that has unit x of `units`, of `shares`.
__device__ __forceinline__ int owner(int64_t x, int64_t units, int shares) {
  return (int)(((x + 1) * shares - 1) / units);
}
__device__ __forceinline__ int64_t first_unit(int p, int64_t units, int shares) { return units * p / shares; }

__device__ __forceinline__ int64_t units_of(const SplitArgs &a, int i) {
  const int64_t len = paging::held(a.lengths[i], a.c.max_pages, a.c.shift);
  return len > kUnit ? (len + kUnit - 1) / kUnit : 1;  // a sequence without tokens has a row to write too
}

// A thread of a join has head c = tid / 16 and, of each 64 columns, 4 x .. + 3 with x = tid % 16.
template <int DP>
struct Row {
  static constexpr int NU = (DP + 63) / 64;
  float m, l;  // l < 0: no token
  f4 o[NU];
  __device__ __forceinline__ static bool in(int u) { return DP % 64 == 0 || 64 * u + 4 * (threadIdx.x & 15) < DP; }
};

// Adds up to kJoin parts in order; part(j) is the j-th's place.  All loads go out before any is used:
// they come from memory, whichever cache another workgroup's XCD has.
template <int DP, class At>
__device__ __forceinline__ Row<DP> join(__amdgpu_buffer_rsrc_t parts, int count, bool live, At part) {
  using R = Row<DP>;
  const int c = threadIdx.x >> 4, x = threadIdx.x & 15;
  float ms[kJoin], ls[kJoin];
  f4 v[kJoin][R::NU];
#pragma unroll
  for (int i = 0; i < kJoin; ++i) {
    ms[i] = kNever, ls[i] = -1.f;
    if (i < count && live) {
      const int at = (int)part(i) * kPart<DP> * 4;
      ms[i] = numrs_hip::ld_dev1(parts, at + 4 * c), ls[i] = numrs_hip::ld_dev1(parts, at + 64 + 4 * c);
#pragma unroll
      for (int u = 0; u < R::NU; ++u)
        if (R::in(u)) v[i][u] = numrs_hip::ld_dev4(parts, at + 128 + (c * DP + 64 * u + 4 * x) * 4);
    }
  }
  R r;
  r.m = kNever, r.l = -1.f;
#pragma unroll
  for (int u = 0; u < R::NU; ++u) r.o[u] = f4{};
#pragma unroll
  for (int i = 0; i < kJoin; ++i) r.m = fmaxf(r.m, ms[i]);
#pragma unroll
  for (int i = 0; i < kJoin; ++i) {
    if (ls[i] < 0.f) continue;
    const float w = __builtin_amdgcn_exp2f(ms[i] - r.m);
    r.l = fmaf(ls[i], w, fmaxf(r.l, 0.f));
#pragma unroll
    for (int u = 0; u < R::NU; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) r.o[u][j] = fmaf(v[i][u][j], w, r.o[u][j]);
  }
  return r;
}

// The result, or a part for a later join.
template <int DP>
__device__ __forceinline__ void put_row(const SplitArgs &a, int i, int head, bool live, const Row<DP> &r) {
  const int x = threadIdx.x & 15;
  if (!live) return;
  float *p = a.out + i * a.ld_out + (int64_t)head * a.c.dh;
#pragma unroll
  for (int u = 0; u < Row<DP>::NU; ++u) {
    const int d = 64 * u + 4 * x;
    if (d >= a.c.dh) continue;
    f4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = r.l < 0.f ? 0.f : r.o[u][j] / r.l;
    *reinterpret_cast<f4u *>(p + d) = y;
  }
}
template <int DP>
__device__ __forceinline__ void put_part(__amdgpu_buffer_rsrc_t parts, int64_t place, bool live, const Row<DP> &r) {
  const int c = threadIdx.x >> 4, x = threadIdx.x & 15, at = (int)place * kPart<DP> * 4;
  if (!live) return;
  if (x == 0) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, r.m), parts, at + 4 * c, 0, numrs_hip::kScDevice);
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, r.l), parts, at + 64 + 4 * c, 0,
                                          numrs_hip::kScDevice);
  }
#pragma unroll
  for (int u = 0; u < Row<DP>::NU; ++u)
    if (Row<DP>::in(u))
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, r.o[u]), parts,
                                             at + 128 + (c * DP + 64 * u + 4 * x) * 4, 0, numrs_hip::kScDevice);
}

// Adds one to a counter once this workgroup's stores are out; whether it was the last of `count`,
// which sets the counter back.  Uniform over the workgroup.
__device__ __forceinline__ bool arrive(unsigned *counter, int count, int *flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned was = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = was + 1 == (unsigned)count;
    if (*flag) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *flag != 0;
}

template <bool INT8, int DP>
__global__ void __launch_bounds__(256, 2) split_rows(SplitArgs a) {
  using S = State<INT8, DP>;
  constexpr int kStep = 16 * S::NB;
  __shared__ float sm[4][16], sl[4][16], so[4][16][S::NU * 64 + 4];
  __shared__ int64_t pre[257], total4[4];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hc = blockIdx.x % (a.c.kv_heads * a.blocks), kv = hc / a.blocks, cb = hc % a.blocks;
  const int group = a.heads / a.c.kv_heads;
  const __amdgpu_buffer_rsrc_t parts = numrs_hip::dev_rsrc(
      a.parts, (int64_t)2 * a.c.kv_heads * a.blocks * a.shares * kPart<DP> * 4);

  auto block_sum = [&](int64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if (lane == 0) total4[w] = v;
    __syncthreads();
    return total4[0] + total4[1] + total4[2] + total4[3];
  };
  int64_t units = 0;
  for (int i = tid; i < a.n; i += 256) units += units_of(a, i);
  units = block_sum(units);
  const int shares = (int)min((int64_t)a.shares, units), p = blockIdx.x / (a.c.kv_heads * a.blocks);
  if (p >= shares) return;
  const int64_t lo = first_unit(p, units, shares), hi = first_unit(p + 1, units, shares);
  const int64_t me = (int64_t)blockIdx.x, stride = (int64_t)a.c.kv_heads * a.blocks;  // workgroup p' of this block: hc + p' stride

  int64_t base = 0;
  for (int i0 = 0; i0 < a.n && base < hi; i0 += 256) {
    // units before each of 256 sequences
    const int64_t mine = i0 + tid < a.n ? units_of(a, i0 + tid) : 0;
    int64_t scan = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t below = __shfl_up(scan, d);
      if (lane >= d) scan += below;
    }
    __syncthreads();
    if (lane == 63) total4[w] = scan;
    __syncthreads();
    int64_t ahead = base;
    for (int k = 0; k < w; ++k) ahead += total4[k];
    pre[tid + 1] = ahead + scan;
    if (tid == 0) pre[0] = base;
    __syncthreads();
    const int count = min(256, a.n - i0);
    const int64_t next = pre[count];
    for (int j = 0; j < count && next > lo; ++j) {
      const int64_t u0 = pre[j], u1 = pre[j + 1];
      if (u1 <= lo) continue;
      if (u0 >= hi) break;
      const int i = i0 + j;
      const int64_t ua = max(u0, lo), ub = min(u1, hi);
      const int64_t len = paging::held(a.lengths[i], a.c.max_pages, a.c.shift);
      const int64_t from = (ua - u0) * kUnit, end = min((ub - u0) * kUnit, len);
      const int head = cb * 16 + (lane & 15);
      S st;
      st.begin(a, i, kv * group + min(head, group - 1), head < group);
      const int32_t *row = a.c.table + (int64_t)i * a.c.max_pages;
      int pages[S::NB];
      auto look = [&](int64_t pos) {
#pragma unroll
        for (int b = 0; b < S::NB; ++b)
          pages[b] = __builtin_amdgcn_readfirstlane(
              pos + 16 * b < end ? paging::page_of(row, a.c.max_pages, a.c.shift, a.c.pages, pos + 16 * b) : -1);
      };
      for (int64_t pos = from + w * kStep; pos < end; pos += 4 * kStep) {
        look(pos);
        st.step(a, kv, pos, end, pages);
      }
      // the four waves' states as one
      const float l = rows4(st.l, [](float x, float y) { return x + y; });
      __syncthreads();
      if (lane < 16) sm[w][lane] = st.m, sl[w][lane] = st.seen ? l : -1.f;
#pragma unroll
      for (int u = 0; u < S::NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int r = 0; r < 4; ++r) so[w][lane & 15][64 * u + 16 * (lane >> 4) + 4 * r + e] = st.o[u][e][r];
      __syncthreads();
      const int c = tid >> 4, x = tid & 15;
      Row<DP> r;
      r.m = fmaxf(fmaxf(sm[0][c], sm[1][c]), fmaxf(sm[2][c], sm[3][c])), r.l = -1.f;
#pragma unroll
      for (int u = 0; u < S::NU; ++u) r.o[u] = f4{};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (sl[k][c] < 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(sm[k][c] - r.m);
        r.l = fmaf(sl[k][c], f, fmaxf(r.l, 0.f));
#pragma unroll
        for (int u = 0; u < S::NU; ++u) {
          const f4 y = *reinterpret_cast<const f4 *>(&so[k][c][64 * u + 4 * x]);
#pragma unroll
          for (int e = 0; e < 4; ++e) r.o[u][e] = fmaf(y[e], f, r.o[u][e]);
        }
      }
      const int out_head = kv * group + cb * 16 + c;
      const bool live = cb * 16 + c < group;
      if (ua == u0 && ub == u1) {
        put_row<DP>(a, i, out_head, live, r);
        continue;
      }
      // Places of parts: a workgroup has at most one that begins its sequence (place 1) and one that
      // does not.
      const int pf = owner(u0, units, shares), pl = owner(u1 - 1, units, shares);
      auto wg = [&](int q) { return hc + (int64_t)q * stride; };
      auto at = [&](int q) { return 2 * wg(q) + (q == pf); };
      put_part<DP>(parts, at(p), live, r);
      const int lead = pf + (p - pf) / kJoin * kJoin, members = min(kJoin, pl - lead + 1);
      if (!arrive(a.arrivals + at(lead), members, &flag)) continue;
      r = join<DP>(parts, members, live, [&](int q) { return at(lead + q); });
      const int groups = (pl - pf) / kJoin + 1;
      if (groups > 1) {
        // in place of the leader's part, which no one reads any more
        __syncthreads();
        put_part<DP>(parts, at(lead), live, r);
        if (!arrive(a.arrivals + 2 * stride * a.shares + wg(pf), groups, &flag)) continue;
        r.m = kNever, r.l = -1.f;
#pragma unroll
        for (int u = 0; u < S::NU; ++u) r.o[u] = f4{};
        for (int q = 0; q < groups; q += kJoin) {
          const Row<DP> y = join<DP>(parts, min(kJoin, groups - q), live,
                                     [&](int z) { return at(pf + (q + z) * kJoin); });
          if (y.l < 0.f) continue;
          const float now = fmaxf(r.m, y.m), f0 = __builtin_amdgcn_exp2f(r.m - now), f1 = __builtin_amdgcn_exp2f(y.m - now);
          r.l = fmaf(fmaxf(r.l, 0.f), f0, y.l * f1);
#pragma unroll
          for (int u = 0; u < S::NU; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[u][e] = fmaf(r.o[u][e], f0, y.o[u][e] * f1);
          r.m = now;
        }
      }
      put_row<DP>(a, i, out_head, live, r);
    }
    __syncthreads();
    base = next;
  }
}

}  // namespace paged
