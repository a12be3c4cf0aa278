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
//           a power of two for each head that puts the largest into [2^14, 2^15)), are the
//           products' only rounding: v_mfma_f32_16x16x32_f16.
// S^T's result rows, tokens 4 g .. + 3 of a block, are the second product's operand in place.
//
// The tokens of all sequences, in units of 64, are dealt evenly to the workgroups of a kv head,
// whatever the lengths (which only the device knows): a workgroup's share is a stretch of units over
// one or several sequences.  A sequence cut by stretches leaves parts (m, l, O), and the workgroup
// that finishes last of up to 16 adds theirs in order, the last of those groups the groups': no
// workgroup waits, and the order of the sums does not depend on who is last.
//
// 5.2 GB of fp32 cache (96 sequences of 6000 and 8000 tokens, 8 heads of 128) are read in 780 to 810 us,
// 6.5 TB/s and above (a large copy: 5.54); 134 MB (131072 tokens of one head) in 37, 3.6 TB/s; 70 MB of
// 8-bit cache of 40 sequences of 1 to 5000 tokens in 36; 333 tokens in 11.  In the short ones the way from the
// lengths to the table, the tokens and the joins, each waiting for the one before, is what takes the
// time.  Loads of a step into registers that a second step's leave free spilled (a wave's state, two
// steps' tokens): keys and values are asked for into the place of those just used.
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

// Loads past the caches, where what is read is more than they keep until the next step.
template <class T, bool PAST>
__device__ __forceinline__ T load(const char *p) {
  if constexpr (PAST) return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
  return *reinterpret_cast<const T *>(p);
}
// f(std::bool_constant<past>) with both kinds of loads kept apart, which the compiler would make one.
template <class F>
__device__ __forceinline__ void by_kind(bool past, F &&f) {
  if (past) {
    asm volatile("" ::: "memory");
    f(std::true_type{});
    asm volatile("" ::: "memory");
  } else {
    f(std::false_type{});
  }
}

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
constexpr int kJoin = 16;       // parts that one workgroup adds: two levels for up to kJoin^2 shares
constexpr int kWaves = 8;       // of a workgroup
constexpr float kNever = -__FLT_MAX__;  // a softmax reference before any score: no finite one is below

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
// 16 g + 4 r + e in o[u][e][r].  The heads' queries lie in LDS, a fragment of NT lanes' 16 bytes each
// (fp32: four columns of each 16; 8 bits: eight columns of each 32, two terms).
template <bool INT8, int DP>
struct State {
  static constexpr int NU = (DP + 63) / 64, NT = INT8 ? DP / 32 : DP / 16;
  static constexpr int NB = INT8 ? 2 : 1;  // blocks of 16 tokens a step
  static constexpr int kQueries = DP * 64;  // bytes of the queries' fragments
  float m, l, fq;  // fq: log2(e) / sqrt(dh), less the queries' factor
  f4 o[NU][4];
  bool seen;
  // A step's tokens as loaded.
  struct Load {
    f4 k[NB][INT8 ? 1 : NT], v[NB][INT8 ? 1 : 4][INT8 ? 1 : NU], ks[INT8 ? NB : 1], vs[INT8 ? NB : 1];
    u2 kc[NB][INT8 ? NT : 1];
    u4 vc[NB][INT8 ? NU : 1];
  };

  __device__ __forceinline__ void clear() {
    m = kNever, l = 0.f, seen = false;
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[u][e] = f4{};
  }

  // The queries of head `head` (zeros where it is not live), from memory ...
  struct Queries {
    f4 x[INT8 ? 2 * NT : NT];
  };
  static __device__ __forceinline__ Queries ask(const SplitArgs &a, int i, int head, bool live) {
    const int g = (threadIdx.x & 63) >> 4;
    const float *p = a.q + i * a.ld_q + (int64_t)head * a.c.dh;
    Queries q;
#pragma unroll
    for (int t = 0; t < (INT8 ? 2 * NT : NT); ++t) {
      const int d = INT8 ? 32 * (t >> 1) + 8 * g + 4 * (t & 1) : 16 * t + 4 * g;
      q.x[t] = live && d < a.c.dh ? f4(*reinterpret_cast<const f4u *>(p + d)) : f4{};
    }
    return q;
  }
  // ... into the wave's part of LDS.
  __device__ __forceinline__ void keep(const SplitArgs &a, const Queries &q, char *lds) {
    const int lane = threadIdx.x & 63;
    if constexpr (!INT8) {
      fq = a.alpha;
#pragma unroll
      for (int t = 0; t < NT; ++t) *reinterpret_cast<f4 *>(lds + t * 1024 + lane * 16) = q.x[t];
    } else {
      float big = 0.f;
#pragma unroll
      for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(q.x[t][j]));
      big = rows4(big, [](float y, float z) { return fmaxf(y, z); });
      const int e = big > 0.f && big < INFINITY ? min(12 - __builtin_amdgcn_frexp_expf(big), 120) : 0;
      fq = __builtin_amdgcn_ldexpf(a.alpha, -e);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_ldexpf(q.x[2 * t + (j >> 2)][j & 3], e);
        const Terms y = tiles::split8(x);
        *reinterpret_cast<h8 *>(lds + t * 2048 + lane * 16) = y.h;
        *reinterpret_cast<h8 *>(lds + t * 2048 + 1024 + lane * 16) = y.m;
      }
    }
  }

  // Asks for the keys, or the values, of the tokens pos .. + 16 NB - 1 of kv head `kv` on `pages`, -1
  // for one that the cache does not have (page 0 is read in its place, and masked).  Uniform addresses
  // and 32-bit offsets of the lane.  A lane past the head's last column reads the last ones again: its
  // products are with zeros (fp32 keys are zeroed, since theirs might be with infinity), its results
  // are not written.
  static __device__ __forceinline__ int64_t row_of(const Cache &c, int kv, int64_t pos, int page) {
    return paging::page_base(max(page, 0), c.kv_heads, kv, c.shift, 1) + ((int)pos & ((1 << c.shift) - 1));
  }
  static __device__ __forceinline__ void load_keys(const Cache &c, int kv, int64_t pos, const int (&pages)[NB], bool past, Load &x) {
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    by_kind(past, [&](auto kind) {
      constexpr bool PAST = decltype(kind)::value;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int64_t row = row_of(c, kv, pos + 16 * b, pages[b]);
        if constexpr (!INT8) {
          const char *p = reinterpret_cast<const char *>(static_cast<const float *>(c.k) + row * c.dh);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            x.k[b][t] = load<f4, PAST>(p + (unsigned)(4 * (col * c.dh + min(16 * t + 4 * g, c.dh - 4))));
        } else {
          const char *p = static_cast<const char *>(c.k) + row * c.dh;
#pragma unroll
          for (int t = 0; t < NT; ++t)
            x.kc[b][t] = load<u2, PAST>(p + (unsigned)(col * c.dh + min(32 * t + 8 * g, c.dh - 8)));
          x.ks[b] = *reinterpret_cast<const f4 *>(reinterpret_cast<const char *>(c.ks + row) + (unsigned)(16 * g));
        }
      }
    });
  }
  static __device__ __forceinline__ void load_values(const Cache &c, int kv, int64_t pos, const int (&pages)[NB], bool past, Load &x) {
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    by_kind(past, [&](auto kind) {
      constexpr bool PAST = decltype(kind)::value;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int64_t row = row_of(c, kv, pos + 16 * b, pages[b]);
        if constexpr (!INT8) {
          const char *p = reinterpret_cast<const char *>(static_cast<const float *>(c.v) + row * c.dh);
#pragma unroll
          for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              x.v[b][r][u] = load<f4, PAST>(
                  p + r * c.dh * 4 + (unsigned)(4 * (4 * g * c.dh + min(64 * u + 4 * col, c.dh - 4))));
        } else {
          x.vs[b] = *reinterpret_cast<const f4 *>(reinterpret_cast<const char *>(c.vs + row) + (unsigned)(16 * g));
          // the four slots 4 g .. + 3, columns 4 col .. + 3
          const char *p = static_cast<const char *>(c.v) + row * c.dh;
#pragma unroll
          for (int u = 0; u < NU; ++u)
            x.vc[b][u] = load<u4, PAST>(p + (unsigned)(4 * (g * c.dh + min(64 * u + 4 * col, c.dh - 4))));
        }
      }
    });
  }

  // The loaded keys' scores, in base 2.
  __device__ __forceinline__ void scores(int dh, const Load &x, const char *queries, f4 (&s)[NB]) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = f4{};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (!INT8) {
        const f4 q = *reinterpret_cast<const f4 *>(queries + t * 1024 + lane * 16);
        const bool in = 16 * t + 4 * g < dh;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(in ? x.k[b][t][e] : 0.f, q[e], s[b], 0, 0, 0);
      } else {
        const h8 qh = *reinterpret_cast<const h8 *>(queries + t * 2048 + lane * 16);
        const h8 qm = *reinterpret_cast<const h8 *>(queries + t * 2048 + 1024 + lane * 16);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          u4 w;
          unsigned lo, hi;
          halves(x.kc[b][t][0], lo, hi), w[0] = lo, w[1] = hi;
          halves(x.kc[b][t][1], lo, hi), w[2] = lo, w[3] = hi;
          const h8 kh = __builtin_bit_cast(h8, w);
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qm, s[b], 0, 0, 0);
          s[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh, s[b], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[b][r] *= INT8 ? x.ks[INT8 ? b : 0][r] * fq : fq;
  }

  // Adds the loaded values times the probabilities; `full`: all of them are tokens.
  __device__ __forceinline__ void outputs(int64_t pos, int64_t end, const int (&pages)[NB], bool full, f4 (&s)[NB], Load &x) {
    const int g = (threadIdx.x & 63) >> 4;
    if constexpr (!INT8) {
      if (!full) {  // what lies in slots of no token must not reach the sums
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pages[b] < 0 || pos + 16 * b + 4 * g + r >= end) {
#pragma unroll
              for (int u = 0; u < NU; ++u) x.v[b][r][u] = f4{};
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
            for (int r = 0; r < 4; ++r) t = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[b][r][u][e], s[b][r], t, 0, 0, 0);
          o[u][e] += t;
        }
    } else {
      if (!full) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pages[b] < 0 || pos + 16 * b + 4 * g + r >= end) x.vs[b][r] = 0.f;
      }
      float big = max4(x.vs[0]);
#pragma unroll
      for (int b = 1; b < NB; ++b) big = fmaxf(big, max4(x.vs[b]));
      big = rows4(big, [](float i, float j) { return fmaxf(i, j); });
      const int ev = big > 0.f ? max(__builtin_amdgcn_frexp_expf(big), -110) : 0;
      const float up = __builtin_amdgcn_ldexpf(1.f, -ev);
      // The largest of a head's products comes to [2^14, 2^15) in turn: a token of a large scale and little
      // probability must not cost the others their bits, nor have none itself.
      float y[NB / 2][8], top = 0.f;
#pragma unroll
      for (int b = 0; b < NB; b += 2)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[b / 2][r] = s[b][r] * (x.vs[b][r] * up), y[b / 2][4 + r] = s[b + 1][r] * (x.vs[b + 1][r] * up);
          top = fmaxf(fmaxf(top, y[b / 2][r]), y[b / 2][4 + r]);
        }
      top = rows4(top, [](float i, float j) { return fmaxf(i, j); });
      const int et = max(__builtin_amdgcn_frexp_expf(top), -100);
      const float lift = __builtin_amdgcn_ldexpf(1.f, 15 - et), back = __builtin_amdgcn_ldexpf(1.f, ev + et - 15);
      Terms w[NB / 2];
#pragma unroll
      for (int b = 0; b < NB; b += 2) w[b / 2] = tiles::split8(y[b / 2], lift);
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f4 t{};
#pragma unroll
          for (int b = 0; b < NB; b += 2) {
            u4 z;
            unsigned lo, hi;
            halves(x.vc[b][u][e], lo, hi), z[0] = lo, z[1] = hi;
            halves(x.vc[b + 1][u][e], lo, hi), z[2] = lo, z[3] = hi;
            const h8 vh = __builtin_bit_cast(h8, z);
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
                                                bool &full) {
    const int g = (threadIdx.x & 63) >> 4;
    full = pos + 16 * NB <= end;
    bool any = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      full &= pages[b] >= 0;
      any |= pages[b] >= 0;
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
      const float now = fmaxf(m, rows4(most, [](float i, float j) { return fmaxf(i, j); }));
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

// A value that is the same in every lane, as a scalar.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// The workgroup of a kv head's block of query heads that has unit x of `units`, of `shares`.
__device__ __forceinline__ int owner(int64_t x, int64_t units, int shares) {
  return (int)(((x + 1) * shares - 1) / units);
}
__device__ __forceinline__ int64_t first_unit(int p, int64_t units, int shares) { return units * p / shares; }

// A thread of a join has head c = tid / 32 and columns 4 x .. + 3 with x = tid % 32.
struct Row {
  float m, l;  // l < 0: no token
  f4 o;
};

// Adds up to kJoin parts in order; part(j) is the j-th's place.  All loads go out before any is used:
// they come from memory, whichever cache another workgroup's XCD has.
template <int DP, class At>
__device__ __forceinline__ Row join(__amdgpu_buffer_rsrc_t parts, int count, bool live, At part) {
  const int c = threadIdx.x >> 5, x = threadIdx.x & 31;
  float ms[kJoin], ls[kJoin];
  f4 v[kJoin];
#pragma unroll
  for (int i = 0; i < kJoin; ++i) {
    const int at = (int)part(min(i, count - 1)) * kPart<DP> * 4;  // past the last: read again, not added
    ms[i] = numrs_hip::ld_dev1(parts, at + 4 * c), ls[i] = numrs_hip::ld_dev1(parts, at + 64 + 4 * c);
    v[i] = numrs_hip::ld_dev4(parts, at + 128 + (c * DP + 4 * min(x, DP / 4 - 1)) * 4);
  }
  Row r{kNever, -1.f, {}};
#pragma unroll
  for (int i = 0; i < kJoin; ++i) {
    if (i >= count || !live) ls[i] = -1.f;
    r.m = fmaxf(r.m, ms[i]);
  }
#pragma unroll
  for (int i = 0; i < kJoin; ++i) {
    if (ls[i] < 0.f) continue;
    const float w = __builtin_amdgcn_exp2f(ms[i] - r.m);
    r.l = fmaf(ls[i], w, fmaxf(r.l, 0.f));
#pragma unroll
    for (int j = 0; j < 4; ++j) r.o[j] = fmaf(v[i][j], w, r.o[j]);
  }
  return r;
}

// The result, or a part for a later join.
__device__ __forceinline__ void put_row(const SplitArgs &a, int i, int head, bool live, const Row &r) {
  const int d = 4 * (threadIdx.x & 31);
  if (!live || d >= a.c.dh) return;
  f4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = r.l < 0.f ? 0.f : r.o[j] / r.l;
  *reinterpret_cast<f4u *>(a.out + i * a.ld_out + (int64_t)head * a.c.dh + d) = y;
}
template <int DP>
__device__ __forceinline__ void put_part(__amdgpu_buffer_rsrc_t parts, int64_t place, bool live, const Row &r) {
  const int c = threadIdx.x >> 5, x = threadIdx.x & 31, at = (int)place * kPart<DP> * 4;
  if (!live) return;
  if (x == 0) {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, r.m), parts, at + 4 * c, 0, numrs_hip::kScDevice);
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, r.l), parts, at + 64 + 4 * c, 0,
                                          numrs_hip::kScDevice);
  }
  if (4 * x < DP)
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, r.o), parts, at + 128 + (c * DP + 4 * x) * 4, 0,
                                           numrs_hip::kScDevice);
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
  return __builtin_amdgcn_readfirstlane(*flag) != 0;
}

template <bool INT8, int DP>
__global__ void __launch_bounds__(64 * kWaves, 2) split_rows(SplitArgs a) {
  using S = State<INT8, DP>;
  constexpr int kStep = 16 * S::NB, kThreads = 64 * kWaves, kCols = S::NU * 64 + 4;
  // of each wave: its queries while it takes tokens in, then its outputs
  __shared__ __attribute__((aligned(16))) float so[kWaves][16][kCols];
  static_assert(16 * kCols * 4 >= S::kQueries);
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ int64_t pre[kThreads + 1], sums[kWaves];
  __shared__ int tokens[kThreads];
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hc = blockIdx.x % (a.c.kv_heads * a.blocks), kv = hc / a.blocks, cb = hc % a.blocks;
  const int group = a.heads / a.c.kv_heads;
  const __amdgpu_buffer_rsrc_t parts = numrs_hip::dev_rsrc(
      a.parts, (int64_t)2 * a.c.kv_heads * a.blocks * a.shares * kPart<DP> * 4);

  // Of kThreads sequences from i0 on: their tokens, and the units before each in pre, with `base`
  // before the first; returns their end.
  auto scan = [&](int i0, int64_t base) {
    const int len = i0 + tid < a.n ? (int)paging::held(a.lengths[i0 + tid], a.c.max_pages, a.c.shift) : 0;
    // a sequence without tokens has a row to write too
    int64_t v = i0 + tid < a.n ? max(1, (int)(((unsigned)len + kUnit - 1) / kUnit)) : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t below = __shfl_up(v, d);
      if (lane >= d) v += below;
    }
    __syncthreads();
    tokens[tid] = len;
    if (lane == 63) sums[w] = v;
    __syncthreads();
    for (int k = 0; k < w; ++k) v += sums[k];
    pre[tid + 1] = base + v;
    if (tid == 0) pre[0] = base;
    __syncthreads();
    return uniform(pre[min(kThreads, a.n - i0)]);
  };
  int64_t units = 0;
  for (int i0 = 0; i0 < a.n; i0 += kThreads) units = scan(i0, units);
  const int shares = (int)min((int64_t)a.shares, units), p = blockIdx.x / (a.c.kv_heads * a.blocks);
  if (p >= shares) return;
  const int64_t lo = first_unit(p, units, shares), hi = first_unit(p + 1, units, shares);
  // What all workgroups read, at most the whole cache however many sequences share its pages, against the
  // 256 MB of the last cache.  Past it on MI355X: 5.2 GB in 784 us in place of 866; 70 MB, which that cache
  // holds until the next step, in 42 in place of 38.
  const bool past = min(units * kUnit, a.c.pages << a.c.shift) * (INT8 ? 2 : 8) * a.c.kv_heads * a.c.dh > int64_t{256} << 20;
  const int64_t stride = (int64_t)a.c.kv_heads * a.blocks;  // workgroup q of this block is hc + q stride

  // This workgroup's part of the j-th sequence of those in LDS.
  struct Stretch {
    int64_t u0, u1, ua, ub;  // the sequence's units, and the workgroup's of them
    int64_t from, end;       // its tokens
    int waves;               // that share them
  };
  auto stretch = [&](int j) {
    Stretch s;
    s.u0 = uniform(pre[j]), s.u1 = uniform(pre[j + 1]);
    s.ua = max(s.u0, lo), s.ub = min(s.u1, hi);
    s.from = (s.ua - s.u0) * kUnit;
    s.end = min((s.ub - s.u0) * kUnit, (int64_t)__builtin_amdgcn_readfirstlane(tokens[j]));
    // Two steps a wave at least, so that several short sequences go at once; one where this is all
    // that the workgroup has.  (Each sequence to all waves in turn: 64 us in place of 39 for the 40
    // sequences above.)
    const int64_t steps = (s.end - s.from + kStep - 1) / kStep;
    s.waves = (int)max((int64_t)1, min((int64_t)kWaves, s.ub - s.ua == hi - lo ? steps : (steps + 1) / 2));
    return s;
  };

  int64_t base = 0;
  for (int i0 = 0; i0 < a.n && base < hi; i0 += kThreads) {
    const int count = min(kThreads, a.n - i0);
    const int64_t next_base = a.n > kThreads ? scan(i0, base) : uniform(pre[count]);
    int j = 0;  // the first that ends after the workgroup's first unit
    for (int k = 0; k < count; k += 64) j += __builtin_popcountll(__ballot(k + lane < count && pre[min(k + lane, count - 1) + 1] <= lo));
    while (j < count && uniform(pre[j]) < hi) {
      // As many sequences as the waves go round, and this wave's place.
      int last = j, used = 0, mine = -1, first = 0;
      Stretch my{};
      while (last < count && uniform(pre[last]) < hi) {
        const Stretch s = stretch(last);
        if (used + s.waves > kWaves) break;
        if (w >= used && w < used + s.waves) mine = last, first = used, my = s;
        used += s.waves, ++last;
      }
      S st;
      st.clear();
      if (mine >= 0) {
        const int i = i0 + mine;
        const int32_t *row = a.c.table + (int64_t)i * a.c.max_pages;
        char *queries = reinterpret_cast<char *>(so[w]);
        int32_t entries[S::NB];
        int pages[S::NB], next[S::NB];
        auto look = [&](int64_t at) {
#pragma unroll
          for (int b = 0; b < S::NB; ++b)
            entries[b] = at + 16 * b < my.end ? paging::entry_of(row, a.c.max_pages, a.c.shift, at + 16 * b) : -1;
        };
        auto resolve = [&] {
#pragma unroll
          for (int b = 0; b < S::NB; ++b)
            next[b] = paging::page_in(__builtin_amdgcn_readfirstlane(entries[b]), a.c.pages);
        };
        // The table's entries, the queries and the first tokens are asked for before any is waited for
        // longer than the next needs.
        typename S::Load x;
        const int64_t ahead = my.waves * kStep;
        int64_t pos = my.from + (w - first) * kStep;
        look(pos);
        const int head = cb * 16 + (lane & 15);
        const auto q = S::ask(a, i, kv * group + min(head, group - 1), head < group);
        resolve();
        if (pos < my.end) S::load_keys(a.c, kv, pos, next, past, x), S::load_values(a.c, kv, pos, next, past, x);
        look(pos + ahead);
        st.keep(a, q, queries);
        __builtin_amdgcn_wave_barrier();
        // The next step's keys take this one's place once its scores are formed, and so the values.
        while (pos < my.end) {
          f4 s[S::NB];
          bool full;
#pragma unroll
          for (int b = 0; b < S::NB; ++b) pages[b] = next[b];
          const bool more = pos + ahead < my.end;
          resolve();
          st.scores(a.c.dh, x, queries, s);
          if (more) S::load_keys(a.c, kv, pos + ahead, next, past, x);
          look(pos + 2 * ahead);
          st.probabilities(pos, my.end, pages, s, full);
          st.outputs(pos, my.end, pages, full, s, x);
          if (more) S::load_values(a.c, kv, pos + ahead, next, past, x);
          pos += ahead;
        }
        __builtin_amdgcn_wave_barrier();
        const float l = rows4(st.l, [](float x, float y) { return x + y; });
        if (lane < 16) sm[w][lane] = st.m, sl[w][lane] = st.seen ? l : -1.f;
#pragma unroll
        for (int u = 0; u < S::NU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            f4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = st.o[u][e][r];
            *reinterpret_cast<f4 *>(&so[w][lane & 15][64 * u + 16 * (lane >> 4) + 4 * r]) = y;
          }
      }
      __syncthreads();
      // each sequence's waves' states as one
      used = 0;
      for (; j < last; ++j) {
        const Stretch s = stretch(j);
        const int i = i0 + j, c = tid >> 5, col = tid & 31, w1 = used + s.waves;
        Row r{kNever, -1.f, {}};
        for (int k = used; k < w1; ++k) r.m = fmaxf(r.m, sm[k][c]);
        for (int k = used; k < w1; ++k) {
          if (sl[k][c] < 0.f) continue;
          const float f = __builtin_amdgcn_exp2f(sm[k][c] - r.m);
          r.l = fmaf(sl[k][c], f, fmaxf(r.l, 0.f));
          if (4 * col < DP) {
            const f4 z = *reinterpret_cast<const f4 *>(&so[k][c][4 * col]);
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[e] = fmaf(z[e], f, r.o[e]);
          }
        }
        used = w1;
        const int out_head = kv * group + cb * 16 + c;
        const bool live = cb * 16 + c < group;
        if (s.ua == s.u0 && s.ub == s.u1) {
          put_row(a, i, out_head, live, r);
          continue;
        }
        // Places of parts: a workgroup has at most one that begins its sequence (place 1) and one that
        // does not.
        const int pf = owner(s.u0, units, shares), pl = owner(s.u1 - 1, units, shares);
        auto wg = [&](int k) { return hc + (int64_t)k * stride; };
        auto at = [&](int k) { return 2 * wg(k) + (k == pf); };
        put_part<DP>(parts, at(p), live, r);
        const int lead = pf + (p - pf) / kJoin * kJoin, members = min(kJoin, pl - lead + 1);
        if (!arrive(a.arrivals + at(lead), members, &flag)) continue;
        r = join<DP>(parts, members, live, [&](int k) { return at(lead + k); });
        const int groups = (pl - pf) / kJoin + 1;
        if (groups > 1) {
          // in place of the leader's part, which no one reads any more
          __syncthreads();
          put_part<DP>(parts, at(lead), live, r);
          if (!arrive(a.arrivals + 2 * stride * a.shares + wg(pf), groups, &flag)) continue;
          r = join<DP>(parts, groups, live, [&](int k) { return at(pf + k * kJoin); });
        }
        put_row(a, i, out_head, live, r);
      }
      __syncthreads();
    }
    base = next_base;
  }
}

}  // namespace paged
