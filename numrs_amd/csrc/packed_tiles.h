// Causal attention over packed sequences on the fp16 matrix cores at fp32 accuracy.
//
// An fp32 operand x, times a power of two that puts its 64-token tile's largest magnitude into
// [2^14, 2^15), is the sum h + m of two fp16 values, each rounded to nearest: h holds 11 bits, x -
// h is exact and m holds its next 11, so h + m is x within 2^-23 |x| for |x| down to 2^-17 of the
// largest and within 2^-39 of the largest below. Where a tile's tokens differ by more than 2^6, each
// has an exponent of its own (kMixed), so that none costs another more than 2^-33 of its own largest:
// neither one that its row does not see nor one that has no probability. Products take such a tile's
// rows to one exponent, before and after the softmax, in a form of each walk that only workgroups
// with such a tile take (its tests in the common one cost training on 2 x 4096 tokens 5 %).
//
// Of the four products of two such operands the matrix cores form three, m h + h m + h h (the fourth
// is below 2^-22 of the product and of either sign), each with fp32 accumulation: half of what three
// bf16 terms and six products take. v_mfma_f32_32x32x16_f16 sums of at most 64 tokens (or one head)
// start from zero and are added to fp32 totals: the matrix cores' own sum is cut off, not rounded.
//
// `pack` splits what the kernels walk over once a call, in the order in which the products read it: a
// fragment is the 32 tokens x 16 columns of a term, lane (g, c)'s 16 bytes being token c's columns 8 g
// .. + 7, so a tile goes to LDS by a plain copy.  The products over tokens need columns: the transposing
// LDS read gives lane (g, c) column c of the tokens 4 g .. + 3 and 8 + 4 g .. + 3, which is the order in
// which a product leaves its results' rows, so the probabilities of one product are the next one's
// operand in the lane that formed them.  Token c's second 16 bytes lie at place c ^ 4 of their half, so
// that the 16 lanes of a transposing read, four tokens' 32 bytes each, meet no bank twice.
#pragma once

#include "packed.h"

namespace tiles {

using numrs_hip::kTile;
using numrs_hip::SeqTile;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));

// A value that an earlier kernel left at an address that is the same in every lane: a scalar load, which
// waits for no copy to LDS in flight.
__device__ __forceinline__ int scalar(const int *p) {
  return *(const __attribute__((address_space(4))) int *)p;
}

// A tile's exponent where its values do not split: one that is not finite, or so large that a
// product might pass fp32's range.  Workgroups that meet one take the row kernels' arithmetic.
constexpr int kOdd = 1 << 20;
// Added to the exponent of a tile whose tokens have exponents of their own: the largest token's. Tokens of zeros
// have it too. Past a difference of 2^140 a tile is odd: what such exponents make of scores and of probabilities
// would leave fp32's range.
constexpr int kMixed = 1 << 16, kSpread = 6, kMostSpread = 140;
__device__ __forceinline__ bool is_mixed(int word) { return word > kMixed / 2; }
__device__ __forceinline__ int base_of(int word) { return is_mixed(word) ? word - kMixed : word; }

// And out . dout, at its gradient's exponent: what values below 2^80 give is below 2^103.
constexpr float kMostTotal = 0x1p110f;
// A softmax reference before any score: below every score of a tile that is not odd.
constexpr float kNone = -0x1p110f;

// x = h + m of a pair.
__device__ __forceinline__ void split(float a, float b, unsigned &h, unsigned &m) {
  const h2 t = __builtin_convertvector(f2{a, b}, h2);
  h = __builtin_bit_cast(unsigned, t);
  // a - h with h taken from its half of the pair: one instruction instead of two
  float r0, r1;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(h), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(h), "v"(b));
  m = __builtin_bit_cast(unsigned, __builtin_convertvector(f2{r0, r1}, h2));
}

// The same of a c and b c, whose products are not rounded before.
__device__ __forceinline__ void split(float a, float b, float c, unsigned &h, unsigned &m) {
  asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(h) : "v"(a), "v"(c));
  asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(h) : "v"(b), "v"(c));
  asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(m) : "v"(a), "v"(c), "v"(h));
  asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(m) : "v"(b), "v"(c), "v"(h));
}

struct Terms {
  h8 h, m;
};

__device__ __forceinline__ Terms split8(const float *x, float c) {
  u4 h, m;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unsigned a, b;
    split(x[2 * j], x[2 * j + 1], c, a, b);
    h[j] = a, m[j] = b;
  }
  return {__builtin_bit_cast(h8, h), __builtin_bit_cast(h8, m)};
}
__device__ __forceinline__ Terms split8(const float *x) {
  u4 h, m;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unsigned a, b;
    split(x[2 * j], x[2 * j + 1], a, b);
    h[j] = a, m[j] = b;
  }
  return {__builtin_bit_cast(h8, h), __builtin_bit_cast(h8, m)};
}

// acc += a b, the small products first: a's second term's, then b's. SWAPPED: b's first, so that a b^T and b a^T
// have the same bits.
template <bool SWAPPED = false>
__device__ __forceinline__ void mma(f16 &acc, const Terms &a, const Terms &b) {
  if constexpr (!SWAPPED) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.m, b.h, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.m, acc, 0, 0, 0);
  if constexpr (SWAPPED) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.m, b.h, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, acc, 0, 0, 0);
}

// The power of two that puts a largest magnitude into [2^14, 2^15). Not above 126, where its inverse is
// still normal: fp16's smallest step is then below fp32's, and the terms hold all of a smaller value.
__device__ __forceinline__ int exponent_for(float big) {
  return big > 0.f ? min(15 - __builtin_amdgcn_frexp_expf(big), 126) : 0;
}

// A tile's word from its tokens' largest and smallest magnitudes that are not 0 (infinity if all are), and a
// token's exponent from its own.
__device__ __forceinline__ int tile_word(float big, float small) {
  const int e = exponent_for(big), spread = exponent_for(fminf(big, small)) - e;
  return spread <= kSpread ? e : spread <= kMostSpread ? e + kMixed : kOdd;
}
__device__ __forceinline__ float not_zero(float top) { return top > 0.f ? top : INFINITY; }
__device__ __forceinline__ float lower(float a, float b) { return fminf(a, b); }

// Row of a 32x32 result that register i of lane group g holds.
__device__ __forceinline__ constexpr int out_row(int i, int g) { return 8 * (i >> 2) + 4 * g + (i & 3); }

// Rows of a result, those of 32 tokens whose own exponents are at `each`, brought to the exponent `base`.
__device__ __forceinline__ void level(f16 &x, const int *each, int base, int hi) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const i4 e = *reinterpret_cast<const i4 *>(each + out_row(4 * i, hi));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * i + j] = __builtin_amdgcn_ldexpf(x[4 * i + j], base - e[j]);
  }
}

// A head size rounded up to DP: 64-token tiles of fragments, the two terms of each side by side.
template <int DP>
struct Shape {
  static constexpr int NS = DP / 16, NB = DP / 32;  // steps of a product over the head, blocks of 32 columns
  static constexpr int kBytes = kTile * DP * 4;     // a tile's fragments
  static constexpr int kHalf = kBytes / 2;          // 32 tokens'
};

// Byte offset of token c's columns 8 g .. + 7 in a fragment.
__device__ __forceinline__ int place(int g, int c) { return (32 * g + (c ^ 4 * g)) * 16; }

// Step s of 32 tokens' rows at p: lane (g, c) has token c, columns 16 s + 8 g .. + 7.  off: place(g, c).
__device__ __forceinline__ Terms rows_of(const char *p, int s, int off) {
  p += s * 2048 + off;
  return {*reinterpret_cast<const h8 *>(p), *reinterpret_cast<const h8 *>(p + 1024)};
}

// Columns 32 b + c of 16 tokens (the st-th 16 of the 32 at p).  off: columns_place(lane).
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4 lds_s4;
__device__ __forceinline__ int columns_place(int lane) {
  // lane 4 r + x of a group of 16 reads four columns 4 x .. + 3 of token 4 g + r
  const int g = lane >> 5, r = (lane & 15) >> 2, x = lane & 3;
  return place(x >> 1, 4 * g + r) + (x & 1) * 8 + (lane >> 4 & 1) * 2048;
}
__device__ __forceinline__ h8 columns_term(const char *p) {
  const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p);
  const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(p + 128));
  return __builtin_bit_cast(h8, s8(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)));
}
__device__ __forceinline__ Terms columns_of(const char *p, int b, int st, int off) {
  p += b * 4096 + st * 256 + off;
  return {columns_term(p), columns_term(p + 1024)};
}

// A lane's row of an operand from memory, columns 16 s + 8 g .. + 7 of each step; zeros past the head.
template <int DP>
struct RowValues {
  float x[DP / 16][8];
  __device__ __forceinline__ void load(const float *p, bool live, int dh, int g) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * g;
      f4 lo{}, hi{};
      if (live && d < dh) lo = *reinterpret_cast<const f4u *>(p + d), hi = *reinterpret_cast<const f4u *>(p + d + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[s][j] = lo[j], x[s][4 + j] = hi[j];
    }
  }
  // Its largest magnitude; odd: see kOdd.
  __device__ __forceinline__ float top(float most, bool &odd) const {
    float big = 0.f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        odd |= !(fabsf(x[s][j]) < most);
        big = fmaxf(big, fabsf(x[s][j]));
      }
    return half_pair(big, [](float a, float b) { return fmaxf(a, b); });
  }
  // Its terms times `by`.
  __device__ __forceinline__ void split_into(Terms (&t)[DP / 16], float by) const {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) t[s] = split8(x[s], by);
  }
};

// One operand to split: heads x tiles.
struct Source {
  const float *x;
  int64_t ld;
  char *rows;   // fragments [tiles, heads]
  int *exps;    // [tiles, heads]: an exponent, plus kMixed where each token has its own, or kOdd
  int *each;    // [tiles, heads, 64]: those
  float most;   // larger magnitudes make a tile odd
  float by;     // a factor in [0.5, 1] that the terms have besides the exponent's
  int heads;
  // The output's gradient: its rows are divided by their softmax sum l, which turns the backward's
  // p into 2^(s - m), and the rows' references and totals go to `rowstat` [tiles, heads, 64]: (m,
  // out . dout / l) with the tile's factor; a row past the sequence has m = infinity (p = 0).
  const float *out, *stats;
  float *rowstat;
};

struct PackArgs {
  const SeqTile *tiles;
  Source src[4];
  int slots, dh;  // heads of all sources
};

// A workgroup a tile and head.  Bound by memory, one read and one write of each operand (the gradient's
// tiles read the output too): the backward's four of 2 x 4096 tokens, 16 heads of 128 on 4, 400 MB in 74 us,
// 5.4 TB/s; of 16 x 256 tokens, 8 heads of 64, 75 MB in 14 us.
template <int DP>
__global__ void __launch_bounds__(256) pack(PackArgs a) {
  using S = Shape<DP>;
  constexpr int NI = DP / 32, NC = DP / 8;  // a thread's chunks of 8 columns; chunks of a row
  __shared__ float tops[kTile][NC + 1];  // of 8 columns
  __shared__ float part[kTile][NC + 1];  // out . dout of 8 columns
  const int tile = blockIdx.x / a.slots, tid = threadIdx.x;
  int head = blockIdx.x % a.slots, which = 0;
  while (head >= a.src[which].heads) head -= a.src[which++].heads;
  const Source s = a.src[which];
  const SeqTile t = a.tiles[tile];
  const int rows = min(kTile, t.len - t.t0);
  const float *x = s.x + (int64_t)(t.row0 + t.t0) * s.ld + (int64_t)head * a.dh;
  float v[NI][8];
  bool odd = false;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = (i * 256 + tid) / NC, c = (i * 256 + tid) % NC;
    f4 lo{}, hi{};
    if (row < rows && c * 8 < a.dh) {
      const float *p = x + row * s.ld + c * 8;
      lo = *reinterpret_cast<const f4u *>(p), hi = *reinterpret_cast<const f4u *>(p + 4);
    }
    float inv = 1.f, dot = 0.f;
    if (s.stats != nullptr && row < rows) {
      const int64_t at = t.row0 + t.t0 + row;
      inv = 1.f / s.stats[(at * s.heads + head) * 2 + 1];
      if (c * 8 < a.dh) {
        const float *p = s.out + at * s.ld + (int64_t)head * a.dh + c * 8;
        const f4 x0 = *reinterpret_cast<const f4u *>(p), x1 = *reinterpret_cast<const f4u *>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) dot = fmaf(x0[j], lo[j], dot);
#pragma unroll
        for (int j = 0; j < 4; ++j) dot = fmaf(x1[j], hi[j], dot);
      }
      odd |= !__builtin_isfinite(dot);
    }
    if (s.stats != nullptr) part[row][c] = dot;
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = (j < 4 ? lo[j] : hi[j - 4]) * inv;
      const float m = fabsf(v[i][j]);
      odd |= !(m < s.most);
      big = fmaxf(big, m);
    }
    tops[row][c] = big;
  }
  const int any = __syncthreads_or(odd), lane = tid & 63;
  // every wave has all rows, one a lane
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) top = fmaxf(top, tops[lane][c]);
  const int word = any ? kOdd : tile_word(wave_max(top), wave_butterfly(not_zero(top), lower));
  if (word == kOdd) {
    if (tid == 0) s.exps[(int64_t)tile * s.heads + head] = kOdd;
    return;
  }
  const bool mixed = is_mixed(word);
  const int e = base_of(word), mine = mixed && top > 0.f ? exponent_for(top) : e;
  if (tid < kTile) {
    if (mixed) s.each[((int64_t)tile * s.heads + head) * kTile + tid] = mine;
    float m = INFINITY, d = 0.f;
    if (s.stats != nullptr) {
      if (tid < rows) {
        const float *st = s.stats + ((int64_t)(t.row0 + t.t0 + tid) * s.heads + head) * 2;
        for (int c = 0; c < NC; ++c) d += part[tid][c];
        m = st[0], d = __builtin_amdgcn_ldexpf(d / st[1], e);
      }
      *reinterpret_cast<f2 *>(s.rowstat + (((int64_t)tile * s.heads + head) * kTile + tid) * 2) = f2{m, d};
    }
    const bool far = __any(!(fabsf(d) < kMostTotal));
    if (tid == 0) s.exps[(int64_t)tile * s.heads + head] = far ? kOdd : word;
  }
  const int64_t at = ((int64_t)tile * s.heads + head) * S::kBytes;
  float by = __builtin_amdgcn_ldexpf(s.by, e);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = (i * 256 + tid) / NC, c = (i * 256 + tid) % NC;
    if (mixed) by = __builtin_amdgcn_ldexpf(s.by, __shfl(mine, row));
    const Terms p = split8(v[i], by);
    char *o = s.rows + at + (row >> 5) * S::kHalf + (c >> 1) * 2048 + place(c & 1, row & 31);
    *reinterpret_cast<h8 *>(o) = p.h;
    *reinterpret_cast<h8 *>(o + 1024) = p.m;
  }
}

// Copies 64 lanes' 16 (or 4) bytes, each from the lane's address, to 64 consecutive places of LDS,
// without passing through registers.  As an instruction of its own: the compiler's form is waited for
// before any later LDS access, whichever place that reads.  There is no output register, and the
// compiler's waits on its own loads only grow longer by these.
__device__ __forceinline__ void copy16(const void *src, const void *lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src),
               "s"((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)lds)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(const void *src, const void *lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src),
               "s"((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)lds)
               : "memory", "m0");
}

// Copies `bytes` (a multiple of 4096) of fragments to LDS: wave w of four has every fourth kilobyte.
template <int BYTES>
__device__ __forceinline__ void fetch(const char *src, char *lds, int w, int lane) {
  static_assert(BYTES % 4096 == 0);
#pragma unroll
  for (int i = 0; i < BYTES / 4096; ++i) copy16(src + (i * 4 + w) * 1024 + lane * 16, lds + (i * 4 + w) * 1024);
}

// Waits for this wave's copies, then for the other waves': what any of them fetched is there.
__device__ __forceinline__ void fetched() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// What the waves' lanes found, by one barrier: bit 0 a tile that is odd, bit 1 one that is mixed.
__device__ __forceinline__ int found(int (&flags)[4], int w, bool odd, bool mixed) {
  flags[w] = (__any(odd) ? 1 : 0) | (__any(mixed) ? 2 : 0);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]);
}
// f(std::bool_constant<mixed>).
template <class F>
__device__ __forceinline__ void by_tiles(bool mixed, F &&f) {
  if (mixed)
    f(std::true_type{});
  else
    f(std::false_type{});
}

template <class Op>
__device__ __forceinline__ float over16(const f16 &x, Op op) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = op(x[2 * i], x[2 * i + 1]);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = op(r[2 * i], r[2 * i + 1]);
  return op(op(r[0], r[1]), op(r[2], r[3]));
}

// The backward's P and dS are split times a power of two that puts each column's largest of the 32 rows at
// hand into [2^14, 2^15): the split's smallest step is then 2^-38 of that, however little of a row's
// probability the rows have or however large another tile's values are. The scaled split costs what the
// plain one does, so this is eight max3 and a swap for 16 elements.
__device__ __forceinline__ float top_of(const f16 &x, float r) {
#pragma unroll
  for (int i = 0; i < 16; i += 2) r = fmaxf(fmaxf(r, fabsf(x[i])), fabsf(x[i + 1]));
  return r;
}
__device__ __forceinline__ int top_exponent(float lane_top) {
  return max(__builtin_amdgcn_frexp_expf(half_pair(lane_top, [](float a, float b) { return fmaxf(a, b); })), -100);
}

// Weights of such tokens, brought to what the tokens count at the exponent `base`, and returns the power of two
// besides: each column's largest comes to 2^100 at most, so that what tokens 2^140 below another weigh stays
// above fp32's smallest.
constexpr int kWeight = 100;
__device__ __forceinline__ int weigh(f16 &x, const int *each, int base, int hi) {
  const int up = kWeight - top_exponent(top_of(x, 0.f));
  level(x, each, base + up, hi);
  return up;
}

// The exponent of a row of wave w, of largest magnitude `top`, as `pack` has it: waves w and w ^ 1 have a tile.
// (Where that is odd for its tokens' differences alone, the row's own.)
__device__ __forceinline__ int own_exponent(const float (&tops)[4], const float (&lows)[4], int w, float top) {
  const float big = fmaxf(tops[w], tops[w ^ 1]);
  const int word = tile_word(big, fminf(lows[w], lows[w ^ 1]));
  return is_mixed(word) && top > 0.f ? exponent_for(top) : exponent_for(big);
}

struct ForwardArgs {
  const float *q;
  const char *k, *v;  // fragments
  const int *ek, *ev, *each_k, *each_v;
  float *out, *stats;
  int64_t ld_q, ld_out;
  int heads, kv_heads, dh;
  float mant;  // log2(e) / sqrt(dh) is mant 2^exp, mant in [0.5, 1)
  int exp;
  float most;  // a query's largest magnitude
};

// Four waves walk the keys before a block of query rows: Z = 1, one stretch of keys for 32 rows a wave
// (128); Z = 2, two sets of waves with every other 32 keys each for 64 rows, joined at the end, where
// there are few blocks and the longest walk decides.  Keys staged at a time: 64, or 32.
template <int DP, int Z>
struct Walk {
  static constexpr int R = 4 / Z;                                // waves with rows of their own
  static constexpr int KT = Z == 2 || DP <= 64 ? 64 : 32;        // the forward's stage
  static constexpr int KB = KT / 32 / Z;                         // 32-key blocks of a wave
  static constexpr int kForward = 4 * KT * DP * 4;               // LDS: two stages of keys and values
  static constexpr int kBack = 2 * (2 * Z * 32 * DP * 4 + 256 * Z);  // and the backward's
};

// Adds the second set's results to the first's, through LDS: every lane N vectors of 16.  Returns whether
// the wave is of the first set.
template <int Z, int N>
__device__ __forceinline__ void join_sets(f16 *const (&x)[N], char *lds, int r, int z, int lane) {
  if constexpr (Z == 2) {
    __syncthreads();
    f4 *p = reinterpret_cast<f4 *>(lds) + (int64_t)r * N * 4 * 64 + lane;
    if (z == 1) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f4 y;
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] = (*x[i])[4 * e + j];
          p[(4 * i + e) * 64] = y;
        }
    }
    __syncthreads();
    if (z == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f4 y = p[(4 * i + e) * 64];
#pragma unroll
          for (int j = 0; j < 4; ++j) (*x[i])[4 * e + j] += y[j];
        }
    }
  }
}

// S^T = K Q^T leaves a query's scores in two lanes. The scale's mantissa is in the queries' terms, so that a
// score in base 2 is its sum times a power of two, exactly, and 2^(score - x) takes one fma however large
// the score: the largest's own exponent is never off by a product's rounding, which from 2^28 on would pass
// what fp16 holds. O^T += V^T P^T with P = 2^(score - top + 14) for the stage's largest score `top`, whatever
// the row's before: the split's smallest step, 2^-24, is then 2^-38 of the stage's largest probability. Sums
// are 2^14 times those relative to a reference m, which moves only when a score passes it by 2^8.
//
// The queries have the exponent that `pack` gives their 64 (two waves have a tile), as in the backward, where
// they are packed: all three kernels then form a score from the same terms in the same order, to the same
// bits, and a row whose largest score is all there is has p = 1.
//
// 8192 tokens, 16 heads of 128 on 4: 0.77 to 0.84 ms by card, 327 to 357 TFLOP/s of fp32 work and three
// times that on the fp16 matrix cores, which are busy 64 % of the cycles at the 1.6 GHz that the card's
// power leaves (a large fp16 library product: 1085 TFLOP/s).  13 prompts of 1 to 1290 tokens, 16 heads of
// 64, take 48 us, of which the longest walk, 21 stages of 64 keys, is most.  Stages of 64 keys twice in LDS
// against 32 four times, 64 and 32 three times, there, with earlier splits: 47, 54, 62, 58 us.
//
// Returns false, before any write, where a tile is odd.
template <int DP, int Z>
__device__ __forceinline__ bool forward_tile(const ForwardArgs &a, const SeqTile &t, int h, char *lds) {
  using S = Shape<DP>;
  using W = Walk<DP, Z>;
  constexpr int KT = W::KT, KB = W::KB, kStage = KT * DP * 4;
  __shared__ float joint[Z == 2 ? 3 : 1][64], tops[4], lows[4];
  __shared__ int flags[4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % W::R, z = w / W::R;
  const int c = lane & 31, hi = lane >> 5, g = h / (a.heads / a.kv_heads);
  const int end = min(t.t0 + 32 * W::R, t.len), q0 = t.t0 + 32 * rw;
  const int64_t kv0 = (int64_t)t.tile0 * a.kv_heads + g;  // the sequence's first tile of this head
  const int last = (end - 1) / kTile;
  Terms q[S::NS];
  bool odd = false;
  RowValues<DP> qx;
  qx.load(a.q + (int64_t)(t.row0 + q0 + c) * a.ld_q + (int64_t)h * a.dh, q0 + c < t.len, a.dh, hi);
  bool mixed = false;
  for (int i = tid; i <= last; i += 256) {
    const int wk = a.ek[kv0 + (int64_t)i * a.kv_heads], wv = a.ev[kv0 + (int64_t)i * a.kv_heads];
    odd |= wk == kOdd || wv == kOdd, mixed |= is_mixed(wk) || is_mixed(wv);
  }
  const float row_top = qx.top(a.most, odd);
  tops[w] = wave_max(row_top), lows[w] = wave_butterfly(not_zero(row_top), lower);
  const int kinds = found(flags, w, odd, mixed);
  if (kinds & 1) return false;
  const int eq = own_exponent(tops, lows, w, row_top);
  qx.split_into(q, __builtin_amdgcn_ldexpf(a.mant, eq));
  const bool live = q0 < t.len;
  const int ro = place(hi, c), co = columns_place(lane);

  f16 o[S::NB] = {};
  float m = kNone, top = kNone, l = 0.f;
  const int n = (end + KT - 1) / KT;              // key blocks of the workgroup
  const int mine = live ? (q0 + 31) / KT + 1 : 0;  // and of the wave
  auto tile_of = [&](int i) { return kv0 + (int64_t)(i * KT / kTile) * a.kv_heads; };
  auto issue = [&](int i) {
    const int64_t at = tile_of(i) * S::kBytes + (i * KT % kTile) * DP * 4;
    char *to = lds + (i & 1) * 2 * kStage;
    fetch<kStage>(a.k + at, to, w, lane);
    fetch<kStage>(a.v + at, to + kStage, w, lane);
  };
  issue(0);
  by_tiles(kinds & 2, [&](auto kind) {
    constexpr bool MIXED = decltype(kind)::value;
    for (int i = 0; i < n; ++i) {
      fetched();
      if (i + 1 < n) issue(i + 1);
      if (i >= mine) continue;
      const char *kf = lds + (i & 1) * 2 * kStage + z * S::kHalf, *vf = kf + kStage;
      const int key0 = i * KT + 32 * z;
      if (key0 > q0 + 31) continue;  // all after the wave's rows
      const int64_t tile = tile_of(i);
      const int wk = scalar(a.ek + tile), wv = scalar(a.ev + tile);
      const int ek = MIXED ? base_of(wk) : wk, ev = MIXED ? base_of(wv) : wv;
      const int64_t in_tile = tile * kTile + i * KT % kTile + 32 * z;
      f16 s[KB] = {};
      Terms x[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) x[kb] = rows_of(kf + kb * S::kHalf, 0, ro);
#pragma unroll
      for (int st = 0; st < S::NS; ++st) {
        Terms y[KB];
        if (st + 1 < S::NS) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) y[kb] = rows_of(kf + kb * S::kHalf, st + 1, ro);
        }
        __builtin_amdgcn_sched_barrier(0);  // the next step's operands are asked for before this one's products
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) mma(s[kb], x[kb], q[st]);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) x[kb] = y[kb];
      }
      if (MIXED && is_mixed(wk)) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) level(s[kb], a.each_k + in_tile + 32 * kb, ek, hi);
      }
      // an underflow of f must not make -inf * f NaN
      const float f = fmaxf(__builtin_amdgcn_ldexpf(1.f, a.exp - eq - ek), 1.17549435e-38f);
      if (key0 + 32 * KB > q0 + 1) {  // keys after a row of the wave
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (key0 + 32 * kb + out_row(e, hi) > q0 + c) s[kb][e] = -INFINITY;
      }
      float most = over16(s[0], [](float x, float y) { return fmaxf(x, y); });
      if constexpr (KB == 2) most = fmaxf(most, over16(s[1], [](float x, float y) { return fmaxf(x, y); }));
      most = half_pair(most, [](float x, float y) { return fmaxf(x, y); }) * f;
      top = fmaxf(top, most);
      if (__any(most > m + 8.f)) {
        const float now = fmaxf(m, most);
        const float r = __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= r;
#pragma unroll
        for (int b = 0; b < S::NB; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[b][e] *= r;
      }
      Terms p[KB][2];
      // from 2^24 on, where a float's steps pass 14, P is at most 1; every other score is then 2 below or more
      const float ref = fabsf(most) < 0x1p24f ? most - 14.f : most;
      // from the reference as rounded
      const float back = __builtin_amdgcn_exp2f(ref - m + 14.f);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = __builtin_amdgcn_exp2f(fmaf(s[kb][e], f, -ref));
        l = fmaf(over16(s[kb], [](float x, float y) { return x + y; }), back, l);
      }
      float fv = __builtin_amdgcn_ldexpf(back, -ev);
      if (MIXED && is_mixed(wv)) {
        float lane_top = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          level(s[kb], a.each_v + in_tile + 32 * kb, ev + kWeight - 15, hi);
          lane_top = top_of(s[kb], lane_top);
        }
        const int big = top_exponent(lane_top);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[kb][e] = __builtin_amdgcn_ldexpf(s[kb][e], 15 - big);
        fv = __builtin_amdgcn_ldexpf(back, big - kWeight - ev);
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = s[kb][e];
        p[kb][0] = split8(x), p[kb][1] = split8(x + 8);
      }
      constexpr int kSteps = 2 * KB;  // of 16 keys
      Terms v = columns_of(vf, 0, 0, co);
#pragma unroll
      for (int b = 0; b < S::NB; ++b) {
        f16 z = {};
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const int nb = st + 1 < kSteps ? b : b + 1, ns = (st + 1) % kSteps;
          Terms y;
          if (nb < S::NB) y = columns_of(vf + (ns >> 1) * S::kHalf, nb, ns & 1, co);
          __builtin_amdgcn_sched_barrier(0);
          mma(z, v, p[st >> 1][st & 1]);
          v = y;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[b][e] = fmaf(z[e], fv, o[b][e]);
      }
    }
  });
  const int row = q0 + c;
  l = half_pair(l, [](float x, float y) { return x + y; });
  if constexpr (Z == 2) {
    // both sets relative to the larger reference
    __syncthreads();
    if (z == 1 && hi == 0) joint[0][32 * rw + c] = m, joint[1][32 * rw + c] = l, joint[2][32 * rw + c] = top;
    if (z == 0 && hi == 0) reinterpret_cast<float *>(lds)[32 * rw + c] = m;
    __syncthreads();
    const float m0 = reinterpret_cast<float *>(lds)[32 * rw + c], m1 = joint[0][32 * rw + c];
    const float now = fmaxf(m0, m1), f = __builtin_amdgcn_exp2f(m - now);
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] *= f;
    l = fmaf(l, f, z == 0 ? joint[1][32 * rw + c] * __builtin_amdgcn_exp2f(m1 - now) : 0.f);
    top = fmaxf(top, joint[2][32 * rw + c]);
    m = now;
    f16 *all[S::NB];
#pragma unroll
    for (int b = 0; b < S::NB; ++b) all[b] = &o[b];
    join_sets<Z>(all, lds, rw, z, lane);
    if (z == 1) return true;
  }
  if (row >= t.len) return true;
  const float inv = 1.f / l;
  float *p = a.out + (int64_t)(t.row0 + row) * a.ld_out + (int64_t)h * a.dh;
#pragma unroll
  for (int b = 0; b < S::NB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 32 * b + 8 * e + 4 * hi;
      if (d < a.dh) {
        f4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = o[b][4 * e + j] * inv;
        *reinterpret_cast<f4u *>(p + d) = x;
      }
    }
  if (a.stats != nullptr && hi == 0) {
    // relative to the largest score
    float *st = a.stats + ((int64_t)(t.row0 + row) * a.heads + h) * 2;
    st[0] = top, st[1] = l * 0x1p-14f * __builtin_amdgcn_exp2f(m - top);
  }
  return true;
}

struct BackwardArgs {
  const float *xq, *xk, *xv, *out, *dout, *stats;
  int64_t ld_xq, ld_xkv, ld_out;
  const char *q, *k, *v, *g;  // fragments; g: the output's gradient
  const int *eq, *ek, *ev, *eg, *each_q, *each_k, *each_v, *each_g;
  const float *rowstat;
  float *dq, *dk, *dv;
  int64_t ld_q, ld_k, ld_v, total;
  int heads, kv_heads, dh, accumulate, acc_kv;  // acc_kv: for dk and dv
  int each;             // query heads of a workgroup of key rows: its group, or one
  float alpha, scale;   // log2(e) / sqrt(dh), 1 / sqrt(dh)
  float mant;           // alpha is mant 2^exp, mant in [0.5, 1)
  int exp;
  float scale_q;        // scale / mant: of sums over the packed queries
  float most_score, most_value;  // see Source
};

// dS comes as dS'' = p (raw 2^-ev - D 2^eg) = dS 2^eg: with V's factor 2^ev and the gradient's 2^eg, raw = dP
// 2^(ev + eg) is below 2^37 and ev in -65..126; D 2^eg, which may come from other tiles of V than the one at
// hand, is below 2^110 (`kMostTotal`).

// A probability times the row's sum, from a score and the row's largest. It is at most 1 as the forward has
// it; where the row kernels had the row, whose sums run in another order, a score may be above.
__device__ __forceinline__ float score(float s, float f, float m) {
  return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(fmaf(s, f, -m)), 0.f, 1.f);
}
__device__ __forceinline__ float dscore(float p, float raw, float graw, float d) { return p * fmaf(raw, graw, -d); }

// s = A a^T and r = B b^T of 32 rows at pa and pb; the next step's operands are asked for before this
// one's products. SWAPPED: s with the order of a A^T.
template <int DP, bool SWAPPED>
__device__ __forceinline__ void two_products(f16 &s, f16 &r, const char *pa, const char *pb, const Terms (&a)[DP / 16],
                                             const Terms (&b)[DP / 16], int off) {
  s = f16{}, r = f16{};
  Terms x = rows_of(pa, 0, off), y = rows_of(pb, 0, off);
#pragma unroll
  for (int st = 0; st < DP / 16; ++st) {
    Terms nx, ny;
    if (st + 1 < DP / 16) nx = rows_of(pa, st + 1, off), ny = rows_of(pb, st + 1, off);
    __builtin_amdgcn_sched_barrier(0);
    mma<SWAPPED>(s, x, a[st]);
    mma(r, y, b[st]);
    x = nx, y = ny;
  }
}

// Writes a wave's 32 columns of a transposed result, times `by`, to the row at p. (The sums are added with powers
// of two alone, which are exact down to fp32's smallest: a scale with a mantissa among them lost bits of
// results below 2^-97.)
template <int DP>
__device__ __forceinline__ void put_rows(float *p, const f16 (&x)[DP / 32], float by, int dh, int hi, int accumulate) {
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 32 * b + 8 * e + 4 * hi;
      if (d < dh) {
        f4 y;
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = x[b][4 * e + j] * by;
        if (accumulate) y += f4(*reinterpret_cast<const f4u *>(p + d));
        *reinterpret_cast<f4u *>(p + d) = y;
      }
    }
}

// dQ of a block of query rows of a head: like the forward, with S^T and dP^T of 32 keys at a time, dQ^T
// += K^T dS^T.  Returns false, before any write, where a tile is odd.
//
// The backward forms S and dP twice, here and for the key rows: seven products for the formula's five,
// against writing dS, or adding dQ by atomics whose order would change the result.  2 x 4096 tokens, 16
// heads of 128 on 4: 1.52 to 1.6 ms for both, 301 to 317 TFLOP/s of the seven products' fp32 work (215 to
// 226 of the five's), at one wave a SIMD, matrix cores busy 41 % of the cycles and the VALU 33 %, at 2.17
// GHz.  As many products a second as in the forward: the card's power is what bounds them, so that products a
// stage ahead of their elements, more stages in flight or sums taken in turn (1520, 1850, 1520 us where the
// kernel of then took 1505) gave nothing.
template <int DP, int Z>
__device__ __forceinline__ bool dq_tile(const BackwardArgs &a, const SeqTile &t, int h, char *lds) {
  using S = Shape<DP>;
  constexpr int R = 4 / Z, kPart = Z * S::kHalf, kStage = 2 * kPart;
  __shared__ float tops[4], lows[4];
  __shared__ int flags[4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % R, z = w / R;
  const int c = lane & 31, hi = lane >> 5, g = h / (a.heads / a.kv_heads);
  const int end = min(t.t0 + 32 * R, t.len), q0 = t.t0 + 32 * rw;
  const int64_t kv0 = (int64_t)t.tile0 * a.kv_heads + g, row = t.row0 + q0 + c;
  const int last = (end - 1) / kTile;
  const bool live = q0 < t.len, mine_in = q0 + c < t.len;
  bool odd = false;
  bool mixed = false;
  for (int i = tid; i <= last; i += 256) {
    const int wk = a.ek[kv0 + (int64_t)i * a.kv_heads], wv = a.ev[kv0 + (int64_t)i * a.kv_heads];
    odd |= wk == kOdd || wv == kOdd, mixed |= is_mixed(wk) || is_mixed(wv);
  }
  Terms q[S::NS], go[S::NS];
  float m = INFINITY, D = 0.f;  // a row past the sequence: p = 0
  int eg;
  RowValues<DP> qx;
  qx.load(a.xq + row * a.ld_xq + (int64_t)h * a.dh, mine_in, a.dh, hi);
  const float q_top = qx.top(a.most_score, odd);
  tops[w] = wave_max(q_top), lows[w] = wave_butterfly(not_zero(q_top), lower);
  {
    RowValues<DP> x, o;
    x.load(a.dout + row * a.ld_out + (int64_t)h * a.dh, mine_in, a.dh, hi);
    o.load(a.out + row * a.ld_out + (int64_t)h * a.dh, mine_in, a.dh, hi);
    float inv = 1.f;
    if (mine_in) {
      const float *st = a.stats + (row * a.heads + h) * 2;
      m = st[0], inv = 1.f / st[1];
    }
#pragma unroll
    for (int s = 0; s < S::NS; ++s) {
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) part = fmaf(x.x[s][j], o.x[s][j], part), x.x[s][j] *= inv;
      D += part;
    }
    D = half_pair(D, [](float y, float z) { return y + z; }) * inv;
    eg = exponent_for(x.top(a.most_value, odd));
    x.split_into(go, __builtin_amdgcn_ldexpf(1.f, eg));
    D = __builtin_amdgcn_ldexpf(D, eg);
    odd |= !(fabsf(D) < kMostTotal);
  }
  const int kinds = found(flags, w, odd, mixed);
  if (kinds & 1) return false;
  const int eq = own_exponent(tops, lows, w, q_top);
  qx.split_into(q, __builtin_amdgcn_ldexpf(a.mant, eq));
  const int ro = place(hi, c), co = columns_place(lane);

  f16 x[S::NB] = {};
  const int n = (end + 32 * Z - 1) / (32 * Z), mine = live ? q0 / 32 + 1 : 0;  // blocks of 32 Z keys, of 32
  auto tile_of = [&](int i) { return kv0 + (int64_t)(i * Z >> 1) * a.kv_heads; };
  auto issue = [&](int i) {
    const int64_t at = tile_of(i) * S::kBytes + (i * Z & 1) * kPart;
    char *to = lds + (i & 1) * kStage;
    fetch<kPart>(a.k + at, to, w, lane);
    fetch<kPart>(a.v + at, to + kPart, w, lane);
  };
  issue(0);
  by_tiles(kinds & 2, [&](auto kind) {
    constexpr bool MIXED = decltype(kind)::value;
    for (int i = 0; i < n; ++i) {
      fetched();
      if (i + 1 < n) issue(i + 1);
      const int kb = i * Z + z;  // the wave's 32 keys
      if (kb >= mine) continue;
      const char *kf = lds + (i & 1) * kStage + z * S::kHalf, *vf = kf + kPart;
      const int64_t tile = tile_of(i), in_tile = tile * kTile + 32 * (kb & 1);
      const int wk = scalar(a.ek + tile), wv = scalar(a.ev + tile);
      const int ek = MIXED ? base_of(wk) : wk, ev = MIXED ? base_of(wv) : wv;
      f16 s, r;
      two_products<DP, false>(s, r, kf, vf, q, go, ro);
      if (MIXED && is_mixed(wk)) level(s, a.each_k + in_tile, ek, hi);
      if (MIXED && is_mixed(wv)) level(r, a.each_v + in_tile, ev, hi);
      f16 p, ds;
      const float f = __builtin_amdgcn_ldexpf(1.f, a.exp - eq - ek), graw = __builtin_amdgcn_ldexpf(1.f, -ev);
#pragma unroll
      for (int e = 0; e < 16; ++e) p[e] = score(s[e], f, m), ds[e] = dscore(p[e], r[e], graw, D);
      if (32 * kb + 31 > q0) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * kb + out_row(e, hi) > q0 + c) ds[e] = 0.f;
      }
      int shift = 0;
      if (MIXED && is_mixed(wk)) shift = weigh(ds, a.each_k + in_tile, ek, hi);
      float y[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = ds[e];
      const int top = top_exponent(top_of(ds, 0.f));
      const float up = __builtin_amdgcn_ldexpf(1.f, 15 - top);
      const Terms b[2] = {split8(y, up), split8(y + 8, up)};
      const float back = __builtin_amdgcn_ldexpf(1.f, top - 15 - shift - eg - ek);
      Terms k0 = columns_of(kf, 0, 0, co), k1 = columns_of(kf, 0, 1, co);
#pragma unroll
      for (int nb = 0; nb < S::NB; ++nb) {
        Terms na, nc;
        if (nb + 1 < S::NB) na = columns_of(kf, nb + 1, 0, co), nc = columns_of(kf, nb + 1, 1, co);
        __builtin_amdgcn_sched_barrier(0);
        f16 u = {};
        mma(u, k0, b[0]);
        mma(u, k1, b[1]);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[nb][e] = fmaf(u[e], back, x[nb][e]);
        k0 = na, k1 = nc;
      }
    }
  });
  f16 *sets[S::NB];
#pragma unroll
  for (int b = 0; b < S::NB; ++b) sets[b] = &x[b];
  join_sets<Z>(sets, lds, rw, z, lane);
  if (mine_in && z == 0) put_rows<DP>(a.dq + row * a.ld_q + (int64_t)h * a.dh, x, a.scale, a.dh, hi, a.accumulate);
  return true;
}

// dK and dV of a block of key rows: the waves own 32 keys each and walk the queries from theirs on, for
// each query head in turn: S = Q K^T and dP = dO V^T of 32 queries, dV^T += dO^T P, dK^T += Q^T dS.
template <int DP, int Z>
__device__ __forceinline__ bool dkv_tile(const BackwardArgs &a, const SeqTile &t, int h0, char *lds) {
  using S = Shape<DP>;
  constexpr int R = 4 / Z, kPart = Z * S::kHalf, kStage = 2 * kPart + 256 * Z;
  __shared__ int flags[4];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % R, z = w / R;
  const int c = lane & 31, hi = lane >> 5, g = h0 / (a.heads / a.kv_heads);
  const int k0 = t.t0 + 32 * rw;
  const int64_t kv0 = (int64_t)t.tile0 * a.kv_heads + g, row = t.row0 + k0 + c;
  const int first = t.t0 / kTile, all = (t.len - 1) / kTile;
  const bool live = k0 < t.len, mine_in = k0 + c < t.len;
  bool odd = false, mixed = false;
  for (int i = first + tid; i <= all; i += 256)
    for (int h = h0; h < h0 + a.each; ++h) {
      const int64_t at = (int64_t)(t.tile0 + i) * a.heads + h;
      const int wq = a.eq[at], wg = a.eg[at];
      odd |= wq == kOdd || wg == kOdd, mixed |= is_mixed(wq) || is_mixed(wg);
    }
  Terms k[S::NS], v[S::NS];
  // the keys' terms as they are packed
  const int64_t own = kv0 + (int64_t)((live ? k0 : t.t0) / kTile) * a.kv_heads;
  const int wk = scalar(a.ek + own), ek = is_mixed(wk) ? a.each_k[own * kTile + (k0 & 32) + c] : wk;
  odd |= wk == kOdd;
  int ev;
  {
    RowValues<DP> x;
    x.load(a.xk + row * a.ld_xkv + (int64_t)g * a.dh, mine_in, a.dh, hi);
    x.split_into(k, __builtin_amdgcn_ldexpf(1.f, ek));
    x.load(a.xv + row * a.ld_xkv + (int64_t)g * a.dh, mine_in, a.dh, hi);
    ev = exponent_for(x.top(a.most_value, odd));
    x.split_into(v, __builtin_amdgcn_ldexpf(1.f, ev));
  }
  const int kinds = found(flags, w, odd, mixed);
  if (kinds & 1) return false;
  const float graw = __builtin_amdgcn_ldexpf(1.f, -ev);
  const int ro = place(hi, c), co = columns_place(lane);

  f16 xk[S::NB] = {}, xv[S::NB] = {};
  // stages of 32 Z queries
  const int b0 = t.t0 / (32 * Z), per = (t.len + 32 * Z - 1) / (32 * Z) - b0, n = per * a.each;
  auto tile_of = [&](int i) {  // the query tile of stage i
    return (int64_t)(t.tile0 + (b0 + i % per) * Z / 2) * a.heads + h0 + i / per;
  };
  auto issue = [&](int i) {
    const int half = (b0 + i % per) * Z & 1;
    const int64_t qt = tile_of(i), at = qt * S::kBytes + half * kPart;
    char *to = lds + (i & 1) * kStage;
    fetch<kPart>(a.q + at, to, w, lane);
    fetch<kPart>(a.g + at, to + kPart, w, lane);
    if (w < Z) copy4(a.rowstat + (qt * kTile + 32 * (half + w)) * 2 + lane, to + 2 * kPart + 256 * w);
  };
  issue(0);
  by_tiles(kinds & 2, [&](auto kind) {
    constexpr bool MIXED = decltype(kind)::value;
    for (int i = 0; i < n; ++i) {
      fetched();
      if (i + 1 < n) issue(i + 1);
      const int q0 = 32 * ((b0 + i % per) * Z + z);
      if (!live || q0 + 31 < k0 || q0 >= t.len) continue;
      const char *stage = lds + (i & 1) * kStage, *qf = stage + z * S::kHalf, *gf = qf + kPart;
      const float *rs = reinterpret_cast<const float *>(stage + 2 * kPart + 256 * z);
      const int64_t qt = tile_of(i);
      const int64_t in_tile = qt * kTile + (q0 & 32);
      const int wq = scalar(a.eq + qt), wg = scalar(a.eg + qt);
      const int eq = MIXED ? base_of(wq) : wq, eg = MIXED ? base_of(wg) : wg;
      f16 s, r;
      two_products<DP, true>(s, r, qf, gf, k, v, ro);
      if (MIXED && is_mixed(wq)) level(s, a.each_q + in_tile, eq, hi);
      if (MIXED && is_mixed(wg)) level(r, a.each_g + in_tile, eg, hi);
      float m[16], d[16];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const f4 y = *reinterpret_cast<const f4 *>(rs + 2 * out_row(e, hi));
        m[e] = y[0], d[e] = y[1], m[e + 1] = y[2], d[e + 1] = y[3];
      }
      f16 p, ds;
      const float f = __builtin_amdgcn_ldexpf(1.f, a.exp - eq - ek);
#pragma unroll
      for (int e = 0; e < 16; ++e) p[e] = score(s[e], f, m[e]), ds[e] = dscore(p[e], r[e], graw, d[e]);
      if (q0 < k0 + 31) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (q0 + out_row(e, hi) < k0 + c) p[e] = 0.f, ds[e] = 0.f;
      }
      int pshift = 0, sshift = 0;
      if (MIXED && is_mixed(wg)) pshift = weigh(p, a.each_g + in_tile, eg, hi);
      if (MIXED && is_mixed(wq)) sshift = weigh(ds, a.each_q + in_tile, eq, hi);
      float y[16], z[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = p[e], z[e] = ds[e];
      const int ptop = top_exponent(top_of(p, 0.f)), stop = top_exponent(top_of(ds, 0.f));
      const float pup = __builtin_amdgcn_ldexpf(1.f, 15 - ptop), sup = __builtin_amdgcn_ldexpf(1.f, 15 - stop);
      const Terms pb[2] = {split8(y, pup), split8(y + 8, pup)}, sb[2] = {split8(z, sup), split8(z + 8, sup)};
      const float bv = __builtin_amdgcn_ldexpf(1.f, ptop - 15 - pshift - eg);
      const float bk = __builtin_amdgcn_ldexpf(1.f, stop - 15 - sshift - eg - eq);
      Terms ga = columns_of(gf, 0, 0, co), qa = columns_of(qf, 0, 0, co);
#pragma unroll
      for (int nb = 0; nb < S::NB; ++nb) {
        f16 u = {}, x = {};
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          Terms gn, qn;
          if (nb + st < S::NB) gn = columns_of(gf, nb + st, 1 - st, co), qn = columns_of(qf, nb + st, 1 - st, co);
          __builtin_amdgcn_sched_barrier(0);
          mma(u, ga, pb[st]);
          mma(x, qa, sb[st]);
          ga = gn, qa = qn;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          xv[nb][e] = fmaf(u[e], bv, xv[nb][e]);
          xk[nb][e] = fmaf(x[e], bk, xk[nb][e]);
        }
      }
    }
  });
  f16 *sets[2 * S::NB];
#pragma unroll
  for (int b = 0; b < S::NB; ++b) sets[2 * b] = &xk[b], sets[2 * b + 1] = &xv[b];
  join_sets<Z>(sets, lds, rw, z, lane);
  if (!mine_in || z != 0) return true;
  // one head of several: its own part, [heads, total, dh]; else the result
  const bool part = a.each < a.heads / a.kv_heads;
  const int64_t at = part ? ((int64_t)h0 * a.total + row) * a.dh : 0;
  const int64_t ck = part ? at : row * a.ld_k + (int64_t)g * a.dh;
  const int64_t cv = part ? at : row * a.ld_v + (int64_t)g * a.dh;
  if (a.dk != nullptr) put_rows<DP>(a.dk + ck, xk, a.scale_q, a.dh, hi, a.acc_kv);
  if (a.dv != nullptr) put_rows<DP>(a.dv + cv, xv, 1.f, a.dh, hi, a.acc_kv);
  return true;
}

}  // namespace tiles
