// New tokens of many sequences over a paged key-value cache, on the fp16 matrix cores at fp32 accuracy.
//
// The query rows of a kv head are the new tokens' heads of its group, token by token: row r of a sequence is head
// r % group of token r / group, so that a block of rows is full whatever the group, and all of it reads the cached
// tokens once.  As in packed_tiles.h a score is S^T = K Q^T and a result O^T += V^T P^T, with 32x32x16 products of
// two-term fp16 splits, h + m, three products each (m h, h m, h h); 8-bit codes are exact in fp16, one term, two
// products.  What the cache holds is split where it is staged:
//   fp32    each token's row of a head, times the power of two that puts its largest magnitude into [2^14, 2^15);
//   8 bits  the codes less 128.
// The row's factor (that power of two's inverse, or its scale) is applied to its scores, and to its probabilities
// before they are split: no token's size costs another its bits, and both formats are one walk.
//
// A workgroup has eight waves: R = 8 / Z of 32 rows, in Z sets with every Z-th 32 tokens of a stage each.  The next
// stage's keys are asked for before this one's scores are formed and split after them, its values before the
// softmax and after the results: sixteen registers hold either on the way.
//
// The work is (kv head, block of rows, stage of tokens), in that order.  It is dealt evenly to one workgroup a CU,
// whatever the lengths, which only the device knows; a block that is cut leaves parts (m, l, O) that
// join_parts adds in order in a second launch: no workgroup waits for another.
#pragma once

#include "packed_tiles.h"
#include "paged_split.h"

namespace chunk {

using numrs_hip::SeqTile;
using paged::Cache;
using paged::kNever;
using paged::uniform;
using tiles::f16;
using tiles::f4;
using tiles::f4u;
using tiles::h8;
using tiles::Terms;
using tiles::u4;
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned long long mask64;

constexpr int kThreads = 512, kStage = 64;  // threads of a workgroup, tokens of a stage

// What a cut block's parts are joined into: written by the workgroup that has its first stage.
struct Cut {
  int parts;       // 0: none
  int row, rows;   // the block's first row in its sequence, and its rows
  int row0, head;  // the sequence's first token, the group's first query head
};

struct Args {
  Cache c;
  const SeqTile *seqs;  // the sequences that have new tokens
  const int32_t *ends;
  const float *q;
  float *out, *parts;
  Cut *cuts;  // [workgroups]
  int64_t ld_q, ld_out;
  int n, heads, group;
  float mant;  // log2(e) / sqrt(dh) is mant 2^exp, mant in [0.5, 1)
  int exp;
};

// Magnitudes within these bounds (or 0) cannot make a product leave fp32's range by themselves.  A stage with a
// token beyond them, with one that is not finite, or on a page that the cache lacks, goes token by token in plain
// fp32 (`take_plain`), and so does what a wave's rows see if one of their queries is beyond them.
constexpr float kSmall = 0x1p-60f, kLarge = 0x1p60f;
__device__ __forceinline__ bool wild(float x) { return !(x == 0.f || (fabsf(x) >= kSmall && fabsf(x) <= kLarge)); }
// The larger; NaN if one is.
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }
// Values from 2^96 on raise the softmax's reference, so that their sums stay below fp32's largest.
constexpr int kRaise = 96;

// Floats of a part: references and sums of a block's rows, then their outputs.
template <int DP, int ROWS>
constexpr int kPart = ROWS * (2 + DP);

__device__ __forceinline__ int log_lanes(int dp) { return dp > 64 ? 4 : dp > 32 ? 3 : 2; }

// A head size rounded up to DP in LDS: a row of keys (or fp32 values) of a term is kRow bytes, its pieces of 16
// bytes out of place by the token, so that neither the reads of a product (one piece of 32 tokens; or of the
// values, 32 columns of 4 tokens) nor the writes (a token's pieces) meet a bank twice.
template <bool INT8, int DP>
struct Shape {
  static constexpr int NS = DP / 16, NB = DP / 32, kTerms = INT8 ? 1 : 2;
  static constexpr int kLanes = DP > 64 ? 4 : DP > 32 ? 3 : 2;  // log2 of the threads of a token's row, 8 columns each
  static constexpr int kRow = 16 << kLanes, kPieces = 1 << kLanes;
  static constexpr int kPass = kThreads >> kLanes, NP = kStage / kPass > 0 ? kStage / kPass : 1;
  static constexpr int kKeys = kTerms * kStage * kRow;
  static constexpr int kValues = INT8 ? kStage * DP * 2 : kKeys;
  static constexpr int kBytes = kKeys + kValues;  // of a stage
  static constexpr int kQuads = kStage / 4 * (DP / 4), NV = (kQuads + kThreads - 1) / kThreads;

  // (A piece 2 st + hi of keys is at the piece hi's place ^ 32 st, a piece 4 b + x of values at x's ^ 64 b.)
  static __device__ __forceinline__ int key_place(int token, int piece) {
    const int turn = kPieces == 16 ? token : kPieces == 8 ? token >> 1 : token >> 2;
    return token * kRow + ((piece ^ turn) & (kPieces - 1)) * 16;
  }
  static __device__ __forceinline__ int value_place(int token, int piece) {
    const int turn = kPieces == 16 ? 4 * (token & 3) : kPieces == 8 ? 4 * (token >> 1 & 1) : 0;
    return token * kRow + (piece ^ turn) * 16;
  }
};

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
template <int LANES>
__device__ __forceinline__ unsigned row_top(unsigned v) {
  v = dpp_max<0x4E>(dpp_max<0xB1>(v));
  if constexpr (LANES > 2) v = dpp_max<0x141>(v);
  if constexpr (LANES > 3) v = dpp_max<0x140>(v);
  return v;
}

// What a workgroup shares.
template <bool INT8, int DP>
struct Lds {
  using S = Shape<INT8, DP>;
  static constexpr int kJoint = 64 * (16 * S::NB + 4) * 4;  // a wave's results, while sets are joined
  // (the stages last: an LDS access has 16 bits for a constant offset)
  float ks[2][kStage], vs[2][kStage];  // the rows' factors
  int plain[4];                        // of three stages in turn: one is read, one written, one cleared
  char stages[2 * S::kBytes > 4 * kJoint ? 2 * S::kBytes : 4 * kJoint];
  __device__ __forceinline__ char *stage(int buf) { return stages + buf * S::kBytes; }
};

// The same value, formed again: what follows from it is not kept in registers around a loop.
__device__ __forceinline__ int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The cached tokens of one sequence and kv head as a block of rows walks over them.
struct Walk {
  const int32_t *pages;
  int held;  // tokens that its pages can hold of it
  int kv;
};

__device__ __forceinline__ int64_t token_row(const Cache &c, int kv, int pos, int page) {
  return paging::page_base(page, c.kv_heads, kv, c.shift, 1) + (pos & ((1 << c.shift) - 1));
}

// A thread's share of a stage on its way from the cache to LDS.
template <bool INT8, int DP>
struct Staging {
  using S = Shape<INT8, DP>;
  static constexpr int NE = INT8 ? S::NP + S::NV + 1 : S::NP;  // places whose pages it needs
  int32_t entries[NE];
  int64_t at[NE];  // the element of the cache that the thread loads first, of a factor its place
  unsigned have;   // places that the cache has, a bit each
  f4 x[INT8 ? 1 : S::NP][2];
  u2 kc[INT8 ? S::NP : 1];
  u4 vc[INT8 ? S::NV : 1];
  float scale;

  // The token of a place within its stage: a row's, a quad's first, or a factor's.
  static __device__ __forceinline__ int token(int i) {
    const int tid = threadIdx.x;
    if (i < S::NP) return i * S::kPass + (tid >> S::kLanes);  // (past the stage where it has fewer rows than threads)
    if (i < S::NP + (INT8 ? S::NV : 0)) return min(((i - S::NP) * kThreads + tid) / (DP / 4), kStage / 4 - 1) * 4;
    return tid & (kStage - 1);
  }
  __device__ __forceinline__ void look(const Cache &c, const Walk &w, int stage) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int pos = stage * kStage + token(i);
      entries[i] = pos < w.held ? paging::entry_of(w.pages, c.max_pages, c.shift, pos) : -1;
    }
  }
  static __device__ __forceinline__ int row_column(const Cache &c) { return 8 * (threadIdx.x & (S::kPieces - 1)); }
  // Loads go out whatever the place is, from the cache's first page where it is none, and are dropped then: what
  // lies in slots of no token must not reach the products.
  __device__ __forceinline__ void resolve(const Cache &c, const Walk &w, int stage) {
    have = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int page = paging::page_in(entries[i], c.pages);
      have |= page >= 0 ? 1u << i : 0u;
      at[i] = token_row(c, w.kv, stage * kStage + token(i), max(page, 0));
      if (i < S::NP)
        at[i] = at[i] * c.dh + min(row_column(c), c.dh - 8);
      else if (i < NE - 1)
        at[i] = at[i] * c.dh + 4 * min(4 * (((i - S::NP) * kThreads + (int)threadIdx.x) % (DP / 4)), c.dh - 4);
    }
  }
  // fp32 rows of keys or values: a thread's eight columns.
  __device__ __forceinline__ void load_rows(const void *from) {
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const float *p = static_cast<const float *>(from) + at[i];
      x[i][0] = *reinterpret_cast<const f4 *>(p), x[i][1] = *reinterpret_cast<const f4 *>(p + 4);
    }
  }
  __device__ __forceinline__ void load_keys(const Cache &c) {
    if constexpr (!INT8) {
      load_rows(c.k);
    } else {
#pragma unroll
      for (int i = 0; i < S::NP; ++i) kc[i] = *reinterpret_cast<const u2 *>(static_cast<const uint8_t *>(c.k) + at[i]);
      scale = (threadIdx.x & kStage ? c.vs : c.ks)[at[NE - 1]];
    }
  }
  __device__ __forceinline__ void load_values(const Cache &c) {
    if constexpr (!INT8) {
      load_rows(c.v);
    } else {
#pragma unroll
      for (int i = 0; i < S::NV; ++i)
        vc[i] = *reinterpret_cast<const u4 *>(static_cast<const uint8_t *>(c.v) + at[S::NP + i]);
    }
  }

  // Rows in fp32 into two terms; whether all of them are ordinary.
  template <bool VALUES>
  __device__ __forceinline__ bool split_rows(const Cache &c, char *to, float *factors) {
    const int piece = threadIdx.x & (S::kPieces - 1);
    bool good = true;
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const int tk = token(i);
      const bool in = (have >> i & 1) != 0 && row_column(c) < c.dh;
      if (__any(!in)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j >> 2][j & 3] = in ? x[i][j >> 2][j & 3] : 0.f;
      }
      float v[8], big = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[i][j >> 2][j & 3];
#pragma unroll
      for (int j = 0; j < 8; j += 2) big = maximum(maximum(big, fabsf(v[j])), fabsf(v[j + 1]));
      const unsigned top = row_top<S::kLanes>(__builtin_bit_cast(unsigned, big));
      // The power of two that puts the largest into [2^14, 2^15), from its exponent's bits; within the bounds
      // neither it nor its inverse leaves the normal numbers (and beyond them the split is not used).
      constexpr unsigned kLow = 127 - 60, kHigh = 127 + 60;
      const unsigned e = max(top >> 23, kLow);
      good &= e < kHigh && (top >> 23 >= kLow || top == 0);
      const Terms t = tiles::split8(v, __builtin_bit_cast(float, (268 - e) << 23));
      if (tk < kStage) {
        char *p = to + (VALUES ? S::value_place(tk, piece) : S::key_place(tk, piece));
        *reinterpret_cast<h8 *>(p) = t.h;
        *reinterpret_cast<h8 *>(p + kStage * S::kRow) = t.m;
        if (piece == 0) factors[tk] = __builtin_bit_cast(float, (e - 14) << 23);
      }
    }
    return good;
  }

  // stage: the one that is written, of the block's walk, and its buffers.
  __device__ __forceinline__ void put_keys(Lds<INT8, DP> &s, const Cache &c, const Walk &w, int stage, int buf, int third) {
    char *to = s.stage(buf);
    bool good = true;
    if constexpr (!INT8) {
      good = split_rows<false>(c, to, s.ks[buf]);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) good &= (have >> i & 1) != 0 || stage * kStage + token(i) >= w.held;
    } else {
      const int piece = threadIdx.x & (S::kPieces - 1);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int tk = token(i);
        u4 h;
        unsigned lo, hi;
        paged::halves(kc[i][0], lo, hi), h[0] = lo, h[1] = hi;
        paged::halves(kc[i][1], lo, hi), h[2] = lo, h[3] = hi;
        if (tk < kStage) *reinterpret_cast<u4 *>(to + S::key_place(tk, piece)) = h;
      }
      const int tk = threadIdx.x & (kStage - 1);
      const bool in = (have >> (NE - 1) & 1) != 0;
      const float y = in ? scale : 0.f;
      if (threadIdx.x < 2 * kStage) (threadIdx.x < kStage ? s.ks : s.vs)[buf][tk] = y;
      good = !wild(y) && (in || stage * kStage + tk >= w.held);
    }
    if (!good) s.plain[third] = 1;
  }
  __device__ __forceinline__ void put_values(Lds<INT8, DP> &s, const Cache &c, int buf, int third) {
    char *to = s.stage(buf) + S::kKeys;
    if constexpr (!INT8) {
      if (!split_rows<true>(c, to, s.vs[buf])) s.plain[third] = 1;
    } else {
      // four tokens' values of a column lie together: eight bytes of a product's operand
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        const int u = i * kThreads + threadIdx.x;
        if (u >= S::kQuads) continue;
        u4 a, b;
        unsigned lo, hi;
        paged::halves(vc[i][0], lo, hi), a[0] = lo, a[1] = hi;
        paged::halves(vc[i][1], lo, hi), a[2] = lo, a[3] = hi;
        paged::halves(vc[i][2], lo, hi), b[0] = lo, b[1] = hi;
        paged::halves(vc[i][3], lo, hi), b[2] = lo, b[3] = hi;
        *reinterpret_cast<u4 *>(to + u * 32) = a;
        *reinterpret_cast<u4 *>(to + u * 32 + 16) = b;
      }
    }
  }
};

// acc += a b: the small products first.
template <bool INT8>
__device__ __forceinline__ void mma_keys(f16 &acc, const Terms &k, const Terms &q) {
  if constexpr (!INT8) {
    tiles::mma(acc, k, q);
  } else {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.h, q.m, acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.h, q.h, acc, 0, 0, 0);
  }
}

// Columns 32 b + c of 16 tokens, those of lane group g being 4 g .. + 3 and 8 + 4 g .. + 3: the order in which a
// product leaves its results' rows.  off: of the first tokens' first columns.
template <bool INT8, int DP>
__device__ __forceinline__ int values_place(int token, int lane) {
  const int g = lane >> 5;
  if constexpr (INT8) return ((token / 4 + g) * DP + (lane & 31)) * 8;
  return Shape<INT8, DP>::value_place(token + 4 * g + (lane >> 2 & 3), 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) + (lane & 1) * 8;
}
template <bool INT8, int DP>
__device__ __forceinline__ Terms values_of(const char *p, int off, int st, int b) {
  using S = Shape<INT8, DP>;
  Terms t;
  if constexpr (INT8) {
    const char *at = p + off + (4 * st * DP + 32 * b) * 8;
    const u2 lo = *reinterpret_cast<const u2 *>(at), hi = *reinterpret_cast<const u2 *>(at + 2 * DP * 8);
    t.h = t.m = __builtin_bit_cast(h8, u4{lo[0], lo[1], hi[0], hi[1]});
  } else {
    const char *at = p + (off ^ 64 * b) + 16 * st * S::kRow;
    auto term = [](const char *at) {
      const auto a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tiles::lds_s4 *)at);
      const auto b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tiles::lds_s4 *)(at + 8 * S::kRow));
      return __builtin_bit_cast(h8, tiles::s8(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)));
    };
    t.h = term(at), t.m = term(at + kStage * S::kRow);
  }
  return t;
}

// A cached key or value.
template <bool INT8>
__device__ __forceinline__ float key_at(const Cache &c, int64_t row, int d) {
  if constexpr (!INT8) return static_cast<const float *>(c.k)[row * c.dh + d];
  return (float)((int)static_cast<const uint8_t *>(c.k)[row * c.dh + d] - 128) * c.ks[row];
}
template <bool INT8>
__device__ __forceinline__ float value_at(const Cache &c, int64_t row, int d) {
  if constexpr (!INT8) return static_cast<const float *>(c.v)[row * c.dh + d];
  const int64_t at = (row & ~int64_t{3}) * c.dh + 4 * d + (row & 3);
  return (float)((int)static_cast<const uint8_t *>(c.v)[at] - 128) * c.vs[row];
}

// A wave's 32 rows over some of a block's tokens; lane (hi, c) has row c.
template <bool INT8, int DP>
struct Rows {
  using S = Shape<INT8, DP>;
  Terms q[S::NS];
  float o[S::NB][16];
  float m, l;   // l: of the lane's own half of the tokens
  float f;      // log2(e) / sqrt(dh) over the query's factor, a power of two
  int seen;     // tokens that the lane's row sees; 0: none
  bool some;    // of them in the cache so far
  bool plain;   // a query of the wave is beyond the bounds

  __device__ __forceinline__ void start(const Args &a, const float *row, bool live, int sees) {
    const int hi = (threadIdx.x & 63) >> 5;
    seen = sees, some = false;
    tiles::RowValues<DP> x;
    x.load(row, live, a.c.dh, hi);
    bool not_finite = false;
    const float top = x.top(INFINITY, not_finite);
    const int e = tiles::exponent_for(top);
    f = __builtin_amdgcn_ldexpf(1.f, a.exp - e);
    plain = __any(not_finite || wild(top));
    x.split_into(q, __builtin_amdgcn_ldexpf(a.mant, e));
    m = kNever, l = 0.f;
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] = 0.f;
  }

  __device__ __forceinline__ void raise(float now) {
    const float r = __builtin_amdgcn_exp2f(m - now);
    m = now;
    l *= r;
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] *= r;
  }

  // 32 tokens from `first` of a stage: the products of their keys ...
  __device__ __forceinline__ void products(Lds<INT8, DP> &lds, int buf, int first, f16 &s) const {
    const int lane = threadIdx.x & 63, c = lane & 31, hi = lane >> 5;
    const char *keys = lds.stage(buf);
    const int off = again(S::key_place(first + c, hi));
    auto ask = [&](int st) {
      const char *p = keys + (off ^ 32 * st);
      Terms k;
      k.h = *reinterpret_cast<const h8 *>(p);
      if constexpr (!INT8) k.m = *reinterpret_cast<const h8 *>(p + kStage * S::kRow);
      return k;
    };
    Terms k = ask(0);
    s = f16{};
#pragma unroll
    for (int st = 0; st < S::NS; ++st) {
      Terms next;
      if (st + 1 < S::NS) next = ask(st + 1);
      __builtin_amdgcn_sched_barrier(0);  // the next step's operands are asked for before this one's products
      mma_keys<INT8>(s, k, q[st]);
      k = next;
    }
  }

  // ... and what follows from them; the stage's tokens begin at pos0.
  __device__ __forceinline__ void take(Lds<INT8, DP> &lds, int buf, int first, int pos0, bool masked, f16 &s) {
    const int lane = threadIdx.x & 63, hi = lane >> 5;
    const char *values = lds.stage(buf) + S::kKeys;
    // factors of the rows that a lane's results are, four at a time
    auto by_factors = [&](const float *factors) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 x = *reinterpret_cast<const f4 *>(factors + first + 8 * i + 4 * hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * i + j] *= x[j];
      }
    };
    by_factors(lds.ks[buf]);
    const int left = seen - pos0 - first;  // tokens from the first that the row sees
    if (masked) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (tiles::out_row(e, hi) >= left) s[e] = -INFINITY;
    }
    some |= left > 0;
    const float most = half_pair(tiles::over16(s, [](float x, float y) { return fmaxf(x, y); }),
                                 [](float x, float y) { return fmaxf(x, y); }) * f;
    if (__any(most > m + 8.f)) raise(fmaxf(m, most));
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], f, -m));
    l += tiles::over16(s, [](float x, float y) { return x + y; });
    // the probabilities times the values' factors, the largest of a row brought to [2^14, 2^15)
    by_factors(lds.vs[buf]);
    const float top = half_pair(tiles::top_of(s, 0.f), [](float x, float y) { return fmaxf(x, y); });
    const int et = max(__builtin_amdgcn_frexp_expf(top), -100);
    const float lift = __builtin_amdgcn_ldexpf(1.f, 15 - et), back = __builtin_amdgcn_ldexpf(1.f, et - 15);
    float x[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = s[e];
    const Terms p[2] = {tiles::split8(x, lift), tiles::split8(x + 8, lift)};
    constexpr int kSteps = 2;  // of 16 tokens
    const int off = again(values_place<INT8, DP>(first, lane));
    Terms v = values_of<INT8, DP>(values, off, 0, 0);
#pragma unroll
    for (int b = 0; b < S::NB; ++b) {
      f16 z = {};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const int nb = st + 1 < kSteps ? b : b + 1, ns = (st + 1) % kSteps;
        Terms next;
        if (nb < S::NB) next = values_of<INT8, DP>(values, off, ns, nb);
        __builtin_amdgcn_sched_barrier(0);
        mma_keys<INT8>(z, v, p[st]);
        v = next;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] = fmaf(z[e], back, o[b][e]);
    }
  }

  // The same in plain fp32, a token after the other: a lane forms half of its row's score, and adds to its columns
  // of the result.  What is not finite does what it does in fp32, and only to the rows that see it.
  __device__ __forceinline__ void take_plain(const Args &a, const Walk &w, const float *row, int from, int to) {
    const int hi = (threadIdx.x & 63) >> 5, half = (a.c.dh / 8 + 1) / 2 * 8;
    const float scale = __builtin_amdgcn_ldexpf(a.mant, a.exp);
#pragma unroll 1
    for (int pos = from; pos < to; ++pos) {
      int dh = a.c.dh;
      asm volatile("" : "+s"(dh));  // what follows from it is formed here, not kept in registers throughout
      const int page = pos < w.held ? paging::page_of(w.pages, a.c.max_pages, a.c.shift, a.c.pages, pos) : -1;
      if (page < 0) continue;
      const int64_t at = token_row(a.c, w.kv, pos, page);
      float x = 0.f, big = 0.f;
#pragma unroll 1
      for (int d = hi * half; d < min(dh, (hi + 1) * half); ++d) {
        x = fmaf(row[d], key_at<INT8>(a.c, at, d), x);
        const float v = fabsf(value_at<INT8>(a.c, at, d));
        if (v < INFINITY) big = fmaxf(big, v);
      }
      x = half_pair(x, [](float x, float y) { return x + y; }) * scale;
      big = half_pair(big, [](float x, float y) { return fmaxf(x, y); });
      if (pos < seen) {
        some = true;
        // values from 2^96 on raise the reference, so that their sums stay below fp32's largest
        const float now = x + fmaxf(0.f, (float)(__builtin_amdgcn_frexp_expf(big) - 96));
        if (now > m) raise(now);
        const float p = __builtin_amdgcn_exp2f(x - m);
        if (hi == 0 || p != p) l += p;
#pragma unroll
        for (int b = 0; b < S::NB; ++b) {
          asm volatile("" : "+s"(dh));
#pragma unroll
          for (int e = 0; e < 16; ++e)  // (a column past the head reads the last one again: it is not written)
            o[b][e] = fmaf(p, value_at<INT8>(a.c, at, min(32 * b + tiles::out_row(e, hi), dh - 1)), o[b][e]);
        }
      }
    }
  }
};

// Tokens that a sequence's row of token t sees, and the stages that a block of rows takes.
__device__ __forceinline__ int sees(int len, int end, int held, int t) {
  return (int)max((int64_t)0, min((int64_t)end - len + t + 1, (int64_t)held));
}
template <int ROWS>
__device__ __forceinline__ int stages_of(const Cache &c, int group, int len, int end, int block) {
  const int last = min((block + 1) * ROWS, len * group) - 1;
  const int n = sees(len, end, (int)paging::held(end, c.max_pages, c.shift), last / group);
  return max(1, (n + kStage - 1) / kStage);
}

template <bool INT8, int DP, int Z>
__global__ void __launch_bounds__(kThreads, 2) walk_blocks(Args a) {
  using S = Shape<INT8, DP>;
  constexpr int R = 8 / Z, ROWS = 32 * R;
  __shared__ __attribute__((aligned(16))) Lds<INT8, DP> lds;
  __shared__ int64_t pre[kThreads + 1], sums[8];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % R, z = w / R, c = lane & 31, hi = lane >> 5;

  // Of kThreads sequences from i0 on: the stages before each in pre, with `base` before the first; returns
  // their end.
  auto scan = [&](int i0, int64_t base) {
    int64_t v = 0;
    if (i0 + tid < a.n) {
      const SeqTile t = a.seqs[i0 + tid];
      const int end = a.ends[t.seq], blocks = (t.len * a.group + ROWS - 1) / ROWS;
      for (int b = 0; b < blocks; ++b) v += stages_of<ROWS>(a.c, a.group, t.len, end, b);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t below = __shfl_up(v, d);
      if (lane >= d) v += below;
    }
    __syncthreads();
    if (lane == 63) sums[w] = v;
    __syncthreads();
    for (int k = 0; k < w; ++k) v += sums[k];
    pre[tid + 1] = base + v;
    if (tid == 0) pre[0] = base;
    __syncthreads();
    return uniform(pre[min(kThreads, a.n - i0)]);
  };
  int64_t units = 0;  // of a kv head
  for (int i0 = 0; i0 < a.n; i0 += kThreads) units = scan(i0, units);
  const int64_t all = units * a.c.kv_heads;
  const int shares = (int)min((int64_t)gridDim.x, all);
  // A kv head's blocks, which read the same tokens, go to neighbours, and those to one XCD where all take part.
  int p = blockIdx.x;
  if (shares == (int)gridDim.x && gridDim.x % 8 == 0) p = p % 8 * (gridDim.x / 8) + p / 8;
  if (tid == 0) a.cuts[p].parts = 0;
  if (p >= shares) return;
  const int64_t lo = all * p / shares, end_unit = all * (p + 1) / shares;
  auto owner = [&](int64_t x) { return (int)(((x + 1) * shares - 1) / all); };

  int i0 = a.n > kThreads ? a.n : 0;  // the sequences in LDS; none yet where there are several times as many
  int64_t base = a.n > kThreads ? all : 0, next = a.n > kThreads ? all : units;
  for (int64_t u = lo; u < end_unit;) {
    const int kv = (int)(u / units);
    int64_t x = u - kv * units;
    if (x < base) i0 = 0, base = 0, next = scan(0, 0);
    while (x >= next) i0 += kThreads, base = next, next = scan(i0, base);
    const int count = min(kThreads, a.n - i0);
    int j = 0;  // the sequence that has x
    for (int k = 0; k < count; k += 64) j += __builtin_popcountll(__ballot(k + lane < count && pre[min(k + lane, count - 1) + 1] <= x));
    const SeqTile t = a.seqs[i0 + j];
    const int end = __builtin_amdgcn_readfirstlane(a.ends[t.seq]), rows = t.len * a.group;
    const Walk walk{a.c.table + (int64_t)t.seq * a.c.max_pages, (int)paging::held(end, a.c.max_pages, a.c.shift), kv};
    int64_t at = uniform(pre[j]);
    int block = 0, stages;
    for (;; ++block) {
      stages = stages_of<ROWS>(a.c, a.group, t.len, end, block);
      if (x < at + stages) break;
      at += stages;
    }
    for (; u < end_unit && block * ROWS < rows; ++block) {
      stages = stages_of<ROWS>(a.c, a.group, t.len, end, block);
      const int s0 = (int)(x - at), s1 = (int)min((int64_t)stages, s0 + (end_unit - u));
      const int64_t first_unit = u - s0;  // of the block

      // the lane's row, and what the wave's first and last see
      const int row = block * ROWS + 32 * rw + c;
      const bool live = row < rows;
      // The token and head of the lane's row; formed again where they are needed.
      auto token_of = [&](int &head) {
        const int of = again(live ? row : 0), token = of / a.group;
        head = kv * a.group + of - token * a.group;
        return t.row0 + token;
      };
      auto query = [&] {
        int head;
        const int64_t at = token_of(head);
        return a.q + at * a.ld_q + (int64_t)head * a.c.dh;
      };
      const int n_seen = live ? sees(t.len, end, walk.held, row / a.group) : 0;
      const int live_rows = min(32, rows - block * ROWS - 32 * rw);
      const int least = live_rows < 32 ? 0 : __builtin_amdgcn_readlane(n_seen, 0);
      const int most = live_rows > 0 ? __builtin_amdgcn_readlane(n_seen, live_rows - 1) : 0;
      Staging<INT8, DP> g;
      g.look(a.c, walk, s0);
      if (tid < 3) lds.plain[tid] = 0;
      Rows<INT8, DP> r;
      r.start(a, query(), live, n_seen);
      g.resolve(a.c, walk, s0);
      __syncthreads();  // the marks are cleared, the last block's buffers free
      g.load_keys(a.c);
      g.put_keys(lds, a.c, walk, s0, 0, 0);
      g.load_values(a.c);
      g.put_values(lds, a.c, 0, 0);
      g.look(a.c, walk, s0 + 1);
      for (int i = s0; i < s1; ++i) {
        const int buf = (i - s0) & 1, third = (i - s0) % 3, after = (i - s0 + 1) % 3;
        const bool more = i + 1 < s1;
        __syncthreads();
        const bool plain = __builtin_amdgcn_readfirstlane(lds.plain[third]) != 0 || r.plain;
        if (tid == 0) lds.plain[(i - s0 + 2) % 3] = 0;
        const int pos0 = i * kStage;
        if (more) {
          g.resolve(a.c, walk, i + 1);
          g.load_keys(a.c);
        }
        if (plain) r.take_plain(a, walk, query(), pos0 + 32 * z, min(pos0 + 32 * z + kStage / Z, most));
        f16 s;
        auto products = [&](int first) {
          if (pos0 + first < most && !plain) r.products(lds, buf, first, s);
        };
        auto take = [&](int first) {
          if (pos0 + first < most && !plain) r.take(lds, buf, first, pos0, pos0 + first + 32 > least, s);
        };
        products(32 * z);
        if constexpr (Z == 1) take(0);
        if (more) {
          g.put_keys(lds, a.c, walk, i + 1, buf ^ 1, after);
          g.load_values(a.c);
          g.look(a.c, walk, i + 2);
        }
        if constexpr (Z == 1) products(32);
        take(Z == 1 ? 32 : 32 * z);
        if (more) g.put_values(lds, a.c, buf ^ 1, after);
      }
      float l = half_pair(r.l, [](float x, float y) { return x + y; });
      __syncthreads();
      if constexpr (Z > 1) {
        // the sets' results as one, relative to the largest reference, in order
        char *joint = lds.stages;  // [Z - 1][R]
        constexpr int kEach = Lds<INT8, DP>::kJoint;
        static_assert((Z - 1) * R * kEach <= (int)sizeof(lds.stages), "the sets' results fit the stages' place");
        if (z > 0) {
          f4 *to = reinterpret_cast<f4 *>(joint + ((z - 1) * R + rw) * kEach);
#pragma unroll
          for (int b = 0; b < S::NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f4 y;
#pragma unroll
              for (int j = 0; j < 4; ++j) y[j] = r.o[b][4 * i + j];
              to[(4 * b + i) * 64 + lane] = y;
            }
          to[4 * S::NB * 64 + lane] = f4{r.m, l, r.some ? 1.f : 0.f, 0.f};
        }
        __syncthreads();
        if (z == 0) {
#pragma unroll
          for (int k = 1; k < Z; ++k) {
            const f4 *of = reinterpret_cast<const f4 *>(joint + ((k - 1) * R + rw) * kEach);
            const f4 st = of[4 * S::NB * 64 + lane];
            const float now = fmaxf(r.m, st[0]), f0 = __builtin_amdgcn_exp2f(r.m - now), f1 = __builtin_amdgcn_exp2f(st[0] - now);
            r.m = now, l = fmaf(st[1], f1, l * f0), r.some |= st[2] != 0.f;
#pragma unroll
            for (int b = 0; b < S::NB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const f4 y = of[(4 * b + i) * 64 + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) r.o[b][4 * i + j] = fmaf(y[j], f1, r.o[b][4 * i + j] * f0);
              }
          }
        }
      }
      const bool whole = s0 == 0 && s1 == stages;
      if (z == 0 && live) {
        float *to;
        float by = 1.f;
        if (whole) {
          int head;
          const int64_t at = token_of(head);
          to = a.out + at * a.ld_out + (int64_t)head * a.c.dh;
          by = 1.f / l;
        } else {
          // a workgroup has at most one part that begins its block (place 1) and one that does not
          float *part = a.parts + (int64_t)(2 * p + (s0 == 0)) * kPart<DP, ROWS>;
          const int in = 32 * rw + c;
          if (hi == 0) part[in] = r.m, part[ROWS + in] = r.some ? l : -1.f;
          to = part + 2 * ROWS + in * DP;
        }
#pragma unroll
        for (int b = 0; b < S::NB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 32 * b + 8 * i + 4 * hi;
            if (d >= a.c.dh) continue;
            f4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = whole && !r.some ? 0.f : r.o[b][4 * i + j] * by;
            *reinterpret_cast<f4u *>(to + d) = y;
          }
      }
      if (tid == 0 && s0 == 0 && !whole)
        a.cuts[p] = {owner(first_unit + stages - 1) - p + 1, block * ROWS, min(ROWS, rows - block * ROWS), t.row0, kv * a.group};
      u += s1 - s0;
      x += s1 - s0, at += stages;
    }
  }
}

// The parts of blocks that were cut, added in order: a workgroup a row, 32 threads with four columns each in eight
// sets of every eighth part, whose loads go out eight at a time.
template <int DP, int ROWS>
__global__ void __launch_bounds__(256) join_parts(Args a) {
  constexpr int kAhead = 8;
  const Cut cut = a.cuts[blockIdx.x];
  const int tid = threadIdx.x, lane = tid & 63, set = tid >> 5, d = 4 * (tid & 31);
  __shared__ float tops[4], sums[8];
  __shared__ f4 outs[8][32];
  for (int r = blockIdx.y; cut.parts > 0 && r < cut.rows; r += gridDim.y) {
    // the first part is the owner's place 1, the others the next ones' places 0
    auto part = [&](int k) { return a.parts + (int64_t)(k == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + k)) * kPart<DP, ROWS>; };
    float m = kNever;
    for (int k = tid; k < cut.parts; k += 256) m = fmaxf(m, part(k)[r]);
    m = wave_max(m);
    if (lane == 0) tops[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    float l = -1.f;  // below 0: no token
    f4 o{};
    for (int k0 = set; k0 < cut.parts; k0 += 8 * kAhead) {
      float ms[kAhead], ls[kAhead];
      f4 y[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float *x = part(min(k0 + 8 * i, cut.parts - 1));  // past the last: read again, not added
        ms[i] = x[r], ls[i] = x[ROWS + r];
        y[i] = *reinterpret_cast<const f4 *>(x + 2 * ROWS + r * DP + min(d, DP - 4));
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (k0 + 8 * i >= cut.parts || ls[i] < 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(ms[i] - m);
        l = fmaf(ls[i], f, fmaxf(l, 0.f));
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(y[i][j], f, o[j]);
      }
    }
    if ((tid & 31) == 0) sums[set] = l;
    outs[set][tid & 31] = o;
    __syncthreads();
    if (set == 0 && d < a.c.dh) {
      bool some = false;
      l = 0.f, o = f4{};
      for (int i = 0; i < 8; ++i) {
        if (sums[i] < 0.f) continue;
        some = true, l += sums[i];
        const f4 y = outs[i][tid];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += y[j];
      }
      const int row = cut.row + r;
      *reinterpret_cast<f4u *>(a.out + (int64_t)(cut.row0 + row / a.group) * a.ld_out + (int64_t)(cut.head + row % a.group) * a.c.dh + d) =
          some ? o / l : f4{};
    }
    __syncthreads();
  }
}

}  // namespace chunk
