// New tokens of many sequences over a paged key-value cache, on the fp16 matrix cores at fp32 accuracy.
//
// The query rows of a kv head are the new tokens' heads of its group, token by token: row r of a sequence is head
// r % group of token r / group, so that a block of rows is full whatever the group, and all of it reads the cached
// tokens once.  As in packed_tiles.h a score is S^T = K Q^T and a result O^T += V^T P^T, with 32x32x16 products of
// two-term fp16 splits, h + m, three products each (m h, h m, h h); 8-bit codes are exact in fp16, one term, two
// products.  What the cache holds is split a stage of 64 tokens at a time:
//   fp32    tokens times a power of two that they share, the base, or one of their own where their size is far from it
//           (kBelow), which is then a factor of theirs;
//   8 bits  the codes less 128; the scale is the token's factor.
// A factor is applied to the token's scores, and to its probabilities before they are split: no token's size costs
// another its bits, and both formats are one walk.
//
// A workgroup has eight waves: R = 8 / Z of 32 rows, in Z sets with every Z-th 32 tokens of a stage each.  Z is 1 for
// many rows, where a stage that is read feeds twice as many products, and 2 for few.  Stages lie in LDS twice.  The next
// one's keys are asked for before this one's scores are formed and split after them, its values before the softmax
// and after the results.  Where many blocks of rows read the same tokens, pack_stages splits them once, into images of
// what a stage is in LDS, and a walk copies those: neither registers nor instructions are spent on them.
//
// The work is (kv head, block of rows, stage of tokens), in that order.  It is dealt evenly to one workgroup a CU,
// whatever the lengths, which only the device knows; a block that is cut leaves parts (m, l, O) that
// join_parts adds in order in a second launch: no workgroup waits for another.
//
// What bounds it, on MI355X: 8192 tokens over 6144 cached on the mean, 16 heads of 128 in groups of 8, fp32, take 1352
// us, 355 TFLOP/s of the formula's and so 1066 of the matrix cores' fp16, where a large library product in fp16 reaches
// 1085 to 1295: the power, at which the clock is 1.4 GHz.  Waves half a stage apart, scores formed beside the stage
// before's softmax, wave priorities and deeper prefetch gave nothing.  512 tokens over 8192, 32 heads in groups of 4:
// 251 us, 27 of it images, 14 joins.  16 tokens over 131072, one kv head: 70 to 77 us, 134 MB, 61 of it the walk.
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
// Units that a block counts beside its stages, for its queries, its first stage's wait and its results: without them the
// workgroups with many short blocks were the last.  None, 1, 2, 3 and 4 of them, us: five pieces of prompts beside 24
// single tokens over 8 bits 164, 139, 126, 129, 129; 2048 tokens each over 6144, 0, 16384 and 2000 1629, 1502, 1400,
// 1376, 1386; 512 over 8192 257, 254, 248, 247, 250; 100 each over 500, six times, 46, 37, 40, 39, 39; 16 over
// 131056, one block, 71, 72, 74, 73, 74 (2048 stages are 8 for each workgroup, 2051 are 9 for some).
constexpr int kTurn = 3;

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
  char *images;  // of stages, [n][kv_heads][most_stages]
  int most_stages;
  Cut *cuts;  // [workgroups]
  int64_t ld_q, ld_out;
  int n, group;
  float mant;  // log2(e) / sqrt(dh) is mant 2^exp, mant in [0.5, 1)
  int exp;
};

// Magnitudes within these bounds (or 0) cannot make a product leave fp32's range by themselves.  A workgroup's walk
// that meets a token or a query beyond them, one that is not finite, or a page that the cache lacks, is given up and
// made again in plain fp32, token by token (`take_plain`): some hundred times slower, and it does to each row
// what fp32 arithmetic does.  (Such a stage alone in that form, within the walk, cost the ordinary ones their
// registers.)
constexpr float kSmall = 0x1p-60f, kLarge = 0x1p60f;
__device__ __forceinline__ bool wild(float x) { return !(x == 0.f || (fabsf(x) >= kSmall && fabsf(x) <= kLarge)); }
// The larger; NaN if one is.
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A magnitude's exponent as its bits have it, 127 for [1, 2).  Tokens whose largest magnitude has one of base - kBelow
// to base + 1 are split at the base, the largest of the walk's first stage or an image's own, which brings that to
// [2^13, 2^14) (so theirs to [2^5, 2^15), and the split's smallest step to 2^-29 of it at most); others at their own,
// and have a factor.  Past kApart it is odd.
constexpr unsigned kLow = 127 - 60, kHigh = 127 + 60, kBelow = 8, kApart = 64, kScaled = 13;
__device__ __forceinline__ float power(unsigned bits) { return __builtin_bit_cast(float, bits << 23); }
// The base of what a first stage was raised to.  One of zeros only says nothing of those after it: from [1, 2) no
// size that is ordinary is past kApart.
__device__ __forceinline__ unsigned base_of(unsigned raised) { return raised == 0 ? 127 : raised; }
// What a stage's rows may be besides.
enum : int { kOdd = 1, kMixedKeys = 2, kMixedValues = 4 };

// Floats of a part: references and sums of a block's rows, then their outputs.
template <int DP, int ROWS>
constexpr int kPart = ROWS * (2 + DP);

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
  // steps whose queries' second terms lie in LDS: what registers lack for heads above 96
  static constexpr int kKept = DP > 96 ? 3 : 0;
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

// A stage's bases, marks and factors, the last kilobyte of its image where it has one.
struct Head {
  unsigned base[2];  // of keys and of values
  int marks, none[61];
  float ks[kStage], vs[kStage];
  char rest[256];
};
static_assert(sizeof(Head) == 1024);
template <int DP>
constexpr int kImage = Shape<false, DP>::kBytes + (int)sizeof(Head);

// What a workgroup shares.
template <bool INT8, int DP>
struct Lds {
  using S = Shape<INT8, DP>;
  static constexpr int kJoint = 64 * (16 * S::NB + 4) * 4;  // a wave's results, while sets are joined
  // (the stages last: an LDS access has 16 bits for a constant offset)
  Head heads[2] __attribute__((aligned(256)));
  int marks[3];      // of three stages in turn: one is read, one written, one cleared
  unsigned base[2];  // the walk's, of keys and of values
  char kept[8][S::kKept > 0 ? S::kKept : 1][1024] __attribute__((aligned(256)));  // of each wave's queries
  char stages[2 * S::kBytes > 4 * kJoint ? 2 * S::kBytes : 4 * kJoint] __attribute__((aligned(256)));
  __device__ __forceinline__ char *stage(int buf) { return stages + buf * S::kBytes; }
};

// The same value, formed again: what follows from it is not kept in registers around a loop.
__device__ __forceinline__ int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ int again_scalar(int v) {
  asm volatile("" : "+s"(v));
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

// A thread's share of a stage on its way from the cache to LDS.  BOTH: keys and values are asked for at once, else
// one after the other.
template <bool INT8, int DP, bool BOTH>
struct Staging {
  using S = Shape<INT8, DP>;
  // places whose pages it needs: rows; in 8 bits also quads of values, a factor
  static constexpr int NE = INT8 ? S::NP + S::NV + 1 : S::NP;
  int32_t entries[NE];  // the places' pages, -1: the cache has none
  bool whole;      // of the wave's places all are, and all of its columns the head's
  f4 x[INT8 ? 1 : BOTH ? 2 : 1][INT8 ? 1 : S::NP][2];
  u2 kc[INT8 ? S::NP : 1];
  u4 vc[INT8 ? S::NV : 1];
  float scale;

  // The token of a place within its stage.
  static __device__ __forceinline__ int token(int tid, int i) {
    if (i < S::NP) return i * S::kPass + (tid >> S::kLanes);  // (past the stage where it has fewer rows than threads)
    if (i < NE - 1) return min(((i - S::NP) * kThreads + tid) / (DP / 4), kStage / 4 - 1) * 4;
    return tid & (kStage - 1);
  }
  static __device__ __forceinline__ int row_column(int tid) { return 8 * (tid & (S::kPieces - 1)); }
  static __device__ __forceinline__ int quad_column(int tid, int i) { return 4 * ((i * kThreads + tid) % (DP / 4)); }
  __device__ __forceinline__ void look(const Cache &c, const Walk &w, int stage) {
    const int tid = again(threadIdx.x);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int pos = stage * kStage + token(tid, i);
      entries[i] = pos < w.held ? paging::entry_of(w.pages, c.max_pages, c.shift, pos) : -1;
    }
  }
  // Loads go out whatever the place is, from the cache's first page where it is none, and are dropped then: what
  // lies in slots of no token must not reach the products.
  __device__ __forceinline__ void resolve(const Cache &c) {
    const int tid = again(threadIdx.x);
    bool all = row_column(tid) < c.dh;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      entries[i] = paging::page_in(entries[i], c.pages);
      all &= entries[i] >= 0;
    }
    whole = __all(all);
  }
  // The element that a place's load begins at, of a factor its place.
  __device__ __forceinline__ int64_t at(const Cache &c, const Walk &w, int stage, int i) const {
    const int tid = again(threadIdx.x);
    // (page * kv_heads + kv) * page size + slot: a factor of 32 bits, so one multiplication
    const uint32_t slot = (uint32_t)(stage * kStage + token(tid, i)) & ((1u << c.shift) - 1);
    const uint64_t row = (uint64_t)(uint32_t)max(entries[i], 0) * ((uint32_t)c.kv_heads << c.shift) +
                         (((uint32_t)w.kv << c.shift) + slot);
    if (INT8 && i == NE - 1) return (int64_t)row;
    return (int64_t)(row * (uint32_t)c.dh + (uint32_t)(i < S::NP ? min(row_column(tid), c.dh - 8) : 4 * min(quad_column(tid, i - S::NP), c.dh - 4)));
  }
  // fp32 rows of keys or values: a thread's eight columns.
  __device__ __forceinline__ void load_rows(const Cache &c, const Walk &w, int stage, const void *from, int which) {
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const float *p = static_cast<const float *>(from) + at(c, w, stage, i);
      x[which][i][0] = *reinterpret_cast<const f4 *>(p), x[which][i][1] = *reinterpret_cast<const f4 *>(p + 4);
    }
  }
  __device__ __forceinline__ void load_keys(const Cache &c, const Walk &w, int stage) {
    if constexpr (!INT8) {
      load_rows(c, w, stage, c.k, 0);
    } else {
#pragma unroll
      for (int i = 0; i < S::NP; ++i)
        kc[i] = *reinterpret_cast<const u2 *>(static_cast<const uint8_t *>(c.k) + at(c, w, stage, i));
      scale = (threadIdx.x & kStage ? c.vs : c.ks)[at(c, w, stage, NE - 1)];
    }
  }
  __device__ __forceinline__ void load_values(const Cache &c, const Walk &w, int stage) {
    if constexpr (!INT8) {
      load_rows(c, w, stage, c.v, BOTH);
    } else {
#pragma unroll
      for (int i = 0; i < S::NV; ++i)
        vc[i] = *reinterpret_cast<const u4 *>(static_cast<const uint8_t *>(c.v) + at(c, w, stage, S::NP + i));
    }
  }
  // What lies in no token's slot, and past the head, becomes zeros.
  template <bool VALUES>
  __device__ __forceinline__ void drop(const Cache &c, const Walk &w, int stage) {
    if (whole) return;
    const int tid = again(threadIdx.x);
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const bool in = stage * kStage + token(tid, i) < w.held && row_column(tid) < c.dh;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[BOTH && VALUES][i][j >> 2][j & 3] = in ? x[BOTH && VALUES][i][j >> 2][j & 3] : 0.f;
    }
  }
  // The bits of a row's largest magnitude, in all of its lanes.
  template <bool VALUES>
  __device__ __forceinline__ unsigned top_of_row(int i) const {
    const f4(&v)[2] = x[BOTH && VALUES][i];
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) big = maximum(maximum(big, fabsf(v[j >> 2][j & 3])), fabsf(v[j >> 2][(j & 3) + 1]));
    return row_top<S::kLanes>(__builtin_bit_cast(unsigned, big));
  }
  // Raises the walk's base to the largest exponent of these rows; rows of zeros leave it at 0 (see base_of).
  template <bool VALUES>
  __device__ __forceinline__ void raise_base(unsigned (&base)[2], const Cache &c, const Walk &w, int stage) {
    if constexpr (!INT8) {
      drop<VALUES>(c, w, stage);
      unsigned e = 0;
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const unsigned top = top_of_row<VALUES>(i);
        if (top != 0) e = max(e, min(max(top >> 23, kLow), kHigh));
      }
      atomicMax(&base[VALUES], e);
    }
  }

  // Rows in fp32 into two terms; returns their marks.
  template <bool VALUES>
  __device__ __forceinline__ int split_rows(const Cache &c, const Walk &w, int stage, char *to, float *factors, unsigned base) {
    const int tid = again(threadIdx.x);
    const int piece = tid & (S::kPieces - 1);
    bool odd = false, mixed = false;
    drop<VALUES>(c, w, stage);
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const int tk = token(tid, i);
      const unsigned top = top_of_row<VALUES>(i), e = top >> 23;
      const bool near = e - (base - kBelow) <= kBelow + 1 || top == 0;
      odd |= !near && (e < kLow || e >= kHigh || e - (base - kApart) > 2 * kApart);
      mixed |= !near;
      const unsigned own = near ? base : e;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[BOTH && VALUES][i][j >> 2][j & 3];
      const Terms t = tiles::split8(v, power(kScaled + 2 * 127 - own));
      if (S::kPass <= kStage || tk < kStage) {
        char *p = to + (VALUES ? S::value_place(tk, piece) : S::key_place(tk, piece));
        *reinterpret_cast<h8 *>(p) = t.h;
        *reinterpret_cast<h8 *>(p + kStage * S::kRow) = t.m;
        if (piece == 0) factors[tk] = power(127 + own - base);
      }
    }
    return (odd ? kOdd : 0) | (mixed ? VALUES ? kMixedValues : kMixedKeys : 0);
  }
  static __device__ __forceinline__ void mark(int *to, int marks) {
    if (marks != 0) atomicOr(to, marks);
  }

  // Marks of tokens of the sequence on pages that the cache lacks.
  __device__ __forceinline__ int lacking(const Walk &w, int stage) const {
    const int tid = again(threadIdx.x);
    int marks = 0;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < S::NP; ++i)
        if (entries[i] < 0 && stage * kStage + token(tid, i) < w.held) marks |= kOdd;
    }
    return marks;
  }
  // stage: the one that is written, of the block's walk, and its buffers.
  __device__ __forceinline__ void put_keys(Lds<INT8, DP> &s, const Cache &c, const Walk &w, int stage, int buf, int third,
                                           unsigned base) {
    const int tid = again(threadIdx.x);
    char *to = s.stage(buf);
    int marks = 0;
    if constexpr (!INT8) {
      marks = split_rows<false>(c, w, stage, to, s.heads[buf].ks, base);
    } else {
      const int piece = tid & (S::kPieces - 1);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int tk = token(tid, i);
        u4 h;
        unsigned lo, hi;
        paged::halves(kc[i][0], lo, hi), h[0] = lo, h[1] = hi;
        paged::halves(kc[i][1], lo, hi), h[2] = lo, h[3] = hi;
        if (S::kPass <= kStage || tk < kStage) *reinterpret_cast<u4 *>(to + S::key_place(tk, piece)) = h;
      }
      const float y = entries[NE - 1] >= 0 ? scale : 0.f;
      if (threadIdx.x < 2 * kStage) {
        (threadIdx.x < kStage ? s.heads[buf].ks : s.heads[buf].vs)[threadIdx.x & (kStage - 1)] = y;
        if (wild(y)) marks = kOdd;
      }
    }
    mark(&s.marks[third], marks | lacking(w, stage));
  }
  __device__ __forceinline__ void put_values(Lds<INT8, DP> &s, const Cache &c, const Walk &w, int stage, int buf, int third,
                                             unsigned base) {
    char *to = s.stage(buf) + S::kKeys;
    if constexpr (!INT8) {
      mark(&s.marks[third], split_rows<true>(c, w, stage, to, s.heads[buf].vs, base));
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
__device__ __forceinline__ h8 values_term(const char *p, int off, int st, int b, int term) {
  using S = Shape<INT8, DP>;
  if constexpr (INT8) {
    const char *at = p + off + (4 * st * DP + 32 * b) * 8;
    const u2 lo = *reinterpret_cast<const u2 *>(at), hi = *reinterpret_cast<const u2 *>(at + 2 * DP * 8);
    return __builtin_bit_cast(h8, u4{lo[0], lo[1], hi[0], hi[1]});
  } else {
    const char *at = p + (off ^ 64 * b) + 16 * st * S::kRow + term * kStage * S::kRow;
    const auto a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tiles::lds_s4 *)at);
    const auto b4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tiles::lds_s4 *)(at + 8 * S::kRow));
    return __builtin_bit_cast(h8, tiles::s8(__builtin_shufflevector(a, b4, 0, 1, 2, 3, 4, 5, 6, 7)));
  }
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
  int fe;       // log2(e) / sqrt(dh) over the query's factor is a power of two, this one
  float f;      // and with the keys' base

  __device__ __forceinline__ void clear() {
    m = kNever, l = 0.f;
#pragma unroll
    for (int b = 0; b < S::NB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] = 0.f;
  }
  static __device__ __forceinline__ char *kept(Lds<INT8, DP> &lds, int st) {
    const int tid = again(threadIdx.x);
    return lds.kept[tid >> 6][st - (S::NS - S::kKept)] + (tid & 63) * 16;
  }
  // Returns whether the row's query is ordinary.
  __device__ __forceinline__ bool start(const Args &a, Lds<INT8, DP> &lds, const float *row, bool live) {
    const int hi = (threadIdx.x & 63) >> 5;
    tiles::RowValues<DP> x;
    x.load(row, live, again_scalar(a.c.dh), hi);
    bool not_finite = false;
    const float top = x.top(INFINITY, not_finite);
    const int e = tiles::exponent_for(top);
    fe = a.exp - e;
    x.split_into(q, __builtin_amdgcn_ldexpf(a.mant, e));
#pragma unroll
    for (int st = S::NS - S::kKept; st < S::NS; ++st) *reinterpret_cast<h8 *>(kept(lds, st)) = q[st].m;
    clear();
    return !(not_finite || wild(top));
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

  // KB blocks of 32 tokens from `first` of a stage: the products of their keys ...
  template <int KB>
  __device__ __forceinline__ void products(Lds<INT8, DP> &lds, int buf, int first, f16 (&s)[KB]) const {
    const int lane = again(threadIdx.x & 63), off = again(S::key_place(first + (lane & 31), lane >> 5));
    const char *keys = lds.stage(buf);
    auto ask = [&](int n) {  // of step n / KB, block n % KB
      const char *p = keys + (off ^ 32 * (n / KB)) + n % KB * 32 * S::kRow;
      Terms k;
      k.h = *reinterpret_cast<const h8 *>(p);
      if constexpr (!INT8) k.m = *reinterpret_cast<const h8 *>(p + kStage * S::kRow);
      return k;
    };
    auto query = [&](int st) {
      Terms t = q[st];
      if (st >= S::NS - S::kKept) t.m = *reinterpret_cast<const h8 *>(kept(lds, st));
      return t;
    };
    constexpr int kAll = S::NS * KB;
    Terms k = ask(0), now = query(0);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = f16{};
#pragma unroll
    for (int n = 0; n < kAll; ++n) {
      Terms next;
      if (n + 1 < kAll) next = ask(n + 1);
      __builtin_amdgcn_sched_barrier(0);  // the next step's operands are asked for before this one's products
      mma_keys<INT8>(s[n % KB], k, now);
      k = next;
      if (n % KB == KB - 1 && n + 1 < kAll) now = query(n / KB + 1);
    }
  }

  // ... and what follows from them; the stage's tokens begin at pos0.
  // seen(): the tokens that the lane's row sees.
  template <int KB, class Seen>
  __device__ __forceinline__ void take(Lds<INT8, DP> &lds, int buf, int first, int pos0, bool masked, int marks,
                                       int values_base, f16 (&s)[KB], Seen &&seen) {
    const int hi = again(threadIdx.x & 63) >> 5;
    const char *values = lds.stage(buf) + S::kKeys;
    // factors of the rows that a lane's results are, four at a time
    auto by_factors = [&](const float *factors) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f4 x = *reinterpret_cast<const f4 *>(factors + first + 32 * kb + 8 * i + 4 * hi);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[kb][4 * i + j] *= x[j];
        }
    };
    if (INT8 || (marks & kMixedKeys)) by_factors(lds.heads[buf].ks);
    if (masked) {
      const int left = seen() - pos0 - first;  // tokens from the first that the row sees
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * kb + tiles::out_row(e, hi) >= left) s[kb][e] = -INFINITY;
    }
    float most = s[0][0];
#pragma unroll
    for (int n = 1; n + 1 < 16 * KB; n += 2) most = maximum(maximum(most, s[n / 16][n % 16]), s[(n + 1) / 16][(n + 1) % 16]);
    most = maximum(most, s[KB - 1][15]);
    most = half_pair(most, [](float x, float y) { return maximum(x, y); }) * f;
    if (__any(most > m + 8.f)) raise(fmaxf(m, most));
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[kb][e] = __builtin_amdgcn_exp2f(fmaf(s[kb][e], f, -m));
        sums[e & 1] += s[kb][e];
      }
    l += sums[0] + sums[1];
    // the probabilities times the values' factors, the largest of a row brought to [2^14, 2^15)
    float top;
    if (INT8 || (marks & kMixedValues)) {
      by_factors(lds.heads[buf].vs);
      top = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) top = tiles::top_of(s[kb], top);
      top = half_pair(top, [](float x, float y) { return fmaxf(x, y); });
    } else {
      top = __builtin_amdgcn_exp2f(most - m);
    }
    const int et = max(__builtin_amdgcn_frexp_expf(top), -100);
    const float lift = __builtin_amdgcn_ldexpf(1.f, 15 - et), back = __builtin_amdgcn_ldexpf(1.f, et - 15 + values_base);
    Terms p[KB][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = s[kb][e];
      p[kb][0] = tiles::split8(x, lift), p[kb][1] = tiles::split8(x + 8, lift);
    }
    const int off = again(values_place<INT8, DP>(first, again(threadIdx.x & 63)));
    constexpr int kSteps = 2 * KB;  // of 16 tokens
    h8 h = values_term<INT8, DP>(values, off, 0, 0, 0);
#pragma unroll
    for (int b = 0; b < S::NB; ++b) {
      f16 z = {};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const int nb = st + 1 < kSteps ? b : b + 1, ns = (st + 1) % kSteps;
        const Terms &w = p[st >> 1][st & 1];
        h8 low, next;
        if constexpr (!INT8) low = values_term<INT8, DP>(values, off, st, b, 1);
        if (nb < S::NB) next = values_term<INT8, DP>(values, off, ns, nb, 0);
        __builtin_amdgcn_sched_barrier(0);
        z = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, w.m, z, 0, 0, 0);
        if constexpr (!INT8) z = __builtin_amdgcn_mfma_f32_32x32x16_f16(low, w.h, z, 0, 0, 0);
        z = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, w.h, z, 0, 0, 0);
        h = next;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] = fmaf(z[e], back, o[b][e]);
    }
  }

  // The same in plain fp32, a token after the other: a lane forms half of its row's score, and adds to its columns
  // of the result.  What is not finite does what it does in fp32, and only to the rows that see it.
  // Returns whether the row sees any of them.
  __device__ __forceinline__ bool take_plain(const Args &a, const Walk &w, const float *row, int seen, int from, int to) {
    bool some = false;
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
    return some;
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

// The images of the stages that the walks will take: split once for all blocks of rows.  A workgroup a stage.
template <int DP>
__global__ void __launch_bounds__(kThreads) pack_stages(Args a) {
  using S = Shape<false, DP>;
  __shared__ unsigned base[2];
  __shared__ int marks;
  const int tid = threadIdx.x, i = (int)(blockIdx.x / a.most_stages), stage = (int)(blockIdx.x % a.most_stages), kv = i % a.c.kv_heads;
  const SeqTile t = a.seqs[i / a.c.kv_heads];
  const int end = __builtin_amdgcn_readfirstlane(a.ends[t.seq]);
  const Walk walk{a.c.table + (int64_t)t.seq * a.c.max_pages, (int)paging::held(end, a.c.max_pages, a.c.shift), kv};
  if (stage > 0 && stage * kStage >= walk.held) return;
  Staging<false, DP, true> g;
  g.look(a.c, walk, stage);
  if (tid < 2) base[tid] = 0;
  if (tid == 2) marks = 0;
  g.resolve(a.c);
  g.load_keys(a.c, walk, stage);
  g.load_values(a.c, walk, stage);
  __syncthreads();
  g.template raise_base<false>(base, a.c, walk, stage);
  g.template raise_base<true>(base, a.c, walk, stage);
  __syncthreads();
  char *image = a.images + (int64_t)blockIdx.x * kImage<DP>;
  Head *head = reinterpret_cast<Head *>(image + S::kBytes);
  const unsigned kbase = base_of(base[0]), vbase = base_of(base[1]);
  int found = g.template split_rows<false>(a.c, walk, stage, image, head->ks, kbase);
  found |= g.template split_rows<true>(a.c, walk, stage, image + S::kKeys, head->vs, vbase);
  g.mark(&marks, found | g.lacking(walk, stage));
  __syncthreads();
  if (tid == 0) head->base[0] = kbase, head->base[1] = vbase, head->marks = marks;
}

// PACKED: the stages are images already.
template <bool INT8, int DP, int Z, bool PACKED>
__global__ void __launch_bounds__(kThreads, 2) walk_blocks(Args a) {
  using S = Shape<INT8, DP>;
  constexpr int R = 8 / Z, ROWS = 32 * R, KB = 2 / Z;
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
      for (int b = 0; b < blocks; ++b) v += kTurn + stages_of<ROWS>(a.c, a.group, t.len, end, b);
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
      if (x < at + kTurn + stages) break;
      at += kTurn + stages;
    }
    for (; u < end_unit && block * ROWS < rows; ++block) {
      stages = stages_of<ROWS>(a.c, a.group, t.len, end, block);
      const int u0 = (int)(x - at), u1 = (int)min((int64_t)(kTurn + stages), u0 + (end_unit - u));
      const int64_t first_unit = u - u0;  // of the block
      u += u1 - u0, x += u1 - u0, at += kTurn + stages;
      const int s0 = max(0, u0 - kTurn), s1 = u1 - kTurn;
      if (s0 >= s1) continue;

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
      auto row_sees = [&] { return live ? sees(t.len, end, walk.held, again(row) / a.group) : 0; };
      const int n_seen = row_sees();
      const int live_rows = min(32, rows - block * ROWS - 32 * rw);
      const int least = live_rows < 32 ? 0 : __builtin_amdgcn_readlane(n_seen, 0);
      const int most = live_rows > 0 ? __builtin_amdgcn_readlane(n_seen, live_rows - 1) : 0;
      constexpr bool kBoth = INT8 || Z > 1;
      Staging<INT8, DP, kBoth> g;
      Rows<INT8, DP> r;
      // A stage's image on its way to LDS.
      auto fetch = [&](int stage, int buf) {
        const char *from = a.images + ((int64_t)((i0 + j) * a.c.kv_heads + kv) * a.most_stages + stage) * kImage<DP> + lane * 16;
#pragma unroll
        for (int k = 0; k < S::kBytes / 8192; ++k) tiles::copy16(from + (k * 8 + w) * 1024, lds.stage(buf) + (k * 8 + w) * 1024);
        if (w == 0) tiles::copy16(from + S::kBytes, &lds.heads[buf]);
      };
      unsigned kbase = 0, vbase = 0;
      if constexpr (PACKED) {
        __syncthreads();  // the last block's buffers are free
        if (tid == 0) lds.marks[0] = 0;
        fetch(s0, 0);
        const bool good = r.start(a, lds, query(), live);
        __syncthreads();
        if (!good) g.mark(&lds.marks[0], kOdd);
      } else {
        g.look(a.c, walk, s0);
        if (tid < 3) lds.marks[tid] = 0;
        if (tid < 2) lds.base[tid] = 0;
        const bool good = r.start(a, lds, query(), live);
        g.resolve(a.c);
        __syncthreads();  // what is marked is cleared, the last block's buffers free
        if (!good) Staging<INT8, DP, kBoth>::mark(&lds.marks[0], kOdd);
        g.load_keys(a.c, walk, s0);
        if constexpr (kBoth) g.load_values(a.c, walk, s0);
        g.template raise_base<false>(lds.base, a.c, walk, s0);
        if constexpr (kBoth) g.template raise_base<true>(lds.base, a.c, walk, s0);
        if constexpr (!INT8) __syncthreads();
        kbase = base_of(__builtin_amdgcn_readfirstlane(lds.base[0]));
        g.put_keys(lds, a.c, walk, s0, 0, 0, kbase);
        if constexpr (!kBoth) {
          g.load_values(a.c, walk, s0);
          g.template raise_base<true>(lds.base, a.c, walk, s0);
          __syncthreads();
        }
        vbase = base_of(__builtin_amdgcn_readfirstlane(lds.base[1]));
        g.put_values(lds, a.c, walk, s0, 0, 0, vbase);
        g.look(a.c, walk, s0 + 1);
      }
      constexpr int kUnscale = INT8 ? 0 : 127 + (int)kScaled;
      auto based = [&] { r.f = __builtin_amdgcn_ldexpf(1.f, r.fe + (INT8 ? 0 : (int)kbase - kUnscale)); };
      based();
      bool odd = false;
      for (int i = s0; i < s1; ++i) {
        const int buf = (i - s0) & 1, third = (i - s0) % 3, after = (i - s0 + 1) % 3;
        const int pos0 = i * kStage, first = 32 * z;
        const bool more = i + 1 < s1;
        if constexpr (PACKED)
          tiles::fetched();
        else
          __syncthreads();
        const int marks = __builtin_amdgcn_readfirstlane(PACKED ? lds.marks[0] | lds.heads[buf].marks : lds.marks[third]);
        odd = (marks & kOdd) != 0;
        if (odd) break;
        if constexpr (PACKED) {
          if (more) fetch(i + 1, buf ^ 1);
          kbase = __builtin_amdgcn_readfirstlane(lds.heads[buf].base[0]);
          vbase = __builtin_amdgcn_readfirstlane(lds.heads[buf].base[1]);
          based();
        } else if (tid == 0) {
          lds.marks[(i - s0 + 2) % 3] = 0;
        }
        const int values_base = INT8 ? 0 : (int)vbase - kUnscale;
        if (!PACKED && more) {
          g.resolve(a.c);
          g.load_keys(a.c, walk, i + 1);
          if constexpr (kBoth) g.load_values(a.c, walk, i + 1);
        }
        const bool mine = pos0 + first < most;
        f16 s[KB];
        if (mine) r.template products<KB>(lds, buf, first, s);
        if (!PACKED && more) {
          g.put_keys(lds, a.c, walk, i + 1, buf ^ 1, after, kbase);
          if constexpr (!kBoth) g.load_values(a.c, walk, i + 1);
          g.look(a.c, walk, i + 2);
        }
        if (mine) r.template take<KB>(lds, buf, first, pos0, pos0 + first + 32 * KB > least, marks, values_base, s, row_sees);
        if (!PACKED && more) g.put_values(lds, a.c, walk, i + 1, buf ^ 1, after, vbase);
      }
      bool some = row_sees() > s0 * kStage + 32 * z;  // whether the row sees a token of the wave's
      if (odd) {
        r.clear();
        some = false;
        const float *row = query();
        for (int pos = s0 * kStage + 32 * z; pos < min(s1 * kStage, most); pos += 32 * Z)
          some |= r.take_plain(a, walk, row, row_sees(), pos, min(pos + 32, most));
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
          to[4 * S::NB * 64 + lane] = f4{r.m, l, some ? 1.f : 0.f, 0.f};
        }
        __syncthreads();
        if (z == 0) {
#pragma unroll
          for (int k = 1; k < Z; ++k) {
            const f4 *of = reinterpret_cast<const f4 *>(joint + ((k - 1) * R + rw) * kEach);
            const f4 st = of[4 * S::NB * 64 + lane];
            const float now = fmaxf(r.m, st[0]), f0 = __builtin_amdgcn_exp2f(r.m - now), f1 = __builtin_amdgcn_exp2f(st[0] - now);
            r.m = now, l = fmaf(st[1], f1, l * f0), some |= st[2] != 0.f;
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
      const int dh = again_scalar(a.c.dh), lane_half = again(lane) >> 5;
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
          if (hi == 0) part[in] = r.m, part[ROWS + in] = some ? l : -1.f;
          to = part + 2 * ROWS + in * DP;
        }
#pragma unroll
        for (int b = 0; b < S::NB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 32 * b + 8 * i + 4 * lane_half;
            if (d >= dh) continue;
            f4 y;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = whole && !some ? 0.f : r.o[b][4 * i + j] * by;
            *reinterpret_cast<f4u *>(to + d) = y;
          }
      }
      if (tid == 0 && s0 == 0 && !whole)
        a.cuts[p] = {owner(first_unit + kTurn + stages - 1) - p + 1, block * ROWS, min(ROWS, rows - block * ROWS), t.row0, kv * a.group};
    }
  }
}

// The parts of blocks that were cut, added in order.  Every workgroup lists the cut blocks' rows; a row of up to
// kFew parts goes to a wave, its halves every other part, a row of more to a workgroup, 32 threads with four columns
// each in eight sets of every eighth part.  Loads go out eight parts at a time.
constexpr int kFew = 32;

template <int DP, int ROWS>
__global__ void __launch_bounds__(256) join_parts(Args a, int wgs) {
  constexpr int kAhead = 8;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  __shared__ int rows[2][257], sums[2][4];
  __shared__ float tops[4], ls[8];
  __shared__ f4 outs[8][32];
  auto part = [&](int p, int k) {  // the first part is its workgroup's place 1, the others the next ones' places 0
    return a.parts + (int64_t)(k == 0 ? 2 * p + 1 : 2 * (p + k)) * kPart<DP, ROWS>;
  };
  auto put = [&](const Cut &cut, int r, int d, bool some, f4 o, float l) {
    const int row = cut.row + r;
    if (d < a.c.dh)
      *reinterpret_cast<f4u *>(a.out + (int64_t)(cut.row0 + row / a.group) * a.ld_out + (int64_t)(cut.head + row % a.group) * a.c.dh + d) =
          some ? o / l : f4{};
  };
  for (int p0 = 0; p0 < wgs; p0 += 256) {
    // rows before each cut block, of few parts and of many
    const Cut mine = p0 + tid < wgs ? a.cuts[p0 + tid] : Cut{};
    int v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[k] = mine.parts > 0 && (mine.parts > kFew) == (k == 1) ? mine.rows : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int below = __shfl_up(v[k], d);
        if (lane >= d) v[k] += below;
      }
      if (lane == 63) sums[k][w] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      for (int i = 0; i < w; ++i) v[k] += sums[k][i];
      rows[k][tid + 1] = v[k];
      if (tid == 0) rows[k][0] = 0;
    }
    __syncthreads();
    auto find = [&](int k, int row) {  // the cut block that has it
      int lo = 0, hi = 256;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (rows[k][mid] <= row ? lo : hi) = mid;
      }
      return lo;
    };
    // a wave's rows follow each other: the block is looked up once
    const int waves = gridDim.x * 4, share = (rows[0][256] + waves - 1) / waves;
    const int i0 = min((int)(blockIdx.x * 4 + w) * share, rows[0][256]), i1 = min(i0 + share, rows[0][256]);
    int at = i0 < i1 ? __builtin_amdgcn_readfirstlane(find(0, i0)) : 0;
    for (int i = i0; i < i1; ++i) {
      while (rows[0][at + 1] <= i) ++at;
      const int p = p0 + at, r = i - rows[0][at], half = lane >> 5, d = 4 * (lane & 31);
      const Cut cut = a.cuts[p];
      f4 y[kAhead / 2];
      auto ask = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kAhead / 2; ++k)  // past the last: read again, not added
          y[k] = *reinterpret_cast<const f4 *>(part(p, min(k0 + 2 * k + half, cut.parts - 1)) + 2 * ROWS + r * DP + min(d, DP - 4));
      };
      float m = kNever, l = -1.f;
      if (lane < cut.parts) m = part(p, lane)[r], l = part(p, lane)[ROWS + r];
      ask(0);
      // (a part without a token has the factor -1: only such a part is left out, since 0 times what is not finite is NaN)
      const float top = wave_max(l < 0.f ? kNever : m), f = l < 0.f ? -1.f : __builtin_amdgcn_exp2f(m - top);
      const bool some = __any(!(l < 0.f));  // (NaN too)
      f4 o{};
      for (int k0 = 0; k0 < cut.parts; k0 += kAhead) {
        if (k0 > 0) ask(k0);
#pragma unroll
        for (int k = 0; k < kAhead / 2; ++k) {
          const float by = __shfl(f, k0 + 2 * k + half);
          if (k0 + 2 * k + half >= cut.parts || by < 0.f) continue;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = fmaf(y[k][j], by, o[j]);
        }
      }
      auto add = [](float x, float y) { return x + y; };
      l = wave_sum(l < 0.f ? 0.f : l * f);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = half_pair(o[j], add);
      if (half == 0) put(cut, r, d, some, o, l);
    }
    for (int i = blockIdx.x; i < rows[1][256]; i += gridDim.x) {
      const int at = find(1, i), p = p0 + at, r = i - rows[1][at], set = tid >> 5, d = 4 * (tid & 31);
      const Cut cut = a.cuts[p];
      float m = kNever;
      for (int k = tid; k < cut.parts; k += 256) m = fmaxf(m, part(p, k)[r]);
      m = wave_max(m);
      if (lane == 0) tops[w] = m;
      __syncthreads();
      m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      float l = -1.f;  // below 0: no token
      f4 o{};
      for (int k0 = set; k0 < cut.parts; k0 += 8 * kAhead) {
        float mk[kAhead], lk[kAhead];
        f4 y[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const float *x = part(p, min(k0 + 8 * k, cut.parts - 1));
          mk[k] = x[r], lk[k] = x[ROWS + r];
          y[k] = *reinterpret_cast<const f4 *>(x + 2 * ROWS + r * DP + min(d, DP - 4));
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (k0 + 8 * k >= cut.parts || lk[k] < 0.f) continue;
          const float f = __builtin_amdgcn_exp2f(mk[k] - m);
          l = fmaf(lk[k], f, fmaxf(l, 0.f));
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = fmaf(y[k][j], f, o[j]);
        }
      }
      if ((tid & 31) == 0) ls[set] = l;
      outs[set][tid & 31] = o;
      __syncthreads();
      if (set == 0) {
        bool some = false;
        l = 0.f, o = f4{};
        for (int k = 0; k < 8; ++k) {
          if (ls[k] < 0.f) continue;
          some = true, l += ls[k];
          const f4 y = outs[k][tid];
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] += y[j];
        }
        put(cut, r, d, some, o, l);
      }
      __syncthreads();
    }
    __syncthreads();
  }
}

}  // namespace chunk
