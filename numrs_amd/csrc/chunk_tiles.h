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

// Rows of a stage whose factors or positions are out of the ordinary: such a stage takes a longer form.
enum : int { kWild = 1, kOddKey = 2, kOddValue = 4, kMissing = 8 };
// Factors within these bounds, and queries likewise, cannot make a product leave fp32's range by themselves.
constexpr float kSmall = 0x1p-60f, kLarge = 0x1p60f;
__device__ __forceinline__ bool wild(float x) { return !(x == 0.f || (fabsf(x) >= kSmall && fabsf(x) <= kLarge)); }
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
  char stages[2 * S::kBytes > 4 * kJoint ? 2 * S::kBytes : 4 * kJoint];
  __device__ __forceinline__ char *stage(int buf) { return stages + buf * S::kBytes; }
  float ks[2][kStage], vs[2][kStage];  // the rows' factors
  int flags[3];                        // of three stages in turn: one is read, one written, one cleared
  mask64 odd_key[3], odd_value[3], missing[3];
};

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
  int pages[NE];
  f4 x[INT8 ? 1 : S::NP][2];
  u2 kc[INT8 ? S::NP : 1];
  u4 vc[INT8 ? S::NV : 1];
  float scale;

  // The token of a place within its stage: a row's, a quad's first, or a factor's.
  static __device__ __forceinline__ int token(int i) {
    const int tid = threadIdx.x;
    if (i < S::NP) return i * S::kPass + (tid >> S::kLanes);
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
  __device__ __forceinline__ void resolve(const Cache &c) {
#pragma unroll
    for (int i = 0; i < NE; ++i) pages[i] = paging::page_in(entries[i], c.pages);
  }

  // fp32 rows of keys or values: a thread's eight columns.
  __device__ __forceinline__ void load_rows(const Cache &c, const Walk &w, int stage, const void *from) {
    const int col = 8 * (threadIdx.x & (S::kPieces - 1));
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      x[i][0] = x[i][1] = f4{};
      const int tk = token(i);
      if (pages[i] < 0 || col >= c.dh || tk >= kStage) continue;
      const float *p = static_cast<const float *>(from) + token_row(c, w.kv, stage * kStage + tk, pages[i]) * c.dh + col;
      x[i][0] = *reinterpret_cast<const f4 *>(p), x[i][1] = *reinterpret_cast<const f4 *>(p + 4);
    }
  }
  __device__ __forceinline__ void load_keys(const Cache &c, const Walk &w, int stage) {
    if constexpr (!INT8) {
      load_rows(c, w, stage, c.k);
    } else {
      const int col = 8 * (threadIdx.x & (S::kPieces - 1));
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int tk = token(i);
        kc[i] = u2{0x80808080u, 0x80808080u};
        if (pages[i] < 0 || col >= c.dh || tk >= kStage) continue;
        kc[i] = *reinterpret_cast<const u2 *>(static_cast<const uint8_t *>(c.k) +
                                              token_row(c, w.kv, stage * kStage + tk, pages[i]) * c.dh + col);
      }
      scale = 0.f;
      const int page = pages[NE - 1], pos = stage * kStage + token(NE - 1);
      if (threadIdx.x < 2 * kStage && page >= 0) scale = (threadIdx.x < kStage ? c.ks : c.vs)[token_row(c, w.kv, pos, page)];
    }
  }
  __device__ __forceinline__ void load_values(const Cache &c, const Walk &w, int stage) {
    if constexpr (!INT8) {
      load_rows(c, w, stage, c.v);
    } else {
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        const int u = i * kThreads + threadIdx.x, col = 4 * (u % (DP / 4));
        vc[i] = u4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
        if (pages[S::NP + i] < 0 || col >= c.dh || u >= S::kQuads) continue;
        vc[i] = *reinterpret_cast<const u4 *>(static_cast<const uint8_t *>(c.v) +
                                              token_row(c, w.kv, stage * kStage + token(S::NP + i), pages[S::NP + i]) * c.dh +
                                              4 * col);
      }
    }
  }

  // Rows in fp32 into two terms; returns what is out of the ordinary.
  template <bool VALUES>
  __device__ __forceinline__ int split_rows(char *to, float *factors, mask64 *odd) {
    const int piece = threadIdx.x & (S::kPieces - 1);
    int flags = 0;
#pragma unroll
    for (int i = 0; i < S::NP; ++i) {
      const int tk = token(i);
      if (tk >= kStage) continue;
      float v[8];
      unsigned top = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = x[i][j >> 2][j & 3];
        top = max(top, __builtin_bit_cast(unsigned, v[j]) & 0x7fffffffu);
      }
      top = row_top<S::kLanes>(top);
      const bool finite = top < 0x7f800000u;
      const float big = __builtin_bit_cast(float, top);
      int e = 0;
      if (finite) {
        e = tiles::exponent_for(big);
      } else {
        flags |= VALUES ? kOddValue : kOddKey;
        if (piece == 0) atomicOr(odd, mask64{1} << tk);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      }
      if (finite && wild(big)) flags |= kWild;
      const Terms t = tiles::split8(v, __builtin_amdgcn_ldexpf(1.f, e));
      char *p = to + (VALUES ? S::value_place(tk, piece) : S::key_place(tk, piece));
      *reinterpret_cast<h8 *>(p) = t.h;
      *reinterpret_cast<h8 *>(p + kStage * S::kRow) = t.m;
      if (piece == 0) factors[tk] = __builtin_amdgcn_ldexpf(1.f, -e);
    }
    return flags;
  }
  static __device__ __forceinline__ void put_flags(int *to, int flags) {
    if (flags != 0) atomicOr(to, flags);
  }

  // stage: the one that is written, of the block's walk, and its buffers.
  __device__ __forceinline__ void put_keys(Lds<INT8, DP> &s, const Cache &c, const Walk &w, int stage, int buf, int third) {
    char *to = s.stage(buf);
    int flags = 0;
    if constexpr (!INT8) {
      flags = split_rows<false>(to, s.ks[buf], &s.odd_key[third]);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int tk = token(i);
        if (tk < kStage && pages[i] < 0 && stage * kStage + tk < w.held) {
          flags |= kMissing;
          atomicOr(&s.missing[third], mask64{1} << tk);
        }
      }
    } else {
      const int piece = threadIdx.x & (S::kPieces - 1);
#pragma unroll
      for (int i = 0; i < S::NP; ++i) {
        const int tk = token(i);
        if (tk >= kStage) continue;
        u4 h;
        unsigned lo, hi;
        paged::halves(kc[i][0], lo, hi), h[0] = lo, h[1] = hi;
        paged::halves(kc[i][1], lo, hi), h[2] = lo, h[3] = hi;
        *reinterpret_cast<u4 *>(to + S::key_place(tk, piece)) = h;
      }
      const int tk = threadIdx.x & (kStage - 1);
      if (threadIdx.x < kStage) {
        s.ks[buf][tk] = scale;
        if (wild(scale)) flags |= kWild;
        if (pages[NE - 1] < 0 && stage * kStage + tk < w.held) {
          flags |= kMissing;
          atomicOr(&s.missing[third], mask64{1} << tk);
        }
      } else if (threadIdx.x < 2 * kStage) {
        const bool finite = fabsf(scale) < INFINITY;
        if (!finite) {
          flags |= kOddValue;
          atomicOr(&s.odd_value[third], mask64{1} << tk);
        } else if (wild(scale)) {
          flags |= kWild;
        }
        s.vs[buf][tk] = finite ? scale : 0.f;
      }
    }
    put_flags(&s.flags[third], flags);
  }
  __device__ __forceinline__ void put_values(Lds<INT8, DP> &s, int buf, int third) {
    char *to = s.stage(buf) + S::kKeys;
    if constexpr (!INT8) {
      put_flags(&s.flags[third], split_rows<true>(to, s.vs[buf], &s.odd_value[third]));
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
// product leaves its results' rows.
template <bool INT8, int DP>
__device__ __forceinline__ Terms values_of(const char *p, int token, int b, int lane) {
  using S = Shape<INT8, DP>;
  Terms t;
  const int g = lane >> 5;
  if constexpr (INT8) {
    const char *at = p + ((token / 4 + g) * DP + 32 * b + (lane & 31)) * 8;
    const u2 lo = *reinterpret_cast<const u2 *>(at), hi = *reinterpret_cast<const u2 *>(at + 2 * DP * 8);
    t.h = t.m = __builtin_bit_cast(h8, u4{lo[0], lo[1], hi[0], hi[1]});
  } else {
    const int tk = token + 4 * g + (lane >> 2 & 3), piece = 4 * b + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
    const char *at = p + S::value_place(tk, piece) + (lane & 1) * 8;
    auto term = [](const char *at) {
      const auto a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tiles::lds_s4 *)at);
      const auto b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tiles::lds_s4 *)(at + 8 * S::kRow));
      return __builtin_bit_cast(h8, tiles::s8(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)));
    };
    t.h = term(at), t.m = term(at + kStage * S::kRow);
  }
  return t;
}

// A cached value, for what the products do not take.
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
  f16 o[S::NB];
  float m, l;
  int fe;    // the scores' exponent
  int seen;  // tokens that the lane's row sees; 0: none
  bool some, odd;
  const float *from;  // the row's query

  __device__ __forceinline__ void start(const Args &a, const float *row, bool live, int sees) {
    const int hi = (threadIdx.x & 63) >> 5;
    from = row, seen = sees, some = false;
    tiles::RowValues<DP> x;
    x.load(row, live, a.c.dh, hi);
    bool not_finite = false;
    const float top = x.top(INFINITY, not_finite);
    const int e = tiles::exponent_for(top);
    fe = a.exp - e;
    odd = __any(wild(top));
    x.split_into(q, __builtin_amdgcn_ldexpf(a.mant, e));
    m = kNever, l = 0.f;
#pragma unroll
    for (int b = 0; b < S::NB; ++b) o[b] = f16{};
  }

  // KB blocks of 32 tokens from `first` of the stage, whose tokens begin at pos0.
  template <bool WILD, int KB>
  __device__ __forceinline__ void take(const Args &a, const Walk &w, Lds<INT8, DP> &lds, int buf, int third, int first,
                                       int pos0, bool masked) {
    const int lane = threadIdx.x & 63, c = lane & 31, hi = lane >> 5;
    const char *keys = lds.stage(buf), *values = keys + S::kKeys;
    f16 s[KB] = {};
#pragma unroll
    for (int st = 0; st < S::NS; ++st)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const char *p = keys + S::key_place(first + 32 * kb + c, 2 * st + hi);
        Terms k;
        k.h = *reinterpret_cast<const h8 *>(p);
        if constexpr (!INT8) k.m = *reinterpret_cast<const h8 *>(p + kStage * S::kRow);
        mma_keys<INT8>(s[kb], k, q[st]);
      }
    // factors of the rows that a lane's results are, four at a time
    auto factors = [&](const float *f, int kb, int i) { return *reinterpret_cast<const f4 *>(f + first + 32 * kb + 8 * i + 4 * hi); };
    float f = 1.f;
    if constexpr (!WILD) f = __builtin_amdgcn_ldexpf(1.f, fe);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 k = factors(lds.ks[buf], kb, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = s[kb][4 * i + j], by = k[j];
          if constexpr (WILD)
            s[kb][4 * i + j] = __builtin_amdgcn_ldexpf(x * __builtin_amdgcn_frexp_mantf(by), __builtin_amdgcn_frexp_expf(by) + fe);
          else
            s[kb][4 * i + j] = x * by;
        }
      }
    int raise = 0;
    mask64 missing = 0, odd_value = 0;
    if constexpr (WILD) {
      missing = uniform((int64_t)lds.missing[third]), odd_value = uniform((int64_t)lds.odd_value[third]);
      if constexpr (!INT8) {
        // keys that are not finite: their scores in plain fp32
        mask64 left = uniform((int64_t)lds.odd_key[third]) >> first;
        if constexpr (KB == 1) left &= 0xffffffffu;
        for (; left != 0; left &= left - 1) {
          const int t = __builtin_ctzll(left), pos = pos0 + first + t;
          const int page = paging::page_of(w.pages, a.c.max_pages, a.c.shift, a.c.pages, pos);
          if (page < 0) continue;
          const float *k = static_cast<const float *>(a.c.k) + token_row(a.c, w.kv, pos, page) * a.c.dh;
          float x = 0.f;
          if (seen > 0)
            for (int d = 0; d < a.c.dh; ++d) x = fmaf(from[d], k[d], x);
          x *= __builtin_amdgcn_ldexpf(a.mant, a.exp);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (32 * kb + tiles::out_row(e, hi) == t) s[kb][e] = x;
        }
      }
      float big = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f4 v = factors(lds.vs[buf], kb, i);
#pragma unroll
          for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(v[j]));
        }
      big = half_pair(big, [](float x, float y) { return fmaxf(x, y); });
      raise = big > 0.f ? __builtin_amdgcn_frexp_expf(big) : 0;  // of the factors for now
    }
    const int left = seen - pos0 - first;  // tokens from the first that the row sees
    if (WILD || masked) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int t = 32 * kb + tiles::out_row(e, hi);
          bool gone = t >= left;
          if constexpr (WILD) gone |= (missing >> (first + t) & 1) != 0;
          if (gone) s[kb][e] = -INFINITY;
        }
    }
    if constexpr (WILD) {
      const int n = min(max(left, 0), 32 * KB);
      const mask64 sees = n == 64 ? ~mask64{0} : (mask64{1} << n) - 1;
      some |= (~missing >> first & sees) != 0;
    } else {
      some |= left > 0;
    }
    float most = tiles::over16(s[0], [](float x, float y) { return fmaxf(x, y); });
    if constexpr (KB == 2) most = fmaxf(most, tiles::over16(s[1], [](float x, float y) { return fmaxf(x, y); }));
    most = half_pair(most, [](float x, float y) { return fmaxf(x, y); });
    if constexpr (!WILD) most *= f;
    const int ev = WILD ? raise : 0;
    if constexpr (WILD) most += (float)max(0, ev + (INT8 ? 7 : 15) - kRaise);
    if (__any(most > m + 8.f)) {
      const float now = fmaxf(m, most), r = __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= r;
#pragma unroll
      for (int b = 0; b < S::NB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[b][e] *= r;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = __builtin_amdgcn_exp2f(fmaf(s[kb][e], f, -m));
      l += tiles::over16(s[kb], [](float x, float y) { return x + y; });
    }
    if constexpr (WILD) {
      // values that are not finite: in plain fp32, for the rows that see them
      mask64 odd = odd_value >> first;
      if constexpr (KB == 1) odd &= 0xffffffffu;
      for (; odd != 0; odd &= odd - 1) {
        const int t = __builtin_ctzll(odd), pos = pos0 + first + t;
        const int page = paging::page_of(w.pages, a.c.max_pages, a.c.shift, a.c.pages, pos);
        if (page < 0) continue;
        const int64_t row = token_row(a.c, w.kv, pos, page);
        float p = 0.f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * kb + tiles::out_row(e, hi) == t) p = s[kb][e];
        p = half_pair(p, [](float x, float y) { return x + y; });
        if (t >= left) continue;
#pragma unroll
        for (int b = 0; b < S::NB; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int d = 32 * b + tiles::out_row(e, hi);
            if (d < a.c.dh) o[b][e] = fmaf(p, value_at<INT8>(a.c, row, d), o[b][e]);
          }
      }
    }
    // the probabilities times the values' factors, the largest of a row brought to [2^14, 2^15)
    float top = 0.f;
    const float down = WILD ? __builtin_amdgcn_ldexpf(1.f, -ev) : 1.f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 v = factors(lds.vs[buf], kb, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[kb][4 * i + j] *= WILD ? v[j] * down : v[j];
      }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) top = tiles::top_of(s[kb], top);
    top = half_pair(top, [](float x, float y) { return fmaxf(x, y); });
    const int et = max(__builtin_amdgcn_frexp_expf(top), -100);
    const float lift = __builtin_amdgcn_ldexpf(1.f, 15 - et), back = __builtin_amdgcn_ldexpf(1.f, et - 15 + ev);
    Terms p[KB][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = s[kb][e];
      p[kb][0] = tiles::split8(x, lift), p[kb][1] = tiles::split8(x + 8, lift);
    }
#pragma unroll
    for (int b = 0; b < S::NB; ++b) {
      f16 z = {};
#pragma unroll
      for (int st = 0; st < 2 * KB; ++st) {
        const Terms v = values_of<INT8, DP>(values, first + 16 * st, b, lane);
        mma_keys<INT8>(z, v, p[st >> 1][st & 1]);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) o[b][e] = fmaf(z[e], back, o[b][e]);
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
      const int token = live ? row / a.group : 0, head = kv * a.group + (live ? row % a.group : 0);
      const int n_seen = live ? sees(t.len, end, walk.held, token) : 0;
      const int live_rows = min(32, rows - block * ROWS - 32 * rw);
      const int least = live_rows < 32 ? 0 : __builtin_amdgcn_readlane(n_seen, 0);
      const int most = live_rows > 0 ? __builtin_amdgcn_readlane(n_seen, live_rows - 1) : 0;
      Staging<INT8, DP> g;
      g.look(a.c, walk, s0);
      if (tid < 3) lds.flags[tid] = 0, lds.odd_key[tid] = lds.odd_value[tid] = lds.missing[tid] = 0;
      Rows<INT8, DP> r;
      r.start(a, a.q + (int64_t)(t.row0 + token) * a.ld_q + (int64_t)head * a.c.dh, live, n_seen);
      g.resolve(a.c);
      __syncthreads();  // the flags are cleared, the last block's buffers free
      g.load_keys(a.c, walk, s0);
      g.put_keys(lds, a.c, walk, s0, 0, 0);
      g.load_values(a.c, walk, s0);
      g.put_values(lds, 0, 0);
      g.look(a.c, walk, s0 + 1);
      for (int i = s0; i < s1; ++i) {
        const int buf = (i - s0) & 1, third = (i - s0) % 3, after = (i - s0 + 1) % 3;
        const bool more = i + 1 < s1;
        __syncthreads();
        const int flags = __builtin_amdgcn_readfirstlane(lds.flags[third]);
        if (tid == 0) {
          const int clear = (i - s0 + 2) % 3;
          lds.flags[clear] = 0, lds.odd_key[clear] = lds.odd_value[clear] = lds.missing[clear] = 0;
        }
        const int pos0 = i * kStage, first = 32 * z;
        if (more) {
          g.resolve(a.c);
          g.load_keys(a.c, walk, i + 1);
        }
        if (pos0 + first < most) {
          const bool masked = pos0 + first + 32 * KB > least;
          if (flags != 0 || r.odd)
            r.template take<true, KB>(a, walk, lds, buf, third, first, pos0, masked);
          else
            r.template take<false, KB>(a, walk, lds, buf, third, first, pos0, masked);
        }
        if (more) {
          g.put_keys(lds, a.c, walk, i + 1, buf ^ 1, after);
          g.load_values(a.c, walk, i + 1);
          g.put_values(lds, buf ^ 1, after);
          g.look(a.c, walk, i + 2);
        }
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
          to = a.out + (int64_t)(t.row0 + token) * a.ld_out + (int64_t)head * a.c.dh;
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

// The parts of blocks that were cut, added in order: a wave a row, its halves every other part.
template <int DP, int ROWS>
__global__ void __launch_bounds__(256) join_parts(Args a) {
  const Cut cut = a.cuts[blockIdx.x];
  const int lane = threadIdx.x & 63, half = lane >> 5, d = 4 * (lane & 31);
  for (int r = blockIdx.y * 4 + (int)(threadIdx.x >> 6); cut.parts > 0 && r < cut.rows; r += gridDim.y * 4) {
    // the first part is the owner's place 1, the others the next ones' places 0
    auto part = [&](int k) { return a.parts + (int64_t)(k == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + k)) * kPart<DP, ROWS>; };
    float m = kNever;
    for (int k = lane; k < cut.parts; k += 64) m = fmaxf(m, part(k)[r]);
    m = wave_max(m);
    float l = 0.f;
    bool some = false;
    f4 o{};
    for (int k = half; k < cut.parts; k += 2) {
      const float *x = part(k);
      const float lk = x[ROWS + r];
      if (lk < 0.f) continue;
      const float f = __builtin_amdgcn_exp2f(x[r] - m);
      some = true, l = fmaf(lk, f, l);
      if (d < a.c.dh) {
        const f4 y = *reinterpret_cast<const f4 *>(x + 2 * ROWS + r * DP + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(y[j], f, o[j]);
      }
    }
    auto add = [](float x, float y) { return x + y; };
    l = half_pair(l, add);
    some = __any(some);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = half_pair(o[j], add);
    if (half == 0 && d < a.c.dh) {
      const int row = cut.row + r;
      const f4 y = some ? o / l : f4{};
      *reinterpret_cast<f4u *>(a.out + (int64_t)(cut.row0 + row / a.group) * a.ld_out + (int64_t)(cut.head + row % a.group) * a.c.dh + d) = y;
    }
  }
}

}  // namespace chunk
