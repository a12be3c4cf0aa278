// A packed batch of sequences, and attention over it as the tensor engine calls it.
#pragma once

#include <memory>
#include <new>

#include "common.h"

namespace numrs_hip {

// kTile tokens of one sequence: the unit of work of the packed kernels.
struct SeqTile {
  int row0;   // the sequence's first row
  int len;    // its tokens
  int t0;     // the tile's first token within it
  int tile0;  // the number of the sequence's first tile
  int seq;    // the sequence's number
  int pad[3];
};
constexpr int kTile = 64;

// Lists of a batch's tiles on the device.
struct Seqs : std::enable_shared_from_this<Seqs> {
  numrs_hip_ctx *ctx = nullptr;
  int64_t n = 0, total = 0, tiles = 0, blocks = 0;
  SeqTile *in_order = nullptr;  // [tiles]; a tile's number is its place
  SeqTile *by_work = nullptr;   // [blocks] of 128 tokens, those with the most tokens before them first
  SeqTile *by_rest = nullptr;   // [blocks], those with the most tokens after them first
  SeqTile *few_by_work = nullptr, *few_by_rest = nullptr;  // the same of the tiles
  SeqTile *several = nullptr, *single = nullptr;  // the sequences of several tokens, and of one
  int64_t severals = 0, singles = 0, longest = 0;
  size_t bytes = 0;
  ~Seqs() { block_free(ctx, in_order, bytes); }
  // Called before a launch that reads the lists: a graph being recorded keeps them for its replays,
  // whatever becomes of the handle.
  int keep() const {
    if (!ctx->capturing) return NUMRS_HIP_OK;
    try {
      ctx->capture_kept.push_back(shared_from_this());
    } catch (const std::bad_alloc &) {
      return fail(ctx, NUMRS_HIP_E_NOMEM, "out of host memory");
    }
    return NUMRS_HIP_OK;
  }
};

struct PackedHeads {
  int64_t heads, kv_heads, dh;
};

int packed_forward(numrs_hip_ctx *ctx, const Seqs &s, const float *q, int64_t ld_q, const float *k,
                   const float *v, int64_t ld_kv, float *out, int64_t ld_out, float *stats,
                   PackedHeads h);
int packed_backward(numrs_hip_ctx *ctx, const Seqs &s, const float *q, int64_t ld_q, const float *k,
                    const float *v, int64_t ld_kv, const float *out, const float *dout,
                    int64_t ld_out, const float *stats, float *dq, float *dk, float *dv,
                    PackedHeads h, int accumulate);

// numrs_hip_attention_paged without its checks; with a list, of those n sequences of one row each of a packed batch.
int paged_steps(numrs_hip_ctx *ctx, const numrs_hip_kv_cache &cache, const float *q, int64_t ld_q, int64_t heads,
                const int32_t *table, int64_t max_pages, const int32_t *lengths, int64_t n, const SeqTile *list,
                float *out, int64_t ld_out);

// Makes the context's device current for a call, and the caller's again after it.
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(numrs_hip_ctx *ctx) {
    int d = -1;
    if (hipGetDevice(&d) == hipSuccess && d != ctx->device && hipSetDevice(ctx->device) == hipSuccess)
      before = d;
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;
};

}  // namespace numrs_hip

struct numrs_hip_seqs {
  std::shared_ptr<const numrs_hip::Seqs> s;
};
