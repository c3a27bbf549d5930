// hh_hist.hpp — argument blocks and device helpers of the history kernels (hh_hist_rows.hip, hh_hist_attn.hip) and of the
// rotary kernel (hh_rotary.hip), shared with their C entries (hh_history.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

enum HistFormat { H_F16 = 1, H_BF16 = 2, H_MXFP8 = 3, H_MXFP4 = 4 };
constexpr int kHistLength = 1 << 30;   // lengths count as at most this
constexpr int kFewRows = 32;           // rows of a kv head up to which a wave takes all of them, 16 or 32
constexpr int kHistChunks = 256;       // most chunks of an attention pass

// A history as kernels take it: [S][kvh][rows][d].
struct HistView {
  uint8_t *k, *v, *ks, *vs;
  const int32_t *lengths;
  int rows, ring, pinned;
};

struct HistRowsArgs {
  HistView h;
  const void *k, *v;                   // write: [S][N][kvh][d], kv_stride between tokens
  void *ko, *vo;                       // read: packed
  const int32_t *starts, *counts;      // starts: read
  int S, N, kvh, d, format, type;
  int64_t kv_stride;
};

struct HistAttnArgs {
  HistView h, p;                       // p.k NULL: no prefix
  const void *q;
  const int32_t *counts;
  const uint16_t *sinks;
  void *out;
  float *lse;
  int S, N, qh, kvh, d, qm, window, first, format;
  float scale;
  int64_t q_stride;
  // How the work is split (history_plan). A pass is over the sequences' own histories or over the prefix, whose rows are those of
  // all sequences' tokens; its keys are cut into chunks of `per` keys, whole tiles.
  struct Pass {
    int chunks, per, tile, block_rows, row_blocks, blocks;
  } own, pre;
  int chunks;                          // of a row, the prefix's first
  float *pm, *pl, *po;                 // chunk states [S][N][qh][chunks], their sums [..][chunks][d]
};

struct RotaryRows {
  const void *x;
  void *y;
  int heads;
  int64_t x_stride, y_stride;
};
struct RotaryArgs {
  RotaryRows r[2];
  const double *turns;
  const int32_t *positions;
  float magnitude;
  int tokens, count, d, rotated, span, interleaved, type;
  int per_block, parts, lanes;         // tokens a workgroup, workgroups that share them, log2 of a row's lanes
};

__device__ __forceinline__ int hist_length(const int32_t *lengths, int s) { return min(max(lengths[s], 0), kHistLength); }
__device__ __forceinline__ int step_count(const int32_t *counts, int s, int n) { return min(max(counts[s], 0), n); }
// The row of a position (>= 0), or −1 where it is not held.
__device__ __forceinline__ int hist_row(const HistView &h, int p) {
  if (h.ring) return p < h.pinned ? p : h.pinned + (int)((uint32_t)(p - h.pinned) % (uint32_t)(h.rows - h.pinned));
  return p < h.rows ? p : -1;
}
__host__ __device__ inline int hist_row_bytes(int format, int d) { return format == H_MXFP8 ? d : format == H_MXFP4 ? d / 2 : 2 * d; }
// A scale byte's number; 255 is NaN.
__device__ __forceinline__ float hist_scale(uint32_t b) { return b == 255 ? __uint_as_float(0x7FC00000u) : e8m0_to_f32(b); }

hipError_t launch_history_write(const HistRowsArgs &a, hipStream_t s);
hipError_t launch_history_read(const HistRowsArgs &a, hipStream_t s);
hipError_t launch_history_advance(int32_t *lengths, const int32_t *counts, int S, int N, hipStream_t s);
void history_plan(HistAttnArgs &a, int64_t length, int64_t prefix_rows);
size_t history_workspace(const HistAttnArgs &a);
size_t history_reserve(const HistAttnArgs &a, int64_t length, int64_t prefix_rows);   // of every call up to these sizes
hipError_t launch_history_attention(HistAttnArgs a, int type, hipStream_t s, int *launches);
template <int D> hipError_t launch_history_attention_d(HistAttnArgs a, int type, hipStream_t s, int *launches);
hipError_t launch_rotary(RotaryArgs a, hipStream_t s);

}  // namespace hh
