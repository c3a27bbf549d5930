// hh_draft.hpp — argument blocks of the drafted-token kernels (hh_tree.hip, hh_verify.hip,
// hh_cache.hip), shared with their C entries (hh_draft.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hh {

enum Elem { E_F32 = 0, E_F16 = 1, E_BF16 = 2 };
constexpr int kTreeNodes = 64;    // most nodes of a tree: an ancestor set is one 64-bit mask
constexpr int kTreeQM = 16;       // most query heads per kv head
constexpr int kTreeGroups = 256;  // workgroups that a call's keys are split for
constexpr int kTreeTiles = 4;     // tiles of keys that one workgroup takes without a split
constexpr int kWeightGroups = 1024; // workgroups of the accumulation
constexpr int kTreeChunks = 256;  // most chunks of a sequence

struct TreeArgs {
  const void *q, *dk, *dv;          // [S][N][qh][d] and [S][N][kvh][d], strides below
  const uint16_t *k, *v;            // [S][rows][kvh][d]
  const int32_t *lengths, *parents, *counts;
  const uint16_t *sinks;            // bf16 [qh] or null
  void *out;                        // [S][N][qh][d]
  float *lse;                       // [S][N][qh] or null
  int S, N, qh, kvh, d, rows, ring, window;
  float scale;
  int64_t q_stride, kv_stride, seq_stride;   // elements between nodes, nodes, sequences
  // How a call's keys are split (tree_plan): chunks of per_chunk keys, whole tiles; blocks of rows.
  int chunks, per_chunk, tile, row_blocks, qm;
  float inv_qm;
  float *pm, *pl, *po;              // chunk states [S][N][qh][chunks], their sums [..][chunks][d]
  // hh_attention_weights
  const float *lse_in;
  const int32_t *path, *accepted;
  float *weights;                   // [S][kvh][rows]
};

// One layer of a commit or an eviction.
struct RowsLayer {
  uint16_t *k, *v;
  const uint16_t *dk, *dv;
  int32_t *lengths;
  float *weights;
  int32_t *positions, *next;
  int64_t seq_stride;
  int32_t rows, ring;
  int32_t limit;                    // most rows that `lengths` may count
  int32_t last;                     // of the call's layers that share `lengths`
};
constexpr int kRowsLayers = 44;     // layers per launch: their blocks are kernel arguments (4 KB)

struct RowsArgs {
  RowsLayer layer[kRowsLayers];
  const int32_t *path, *accepted;
  int layers, S, N, kvh, d;
  int64_t kv_stride;
  uint32_t *arrivals;               // a commit's workgroups by sequence, zero between launches; NULL: lengths advance later
  // Eviction.
  int keep, recent, max_moves;
  int32_t *moves;                   // [layer][S][kvh]: rows that move
  int32_t *from, *to;               // [layer][S][kvh][max_moves]
};

static_assert(sizeof(RowsArgs) <= 4096, "kernel arguments");

struct VerifyArgs {
  const void *target, *draft;
  int64_t t_stride, d_stride;       // elements between nodes
  const int32_t *tokens, *parents, *counts;
  const float *u, *u_final;
  int32_t *path, *accepted, *next;
  int S, N, V, type, mode, children;
  bool late_leaves;                 // the statistics of leaves after the rounds
  double inv_t, k;                  // 1 / temperature (0: greedy), 256 log2(e) / temperature
  uint8_t *ws;
};

size_t verify_workspace(int S, int N, int V);
size_t verify_reserve(int S, int N, int V);   // of every call up to these sizes
bool verify_fits(int S, int N, int V);   // launches' block counts
void tree_plan(TreeArgs &a, int64_t length);
size_t tree_workspace(const TreeArgs &a);
size_t tree_reserve(const TreeArgs &a, int64_t length);   // of every call up to these sizes
hipError_t launch_tree(const TreeArgs &a, int type, hipStream_t s);
hipError_t launch_weights(TreeArgs a, int type, hipStream_t s);
hipError_t launch_verify(VerifyArgs a, hipStream_t s, int *launches);
hipError_t launch_commit(const RowsArgs &a, bool last, hipStream_t s);
hipError_t launch_evict(const RowsArgs &a, hipStream_t s);

}  // namespace hh
