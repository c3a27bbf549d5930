// hh_ctx.hpp — the context and graph objects behind the C ABI, and its error reporting.
#pragma once
#include <hip/hip_runtime.h>

#include <string>
#include <vector>

#include "hydra_hip.h"

namespace hh {
// Sets hh_last_error()'s message of the calling thread; returns `code`.
int fail(int code, const std::string &msg);
int hip_fail(hipError_t e, const char *what);
}  // namespace hh

#define HH_HIP(call)                                      \
  do {                                                    \
    hipError_t e_ = (call);                               \
    if (e_ != hipSuccess) return hh::hip_fail(e_, #call); \
  } while (0)

struct hh_ctx {
  // Flags of the fused decode kernel: allocated and zeroed once, then only ever written with
  // flag values; `epoch` is the value of the last call.
  uint32_t *flags = nullptr;
  uint32_t epoch = 0;
  uint32_t fused_calls = 0;    // one-launch decode calls so far (the counter region parity)
  int decode_fused = -1;   // 1 on, 0 off, -1 the environment's choice
  int device = 0;
  hipStream_t stream = nullptr;
  uint8_t *arena = nullptr;
  size_t arena_bytes = 0;
  int64_t dispatches = 0;
  // Profiling: a pool of events, a start/stop pair per phase of each profiled forward call.
  bool profile = false;
  std::vector<hipEvent_t> events;
  size_t events_used = 0;
  // Graph capture: calls are recorded, not run; dispatches counted while recording are moved
  // to the graph and added back per launch.
  bool capturing = false;
  int64_t capture_base = 0;
  // Decode attention partials (per query head and chunk), grown on demand.
  float *attn = nullptr;
  size_t attn_bytes = 0;
  // Workspace of the drafted-token entries (hh_draft.hip), grown on demand.
  uint8_t *draft = nullptr;
  size_t draft_bytes = 0;
  uint32_t *arrivals = nullptr;   // hh_cache_commit's counters, zero between its launches
  // Workspace of hh_history_attention (hh_history.hip), grown on demand.
  uint8_t *hist = nullptr;
  size_t hist_bytes = 0;
  // Instantiated graphs of this context that are not yet destroyed: they hold the arena's,
  // the attention partials' and the draft and history workspaces' device addresses, so none may be reallocated while any exist.
  int live_graphs = 0;
  // This device's copy of the static scratch array (hh_moe_forward_noalloc), or NULL when its
  // address could not be resolved (scratch_error then says why).
  uint8_t *scratch = nullptr;
  std::string scratch_error;
};

struct hh_graph {
  hh_ctx *ctx = nullptr;
  hipGraph_t graph = nullptr;
  hipGraphExec_t exec = nullptr;
  int64_t dispatches = 0;
};
