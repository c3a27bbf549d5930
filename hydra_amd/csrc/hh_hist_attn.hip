// hh_hist_attn.hip — how an attention call over histories is split, and its launch.
#include "hh_hist.hpp"

namespace hh {

// Workgroups that a pass's keys are split for: those that the chip holds at once, by the kernels' registers (256 tokens behind 16384, bf16 over
// 8 bits: heads of 64 162 us, with 512 workgroups 163, with 1024 158; heads of 128 115 us, with 384 133, with 768 127; of 256 161, with 128 289, with 512 180).
static int wanted_groups(int d, bool few) { return few ? (d == 64 ? 768 : 512) : d == 64 ? 768 : d == 128 ? 512 : 256; }

static HistAttnArgs::Pass plan_pass(const HistAttnArgs &a, int64_t rows, int64_t heads, int64_t keys) {
  HistAttnArgs::Pass p{};
  // With a prefix both passes are one launch, of workgroups for 16 rows and for 128.
  const bool few = rows <= (a.p.k ? 16 : kFewRows);
  p.block_rows = rows <= 16 ? 16 : few ? kFewRows : 128;
  p.row_blocks = (int)((rows + p.block_rows - 1) / p.block_rows);
  p.tile = few ? 128 : a.d == 256 ? 32 : 64;
  const int64_t most = (keys + p.tile - 1) / p.tile;
  int64_t chunks = wanted_groups(a.d, few) / (heads * p.row_blocks);
  // A few tiles one after the other take less than a launch that joins them.
  if (chunks > most / 2) chunks = most / 2;
  if (chunks > kHistChunks) chunks = kHistChunks;
  if (chunks < 1) chunks = 1;
  int64_t per = ((keys + chunks - 1) / chunks + p.tile - 1) / p.tile * p.tile;
  if (per < p.tile) per = p.tile;
  p.per = (int)per;
  p.chunks = (int)((keys + per - 1) / per);
  if (p.chunks < 1) p.chunks = 1;
  // The workgroups of many rows are dealt to the eight XCDs (history_many).
  const int64_t groups = heads * p.chunks, parts = groups >= 8 ? 1 : (8 + groups - 1) / groups, share = (p.row_blocks + parts - 1) / parts;
  p.blocks = (int)(few ? groups : 8 * ((groups * share * parts + 7) / 8));
  return p;
}

void history_plan(HistAttnArgs &a, int64_t length, int64_t prefix_rows) {
  int64_t keys = length;
  if (!a.h.ring && keys > a.h.rows) keys = a.h.rows;
  const int64_t rows = (int64_t)a.N * a.qm;
  if (a.window) {
    // A block of rows sees its window, the tokens that it spans besides the first, and the first tokens.
    const int64_t spanned = rows <= kFewRows ? a.N : 128 / a.qm + 2, seen = (int64_t)a.window + spanned + a.first;
    if (keys > seen) keys = seen;
  }
  a.own = plan_pass(a, rows, (int64_t)a.S * a.kvh, keys);
  a.pre = HistAttnArgs::Pass{};
  if (a.p.k) a.pre = plan_pass(a, rows * a.S, a.kvh, prefix_rows);
  a.chunks = a.own.chunks + a.pre.chunks;
}

size_t history_workspace(const HistAttnArgs &a) {
  return a.chunks > 1 ? sizeof(float) * (size_t)a.S * a.N * a.qh * a.chunks * (a.d + 2) : 0;
}

// A pass that is cut has at most wanted_groups workgroups of at most 128 rows each, and a row at most as many chunks as half its tiles, of
// 32 keys or more; one that is not cut a state a row, or, without a prefix, none.
size_t history_reserve(const HistAttnArgs &a, int64_t length, int64_t prefix_rows) {
  const int64_t rows = (int64_t)a.S * a.N * a.qh;
  auto states = [&](int64_t keys) {
    int64_t chunks = (keys + 31) / 32 / 2;
    if (chunks > kHistChunks) chunks = kHistChunks;
    if (chunks < 2) return (int64_t)0;
    const int64_t groups = (int64_t)wanted_groups(a.d, true) * 128;
    return rows * chunks < groups ? rows * chunks : groups;
  };
  // A block of rows over a ring sees its window and no more than 130 tokens beside it, whatever the length.
  if (a.h.ring) length = (int64_t)a.h.rows + 130;
  else if (length > a.h.rows) length = a.h.rows;
  int64_t n = states(length);
  if (a.p.k) n = (n > rows ? n : rows) + (states(prefix_rows) > rows ? states(prefix_rows) : rows);
  return sizeof(float) * (size_t)n * (a.d + 2);
}

hipError_t launch_history_attention(HistAttnArgs a, int type, hipStream_t s, int *launches) {
  if (a.d == 64) return launch_history_attention_d<64>(a, type, s, launches);
  return a.d == 128 ? launch_history_attention_d<128>(a, type, s, launches) : launch_history_attention_d<256>(a, type, s, launches);
}

}  // namespace hh
