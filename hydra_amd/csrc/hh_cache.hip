// hh_cache.hip — the accepted rows of a drafted tree into the histories of many layers, and the
// eviction of the rows of least accumulated weight.
#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

// Rows that a sequence's histories take: `accepted`, bounded by the path and the room left.
__device__ __forceinline__ int committed(const RowsLayer &y, const RowsArgs &a, int s) {
  const int acc = min(max(a.accepted[s], 0), a.N);
  return min(acc, max(0, y.limit - max(y.lengths[s], 0)));
}

// One workgroup per (layer, sequence, place on the path).
__global__ __launch_bounds__(256) void commit_kernel(RowsArgs a) {
  const int i = blockIdx.x % a.N, s = blockIdx.x / a.N % a.S;
  const RowsLayer &y = a.layer[blockIdx.x / (a.N * a.S)];
  const int c = committed(y, a, s);
  const int node = a.path[(int64_t)s * a.N + i];
  // A ring takes the last rows of a path longer than itself.
  if (i >= c || node < 0 || node >= a.N || i < c - y.rows) return;
  const int64_t pos = (int64_t)max(y.lengths[s], 0) + i;
  const int64_t row = y.ring ? pos % y.rows : pos;
  if (row >= y.rows) return;
  const int vecs = a.kvh * a.d / 8;
  const int64_t src = ((int64_t)s * a.N + node) * a.kv_stride, dst = (int64_t)s * y.seq_stride + row * a.kvh * a.d;
  for (int e = threadIdx.x; e < 2 * vecs; e += 256) {
    const bool v = e >= vecs;
    const int o = 8 * (v ? e - vecs : e);
    *(u32x4 *)((v ? y.v : y.k) + dst + o) = *(const u32x4 *)((v ? y.dv : y.dk) + src + o);
  }
  if ((int)threadIdx.x < a.kvh) {
    const int64_t at = ((int64_t)s * a.kvh + threadIdx.x) * y.rows + row;
    if (y.weights) y.weights[at] = 0.f;
    if (y.positions) y.positions[at] = y.next[s] + i;
  }
}

// The lengths and next positions, once for the layers that share them.
__global__ __launch_bounds__(64) void advance_kernel(RowsArgs a) {
  const RowsLayer &y = a.layer[blockIdx.x];
  if (!y.last) return;
  for (int s = threadIdx.x; s < a.S; s += 64) {
    const int c = committed(y, a, s);
    y.lengths[s] = max(y.lengths[s], 0) + c;
    if (y.next) y.next[s] += c;
  }
}

// Eviction's order as an unsigned key: recent rows above every weight, NaN as minus infinity, the two
// zeros equal.
__device__ __forceinline__ uint32_t rank_key(float w, int pos, int64_t oldest) {
  if (pos >= oldest) return 0xFFFFFFFFu;
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelT = 1024;

// Exclusive prefix of `flag` over the workgroup in thread order, and its total.
__device__ __forceinline__ int block_rank(bool flag, int *s_w, int &total) {
  const uint64_t b = __ballot(flag);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (lane == 0) s_w[wave] = __popcll(b);
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < kSelT / 64; ++w) {
    if (w < wave) before += s_w[w];
    total += s_w[w];
  }
  __syncthreads();
  return before + __popcll(b & ((1ull << lane) - 1));
}

// One workgroup per (layer, sequence, kv head): the key of the keep-th row by radix selection, eight
// bits a pass, then the rows below `keep` that go and those from `keep` on that stay, in order.
__global__ __launch_bounds__(kSelT) void select_kernel(RowsArgs a) {
  __shared__ int s_hist[256], s_w[kSelT / 64], s_bin, s_left;
  const int head = blockIdx.x, g = head % a.kvh, s = head / a.kvh % a.S;
  const RowsLayer &y = a.layer[head / (a.kvh * a.S)];
  const int tid = threadIdx.x;
  const int n = min(max(y.lengths[s], 0), y.rows);
  if (n <= a.keep) {
    if (tid == 0) a.moves[head] = 0;
    return;
  }
  const int64_t oldest = (int64_t)y.next[s] - a.recent;
  const int64_t base = ((int64_t)s * a.kvh + g) * y.rows;
  const float *w = y.weights + base;
  const int *pos = y.positions + base;
  uint32_t prefix = 0;
  int left = a.keep;   // rows still to take among those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) s_hist[tid] = 0;
    __syncthreads();
    for (int r = tid; r < n; r += kSelT) {
      const uint32_t key = rank_key(w[r], pos[r], oldest);
      if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s_hist[key >> shift & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int bin = 255, need = left;
      while (bin > 0 && s_hist[bin] < need) need -= s_hist[bin--];
      s_bin = bin;
      s_left = need;
    }
    __syncthreads();
    prefix |= (uint32_t)s_bin << shift;
    left = s_left;
  }
  // Rows above `prefix` stay, and the first `left` of those equal to it.
  int equal = 0, holes = 0, from = 0;
  int32_t *src = a.from + (int64_t)head * a.max_moves, *dst = a.to + (int64_t)head * a.max_moves;
  for (int t = 0; t < n; t += kSelT) {
    const int r = t + tid;
    const uint32_t key = r < n ? rank_key(w[r], pos[r], oldest) : 0;
    int total;
    const bool eq = r < n && key == prefix;
    const int e = equal + block_rank(eq, s_w, total);
    equal += total;
    const bool stay = r < n && (key > prefix || (eq && e < left));
    const bool hole = r < n && r < a.keep && !stay, move = r >= a.keep && stay;
    const int i = holes + block_rank(hole, s_w, total);
    if (hole && i < a.max_moves) dst[i] = r;
    holes += total;
    const int j = from + block_rank(move, s_w, total);
    if (move && j < a.max_moves) src[j] = r;
    from += total;
  }
  if (tid == 0) a.moves[head] = min(min(holes, from), a.max_moves);
}

// Moves the rows of a head, a group of lanes per row; the sources, at `keep` and above, and the
// destinations, below it, do not overlap. One workgroup of the last layer that shares them shortens the lengths.
__global__ __launch_bounds__(256) void move_kernel(RowsArgs a, int parts) {
  const int head = blockIdx.x / parts, part = blockIdx.x % parts;
  const int g = head % a.kvh, s = head / a.kvh % a.S;
  const RowsLayer &y = a.layer[head / (a.kvh * a.S)];
  const int moves = a.moves[head];
  const int32_t *src = a.from + (int64_t)head * a.max_moves, *dst = a.to + (int64_t)head * a.max_moves;
  const int lanes = a.d / 8, per = 256 / lanes, lane = threadIdx.x % lanes;
  const int64_t base = (int64_t)s * y.seq_stride + (int64_t)g * a.d + 8 * lane, meta = ((int64_t)s * a.kvh + g) * y.rows;
  for (int i = part * per + threadIdx.x / lanes; i < moves; i += parts * per) {
    const int f = src[i], t = dst[i];
    const int64_t fo = base + (int64_t)f * a.kvh * a.d, to = base + (int64_t)t * a.kvh * a.d;
    *(u32x4 *)(y.k + to) = *(const u32x4 *)(y.k + fo);
    *(u32x4 *)(y.v + to) = *(const u32x4 *)(y.v + fo);
    if (lane == 0) {
      y.weights[meta + t] = y.weights[meta + f];
      y.positions[meta + t] = y.positions[meta + f];
    }
  }
  if (y.last && g == 0 && part == 0 && threadIdx.x == 0) y.lengths[s] = min(y.lengths[s], a.keep);
}

hipError_t launch_commit(const RowsArgs &a, bool last, hipStream_t s) {
  if (last) hipLaunchKernelGGL(advance_kernel, dim3(a.layers), dim3(64), 0, s, a);
  else hipLaunchKernelGGL(commit_kernel, dim3(a.layers * a.S * a.N), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_evict(const RowsArgs &a, hipStream_t s) {
  const int heads = a.layers * a.S * a.kvh;
  hipLaunchKernelGGL(select_kernel, dim3(heads), dim3(kSelT), 0, s, a);
  const int parts = 8;
  hipLaunchKernelGGL(move_kernel, dim3(heads * parts), dim3(256), 0, s, a, parts);
  return hipGetLastError();
}

}  // namespace hh
