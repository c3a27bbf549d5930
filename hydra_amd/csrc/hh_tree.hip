// hh_tree.hip — attention of a tree of drafted tokens over the history, and the accumulation of
// the accepted tokens' attention weights.
#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

__device__ __forceinline__ float elem_f32(const _Float16 *p) { return (float)*p; }
__device__ __forceinline__ float elem_f32(const float *p) { return *p; }
__device__ __forceinline__ float elem_f32(const __bf16 *p) { return (float)*p; }

__device__ __forceinline__ float wsum(float v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ float wmax(float v) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// The ancestors-or-self of every node as bit masks, lane i node i (i < N).
__device__ __forceinline__ uint64_t ancestors(const int32_t *parents, int N, int lane) {
  int up = lane < N ? parents[lane] : -1;
  if (up < 0 || up >= lane) up = -1;
  uint64_t mask = 1ull << lane;
  for (int r = 0; r < 6; ++r) {
    const int at = up < 0 ? lane : up;
    const uint32_t lo = __shfl((uint32_t)mask, at), hi = __shfl((uint32_t)(mask >> 32), at);
    const int next = __shfl(up, at);
    if (up >= 0) {
      mask |= ((uint64_t)hi << 32) | lo;
      up = next;
    }
  }
  return mask;
}

// One wave per (sequence, node, head).
template <class Q, class C>
__global__ __launch_bounds__(64) void tree_kernel(TreeArgs a) {
  const int lane = threadIdx.x, h = blockIdx.x % a.qh, n = blockIdx.x / a.qh % a.N, s = blockIdx.x / (a.qh * a.N);
  if (n >= a.counts[s]) return;
  __shared__ float s_q[256], s_p[64];
  const int g = h / (a.qh / a.kvh), D = a.d;
  const Q *q = (const Q *)a.q + ((int64_t)s * a.N + n) * a.q_stride + (int64_t)h * D;
  for (int i = lane; i < D; i += 64) s_q[i] = elem_f32(q + i) * a.scale;
  const uint64_t mask = ancestors(a.parents + (int64_t)s * a.N, a.N, lane);
  const uint64_t own = ((uint64_t)(uint32_t)__shfl((uint32_t)(mask >> 32), n) << 32) | (uint32_t)__shfl((uint32_t)mask, n);
  const int depth = __popcll(mask) - 1;
  const int64_t length = a.ring ? max(a.lengths[s], 0) : min(max(a.lengths[s], 0), a.rows);
  const int64_t pos = length + __popcll(own) - 1;
  int64_t first = a.ring ? max((int64_t)0, length - a.rows) : 0;
  if (a.window) first = max(first, pos - a.window + 1);
  const int64_t keys = max((int64_t)0, length - first);
  __syncthreads();
  float M = a.sinks ? bf16_bits_to_f32(a.sinks[h]) : -INFINITY, L = a.sinks ? 1.f : 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int64_t base = (int64_t)s * a.seq_stride + (int64_t)g * D;
  for (int64_t t = 0; t < keys + a.N; t += 64) {
    const int64_t j = t + lane;
    const C *kr = nullptr;
    if (j < keys) {
      const int64_t row = a.ring ? (first + j) % a.rows : first + j;
      kr = (const C *)a.k + base + row * a.kvh * D;
    } else if (j < keys + a.N) {
      const int m = (int)(j - keys);
      const int dm = __popcll(own & ((2ull << m) - 1)) - 1;   // the ancestor's depth
      if ((own >> m & 1) && (!a.window || dm + length > pos - a.window))
        kr = (const C *)a.dk + ((int64_t)s * a.N + m) * a.kv_stride + (int64_t)g * D;
    }
    float x = -INFINITY;
    if (kr) {
      x = 0.f;
      for (int i = 0; i < D; ++i) x = fmaf(s_q[i], elem_f32(kr + i), x);
    }
    const float mn = fmaxf(M, wmax(x));
    const float p = kr ? __expf(x - mn) : 0.f;
    const float corr = mn == -INFINITY ? 1.f : __expf(M - mn);
    L = L * corr + wsum(p);
    M = mn;
    s_p[lane] = p;
    const uint64_t used = __ballot(kr != nullptr);
    __syncthreads();
    for (int i = 0; i < 4; ++i) acc[i] *= corr;
    for (int jj = 0; jj < 64; ++jj) {
      if (!(used >> jj & 1)) continue;
      const int64_t j2 = t + jj;
      const C *vr;
      if (j2 < keys) {
        const int64_t row = a.ring ? (first + j2) % a.rows : first + j2;
        vr = (const C *)a.v + base + row * a.kvh * D;
      } else {
        vr = (const C *)a.dv + ((int64_t)s * a.N + (j2 - keys)) * a.kv_stride + (int64_t)g * D;
      }
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D) acc[i] = fmaf(s_p[jj], elem_f32(vr + lane + 64 * i), acc[i]);
    }
    __syncthreads();
  }
  const int64_t o = (((int64_t)s * a.N + n) * a.qh + h) * D;
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < D) ((Q *)a.out)[o + lane + 64 * i] = (Q)(acc[i] / L);
  if (lane == 0 && a.lse) a.lse[((int64_t)s * a.N + n) * a.qh + h] = M + __logf(L);
}

// One wave per (sequence, kv head, 64 rows), a lane per row.
template <class Q, class C>
__global__ __launch_bounds__(64) void weights_kernel(TreeArgs a) {
  const int tiles = (a.rows + 63) / 64;
  const int t = blockIdx.x % tiles, g = blockIdx.x / tiles % a.kvh, s = blockIdx.x / (tiles * a.kvh);
  const int row = t * 64 + threadIdx.x, D = a.d, qm = a.qh / a.kvh;
  const int length = min(max(a.lengths[s], 0), a.rows);
  const int acc = min(max(a.accepted[s], 0), min(a.N, length));
  if (row >= length) return;
  const C *kr = (const C *)a.k + (int64_t)s * a.seq_stride + ((int64_t)row * a.kvh + g) * D;
  float w = 0.f;
  for (int i = 0; i < acc; ++i) {
    const int n = a.path[(int64_t)s * a.N + i];
    if (n < 0 || n >= a.N || row > length - acc + i) continue;
    for (int h = g * qm; h < (g + 1) * qm; ++h) {
      const Q *q = (const Q *)a.q + ((int64_t)s * a.N + n) * a.q_stride + (int64_t)h * D;
      float x = 0.f;
      for (int e = 0; e < D; ++e) x = fmaf(elem_f32(q + e), elem_f32(kr + e), x);
      w += __expf(x * a.scale - a.lse_in[((int64_t)s * a.N + n) * a.qh + h]);
    }
  }
  a.weights[((int64_t)s * a.kvh + g) * a.rows + row] += w;
}

hipError_t launch_tree(const TreeArgs &a, int type, hipStream_t s) {
  const dim3 grid(a.S * a.N * a.qh);
  if (type == E_F32) hipLaunchKernelGGL((tree_kernel<float, _Float16>), grid, dim3(64), 0, s, a);
  else if (type == E_F16) hipLaunchKernelGGL((tree_kernel<_Float16, _Float16>), grid, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((tree_kernel<__bf16, __bf16>), grid, dim3(64), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_weights(const TreeArgs &a, int type, hipStream_t s) {
  const dim3 grid(a.S * a.kvh * ((a.rows + 63) / 64));
  if (type == E_F32) hipLaunchKernelGGL((weights_kernel<float, _Float16>), grid, dim3(64), 0, s, a);
  else if (type == E_F16) hipLaunchKernelGGL((weights_kernel<_Float16, _Float16>), grid, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((weights_kernel<__bf16, __bf16>), grid, dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace hh
