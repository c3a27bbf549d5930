// hh_rotary.hip — rotary positions of queries and keys in one launch.
//
// y1 = m (x1 cos a − x2 sin a), y2 = m (x2 cos a + x1 sin a), a = 2 pi · position · turns_i. The angle is formed in turns: the
// fp64 product of position and frequency loses its whole turns exactly, and what is left, within half a turn, is rounded to
// fp32 (2^-25 of a turn) for sine and cosine. A workgroup takes some tokens, puts the sines and cosines of their pairs
// into LDS once for all heads, and passes over the heads' columns in 16-byte pieces; both tensors are read and written once.
#include "hh_hist.hpp"

namespace hh {

constexpr int kRotaryPairs = 2048;   // of a workgroup's tokens: 16 KB of LDS

// T: float, _Float16 or __bf16. MODE 0: pairs of neighbours, 1: halves whose distance is whole pieces, 2: any halves.
template <typename T, int MODE> __global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
  __shared__ float s_cos[kRotaryPairs], s_sin[kRotaryPairs];
  warm_kernargs<sizeof(RotaryArgs)>();
  const int tid = threadIdx.x, part = blockIdx.x % a.parts, half = a.span / 2, pairs = a.rotated / 2;
  const int t0 = blockIdx.x / a.parts * a.per_block, nt = min(a.per_block, a.tokens - t0);
  for (int e = tid; e < nt * pairs; e += 256) {
    const int t = e / pairs, i = e - t * pairs;
    const double x = (double)a.positions[t0 + t] * a.turns[i];
    float sn, cs;
    sincospif((float)(2.0 * (x - rint(x))), &sn, &cs);
    s_cos[e] = a.magnitude * cs;
    s_sin[e] = a.magnitude * sn;
  }
  __syncthreads();
  const int pieces = a.d / V, all = nt * (a.r[0].heads + (a.count > 1 ? a.r[1].heads : 0)) * pieces;
  for (int e = part * 256 + tid; e < all; e += a.parts * 256) {
    int at = e;
    const int first = nt * a.r[0].heads * pieces;
    const bool second = e >= first;
    const RotaryRows &r = a.r[second];
    if (second) at -= first;
    const int c = at % pieces * V, th = at / pieces, hd = th % r.heads, t = th / r.heads;
    const T *x = (const T *)r.x + (int64_t)(t0 + t) * r.x_stride + (int64_t)hd * a.d;
    T *y = (T *)r.y + (int64_t)(t0 + t) * r.y_stride + (int64_t)hd * a.d;
    const float *cs = s_cos + t * pairs, *sn = s_sin + t * pairs;
    if constexpr (MODE == 0) {
      vec v = *(const vec *)(x + c);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const int i = (c + j) / 2;
        if (i >= pairs) break;
        const float x1 = (float)v[j], x2 = (float)v[j + 1];
        v[j] = (T)fmaf(x1, cs[i], -(x2 * sn[i]));
        v[j + 1] = (T)fmaf(x2, cs[i], x1 * sn[i]);
      }
      *(vec *)(y + c) = v;
    } else if constexpr (MODE == 1) {
      // The piece of the pairs' second columns is written by the thread of their first.
      if (c >= half && c < a.span) continue;
      vec v = *(const vec *)(x + c);
      if (c < half) {
        vec w = *(const vec *)(x + c + half);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = c + j;
          if (i >= pairs) break;
          const float x1 = (float)v[j], x2 = (float)w[j];
          v[j] = (T)fmaf(x1, cs[i], -(x2 * sn[i]));
          w[j] = (T)fmaf(x2, cs[i], x1 * sn[i]);
        }
        *(vec *)(y + c + half) = w;
      }
      *(vec *)(y + c) = v;
    } else {
      // Column by column: a pair by the thread of its first column, and columns of no pair.
      for (int j = 0; j < V; ++j) {
        const int k = c + j, i = k;
        if (i < pairs) {
          const float x1 = (float)x[i], x2 = (float)x[i + half];
          y[i] = (T)fmaf(x1, cs[i], -(x2 * sn[i]));
          y[i + half] = (T)fmaf(x2, cs[i], x1 * sn[i]);
        } else if (k < half || k >= half + pairs) {
          y[k] = x[k];
        }
      }
    }
  }
}

template <typename T> static void launch_rotary_t(const RotaryArgs &a, dim3 grid, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  if (a.interleaved) hipLaunchKernelGGL((rotary_kernel<T, 0>), grid, dim3(256), 0, s, a);
  else if (a.span / 2 % V == 0) hipLaunchKernelGGL((rotary_kernel<T, 1>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, 2>), grid, dim3(256), 0, s, a);
}

hipError_t launch_rotary(RotaryArgs a, hipStream_t s) {
  const int heads = a.r[0].heads + (a.count > 1 ? a.r[1].heads : 0), pieces = a.d / (a.type == E_F32 ? 4 : 8);
  a.per_block = kRotaryPairs / (a.rotated / 2);
  int fill = (a.tokens + 1023) / 1024;
  if (fill > 64) fill = 64;
  if (a.per_block > fill) a.per_block = fill;
  if (a.per_block < 1) a.per_block = 1;
  const int blocks = (a.tokens + a.per_block - 1) / a.per_block;
  a.parts = 1;
  while (a.parts * blocks < 512 && a.parts * 256 < a.per_block * heads * pieces) a.parts *= 2;
  const dim3 grid((uint32_t)(blocks * a.parts));
  if (a.type == E_F32) launch_rotary_t<float>(a, grid, s);
  else if (a.type == E_F16) launch_rotary_t<_Float16>(a, grid, s);
  else launch_rotary_t<__bf16>(a, grid, s);
  return hipGetLastError();
}

}  // namespace hh
