// hh_rotary.hip — rotary positions of queries and keys in one launch.
//
// y1 = m (x1 cos a − x2 sin a), y2 = m (x2 cos a + x1 sin a), a = 2 pi · position · turns_i. The angle is formed in turns: the
// fp64 product of position and frequency loses its whole turns exactly, and what is left, within half a turn, is rounded to
// fp32 (2^-25 of a turn) for sine and cosine. A workgroup takes some tokens, puts the sines and cosines of their pairs
// into LDS once for all heads, and passes over the heads' columns in 16-byte pieces; both tensors are read and written once. Bound by the
// bytes: 16384 tokens of 18 heads of 256, 64 columns turned, bf16, 302 MB in 55 us (5.5 TB/s); one token of 72 heads 2.7 us, its latencies. Halves whose
// distance is no whole pieces go column by column: 18 heads of 96, 24 columns turned, 113 MB in 96 us (1.2 TB/s).
#include "hh_hist.hpp"

namespace hh {

constexpr int kRotaryPairs = 2048;   // of a workgroup's tokens: 16 KB of LDS

// T: float, _Float16 or __bf16. MODE 0: pairs of neighbours, 1: halves whose distance is whole pieces, 2: any halves. A row (token, head) has
// 2^lanes lanes, a piece each: of MODE 1 those of the first half, which write the second's too, and those behind the pairs' span.
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
  const int heads = a.r[0].heads + (a.count > 1 ? a.r[1].heads : 0), rows = nt * heads, each = 256 >> a.lanes, stride = a.parts * each;
  const int piece = tid & ((1 << a.lanes) - 1);
  const int c = (MODE == 1 && piece >= half / V ? piece + half / V : piece) * V;
  if (c >= a.d) return;
  // One row at a time: two in flight a lane took 1.2 times as long, four 1.5 times (16384 tokens of 18 heads of 256, bf16).
  for (int r = part * each + (tid >> a.lanes); r < rows; r += stride) {
    const int t = (int)((uint32_t)r / (uint32_t)heads), h = r - t * heads;
    const bool second = h >= a.r[0].heads;
    const RotaryRows &z = a.r[second];
    const int64_t o = (int64_t)(h - (second ? a.r[0].heads : 0)) * a.d;
    const T *x = (const T *)z.x + (int64_t)(t0 + t) * z.x_stride + o;
    T *y = (T *)z.y + (int64_t)(t0 + t) * z.y_stride + o;
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
        const int k = c + j;
        if (k < pairs) {
          const float x1 = (float)x[k], x2 = (float)x[k + half];
          y[k] = (T)fmaf(x1, cs[k], -(x2 * sn[k]));
          y[k + half] = (T)fmaf(x2, cs[k], x1 * sn[k]);
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
  const int heads = a.r[0].heads + (a.count > 1 ? a.r[1].heads : 0), V = a.type == E_F32 ? 4 : 8;
  int pieces = a.d / V;                      // at most 256
  if (!a.interleaved && a.span / 2 % V == 0) pieces -= a.span / 2 / V;
  while (1 << a.lanes < pieces) ++a.lanes;
  const int each = 256 >> a.lanes;
  // Four tokens a workgroup (54 us; one: 62, sixteen: 84), fewer where they fill LDS or there are few: then several share a token's heads.
  a.per_block = kRotaryPairs / (a.rotated / 2);
  const int fill = a.tokens / 1024 < 4 ? a.tokens / 1024 : 4;
  if (a.per_block > fill) a.per_block = fill;
  if (a.per_block < 1) a.per_block = 1;
  const int blocks = (a.tokens + a.per_block - 1) / a.per_block;
  a.parts = 1;
  while ((int64_t)a.parts * blocks < 1024 && a.parts * each < a.per_block * heads) a.parts *= 2;
  const dim3 grid((uint32_t)(blocks * a.parts));
  if (a.type == E_F32) launch_rotary_t<float>(a, grid, s);
  else if (a.type == E_F16) launch_rotary_t<_Float16>(a, grid, s);
  else launch_rotary_t<__bf16>(a, grid, s);
  return hipGetLastError();
}

}  // namespace hh
