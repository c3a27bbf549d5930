// hh_rotary.hip — rotary positions of queries and keys in one launch.
//
// y1 = m (x1 cos a − x2 sin a), y2 = m (x2 cos a + x1 sin a), a = 2 pi · position · turns_i. The angle is formed in turns: the
// fp64 product of position and frequency loses its whole turns exactly, and what is left, within half a turn, is rounded to
// fp32 (2^-25 of a turn) for sine and cosine. A workgroup takes some tokens, puts the sines and cosines of their pairs
// into LDS once for all heads, and passes over the heads' columns in 16-byte pieces; both tensors are read and written once.
#include "hh_hist.hpp"

namespace hh {

constexpr int kRotaryPairs = 2048;   // of a workgroup's tokens: 16 KB of LDS
constexpr int kRotaryAhead = 4;      // rows that a thread has in flight

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
  for (int r0 = part * each + (tid >> a.lanes); r0 < rows; r0 += kRotaryAhead * stride) {
    const T *x[kRotaryAhead];
    T *y[kRotaryAhead];
    vec v[kRotaryAhead], w[kRotaryAhead];
    int at[kRotaryAhead];            // the token's sines, −1: no row
#pragma unroll
    for (int u = 0; u < kRotaryAhead; ++u) {
      const int r = r0 + u * stride;
      at[u] = -1;
      if (r >= rows) continue;
      const int t = (int)((uint32_t)r / (uint32_t)heads), h = r - t * heads;
      const bool second = h >= a.r[0].heads;
      const RotaryRows &z = a.r[second];
      const int64_t o = (int64_t)(h - (second ? a.r[0].heads : 0)) * a.d;
      at[u] = t * pairs;
      x[u] = (const T *)z.x + (int64_t)(t0 + t) * z.x_stride + o;
      y[u] = (T *)z.y + (int64_t)(t0 + t) * z.y_stride + o;
      if constexpr (MODE < 2) v[u] = *(const vec *)(x[u] + c);
      if (MODE == 1 && c < half) w[u] = *(const vec *)(x[u] + c + half);
    }
#pragma unroll
    for (int u = 0; u < kRotaryAhead; ++u) {
      if (at[u] < 0) continue;
      const float *cs = s_cos + at[u], *sn = s_sin + at[u];
      if constexpr (MODE == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const int i = (c + j) / 2;
          if (i >= pairs) break;
          const float x1 = (float)v[u][j], x2 = (float)v[u][j + 1];
          v[u][j] = (T)fmaf(x1, cs[i], -(x2 * sn[i]));
          v[u][j + 1] = (T)fmaf(x2, cs[i], x1 * sn[i]);
        }
        *(vec *)(y[u] + c) = v[u];
      } else if constexpr (MODE == 1) {
        if (c < half) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int i = c + j;
            if (i >= pairs) break;
            const float x1 = (float)v[u][j], x2 = (float)w[u][j];
            v[u][j] = (T)fmaf(x1, cs[i], -(x2 * sn[i]));
            w[u][j] = (T)fmaf(x2, cs[i], x1 * sn[i]);
          }
          *(vec *)(y[u] + c + half) = w[u];
        }
        *(vec *)(y[u] + c) = v[u];
      } else {
        // Column by column: a pair by the thread of its first column, and columns of no pair.
        for (int j = 0; j < V; ++j) {
          const int k = c + j;
          if (k < pairs) {
            const float x1 = (float)x[u][k], x2 = (float)x[u][k + half];
            y[u][k] = (T)fmaf(x1, cs[k], -(x2 * sn[k]));
            y[u][k + half] = (T)fmaf(x2, cs[k], x1 * sn[k]);
          } else if (k < half || k >= half + pairs) {
            y[u][k] = x[u][k];
          }
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
  // Sixteen tokens a workgroup, fewer where they fill LDS or there are few: then several share a token's heads.
  a.per_block = kRotaryPairs / (a.rotated / 2);
  const int fill = a.tokens / 1024 < 16 ? a.tokens / 1024 : 16;
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
