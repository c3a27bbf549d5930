// hh_hist_attn.hip — attention of a step's tokens over a history in 16, 8 or 4 bits, and over a prefix that the batch shares.
//
// One wave a (token, query head), its columns spread over the lanes: one pass over the keys that the token sees, with the running
// maximum and sum.
#include "hh_hist.hpp"

namespace hh {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNone = -3.402823466e38f;

template <int FMT> __device__ __forceinline__ float number_at(const uint8_t *row, const uint8_t *scales, int c) {
  if constexpr (FMT == H_F16) return (float)((const _Float16 *)row)[c];
  else if constexpr (FMT == H_BF16) return bf16_bits_to_f32(((const uint16_t *)row)[c]);
  else if constexpr (FMT == H_MXFP8) return __builtin_amdgcn_cvt_f32_fp8((int)row[c], 0) * hist_scale(scales[c >> 5]);
  else {
    const uint32_t n = row[c >> 1] >> 4 * (c & 1) & 15;
    const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(n, 1.f, 0);
    return (float)v[0] * hist_scale(scales[c >> 5]);
  }
}

template <typename T, int FMT> __global__ __launch_bounds__(256) void history_attention_kernel(HistAttnArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.S * a.N * a.qh) return;
  const int head = (int)(row % a.qh), i = (int)(row / a.qh % a.N), s = (int)(row / ((int64_t)a.qh * a.N)), g = head / a.qm;
  if (i >= step_count(a.counts, s, a.N)) return;
  const int own = hist_length(a.h.lengths, s) + i, n = a.d / 64;
  const T *q = (const T *)a.q + ((int64_t)s * a.N + i) * a.q_stride + (int64_t)head * a.d;
  float x[4], o[4], m = kNone, l = 0.f;
  for (int j = 0; j < n; ++j) x[j] = (float)q[lane + 64 * j], o[j] = 0.f;
  const int rb = hist_row_bytes(FMT, a.d);
  auto key = [&](const HistView &h, int64_t r) {
    const uint8_t *k = h.k + r * rb, *v = h.v + r * rb, *ks = h.ks + r * (a.d / 32), *vs = h.vs + r * (a.d / 32);
    float dot = 0.f;
    for (int j = 0; j < n; ++j) dot = fmaf(x[j], number_at<FMT>(k, ks, lane + 64 * j), dot);
    for (int b = 32; b; b >>= 1) dot += __shfl_xor(dot, b);
    const float y = dot * a.scale * kLog2e, mn = fmaxf(m, y), corr = __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(y - mn);
    m = mn;
    l = fmaf(l, corr, p);
    for (int j = 0; j < n; ++j) o[j] = fmaf(o[j], corr, p * number_at<FMT>(v, vs, lane + 64 * j));
  };
  if (a.p.k) {
    const int length = min(hist_length(a.p.lengths, 0), a.p.rows);
    for (int p = 0; p < length; ++p) key(a.p, (int64_t)g * a.p.rows + p);
  }
  const int last = a.h.ring ? own : min(own, a.h.rows - 1);
  const int low = a.window ? max(0, own - a.window + 1) : 0, first = min(a.first, low);
  const int64_t base = ((int64_t)s * a.kvh + g) * a.h.rows;
  for (int p = 0; p < first && p <= last; ++p) key(a.h, base + hist_row(a.h, p));
  for (int p = low; p <= last; ++p) key(a.h, base + hist_row(a.h, p));
  if (a.sinks) {
    const float y = bf16_bits_to_f32(a.sinks[head]) * kLog2e, mn = fmaxf(m, y), f = __builtin_amdgcn_exp2f(m - mn);
    l = fmaf(l, f, __builtin_amdgcn_exp2f(y - mn));
    for (int j = 0; j < n; ++j) o[j] *= f;
    m = mn;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int j = 0; j < n; ++j) ((T *)a.out)[row * a.d + lane + 64 * j] = (T)(o[j] * inv);
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T> static void launch_t(const HistAttnArgs &a, dim3 grid, hipStream_t s) {
  if (a.format == H_F16) hipLaunchKernelGGL((history_attention_kernel<T, H_F16>), grid, dim3(256), 0, s, a);
  else if (a.format == H_BF16) hipLaunchKernelGGL((history_attention_kernel<T, H_BF16>), grid, dim3(256), 0, s, a);
  else if (a.format == H_MXFP8) hipLaunchKernelGGL((history_attention_kernel<T, H_MXFP8>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((history_attention_kernel<T, H_MXFP4>), grid, dim3(256), 0, s, a);
}

hipError_t launch_history_attention(const HistAttnArgs &a, int type, hipStream_t s, int *launches) {
  const dim3 grid((uint32_t)(((int64_t)a.S * a.N * a.qh + 3) / 4));
  if (type == E_F32) launch_t<float>(a, grid, s);
  else if (type == E_F16) launch_t<_Float16>(a, grid, s);
  else launch_t<__bf16>(a, grid, s);
  *launches = 1;
  return hipGetLastError();
}

}  // namespace hh
