// hh_hist_rows.hip — a step's keys and values into a history, quantised, and rows back as numbers.
//
// Eight columns a lane, four lanes a scale: the largest magnitude of 32 columns by two exchanges, the scale's exponent from
// its bits, and x·2^-e, exact, through the conversion to e4m3 or e2m1, to nearest even. Lanes run over a head's columns, then over
// the tokens, so that both sides move whole stretches: [token][head] on one, [head][row] on the other. Bound by the bytes: two prompts of up to
// 8000 tokens, 8 heads of 128, bf16 into 4 bits 16.5 us and back 14.6 (62 MB in and out each way: 3.8 and 4.3 TB/s, a copy 5.2); a step of 32 tokens
// 3 us each, its latencies.
#include "hh_hist.hpp"

namespace hh {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Eight numbers of a row in a type's bits.
template <int T> __device__ __forceinline__ void load8(const void *p, int64_t at, float (&x)[8]) {
  if constexpr (T == E_F32) {
    const f32x4 *q = (const f32x4 *)((const float *)p + at);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else if constexpr (T == E_F16) {
    const f16x8 a = *(const f16x8 *)((const _Float16 *)p + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  } else {
    const bf16x8 a = *(const bf16x8 *)((const __bf16 *)p + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
  }
}
template <int T> __device__ __forceinline__ void store8(void *p, int64_t at, const float (&x)[8]) {
  if constexpr (T == E_F32) {
    f32x4 *q = (f32x4 *)((float *)p + at);
    q[0] = f32x4{x[0], x[1], x[2], x[3]};
    q[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else if constexpr (T == E_F16) {
    f16x8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (_Float16)x[i];
    *(f16x8 *)((_Float16 *)p + at) = a;
  } else {
    bf16x8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (__bf16)x[i];
    *(bf16x8 *)((__bf16 *)p + at) = a;
  }
}

// Eight columns of a group that the four lanes l & ~3 .. l | 3 hold.
template <int FMT> __device__ __forceinline__ void encode8(float (&x)[8], uint32_t (&w)[2], uint32_t &scale) {
  uint32_t top = 0;   // magnitudes in order as bits: an infinity or a NaN is above every number
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2));
  // top = m·2^t, and the format's largest M·2^E: e = t − E, one more where m > M.
  constexpr uint32_t M = FMT == H_MXFP8 ? 0x600000u : 0x400000u;   // 1.75, 1.5
  constexpr int E = FMT == H_MXFP8 ? 8 : 2;
  const bool odd = top >= 0x7F800000u;
  const int e = max((int)(top >> 23) - E + ((top & 0x7FFFFFu) > M ? 1 : 0), 1);   // biased
  scale = odd ? 255u : (uint32_t)e;
  const float by = odd ? 0.f : __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = odd ? 0.f : x[i] * by;
  if constexpr (FMT == H_MXFP8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], v, true);
    }
  } else {
    uint32_t v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], 1.f, 0);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[2], x[3], 1.f, 1);
    v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[4], x[5], 1.f, 2);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[6], x[7], 1.f, 3);
    w[1] = 0;
  }
}

template <int FMT> __device__ __forceinline__ void decode8(const uint8_t *row, const uint8_t *scales, int c, float (&x)[8]) {
  if constexpr (FMT == H_F16) {
    load8<E_F16>(row, c, x);
  } else if constexpr (FMT == H_BF16) {
    load8<E_BF16>(row, c, x);
  } else if constexpr (FMT == H_MXFP8) {
    const u32x2 w = *(const u32x2 *)(row + c);
    const float by = hist_scale(scales[c >> 5]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 0) * by;
      x[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 1) * by;
      x[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 2) * by;
      x[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)w[i], 3) * by;
    }
  } else {
    const bf16x8 v = mxfp4_to_bf16(*(const uint32_t *)(row + (c >> 1)), 1.f);
    const float by = hist_scale(scales[c >> 5]);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i] * by;
  }
}

// A workgroup's rows: of one sequence's keys or values, heads outermost, U of 256·8 / d at a time each lane.
template <int U> struct RowItems {
  int s, v, c;
  int g[U], i[U];              // head, token; token −1: none
  __device__ __forceinline__ RowItems(const HistRowsArgs &a) {
    const int lanes = a.d / 8, each = 256 / lanes, r0 = (int)blockIdx.x * each * U + (int)threadIdx.x / lanes;
    s = blockIdx.y >> 1, v = blockIdx.y & 1, c = (int)threadIdx.x % lanes * 8;
    const int count = step_count(a.counts, s, a.N), rows = a.kvh * a.N;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * each;
      g[u] = (int)((uint32_t)r / (uint32_t)a.N);
      i[u] = r - g[u] * a.N;
      if (r >= rows || i[u] >= count) i[u] = -1;
    }
  }
};

template <int T, int FMT, int U> __global__ __launch_bounds__(256) void history_write_kernel(HistRowsArgs a) {
  warm_kernargs<sizeof(HistRowsArgs)>();
  const RowItems<U> p(a);      // a group's four lanes together
  const int count = step_count(a.counts, p.s, a.N), length = hist_length(a.h.lengths, p.s);
  const void *from = p.v ? a.v : a.k;
  uint8_t *codes = p.v ? a.h.v : a.h.k, *scales = p.v ? a.h.vs : a.h.ks;
  float x[U][8];
  int row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    row[u] = -1;
    if (p.i[u] < 0) continue;
    const int at = length + p.i[u];
    // Of a step longer than the ring the last.
    if (a.h.ring && at >= a.h.pinned && at < length + count - (a.h.rows - a.h.pinned)) continue;
    row[u] = hist_row(a.h, at);
    if (row[u] >= 0) load8<T>(from, ((int64_t)p.s * a.N + p.i[u]) * a.kv_stride + (int64_t)p.g[u] * a.d + p.c, x[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row[u] < 0) continue;
    const int64_t r = ((int64_t)p.s * a.kvh + p.g[u]) * a.h.rows + row[u];
    uint8_t *to = codes + r * hist_row_bytes(FMT, a.d);
    if constexpr (FMT == H_F16) {
      store8<E_F16>(to, p.c, x[u]);
    } else if constexpr (FMT == H_BF16) {
      store8<E_BF16>(to, p.c, x[u]);
    } else {
      uint32_t w[2], scale;
      encode8<FMT>(x[u], w, scale);
      if constexpr (FMT == H_MXFP8) *(u32x2 *)(to + p.c) = u32x2{w[0], w[1]};
      else *(uint32_t *)(to + p.c / 2) = w[0];
      if ((p.c & 31) == 0) (scales + r * (a.d / 32))[p.c >> 5] = (uint8_t)scale;
    }
  }
}

template <int T, int FMT, int U> __global__ __launch_bounds__(256) void history_read_kernel(HistRowsArgs a) {
  warm_kernargs<sizeof(HistRowsArgs)>();
  const RowItems<U> p(a);
  const uint8_t *codes = p.v ? a.h.v : a.h.k, *scales = p.v ? a.h.vs : a.h.ks;
  void *to = p.v ? a.vo : a.ko;
  float x[U][8];
  int row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    row[u] = -1;
    const int64_t at = (int64_t)a.starts[p.s] + p.i[u];
    if (p.i[u] < 0 || at < 0 || at > INT32_MAX) continue;
    row[u] = hist_row(a.h, (int)at);
    if (row[u] < 0) continue;
    const int64_t r = ((int64_t)p.s * a.kvh + p.g[u]) * a.h.rows + row[u];
    decode8<FMT>(codes + r * hist_row_bytes(FMT, a.d), scales + r * (a.d / 32), p.c, x[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (row[u] >= 0) store8<T>(to, (((int64_t)p.s * a.N + p.i[u]) * a.kvh + p.g[u]) * a.d + p.c, x[u]);
}

__global__ __launch_bounds__(64) void history_advance_kernel(int32_t *lengths, const int32_t *counts, int S, int N) {
  const int s = blockIdx.x * 64 + threadIdx.x;
  if (s < S) lengths[s] = min(hist_length(lengths, s) + step_count(counts, s, N), kHistLength);
}

constexpr int kRowsAhead = 4;  // rows that a lane has in flight, where there are enough to fill the chip (two prompts of 8000: 34 us, 47 with one)
template <int T, int FMT> static void launch_rows_tf(const HistRowsArgs &a, bool write, hipStream_t s) {
  const int64_t rows = (int64_t)a.kvh * a.N, each = 256 / (a.d / 8);
  const bool ahead = 2 * rows * a.S >= 1024 * kRowsAhead * each;
  const int64_t per = ahead ? kRowsAhead * each : each;
  const dim3 grid((uint32_t)((rows + per - 1) / per), 2 * a.S), block(256);
  if (write) {
    if (ahead) hipLaunchKernelGGL((history_write_kernel<T, FMT, kRowsAhead>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((history_write_kernel<T, FMT, 1>), grid, block, 0, s, a);
  } else {
    if (ahead) hipLaunchKernelGGL((history_read_kernel<T, FMT, kRowsAhead>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((history_read_kernel<T, FMT, 1>), grid, block, 0, s, a);
  }
}
template <int T> static void launch_rows_t(const HistRowsArgs &a, bool write, hipStream_t s) {
  if (a.format == H_F16) launch_rows_tf<T, H_F16>(a, write, s);
  else if (a.format == H_BF16) launch_rows_tf<T, H_BF16>(a, write, s);
  else if (a.format == H_MXFP8) launch_rows_tf<T, H_MXFP8>(a, write, s);
  else launch_rows_tf<T, H_MXFP4>(a, write, s);
}
static hipError_t launch_rows(const HistRowsArgs &a, bool write, hipStream_t s) {
  if (a.type == E_F32) launch_rows_t<E_F32>(a, write, s);
  else if (a.type == E_F16) launch_rows_t<E_F16>(a, write, s);
  else launch_rows_t<E_BF16>(a, write, s);
  return hipGetLastError();
}
hipError_t launch_history_write(const HistRowsArgs &a, hipStream_t s) { return launch_rows(a, true, s); }
hipError_t launch_history_read(const HistRowsArgs &a, hipStream_t s) { return launch_rows(a, false, s); }
hipError_t launch_history_advance(int32_t *lengths, const int32_t *counts, int S, int N, hipStream_t s) {
  hipLaunchKernelGGL(history_advance_kernel, dim3((S + 63) / 64), dim3(64), 0, s, lengths, counts, S, N);
  return hipGetLastError();
}

}  // namespace hh
