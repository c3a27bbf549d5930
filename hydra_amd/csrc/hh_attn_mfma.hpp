// hh_attn_mfma.hpp — what the attention kernels on the 32x32 MFMA share (hh_tree.hip, hh_hist_attn.hpp): the product, exchanges
// between a row's two lanes, exponentials, and probabilities as terms of the values' type.
#pragma once
#include "hh_common.hpp"

namespace hh {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <bool BF> __device__ __forceinline__ f32x16 mfma32(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// The value of the other half of the wave (lane ^ 32).
__device__ __forceinline__ float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// M follows a row's maximum by steps of at least kLag: rescaling costs more than what it keeps small, and with
// M moved at every new maximum some row of 32 moved it at nearly every tile. p = 2^(y − M + kOff) fits fp16: at most 2^14.5, and
// no more where the two are rounded to what fp32 holds beside M. The largest p of a row is 2^7 or more, so that fp16's smallest
// step holds each to 2^-32 of it.
constexpr float kOff = 7.f, kLag = 7.5f;
constexpr float kNone = -3.402823466e38f;    // a maximum of nothing: finite, so that no difference of maxima is NaN, and below none

// Two probabilities as fp16 pairs: hi cut off, lo the rest of it, rounded. minus1 is −1 in a register: with
// the constant the compiler makes a conversion and a subtraction of the one mixed-precision instruction.
__device__ __forceinline__ u32x2 split_pair(float p0, float p1, float minus1) {
  const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(p0, p1));
  const f16x2 l = {(_Float16)fmaf((float)h[0], minus1, p0), (_Float16)fmaf((float)h[1], minus1, p1)};
  return u32x2{__builtin_bit_cast(uint32_t, h), __builtin_bit_cast(uint32_t, l)};
}
// The same in bf16: to 2^-15 of each.
__device__ __forceinline__ u32x2 split_pair_bf16(float p0, float p1) {
  const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
  const bf16x2 l = {(__bf16)(p0 - __uint_as_float(u0 & 0xFFFF0000u)), (__bf16)(p1 - __uint_as_float(u1 & 0xFFFF0000u))};
  return u32x2{__builtin_amdgcn_perm(u1, u0, 0x07060302u), __builtin_bit_cast(uint32_t, l)};
}

}  // namespace hh
