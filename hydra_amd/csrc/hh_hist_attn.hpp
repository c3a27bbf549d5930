// hh_hist_attn.hpp — attention of a step's tokens over a history in 16, 8 or 4 bits, and over a prefix that the batch shares: the
// kernels of one head_dim (hh_hist_attn_64/_128/_256.hip).
//
// A kv head's rows are its (token, query head) pairs, r = token·qm + head. Keys are numbered from 0 in the order of their positions:
// the first tokens, then those from the window's start of the block's first row on. One pass with the running maximum M and sum L of
// each row, in the exponent base 2, as in hh_tree.hip: S^T [32 keys × 32 rows] = K·q^T, O^T [D × 32 rows] += V^T·P^T, a row's
// probabilities in its two lanes all the way.
//
// Numbers in 8 and 4 bits become bf16 as they are loaded, exactly (4 and 2 bits of mantissa, any power of two), so products are those
// of the numbers held. Queries enter as the terms of bf16 that hold them (F16: two, F32: three; over F16 histories F32 as two of fp16),
// probabilities as two (outputs of 16 bits: to 2^-15 of each) or three (F32: as exact as the sums) of bf16, or two of fp16.
#pragma once
#include <type_traits>

#include "hh_attn_mfma.hpp"
#include "hh_hist.hpp"

namespace hh {

constexpr int kFewRows = 32;                 // rows of a kv head up to which a wave takes all of them

template <int QT, int FMT> struct HistTypes {
  static constexpr bool BF = FMT != H_F16, MX = FMT >= H_MXFP8;
  static constexpr int E = FMT == H_MXFP8 ? 16 : FMT == H_MXFP4 ? 32 : 8;                       // numbers of 16 bytes
  static constexpr int NQ = QT == E_F32 ? (BF ? 3 : 2) : QT == E_F16 && BF ? 2 : 1;             // terms of a query
  static constexpr int NP = QT == E_F32 && BF ? 3 : 2;                                          // of a probability
};

// 16 bytes of a row and their scale byte as MFMA operands of eight numbers. Scale byte 0 (2^-127) gives 0 or what it stands for; 255 is the
// caller's to see to.
template <int FMT> __device__ __forceinline__ void widen(const u32x4 &raw, uint32_t scale, u32x4 (&out)[HistTypes<0, FMT>::E / 8]) {
  if constexpr (FMT == H_F16 || FMT == H_BF16) {
    out[0] = raw;
  } else {
    const float by = __uint_as_float(scale << 23);
#pragma unroll
    for (int x = 0; x < HistTypes<0, FMT>::E / 8; ++x) {
      if constexpr (FMT == H_MXFP8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          out[x][2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[2 * x + i], by, false));
          out[x][2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[2 * x + i], by, true));
        }
      } else {
        out[x] = __builtin_bit_cast(u32x4, mxfp4_to_bf16(raw[x], by));
      }
    }
  }
}

template <int FMT> __device__ __forceinline__ float number_at(const uint8_t *row, const uint8_t *scales, int c) {
  if constexpr (FMT == H_F16) return (float)((const _Float16 *)row)[c];
  else if constexpr (FMT == H_BF16) return bf16_bits_to_f32(((const uint16_t *)row)[c]);
  else if constexpr (FMT == H_MXFP8) return __builtin_amdgcn_cvt_f32_fp8((int)row[c], 0) * hist_scale(scales[c >> 5]);
  else {
    const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(row[c >> 1] >> 4 * (c & 1) & 15u, 1.f, 0);
    return (float)v[0] * hist_scale(scales[c >> 5]);
  }
}

// What the rows of a block see: keys 0 .. n − 1, the first `fold` of them the first positions, the others from position `low` on.
struct Visible {
  int length, low, fold, last, n;
};
__device__ __forceinline__ Visible visible_of(const HistAttnArgs &a, int s, int i0, int i1) {
  Visible v;
  const HistView &h = a.h;
  v.length = hist_length(h.lengths, s);
  v.last = h.ring ? v.length + i1 : min(v.length + i1, h.rows - 1);
  v.low = a.window ? max(0, v.length + i0 - a.window + 1) : 0;
  v.fold = min(a.first, v.low);
  if (!h.ring) v.fold = min(v.fold, h.rows);
  v.n = v.fold + max(0, v.last - v.low + 1);
  return v;
}
__device__ __forceinline__ Visible visible_prefix(const HistAttnArgs &a) {
  Visible v;
  v.length = v.n = min(hist_length(a.p.lengths, 0), a.p.rows);
  v.low = v.fold = 0;
  v.last = v.n - 1;
  return v;
}
// Keys of a chunk: `per`, or more where the launch was sized for shorter histories.
__device__ __forceinline__ int chunk_keys(const HistAttnArgs::Pass &p, int n) {
  if ((int64_t)p.per * p.chunks >= n) return p.per;
  const int need = (int)((uint32_t)n / (uint32_t)p.chunks) + 1;
  return (int)(((uint32_t)need + p.tile - 1) / (uint32_t)p.tile * (uint32_t)p.tile);
}
__device__ __forceinline__ int used_chunks(int n, int per) { return n <= per ? 1 : (int)(((uint32_t)n + per - 1) / (uint32_t)per); }

// A block of rows of a pass: whose rows, what they see, and which keys of it are this workgroup's.
struct Block {
  int s, g, r0, count, chunk, c0, nc;       // keys c0 .. c0 + nc − 1
  Visible v;
  int first_low, last_low, first_high;      // of the first and the last row
  uint64_t k, v_, ks, vs;                   // the head's rows
  int rows, span, pinned, delta;            // position -> row
};
__device__ __forceinline__ int row_low(const HistAttnArgs &a, const Visible &v, int i) {
  return a.window ? v.fold + max(v.length + i - a.window + 1, v.low) - v.low : 0;
}
__device__ __forceinline__ int row_high(const Visible &v, int i) { return v.fold + max(0, min(v.length + i, v.last) - v.low + 1) - 1; }

template <int FMT, int D> __device__ __forceinline__ bool block_of(const HistAttnArgs &a, int sg, int rb, int chunk, Block &b) {
  const HistAttnArgs::Pass &p = a.shared ? a.pre : a.own;
  const HistView &h = a.shared ? a.p : a.h;
  b.s = a.shared ? 0 : sg / a.kvh;
  b.g = sg - b.s * a.kvh;
  b.r0 = rb * p.block_rows;
  b.chunk = chunk;
  int i0 = 0;
  if (a.shared) {
    b.count = a.S * a.N;
    b.v = visible_prefix(a);
    b.first_low = b.last_low = 0;
    b.first_high = b.v.n - 1;
  } else {
    b.count = step_count(a.counts, b.s, a.N);
    if (b.r0 >= b.count * a.qm) return false;
    i0 = b.r0 / a.qm;
    const int i1 = min(b.count, (b.r0 + p.block_rows - 1) / a.qm + 1) - 1;
    b.v = visible_of(a, b.s, i0, i1);
    b.first_low = row_low(a, b.v, i0);
    b.last_low = row_low(a, b.v, i1);
    b.first_high = row_high(b.v, i0);
  }
  const int per = chunk_keys(p, b.v.n);
  const int64_t c0 = (int64_t)chunk * per;
  if (chunk && c0 >= b.v.n) return false;
  b.c0 = (int)c0;
  b.nc = min(per, b.v.n - b.c0);
  const int64_t base = (int64_t)sg * h.rows;                 // sg counts the prefix's heads too
  b.k = (uint64_t)(h.k + base * hist_row_bytes(FMT, D));
  b.v_ = (uint64_t)(h.v + base * hist_row_bytes(FMT, D));
  b.ks = (uint64_t)(h.ks + base * (D / 32));
  b.vs = (uint64_t)(h.vs + base * (D / 32));
  b.rows = h.rows;
  b.pinned = h.ring ? h.pinned : 0;
  b.span = h.rows - b.pinned;
  b.delta = 0;
  if (h.ring) {
    const int from = max(b.v.low, b.pinned);
    b.delta = (int)((uint32_t)(from - b.pinned) % (uint32_t)b.span) + b.pinned - from;
  }
  return true;
}
// The row of key j, j clamped to those that there are (n > 0).
__device__ __forceinline__ int key_row(const Block &b, int j) {
  j = min(j, b.v.n - 1);
  const int p = j < b.v.fold ? j : j - b.v.fold + b.v.low;
  int r = p < b.pinned ? p : p + b.delta;
  return r >= b.rows ? r - b.span : r;
}
// The first x of 32 keys.
__device__ __forceinline__ uint32_t first_keys(int x) { return x >= 32 ? 0xFFFFFFFFu : x <= 0 ? 0u : (1u << x) - 1; }

// A lane's row: its token and head, and the keys that it sees: those below a.first, and low .. high.
struct Row {
  bool in;
  int s, i, head, low, high;
};
__device__ __forceinline__ Row row_of(const HistAttnArgs &a, const Block &b, int r) {
  Row x;
  const int t = r / a.qm;
  x.in = t < b.count;
  const int tt = x.in ? t : b.r0 / a.qm;                     // rows past the last stand for the block's first
  x.head = b.g * a.qm + (x.in ? r - t * a.qm : 0);
  if (a.shared) {
    x.s = tt / a.N;
    x.i = tt - x.s * a.N;
    x.in = x.in && x.i < step_count(a.counts, x.s, a.N);
    x.low = 0;
    x.high = b.v.n - 1;
  } else {
    x.s = b.s;
    x.i = tt;
    x.low = row_low(a, b.v, tt);
    x.high = row_high(b.v, tt);
  }
  return x;
}

// Eight columns of a query as NQ operands.
template <int QT, bool BF, int NQ> __device__ __forceinline__ void query_terms(const void *q, int64_t at, float scale, u32x4 (&out)[NQ]) {
  if constexpr (NQ == 1) {
    out[0] = *(const u32x4 *)((const uint16_t *)q + at);
  } else {
    float x[8];
    if constexpr (QT == E_F32) {
      const f32x4 *p = (const f32x4 *)((const float *)q + at);
      const f32x4 l = p[0], h = p[1];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = (e < 4 ? l[e & 3] : h[e & 3]) * scale;
        // Rounded to fp32 before it is split: a head from the product by one mixed-precision instruction differs near ties.
        asm volatile("" : "+v"(x[e]));
      }
    } else {
      const f16x8 v = *(const f16x8 *)((const _Float16 *)q + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
    }
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      if constexpr (BF) {
        bf16x8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (__bf16)x[e], x[e] -= (float)h[e];
        out[t] = __builtin_bit_cast(u32x4, h);
      } else {
        f16x8 h;
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] = (_Float16)x[e], x[e] -= (float)h[e];
        out[t] = __builtin_bit_cast(u32x4, h);
      }
    }
  }
}

// Two probabilities as NP terms: bf16 by cutting off, the last rounded.
template <bool BF, int NP> __device__ __forceinline__ void split_terms(float p0, float p1, float minus1, uint32_t (&w)[NP]) {
  if constexpr (!BF) {
    const u32x2 v = split_pair(p0, p1, minus1);
    w[0] = v[0], w[1] = v[1];
  } else {
    if constexpr (NP == 3) {
      const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
      w[0] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
      p0 -= __uint_as_float(u0 & 0xFFFF0000u);
      p1 -= __uint_as_float(u1 & 0xFFFF0000u);
    }
    const u32x2 v = split_pair_bf16(p0, p1);
    w[NP - 2] = v[0], w[NP - 1] = v[1];
  }
}

// A row's four outputs from its joined state: the sink's share of the denominator, the quotient, its rounding.
template <int QT, int D>
__device__ __forceinline__ void finish_history_row(const HistAttnArgs &a, int64_t row, int head, int q4, float m, float den, f32x4 o) {
  if (a.sinks) {
    const float y = bf16_bits_to_f32(a.sinks[head]) * kLog2e, mn = fmaxf(m, y), f = exp2_(m - mn);
    den = fmaf(den, f, exp2_(y - mn));
    o *= f;
    m = mn;
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;            // of nothing: 0
  if constexpr (QT == E_F32) {
    *(f32x4 *)((float *)a.out + row * D + 4 * q4) = o * inv;
  } else if constexpr (QT == E_F16) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *(f16x4 *)((_Float16 *)a.out + row * D + 4 * q4) = f16x4{(_Float16)(o[0] * inv), (_Float16)(o[1] * inv), (_Float16)(o[2] * inv), (_Float16)(o[3] * inv)};
  } else {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *(bf16x4 *)((__bf16 *)a.out + row * D + 4 * q4) = bf16x4{(__bf16)(o[0] * inv), (__bf16)(o[1] * inv), (__bf16)(o[2] * inv), (__bf16)(o[3] * inv)};
  }
  if (q4 == 0 && a.lse) a.lse[row] = den == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(den)) * kLn2;
}

// A row's state of one chunk, or its outputs where there is no other.
template <int QT, int D>
__device__ __forceinline__ void leave_row(const HistAttnArgs &a, const Block &b, const Row &x, int q4, float m, float den, f32x4 o) {
  const int64_t row = ((int64_t)x.s * a.N + x.i) * a.qh + x.head;
  if (a.chunks > 1) {
    const int64_t slot = row * a.chunks + (a.shared ? 0 : a.pre.chunks) + b.chunk;
    *(f32x4 *)(a.po + slot * D + 4 * q4) = o;
    if (q4 == 0) {
      a.pm[slot] = m;
      a.pl[slot] = den;
    }
  } else {
    finish_history_row<QT, D>(a, row, x.head, q4, m, den, o);
  }
}

// Infinities and NaN of an operand's eight numbers taken out: 0·NaN would carry them to rows that do not see them. They are put back
// into the rows that do behind the loop.
template <bool BF> __device__ __forceinline__ bool take_odd(u32x4 &x) {
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t em = BF ? 0x7F80u : 0x7C00u;
    const bool l = (x[e] & em) == em, h = (x[e] >> 16 & em) == em;
    x[e] &= (l ? 0u : 0xFFFFu) | (h ? 0u : 0xFFFF0000u);
    odd |= l || h;
  }
  return odd;
}
// What take_odd took out of keys j0 .. j1 − 1, for one row's four columns.
template <int FMT, int D>
__device__ void put_odd(const Block &b, int first, int low, int high, int j0, int j1, int q4, f32x4 &o) {
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    if (j > high || (j >= first && j < low)) continue;
    const int64_t r = key_row(b, j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = number_at<FMT>((const uint8_t *)b.v_ + r * hist_row_bytes(FMT, D), (const uint8_t *)b.vs + r * (D / 32), 4 * q4 + i);
      if (!(fabsf(v) < INFINITY)) o[i] += v;
    }
  }
}

// The rows' state over a run of 32 keys at a time.
template <int QT, int FMT, int D> struct RowState {
  using T = HistTypes<QT, FMT>;
  static constexpr int NB = D / 32;
  float M = kNone, L = 0.f;
  f32x16 acc[NB];
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x16{};
  }
  // S, in element i the logit of key 8 (i / 4) + 4 hh + i % 4, to probabilities: `sees` has a bit a key, from this lane's first.
  // `mem`: the values [32][D] in LDS, 16-byte pieces XORed by the row; vcol: this lane's part of reading them by columns.
  __device__ __forceinline__ void softmax(f32x16 &S, bool part, uint32_t sees, float scale) {
    if constexpr (QT != E_F32) S *= scale;                   // rounded to y once, before the maximum
    if (part) {
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = sees >> (8 * (i >> 2) + (i & 3)) & 1 ? S[i] : -INFINITY;
    }
    float top = fmaxf(S[0], S[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) top = fmaxf(top, S[i]);
    top = max_halves(top);
    if (__any(top - M > kLag)) {
      const float mn = fmaxf(M, top), corr = exp2_(M - mn);
      M = mn;
      L *= corr;
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[n] *= corr;
    }
    const float sub = kOff - M;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      S[i] = exp2_(S[i] + sub);
      sum[i & 3] += S[i];
    }
    L += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  }
  __device__ __forceinline__ void values(const f32x16 &S, const uint8_t *vcol, int vpiece, float minus1) {
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      u32x4 p[T::NP];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[T::NP];
        split_terms<T::BF, T::NP>(S[8 * kc + 2 * e], S[8 * kc + 2 * e + 1], minus1, w);
#pragma unroll
        for (int t = 0; t < T::NP; ++t) p[t][e] = w[t];
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        u32x4 vf;
#pragma unroll
        for (int x8 = 0; x8 < 2; ++x8) {
          const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4 *)(vcol + (16 * kc + 8 * x8) * 2 * D + ((vpiece ^ (4 * n)) << 4)));
          const u32x2 v = __builtin_bit_cast(u32x2, w);
          vf[2 * x8] = v[0];
          vf[2 * x8 + 1] = v[1];
        }
#pragma unroll
        for (int t = 0; t < T::NP; ++t) acc[n] = mfma32<T::BF>(vf, p[t], acc[n]);
      }
    }
  }
};
__device__ __forceinline__ int piece_xor(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

// Few rows: each wave has all of a kv head's (up to 32) and tiles of 32 keys of its own, W of them a workgroup; the next tile's bytes are
// in flight under this one's products. Keys go from memory to the operands' registers: the order of a product's columns is free, so
// that a lane's 16 bytes are its own; values pass through LDS to be read by columns. No barrier until the waves' states meet.
template <int QT, int FMT, int D, int W, int OCC>
__global__ __launch_bounds__(64 * W, OCC) void history_few_kernel(HistAttnArgs a) {
  using T = HistTypes<QT, FMT>;
  constexpr int E = T::E, U = D / (2 * E), X = E / 8, RB = D * 16 / E, NB = D / 32, ROWS = 32;
  __shared__ __align__(1024) uint8_t s_mem[W * ROWS * D * 4];
  __shared__ float s_m[W][ROWS], s_l[W][ROWS];
  __shared__ int s_lo[ROWS], s_hi[ROWS], s_odd;
  warm_kernargs<sizeof(HistAttnArgs)>();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hh = lane >> 5;
  const int heads = a.shared ? a.kvh : a.S * a.kvh;
  Block b;
  if (!block_of<FMT, D>(a, (int)(blockIdx.x % heads), 0, (int)(blockIdx.x / heads), b)) return;
  const Row row = row_of(a, b, l32);
  u32x4 q[D / 16][T::NQ];                    // fragment u·X + x: columns 2E u + E hh + 8 x
  {
    const int64_t at = ((int64_t)row.s * a.N + row.i) * a.q_stride + (int64_t)row.head * D + E * hh;
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
      query_terms<QT, T::BF, T::NQ>(a.q, at + 2 * E * (f / X) + 8 * (f % X), a.scale * kLog2e, q[f]);
  }
  const float scale = a.scale * kLog2e;
  if (wave == 0 && hh == 0) s_lo[l32] = row.low, s_hi[l32] = row.high;
  if (tid == 0) s_odd = 0;
  __syncthreads();

  const int tiles = (b.nc + 31) / 32;
  struct Raw {
    u32x4 k[U], v[U];
    uint64_t ks, vs;
  } raw;
  typedef typename std::conditional<D == 64, uint16_t, typename std::conditional<D == 128, uint32_t, uint64_t>::type>::type scales_t;
  auto fetch = [&](int t) {
    const uint64_t r = key_row(b, b.c0 + 32 * t + l32);
    const uint64_t at = r * RB + 16 * hh;
#pragma unroll
    for (int u = 0; u < U; ++u) raw.k[u] = *(const u32x4 *)(b.k + at + 32 * u);
    if constexpr (T::MX) raw.ks = *(const scales_t *)(b.ks + r * (D / 32));
#pragma unroll
    for (int u = 0; u < U; ++u) raw.v[u] = *(const u32x4 *)(b.v_ + at + 32 * u);
    if constexpr (T::MX) raw.vs = *(const scales_t *)(b.vs + r * (D / 32));
  };
  auto scale_of = [&](uint64_t s, int u) { return (uint32_t)(s >> (FMT == H_MXFP4 ? 8 * (2 * u + hh) : 8 * u)) & 0xFFu; };
  auto is_part = [&](int t) {
    const int j = b.c0 + 32 * t;
    return j + 31 > b.first_high || (j + 32 > a.first && j < b.last_low);
  };
  RowState<QT, FMT, D> st;
  st.init();
  float minus1 = -1.f;
  asm volatile("" : "+s"(minus1));
  uint8_t *vmem = s_mem + wave * (32 * D * 2);
  const int j16 = lane & 15;
  const int vrow = 4 * hh + (j16 >> 2), vpiece = (2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1)) ^ piece_xor(vrow);
  const uint8_t *vcol = vmem + vrow * (2 * D) + (j16 & 1) * 8;
  if (wave < tiles) fetch(wave);
  for (int t = wave; t < tiles; t += W) {
    const bool part = is_part(t);
    u32x4 kf[D / 16];
    bool bad = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      u32x4 w[X];
      const uint32_t sc = T::MX ? scale_of(raw.ks, u) : 0;
      widen<FMT>(raw.k[u], sc, w);
      if constexpr (T::MX) bad |= sc == 255;
#pragma unroll
      for (int x = 0; x < X; ++x) kf[u * X + x] = w[x];
    }
    if (T::MX && __any(bad)) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (scale_of(raw.ks, u) == 255)
#pragma unroll
          for (int x = 0; x < X; ++x) kf[u * X + x] = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
    }
    f32x16 S = f32x16{};
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
#pragma unroll
      for (int n = 0; n < T::NQ; ++n) S = mfma32<T::BF>(kf[f], q[f][n], S);
    asm volatile("" ::: "memory");           // the wave's last tile has been read: LDS takes its accesses in their order
#pragma unroll
    for (int u = 0; u < U; ++u) {
      u32x4 w[X];
      const uint32_t sc = T::MX ? scale_of(raw.vs, u) : 0;
      widen<FMT>(raw.v[u], sc, w);
      if (T::MX && __any(sc == 255)) {
        if (sc == 255)
#pragma unroll
          for (int x = 0; x < X; ++x) w[x] = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
      }
      if (part) {
        bool odd = false;
#pragma unroll
        for (int x = 0; x < X; ++x) odd |= take_odd<T::BF>(w[x]);
        if (odd) s_odd = 1;
      }
#pragma unroll
      for (int x = 0; x < X; ++x)
        *(u32x4 *)(vmem + l32 * (2 * D) + (((2 * E * u + E * hh + 8 * x) / 8 ^ piece_xor(l32)) << 4)) = w[x];
    }
    asm volatile("" ::: "memory");           // the rows are read by other lanes than wrote them, behind the writes
    if (t + W < tiles) fetch(t + W);
    uint32_t sees = 0;
    if (part) {
      const int j = b.c0 + 32 * t;
      sees = ((~first_keys(row.low - j) | first_keys(a.first - j)) & first_keys(row.high + 1 - j)) >> (4 * hh);
    }
    st.softmax(S, part, sees, scale);
    st.values(S, vcol, vpiece, minus1);
  }

  // The waves' states meet in LDS, the sums of a row in 16-byte pieces XORed by the row.
  st.L += other_half(st.L);
  __syncthreads();
  float *so = (float *)s_mem + (size_t)(wave * ROWS + l32) * D;
  if (hh == 0) {
    s_m[wave][l32] = st.M - kOff;            // the exponent that L and O are relative to
    s_l[wave][l32] = st.L;
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *(f32x4 *)(so + 4 * ((8 * n + 2 * e + hh) ^ (l32 & 7))) =
          f32x4{st.acc[n][4 * e], st.acc[n][4 * e + 1], st.acc[n][4 * e + 2], st.acc[n][4 * e + 3]};
  __syncthreads();
#pragma unroll 1
  for (int e = tid; e < ROWS * (D / 4); e += 64 * W) {
    const int r = e / (D / 4), q4 = e % (D / 4);
    const Row x = row_of(a, b, r);
    if (!x.in) continue;
    float m = s_m[0][r];
#pragma unroll
    for (int k = 1; k < W; ++k) m = fmaxf(m, s_m[k][r]);
    float den = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float f = exp2_(s_m[k][r] - m);
      den = fmaf(s_l[k][r], f, den);
      const f32x4 w = *(const f32x4 *)((const float *)s_mem + (size_t)(k * ROWS + r) * D + 4 * (q4 ^ (r & 7)));
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(w[i], f, o[i]);
    }
    if (s_odd)
      for (int t = 0; t < tiles; ++t)
        if (is_part(t)) put_odd<FMT, D>(b, a.first, s_lo[r], s_hi[r], b.c0 + 32 * t, min(b.c0 + 32 * t + 32, b.c0 + b.nc), q4, o);
    leave_row<QT, D>(a, b, x, q4, m, den, o);
  }
}

// Many rows: 128 a workgroup, 32 a wave; tiles of KT keys, whose 16-byte pieces the threads share, become operands in LDS, two tiles in
// turn, read by every wave. The bytes of the tile after the next are in flight under a tile's products. A tile's one barrier keeps
// the waves of a workgroup in step, so the workgroups are small: several a compute unit, each at its own place.
template <int QT, int FMT, int D, int KT, int OCC>
__global__ __launch_bounds__(256, OCC) void history_many_kernel(HistAttnArgs a) {
  using T = HistTypes<QT, FMT>;
  constexpr int E = T::E, X = E / 8, RB = D * 16 / E, PR = RB / 16, NB = D / 32, ROWS = 128;
  constexpr int ALL = 2 * KT * PR, NPC = (ALL + 255) / 256, STAGE = KT * D * 4;
  constexpr int OUTS = ROWS * D * 4;
  __shared__ __align__(1024) uint8_t s_mem[2 * STAGE > OUTS ? 2 * STAGE : OUTS];
  __shared__ int s_odd;
  warm_kernargs<sizeof(HistAttnArgs)>();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hh = lane >> 5;
  // Each XCD takes a stretch of the list (head and chunk, block of rows), so that what it reads again is in its L2; a block's share of
  // a head that several XCDs have is spread over its rows, the ones that see most first.
  const HistAttnArgs::Pass &pass = a.shared ? a.pre : a.own;
  const int heads = a.shared ? a.kvh : a.S * a.kvh, groups = heads * pass.chunks;
  const int parts = groups >= 8 ? 1 : (8 + groups - 1) / groups, share = (pass.row_blocks + parts - 1) / parts;
  const uint32_t all = (uint32_t)groups * (uint32_t)(share * parts), each = (all + 7) / 8, w = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= each || w >= all) return;
  const int grp = (int)(w / (uint32_t)(share * parts)), at = (int)(w - (uint32_t)grp * (uint32_t)(share * parts));
  const int rb = pass.row_blocks - 1 - (at % share * parts + at / share);
  if (rb < 0) return;
  Block b;
  if (!block_of<FMT, D>(a, grp % heads, rb, grp / heads, b)) return;
  const Row row = row_of(a, b, b.r0 + wave * 32 + l32);
  u32x4 q[D / 16][T::NQ];
  {
    const int64_t from = ((int64_t)row.s * a.N + row.i) * a.q_stride + (int64_t)row.head * D + 8 * hh;
#pragma unroll
    for (int f = 0; f < D / 16; ++f) query_terms<QT, T::BF, T::NQ>(a.q, from + 16 * f, a.scale * kLog2e, q[f]);
  }
  const float scale = a.scale * kLog2e;
  if (tid == 0) s_odd = 0;
  // The keys that any of the wave's rows sees.
  int wlow = row.low, whigh = row.high;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) wlow = min(wlow, __shfl_xor(wlow, o)), whigh = max(whigh, __shfl_xor(whigh, o));
  wlow = __builtin_amdgcn_readfirstlane(wlow);
  whigh = __builtin_amdgcn_readfirstlane(whigh);
  __syncthreads();

  const int tiles = (b.nc + KT - 1) / KT;
  u32x4 raw[NPC];
  uint32_t rs[NPC];
  auto fetch = [&](int t) {
#pragma unroll
    for (int u = 0; u < NPC; ++u) {
      const int e = u * 256 + tid, v = e >= ALL / 2, p = e - v * (ALL / 2), c = p % PR;
      if (ALL < 256 && e >= ALL) continue;
      const uint64_t r = key_row(b, b.c0 + t * KT + p / PR);
      raw[u] = *(const u32x4 *)((v ? b.v_ : b.k) + r * RB + 16 * c);
      if constexpr (T::MX) rs[u] = *(const uint8_t *)((v ? b.vs : b.ks) + r * (D / 32) + (E * c) / 32);
    }
  };
  auto is_part = [&](int j, int n) { return j + n - 1 > b.first_high || (j + n > a.first && j < b.last_low); };
  auto place = [&](int t, int slot) {
    const bool part = is_part(b.c0 + t * KT, KT);
#pragma unroll
    for (int u = 0; u < NPC; ++u) {
      const int e = u * 256 + tid, v = e >= ALL / 2, p = e - v * (ALL / 2), c = p % PR, r = p / PR;
      if (ALL < 256 && e >= ALL) continue;
      u32x4 o[X];
      widen<FMT>(raw[u], T::MX ? rs[u] : 0, o);
      if (T::MX && rs[u] == 255)
#pragma unroll
        for (int x = 0; x < X; ++x) o[x] = u32x4{0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u};
      if (part && v) {
        bool odd = false;
#pragma unroll
        for (int x = 0; x < X; ++x) odd |= take_odd<T::BF>(o[x]);
        if (odd) s_odd = 1;
      }
      uint8_t *to = s_mem + slot * STAGE + v * (KT * D * 2) + r * (2 * D);
#pragma unroll
      for (int x = 0; x < X; ++x) *(u32x4 *)(to + ((c * X + x ^ piece_xor(r)) << 4)) = o[x];
    }
  };
  RowState<QT, FMT, D> st;
  st.init();
  float minus1 = -1.f;
  asm volatile("" : "+s"(minus1));
  const int j16 = lane & 15;
  const int vrow = 4 * hh + (j16 >> 2), vpiece = (2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1)) ^ piece_xor(vrow);
  if (tiles > 0) {
    fetch(0);
    place(0, 0);
    if (tiles > 1) fetch(1);
  }
  __syncthreads();
  for (int t = 0; t < tiles; ++t) {
    const uint8_t *stage = s_mem + (t & 1) * STAGE;
#pragma unroll 1
    for (int k = 0; k < KT / 32; ++k) {
      const int j = b.c0 + t * KT + 32 * k;
      if (j > whigh || (j >= a.first && j + 32 <= wlow)) continue;
      const uint8_t *krow = stage + (32 * k + l32) * (2 * D);
      f32x16 S = f32x16{};
#pragma unroll
      for (int f = 0; f < D / 16; ++f) {
        const u32x4 kf = *(const u32x4 *)(krow + (((2 * f + hh) ^ piece_xor(l32)) << 4));
#pragma unroll
        for (int n = 0; n < T::NQ; ++n) S = mfma32<T::BF>(kf, q[f][n], S);
      }
      const bool part = is_part(j, 32);
      uint32_t sees = 0;
      if (part) sees = ((~first_keys(row.low - j) | first_keys(a.first - j)) & first_keys(row.high + 1 - j)) >> (4 * hh);
      st.softmax(S, part, sees, scale);
      st.values(S, stage + KT * D * 2 + (32 * k + vrow) * (2 * D) + (j16 & 1) * 8, vpiece, minus1);
    }
    if (t + 1 < tiles) {
      place(t + 1, (t + 1) & 1);
      if (t + 2 < tiles) fetch(t + 2);
    }
    __syncthreads();
  }

  // Rows to their columns' order through LDS: a wave's own 32 rows.
  st.L += other_half(st.L);
  float *so = (float *)s_mem + (size_t)(wave * 32) * D;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *(f32x4 *)(so + l32 * D + 4 * ((8 * n + 2 * e + hh) ^ (l32 & 7))) =
          f32x4{st.acc[n][4 * e], st.acc[n][4 * e + 1], st.acc[n][4 * e + 2], st.acc[n][4 * e + 3]};
  asm volatile("" ::: "memory");
#pragma unroll 1
  for (int e = lane; e < 32 * (D / 4); e += 64) {
    const int r = e / (D / 4), q4 = e % (D / 4);             // one row, or a few, for the whole wave
    f32x4 o = *(const f32x4 *)(so + r * D + 4 * (q4 ^ (r & 7)));
    const float m = __shfl(st.M, r) - kOff, den = __shfl(st.L, r);
    const Row x = row_of(a, b, b.r0 + wave * 32 + r);
    if (!x.in) continue;
    if (s_odd)
      for (int t = 0; t < tiles; ++t)
        if (is_part(b.c0 + t * KT, KT))
          put_odd<FMT, D>(b, a.first, x.low, x.high, b.c0 + t * KT, min(b.c0 + t * KT + KT, b.c0 + b.nc), q4, o);
    leave_row<QT, D>(a, b, x, q4, m, den, o);
  }
}

// Joins a row's chunks, in order: a wave per row, D / 4 lanes a chunk.
template <int QT, int D> __global__ __launch_bounds__(256) void history_merge_kernel(HistAttnArgs a) {
  warm_kernargs<sizeof(HistAttnArgs)>();
  constexpr int LR = D / 4, GR = 64 / LR;    // lanes per chunk, chunks at a time
  const int lane = threadIdx.x & 63, q4 = lane % LR, cg = lane / LR;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.S * a.N * a.qh) return;
  const int hd = (int)(row % a.qh), i = (int)(row / a.qh % a.N), s = (int)(row / ((int64_t)a.qh * a.N));
  const int count = step_count(a.counts, s, a.N);
  if (i >= count) return;
  const int r0 = (i * a.qm + hd % a.qm) / a.own.block_rows * a.own.block_rows;
  const Visible v = visible_of(a, s, r0 / a.qm, min(count, (r0 + a.own.block_rows - 1) / a.qm + 1) - 1);
  const int own = used_chunks(v.n, chunk_keys(a.own, v.n));
  int pre = 0;
  if (a.p.k) {
    const int n = visible_prefix(a).n;
    pre = used_chunks(n, chunk_keys(a.pre, n));
  }
  const int used = pre + own;
  auto slot = [&](int c) { return row * a.chunks + (c < pre ? c : a.pre.chunks + c - pre); };
  float m = kNone;
  for (int c = lane; c < used; c += 64) m = fmaxf(m, a.pm[slot(c)]);
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  float den = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = cg; c < used; c += GR) {
    const int64_t at = slot(c);
    const float f = exp2_(a.pm[at] - m);
    den = fmaf(a.pl[at], f, den);
    const f32x4 w = *(const f32x4 *)(a.po + at * D + 4 * q4);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = fmaf(w[k], f, sum[k]);
  }
#pragma unroll
  for (int o = LR; o < 64; o <<= 1) {
    den += __shfl_xor(den, o);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] += __shfl_xor(sum[k], o);
  }
  if (cg == 0) finish_history_row<QT, D>(a, row, hd, q4, m, den, sum);
}

template <int QT, int FMT, int D> static void launch_pass(const HistAttnArgs &a, hipStream_t s) {
  const HistAttnArgs::Pass &p = a.shared ? a.pre : a.own;
  const int64_t groups = (int64_t)(a.shared ? a.kvh : a.S * a.kvh) * p.chunks;
  constexpr int KT = D == 256 ? 32 : 64, OCC_FEW = D == 64 ? 3 : D == 128 ? 2 : 1, OCC_MANY = D == 256 ? 1 : 2;
  if (p.block_rows == kFewRows) {
    hipLaunchKernelGGL((history_few_kernel<QT, FMT, D, 4, OCC_FEW>), dim3((uint32_t)groups), dim3(256), 0, s, a);
  } else {
    const int parts = groups >= 8 ? 1 : (int)((8 + groups - 1) / groups), share = (p.row_blocks + parts - 1) / parts;
    const int64_t all = groups * share * parts;
    hipLaunchKernelGGL((history_many_kernel<QT, FMT, D, KT, OCC_MANY>), dim3((uint32_t)(8 * ((all + 7) / 8))), dim3(256), 0, s, a);
  }
}

template <int QT, int FMT, int D> static hipError_t launch_types(HistAttnArgs a, hipStream_t s, int *launches) {
  *launches = 0;
  for (int shared = a.p.k ? 1 : 0; shared >= 0; --shared) {
    a.shared = shared;
    launch_pass<QT, FMT, D>(a, s);
    ++*launches;
  }
  if (a.chunks > 1) {
    const int64_t rows = (int64_t)a.S * a.N * a.qh;
    hipLaunchKernelGGL((history_merge_kernel<QT, D>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s, a);
    ++*launches;
  }
  return hipGetLastError();
}

template <int QT, int D> static hipError_t launch_format(const HistAttnArgs &a, hipStream_t s, int *launches) {
  if (a.format == H_MXFP8) return launch_types<QT, H_MXFP8, D>(a, s, launches);
  if (a.format == H_MXFP4) return launch_types<QT, H_MXFP4, D>(a, s, launches);
  return launch_types<QT, QT == E_BF16 ? H_BF16 : H_F16, D>(a, s, launches);
}

template <int D> hipError_t launch_history_attention_d(HistAttnArgs a, int type, hipStream_t s, int *launches) {
  if (type == E_F32) return launch_format<E_F32, D>(a, s, launches);
  return type == E_F16 ? launch_format<E_F16, D>(a, s, launches) : launch_format<E_BF16, D>(a, s, launches);
}

}  // namespace hh
