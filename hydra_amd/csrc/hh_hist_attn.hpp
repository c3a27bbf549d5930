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
// probabilities as two (outputs of 16 bits: to 2^-15 of each) or three (F32: as exact as the sums) of bf16, or two of fp16: outputs of 16 bits
// are rounded once, and a token's weights are held alike whether few or many share its call. (One term of many rows would take a fifth off
// a prompt's time: 168 us for 215, but 2.2e-3 from 64 bits for 1.7e-3, the output's own rounding.)
#pragma once
#include <type_traits>
#include <utility>

#include "hh_attn_mfma.hpp"
#include "hh_hist.hpp"

namespace hh {

template <int QT, int FMT> struct HistTypes {
  static constexpr bool BF = FMT != H_F16, MX = FMT >= H_MXFP8;
  static constexpr int E = FMT == H_MXFP8 ? 16 : FMT == H_MXFP4 ? 32 : 8;                       // numbers of 16 bytes
  static constexpr int NQ = QT == E_F32 ? (BF ? 3 : 2) : QT == E_F16 && BF ? 2 : 1;             // terms of a query
  static constexpr int NP = QT == E_F32 && BF ? 3 : 2;                                          // of a probability
};

// Memory that is read as the device's own: a load that could be of LDS too would wait with LDS's.
typedef const uint8_t __attribute__((address_space(1))) *gptr_t;
template <typename V> __device__ __forceinline__ V load_global(gptr_t p) { return *(const V __attribute__((address_space(1))) *)p; }

// N bytes of a row (16, or 8 of MXFP4) and their scale byte as MFMA operands of eight numbers. The conversions take a
// scale's exponent bits as e8m0: 255 makes every number NaN.
template <int FMT, int N> __device__ __forceinline__ void widen(const uint32_t (&raw)[N / 4], uint32_t scale, u32x4 (&out)[HistTypes<0, FMT>::E * N / 128]) {
  if constexpr (FMT == H_F16 || FMT == H_BF16) {
    out[0] = u32x4{raw[0], raw[1], raw[2], raw[3]};
  } else {
    const float by = __uint_as_float(scale << 23);
#pragma unroll
    for (int x = 0; x < HistTypes<0, FMT>::E * N / 128; ++x) {
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

// Columns 4 q4 .. 4 q4 + 3 of a row.
template <int FMT> __device__ __forceinline__ f32x4 numbers_at(gptr_t row, gptr_t scales, int q4) {
  if constexpr (FMT == H_F16) {
    const f16x2 l = __builtin_bit_cast(f16x2, load_global<uint32_t>(row + 8 * q4)), h = __builtin_bit_cast(f16x2, load_global<uint32_t>(row + 8 * q4 + 4));
    return f32x4{(float)l[0], (float)l[1], (float)h[0], (float)h[1]};
  } else if constexpr (FMT == H_BF16) {
    const u32x2 w = load_global<u32x2>(row + 8 * q4);
    return f32x4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xFFFF0000u)};
  } else if constexpr (FMT == H_MXFP8) {
    const int w = (int)load_global<uint32_t>(row + 4 * q4);
    const float by = hist_scale(load_global<uint8_t>(scales + (q4 >> 3)));
    return f32x4{__builtin_amdgcn_cvt_f32_fp8(w, 0) * by, __builtin_amdgcn_cvt_f32_fp8(w, 1) * by, __builtin_amdgcn_cvt_f32_fp8(w, 2) * by,
                 __builtin_amdgcn_cvt_f32_fp8(w, 3) * by};
  } else {
    const uint32_t w = load_global<uint16_t>(row + 2 * q4);
    const float by = hist_scale(load_global<uint8_t>(scales + (q4 >> 3)));
    const bf16x2 l = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 0), h = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.f, 1);
    return f32x4{(float)l[0] * by, (float)l[1] * by, (float)h[0] * by, (float)h[1] * by};
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
  bool shared;
  int s, g, r0, count, chunk, c0, nc;       // keys c0 .. c0 + nc − 1
  Visible v;
  int last_low, first_high;                 // of the last and the first row
  gptr_t k, v_, ks, vs;                     // the head's rows
  int rows, span, pinned, delta;            // position -> row
  int even, even_end, even_row;             // keys even .. even_end − 1 are in consecutive rows from even_row on: all but a few
};
__device__ __forceinline__ int row_low(const HistAttnArgs &a, const Visible &v, int i) {
  return a.window ? v.fold + max(v.length + i - a.window + 1, v.low) - v.low : 0;
}
__device__ __forceinline__ int row_high(const Visible &v, int i) { return v.fold + max(0, min(v.length + i, v.last) - v.low + 1) - 1; }

template <int FMT, int D> __device__ __forceinline__ bool block_of(const HistAttnArgs &a, bool shared, int sg, int rb, int chunk, Block &b) {
  const HistAttnArgs::Pass &p = shared ? a.pre : a.own;
  const HistView &h = shared ? a.p : a.h;
  b.shared = shared;
  b.s = shared ? 0 : sg / a.kvh;
  b.g = sg - b.s * a.kvh;
  b.r0 = rb * p.block_rows;
  b.chunk = chunk;
  int i0 = 0;
  if (shared) {
    b.count = a.S * a.N;
    b.v = visible_prefix(a);
    b.last_low = 0;
    b.first_high = b.v.n - 1;
  } else {
    b.count = step_count(a.counts, b.s, a.N);
    if (b.r0 >= b.count * a.qm) return false;
    i0 = b.r0 / a.qm;
    const int i1 = min(b.count, (b.r0 + p.block_rows - 1) / a.qm + 1) - 1;
    b.v = visible_of(a, b.s, i0, i1);
    b.last_low = row_low(a, b.v, i1);
    b.first_high = row_high(b.v, i0);
  }
  const int per = chunk_keys(p, b.v.n);
  const int64_t c0 = (int64_t)chunk * per;
  if (chunk && c0 >= b.v.n) return false;
  b.c0 = (int)c0;
  b.nc = min(per, b.v.n - b.c0);
  const int64_t base = (int64_t)sg * h.rows;                 // sg counts the prefix's heads too
  b.k = (gptr_t)h.k + base * hist_row_bytes(FMT, D);
  b.v_ = (gptr_t)h.v + base * hist_row_bytes(FMT, D);
  b.ks = (gptr_t)h.ks + base * (D / 32);
  b.vs = (gptr_t)h.vs + base * (D / 32);
  b.rows = h.rows;
  b.pinned = h.ring ? h.pinned : 0;
  b.span = h.rows - b.pinned;
  b.delta = 0;
  if (h.ring) {
    const int from = max(b.v.low, b.pinned);
    b.delta = (int)((uint32_t)(from - b.pinned) % (uint32_t)b.span) + b.pinned - from;
  }
  // From the window's start, or behind the pinned rows, to the end, or to where a ring goes on at its first row.
  const int from = max(b.v.low, b.pinned);
  b.even = b.v.fold + from - b.v.low;
  b.even_row = from + b.delta;
  b.even_end = min(b.v.n, b.even + b.rows - b.even_row);
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
  const int tt = x.in ? t : b.r0 / a.qm;                     // rows past the last see what the block's first sees
  x.head = b.g * a.qm + (x.in ? r - t * a.qm : 0);
  if (b.shared) {
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

// Eight columns of a query as NQ operands. Logits are scaled as fp32 sums: scaled first, a query's terms would be no short numbers any more.
template <int QT, bool BF, int NQ> __device__ __forceinline__ void query_terms(const void *q, int64_t at, u32x4 (&out)[NQ]) {
  if constexpr (NQ == 1) {
    out[0] = *(const u32x4 *)((const uint16_t *)q + at);
  } else {
    float x[8];
    if constexpr (QT == E_F32) {
      const f32x4 *p = (const f32x4 *)((const float *)q + at);
      const f32x4 l = p[0], h = p[1];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = e < 4 ? l[e & 3] : h[e & 3];
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

// Two probabilities as NP terms: bf16 by cutting off, the last rounded. What is left of a probability is exact, as the sum of it and −1
// times its head, which the dot product takes from the packed heads: one instruction in place of a mask and a subtraction. The constants
// are registers: as immediates, (−1, 0) and (0, −1) in bf16 come out alike.
struct SplitConst {
  float minus1;
  uint32_t m0, m1;
  __device__ __forceinline__ SplitConst() : minus1(-1.f), m0(0x0000BF80u), m1(0xBF800000u) { asm volatile("" : "+s"(minus1), "+s"(m0), "+s"(m1)); }
};
template <bool BF, int NP> __device__ __forceinline__ void split_terms(float p0, float p1, const SplitConst &k, uint32_t (&w)[NP]) {
  if constexpr (!BF) {
    const u32x2 v = split_pair(p0, p1, k.minus1);
    w[0] = v[0], w[1] = v[1];
  } else {
    const bf16x2 m0 = __builtin_bit_cast(bf16x2, k.m0), m1 = __builtin_bit_cast(bf16x2, k.m1);
#pragma unroll
    for (int t = 0; t + 1 < NP; ++t) {
      w[t] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
      const bf16x2 h = __builtin_bit_cast(bf16x2, w[t]);
      p0 = __builtin_amdgcn_fdot2_f32_bf16(h, m0, p0, false);
      p1 = __builtin_amdgcn_fdot2_f32_bf16(h, m1, p1, false);
    }
    const bf16x2 l = {(__bf16)p0, (__bf16)p1};
    w[NP - 1] = __builtin_bit_cast(uint32_t, l);
  }
}

// The sink into a row's denominator; returns the factor of what was summed before. The log of a denominator: of nothing −inf.
__device__ __forceinline__ float sink_share(const HistAttnArgs &a, int head, float &m, float &den) {
  if (!a.sinks) return 1.f;
  const float y = bf16_bits_to_f32(a.sinks[head]) * kLog2e, mn = fmaxf(m, y), f = exp2_(m - mn);
  den = fmaf(den, f, exp2_(y - mn));
  m = mn;
  return f;
}
__device__ __forceinline__ float lse_of(float m, float den) { return den == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(den)) * kLn2; }
// Four outputs, rounded once.
template <int QT> __device__ __forceinline__ void store_out(const HistAttnArgs &a, int64_t at, f32x4 o) {
  if constexpr (QT == E_F32) {
    *(f32x4 *)((float *)a.out + at) = o;
  } else if constexpr (QT == E_F16) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *(f16x4 *)((_Float16 *)a.out + at) = f16x4{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
  } else {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *(bf16x4 *)((__bf16 *)a.out + at) = bf16x4{(__bf16)o[0], (__bf16)o[1], (__bf16)o[2], (__bf16)o[3]};
  }
}
// A row's four outputs from its joined state.
template <int QT, int D>
__device__ __forceinline__ void finish_history_row(const HistAttnArgs &a, int64_t row, int head, int q4, float m, float den, f32x4 o) {
  const float f = sink_share(a, head, m, den) * (den == 0.f ? 0.f : 1.f / den);   // of nothing: 0
  store_out<QT>(a, row * D + 4 * q4, o * f);
  if (q4 == 0 && a.lse) a.lse[row] = lse_of(m, den);
}

// A row's state of one chunk, or its outputs where there is no other.
template <int QT, int D>
__device__ __forceinline__ void leave_row(const HistAttnArgs &a, const Block &b, const Row &x, int q4, float m, float den, f32x4 o) {
  const int64_t row = ((int64_t)x.s * a.N + x.i) * a.qh + x.head;
  if (a.chunks > 1) {
    const int64_t slot = row * a.chunks + (b.shared ? 0 : a.pre.chunks) + b.chunk;
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
// into the rows that do behind the loop. An exponent of all ones carries into the sign's place when one is added to it.
template <bool BF> __device__ __forceinline__ bool take_odd(u32x4 &x) {
  constexpr uint32_t em = BF ? 0x7F80u : 0x7C00u, both = em | em << 16, one = BF ? 0x00800080u : 0x04000400u;
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) any |= (x[e] & both) + one;
  const bool odd = any & 0x80008000u;
  if (!__any(odd)) return false;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] &= ((x[e] & em) == em ? 0u : 0xFFFFu) | ((x[e] >> 16 & em) == em ? 0u : 0xFFFF0000u);
  return odd;
}
// A logit, or where bit BIT of `hidden` is set `none`'s bits: two instructions (the bit's extraction in assembly, or the compiler makes a
// comparison and a selection of it, with waits between).
template <int BIT> __device__ __forceinline__ float seen_or(float s, uint32_t hidden, uint32_t none) {
  uint32_t m;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(m) : "v"(hidden), "n"(BIT));
  return __uint_as_float((none & m) | (__float_as_uint(s) & ~m));
}
// The same of N logits: element G k + i is key PER k + i from the lane's first.
template <int G, int PER, int N, int... I>
__device__ __forceinline__ void hide(float (&y)[N], uint32_t hidden, uint32_t none, std::integer_sequence<int, I...>) {
  ((y[I] = seen_or<PER * (I / G) + I % G>(y[I], hidden, none)), ...);
}
// The infinities and NaN among the values of keys j0 .. j1 − 1 (j0 < j1) that a row sees, in four columns, added to `odd`.
template <int FMT, int D>
__device__ __forceinline__ void add_odd(const Block &b, int first, int low, int high, int j0, int j1, int q4, f32x4 &odd) {
#pragma unroll 1
  for (int j = j0; j < j1; j += 4) {
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t r = key_row(b, j + u);
      v[u] = numbers_at<FMT>(b.v_ + r * hist_row_bytes(FMT, D), b.vs + r * (D / 32), q4);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = j + u;
      const bool seen = k < j1 && k <= high && (k < first || k >= low);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (seen && !(fabsf(v[u][i]) < INFINITY)) odd[i] += v[u][i];
    }
  }
}
// A row's four sums with the infinities and NaN of the values that it sees: those that take_odd took out (`taken`) of the tiles that some
// row does not see whole, and, where a sum is NaN though the row's logits are numbers, those of all tiles, since a zero among an
// infinity's probability terms has made it NaN there. KT keys a tile.
template <int FMT, int D, int KT, typename P>
__device__ __forceinline__ void put_odd(const Block &b, int first, int low, int high, int tiles, bool taken, P is_part, float den, int q4, f32x4 &o) {
  const bool lost = den == den && !(o[0] == o[0] && o[1] == o[1] && o[2] == o[2] && o[3] == o[3]);
  if (__builtin_expect(!taken && !lost, 1)) return;   // expected, or the loop before it spills registers for this one
  f32x4 odd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    if (!lost && !is_part(t)) continue;
    add_odd<FMT, D>(b, first, low, high, b.c0 + KT * t, min(b.c0 + KT * t + KT, b.c0 + b.nc), q4, odd);
    bool all = !taken;                       // every sum is a number or NaN for good
#pragma unroll
    for (int i = 0; i < 4; ++i) all = all && (o[i] == o[i] || odd[i] != odd[i]);
    if (all) break;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = o[i] == o[i] ? o[i] + odd[i] : odd[i] != 0.f ? odd[i] : o[i];
}

// Logits S of a run of keys, N of them a lane, its row's shared with the lanes that `top_of` exchanges with, to probabilities
// 2^(y − R), y = S·scale, and their sum to L. R follows the row's maximum y, less `off`, by steps of at least kLag. Whether it has to
// step is seen from the sum of what comes out with the R that there is, so that no maximum is formed but where it does. The product and
// the difference are one fma; where R is so far from zero that the product's lost bits would matter (`far`), y is rounded first, as R
// was, and R follows every new maximum. The wave goes into the branch as one, but each row steps and rounds by its own logits alone, so that
// its bits do not depend on the rows beside it. Returns what the sums so far are to be multiplied with after a step of R (1: none); L is.
//
// The largest probability of fp16 operands is 2^7 to 2^14.5 (kOff, for fp16's smallest steps); bf16 reaches as far down as fp32, and there none is above 1, so that
// the sums of values stay within fp32 wherever the values times the keys do.
constexpr float kFar = 65536.f;
template <bool BF, int N, typename F> __device__ __forceinline__ float to_probabilities(float (&S)[N], float scale, float &R, float &L, bool &far, F top_of) {
  constexpr float off = BF ? -kLag : kOff, kMost = BF ? 1.f : 23170.475f;    // 2^(off + kLag)
  float y[N], corr = 1.f;
  auto sum_of = [&]() {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      y[i] = exp2_(y[i]);
      sum[i & 1] += y[i];
    }
    return sum[0] + sum[1];
  };
#pragma unroll
  for (int i = 0; i < N; ++i) y[i] = fmaf(S[i], scale, -R);
  float sum = sum_of();
  if (__any(far || sum > kMost)) {
    // Nearly never: with a scale of its own, so that its products are not made ahead of the branch.
    float own = scale;
    asm volatile("" : "+v"(own));
    float top = S[0] * own;
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, S[i] * own);
    top = top_of(top);
    const bool moves = far || top_of(sum > kMost ? 1.f : 0.f) > 0.f;
    const float to = moves ? fmaxf(R, top - off) : R;
    corr = moves ? exp2_(R - to) : 1.f;
    R = to;
    L *= corr;
    far = fabsf(R) > kFar && R > kNone;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = far ? S[i] * own - R : fmaf(S[i], own, -R);
    sum = sum_of();
  }
  L += sum;
#pragma unroll
  for (int i = 0; i < N; ++i) S[i] = y[i];
  return corr;
}
// Operands from memory, waited for here: a wait left to a loop's first use would there wait for the loop's own loads each time.
template <int N> __device__ __forceinline__ void arrived(u32x4 (&q)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) asm volatile("" : "+v"(q[n]));
}

__device__ __forceinline__ int piece_xor(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }
template <bool BF> __device__ __forceinline__ f32x4 mfma16(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
  if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ u32x2 read_columns(const uint8_t *p) {   // transposing: four rows of the lane's column
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p));
}

// Few rows: each wave has all of a kv head's, 16·RT, and tiles of 32 keys of its own, W of them a workgroup; the next tile's bytes are
// in flight under this one's products. On the 16x16 MFMA, S^T [16 keys × 16 rows] twice a tile: a head of 64 in 8 bits is 64 bytes, four
// lanes of a key, so that a load is one stretch of memory, and goes to the operands' registers as it is, since the order of a product's
// columns is free. Values pass through LDS to be read by columns. No barrier until the waves' states meet. Bound by the bytes where
// there are enough: eight streams of up to 32768 keys in 8 bits, fp32, 64 / 8 heads of 64, 208 MB in 39 us (5.3 TB/s; the joining launch 5
// more), in fp16 403 MB in 83 (4.9); 131071 keys in 4 bits, 16 / 2 heads of 256, 71 MB in 17.5 us (4.1 TB/s: the LDS that the waves' states meet in
// lets two workgroups onto a unit). By the chain of latencies where
// there are few: 16 windows of 132 keys 6.9 us. Of 32 rows with heads of 256 the sums leave one wave a SIMD, and other types than bf16 over
// codes spill 11 to 129 registers: four streams of 16384 keys over 8 bits 43 us in bf16 and 83 in fp32 (16 rows: 28 and 38). With 64 rows a wave (four of these tiles of 16)
// 64 rows of 32768 keys took 26 us of heads of 64 in bf16, the kernel of many rows 30; but of fp32 42 and 35, and of 1000 keys 14.7 and 13.6: the
// sums and the queries' terms fill the registers.
template <int D, int RT, int W> constexpr int few_lds() { return W * (16 * RT * D * 4 > 64 * D ? 16 * RT * D * 4 : 64 * D); }
template <int QT, int FMT, int D, int RT, int W>
__device__ __forceinline__ void history_few(const HistAttnArgs &a, bool shared, int block, uint8_t *s_mem) {
  using T = HistTypes<QT, FMT>;
  constexpr int E = T::E, RB = D * 16 / E, PB = RB / 4 < 16 ? RB / 4 : 16, U = RB / 4 / PB, EP = PB * E / 16, X = EP / 8;
  constexpr int NF = D / 32, NB = D / 16, ROWS = 16 * RT;   // operands of a query or of 16 keys; blocks of 16 value columns
  __shared__ float s_m[W][ROWS], s_l[W][ROWS];
  __shared__ int s_lo[ROWS], s_hi[ROWS], s_odd;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, quad = lane >> 4;
  const int heads = shared ? a.kvh : a.S * a.kvh;
  Block b;
  if (!block_of<FMT, D>(a, shared, block % heads, 0, block / heads, b)) return;
  u32x4 q[RT][NF][T::NQ];                    // operand u·X + x: columns EP (4 u + quad) + 8 x
  int low[RT], high[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const Row row = row_of(a, b, 16 * r + l16);
    low[r] = row.low, high[r] = row.high;
    if (wave == 0 && quad == 0) s_lo[16 * r + l16] = row.low, s_hi[16 * r + l16] = row.high;
    const int64_t at = ((int64_t)row.s * a.N + row.i) * a.q_stride + (int64_t)row.head * D + EP * quad;
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int n = 0; n < T::NQ; ++n) q[r][f][n] = u32x4{};
    if (row.in)                              // queries of tokens that are not there are not read
#pragma unroll
      for (int f = 0; f < NF; ++f) query_terms<QT, T::BF, T::NQ>(a.q, at + 4 * EP * (f / X) + 8 * (f % X), q[r][f]);
  }
  const float scale = a.scale * kLog2e;
  const uint32_t none = scale < 0.f ? 0x7F800000u : 0xFF800000u;   // the logit of a key that is not seen: y is −inf
  if (tid == 0) s_odd = 0;
  __syncthreads();

  const int tiles = (b.nc + 31) / 32;
  typedef typename std::conditional<D == 64, uint16_t, typename std::conditional<D == 128, uint32_t, uint64_t>::type>::type scales_t;
  typedef typename std::conditional<PB == 16, u32x4, u32x2>::type piece_t;
  piece_t raw[2][2][U];                      // keys and values, 16 keys, pieces
  scales_t rs[2][2];
  auto fetch = [&](int t) {
    const int j = b.c0 + 32 * t;
    gptr_t at[2][2], sc[2][2];
    if (j >= b.even && j + 32 <= b.even_end) {
      const int64_t r = b.even_row + (j - b.even);
      const uint32_t o = (uint32_t)(l16 * RB + quad * PB), so = (uint32_t)(l16 * (D / 32));
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
        at[0][kg] = b.k + r * RB + 16 * kg * RB + o;
        at[1][kg] = b.v_ + r * RB + 16 * kg * RB + o;
        sc[0][kg] = b.ks + r * (D / 32) + 16 * kg * (D / 32) + so;
        sc[1][kg] = b.vs + r * (D / 32) + 16 * kg * (D / 32) + so;
      }
    } else {
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
        const int64_t r = key_row(b, j + 16 * kg + l16);
        at[0][kg] = b.k + r * RB + quad * PB;
        at[1][kg] = b.v_ + r * RB + quad * PB;
        sc[0][kg] = b.ks + r * (D / 32);
        sc[1][kg] = b.vs + r * (D / 32);
      }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
        if constexpr (T::MX) rs[v][kg] = load_global<scales_t>(sc[v][kg]);
#pragma unroll
        for (int u = 0; u < U; ++u) raw[v][kg][u] = load_global<piece_t>(at[v][kg] + 4 * PB * u);
      }
  };
  // The scale byte of piece u: its 32 columns are EP (4 u + quad) / 32.
  const int sshift = 8 * (EP * quad / 32);
  auto scale_of = [&](scales_t s, int u) { return (uint32_t)(s >> sshift >> 8 * (4 * EP * u / 32)) & 0xFFu; };
  auto operands = [&](int v, int kg, int u, u32x4 (&w)[X]) {
    uint32_t x[PB / 4];
#pragma unroll
    for (int i = 0; i < PB / 4; ++i) x[i] = raw[v][kg][u][i];
    const uint32_t sc = T::MX ? scale_of(rs[v][kg], u) : 0;
    widen<FMT, PB>(x, sc, w);
  };
  auto is_part = [&](int t) {
    const int j = b.c0 + 32 * t;
    return j + 31 > b.first_high || (j + 32 > a.first && j < b.last_low);
  };
  float R[RT], L[RT];
  bool far[RT];
  f32x4 acc[RT][NB];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    R[r] = kNone, L[r] = 0.f, far[r] = false;
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[r][n] = f32x4{};
  }
  const SplitConst kSplit;
  uint8_t *vmem = s_mem + wave * (64 * D);
  const int j16 = lane & 15, vrow = 4 * quad + (j16 >> 2), vpiece = ((j16 & 3) >> 1) ^ piece_xor(vrow);
  const uint8_t *vcol = vmem + vrow * (2 * D) + (j16 & 1) * 8;
  if (wave < tiles) fetch(wave);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int f = 0; f < NF; ++f) arrived(q[r][f]);
  for (int t = wave; t < tiles; t += W) {
    const bool part = is_part(t);
    f32x4 S[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) S[r][0] = S[r][1] = f32x4{};
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        u32x4 w[X];
        operands(0, kg, u, w);
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < T::NQ; ++n) S[r][kg] = mfma16<T::BF>(w[x], q[r][u * X + x][n], S[r][kg]);
      }
    asm volatile("" ::: "memory");           // the wave's last tile has been read: LDS takes its accesses in their order
#pragma unroll
    for (int kg = 0; kg < 2; ++kg)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        u32x4 w[X];
        operands(1, kg, u, w);
        if (part) {
          bool odd = false;
#pragma unroll
          for (int x = 0; x < X; ++x) odd |= take_odd<T::BF>(w[x]);
          if (odd) s_odd = 1;
        }
        const int row = 16 * kg + l16;
#pragma unroll
        for (int x = 0; x < X; ++x)
          *(u32x4 *)(vmem + row * (2 * D) + ((EP * (4 * u + quad) / 8 + x ^ piece_xor(row)) << 4)) = w[x];
      }
    asm volatile("" ::: "memory");           // the rows are read by other lanes than wrote them, behind the writes
    if (t + W < tiles) fetch(t + W);
    u32x4 p[RT][T::NP];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      // Element 4 kg + i is key 16 kg + 4 quad + i of the 32.
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = S[r][i >> 2][i & 3];
      if (part) {
        const int j = b.c0 + 32 * t;
        const uint32_t hidden = ~((~first_keys(low[r] - j) | first_keys(a.first - j)) & first_keys(high[r] + 1 - j)) >> (4 * quad);
        hide<4, 16>(y, hidden, none, std::make_integer_sequence<int, 8>{});
      }
      const float corr = to_probabilities<T::BF, 8>(y, scale, R[r], L[r], far[r], [](float v) { return max_lane_groups(v); });
      if (__any(corr != 1.f))
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[r][n] *= corr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[T::NP];
        split_terms<T::BF, T::NP>(y[2 * e], y[2 * e + 1], kSplit, w);
#pragma unroll
        for (int n = 0; n < T::NP; ++n) p[r][n][e] = w[n];
      }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const u32x2 v0 = read_columns(vcol + ((vpiece ^ (2 * n)) << 4)), v1 = read_columns(vcol + 32 * D + ((vpiece ^ (2 * n)) << 4));
      const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int k = 0; k < T::NP; ++k) acc[r][n] = mfma16<T::BF>(vf, p[r][k], acc[r][n]);
    }
  }

  // The waves' states meet in LDS, the sums of a row in 16-byte pieces XORed by the row.
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = 16 * r + l16;
    const float l = sum_lane_groups(L[r]);
    if (quad == 0) {
      s_m[wave][row] = R[r];                 // the exponent that L and O are relative to
      s_l[wave][row] = l;
    }
    float *so = (float *)s_mem + (size_t)(wave * ROWS + row) * D;
#pragma unroll
    for (int n = 0; n < NB; ++n) *(f32x4 *)(so + 4 * ((4 * n + quad) ^ (row & 7))) = acc[r][n];
  }
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
    put_odd<FMT, D, 32>(b, a.first, s_lo[r], s_hi[r], tiles, s_odd, is_part, den, q4, o);
    leave_row<QT, D>(a, b, x, q4, m, den, o);
  }
}

// Which 16 bytes of a tile a thread takes: the row and its piece. Eight lanes one after the other write to eight different places of the
// 128 bytes that LDS takes at a time (piece_xor of rows r and r + 4 is one apart, of r and r + 1 two), and 64 cover whole rows.
template <int X, int PR> __device__ __forceinline__ void piece_place(int e, int &row, int &c) {
  if constexpr (X == 1) {
    c = e % PR, row = e / PR;
  } else if constexpr (X == 2) {             // c0 c1 r2 c2.. r0 r1 r3..
    const int r2 = e >> 2 & 1, rest = e >> 3, hi = rest % (PR / 4), rr = rest / (PR / 4);
    c = (e & 3) + 4 * hi;
    row = (rr & 3) + 4 * r2 + (rr >> 2 << 3);
  } else {                                   // c0 r2 r0 c1.. r1 r3..
    const int r2 = e >> 1 & 1, r0 = e >> 2 & 1, rest = e >> 3, hi = rest % (PR / 2), rr = rest / (PR / 2);
    c = (e & 1) + 2 * hi;
    row = r0 + 2 * (rr & 1) + 4 * r2 + (rr >> 1 << 3);
  }
}

// Many rows: 128 a workgroup, 32 a wave, on the 32x32 MFMA; tiles of KT keys, whose 16-byte pieces the threads share, become operands in
// LDS, two tiles in turn, read by every wave. The bytes of the tile after the next are in flight under a tile's products. A tile's one
// barrier keeps the waves of a workgroup in step, so the workgroups are small: several a compute unit, each at its own place. Bound by the
// VALU's instructions and the matrix unit's cycles, one after the other on a SIMD (a prompt of 4096, 64 / 8 heads of 64, bf16 over 8 bits: 64%
// and 43% of the time, LDS 30%; 127 instructions for a wave's 32 keys: the softmax, and the probabilities' two terms), so what
// changes from tile to tile is kept to scalars and immediate offsets. That prompt takes 215 us (640 TFLOP/s; at a large
// library product's rate it would be 110). Two prompts of 6001, 32 / 8 heads of 128 in fp16 under a window of 1024, take 271 us (560): VALU, matrix unit and
// LDS 37, 37 and 34%, which two waves a SIMD hardly put beside each other. 256 tokens
// behind 16384, 16 / 2 heads of 256, 160 us (430: one wave a SIMD); a prompt of 2048 of those heads 145 us (240: one workgroup a unit, and the first see
// little). In fp32, three terms a query and a probability: a prompt of 2048, heads of 64 over 8 bits, 110 us (310; bf16 72), of 256 300 (115; 61 to 81 registers
// spilled). Tried and slower: scores of the next tile formed under the exponentials of one, with a third place for values (7 to 10%).
template <int D> constexpr int many_keys() { return D == 256 ? 32 : 64; }
template <int D> constexpr int many_lds() { return 2 * many_keys<D>() * D * 4 > 128 * D * 4 ? 2 * many_keys<D>() * D * 4 : 128 * D * 4; }
template <int QT, int FMT, int D> __device__ __forceinline__ void history_many(const HistAttnArgs &a, bool shared, uint32_t block, uint8_t *s_mem) {
  using T = HistTypes<QT, FMT>;
  constexpr int KT = many_keys<D>(), E = T::E, X = E / 8, RB = D * 16 / E, PR = RB / 16, NB = D / 32;
  constexpr int ALL = 2 * KT * PR, NPC = (ALL + 255) / 256, STAGE = KT * D * 4;
  static_assert(ALL % 256 == 0, "whole pieces a thread");
  __shared__ int s_odd;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hh = lane >> 5;
  // Each XCD takes a stretch of the list (head and chunk, block of rows), so that what it reads again is in its L2; a block's share of
  // a head that several XCDs have is spread over its rows, the ones that see most first.
  const HistAttnArgs::Pass &pass = shared ? a.pre : a.own;
  const int heads = shared ? a.kvh : a.S * a.kvh, groups = heads * pass.chunks;
  const int parts = groups >= 8 ? 1 : (8 + groups - 1) / groups, share = (pass.row_blocks + parts - 1) / parts;
  const uint32_t all = (uint32_t)groups * (uint32_t)(share * parts), each = (all + 7) / 8, w = (block & 7) * each + (block >> 3);
  if ((block >> 3) >= each || w >= all) return;
  const int grp = (int)(w / (uint32_t)(share * parts)), at = (int)(w - (uint32_t)grp * (uint32_t)(share * parts));
  // An XCD's 32 compute units take them in turn: where it holds all at once, forth and back, so that those that see most do not meet on one
  // (a prompt of 2048, 64 / 8 heads of 64: 73 us, 74 without); more are dealt as units come free (4096 tokens: 234, 240 forth and back).
  int turn = at % share;
  if (share <= 128 && turn >> 5 & 1) turn = (turn & ~31) + min(32, share - (turn & ~31)) - 1 - (turn & 31);
  const int rb = pass.row_blocks - 1 - (turn * parts + at / share);
  if (rb < 0) return;
  Block b;
  if (!block_of<FMT, D>(a, shared, grp % heads, rb, grp / heads, b)) return;
  const Row row = row_of(a, b, b.r0 + wave * 32 + l32);
  u32x4 q[D / 16][T::NQ];
  {
    const int64_t from = ((int64_t)row.s * a.N + row.i) * a.q_stride + (int64_t)row.head * D + 8 * hh;
#pragma unroll
    for (int f = 0; f < D / 16; ++f)
#pragma unroll
      for (int n = 0; n < T::NQ; ++n) q[f][n] = u32x4{};
    if (row.in)                              // queries of tokens that are not there are not read
#pragma unroll
      for (int f = 0; f < D / 16; ++f) query_terms<QT, T::BF, T::NQ>(a.q, from + 16 * f, q[f]);
  }
  const float scale = a.scale * kLog2e;
  const uint32_t none = scale < 0.f ? 0x7F800000u : 0xFF800000u;   // the logit of a key that is not seen: y is −inf
  if (tid == 0) s_odd = 0;
  // The keys that any of the wave's rows sees.
  int wlow = row.low, whigh = row.high;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) wlow = min(wlow, __shfl_xor(wlow, o)), whigh = max(whigh, __shfl_xor(whigh, o));
  wlow = __builtin_amdgcn_readfirstlane(wlow);
  whigh = __builtin_amdgcn_readfirstlane(whigh);
  // A wave without rows only loads, and leaves its SIMD to other workgroups' (40 rows of 16384 keys in bf16, heads of 64: 25 us, 31 with its
  // products; of 128: 33 and 41). Heads of 256 have one wave a SIMD: nothing to leave it to, and prompts 3% longer.
  const bool idle = D < 256 && b.r0 + wave * 32 >= b.count * a.qm;
  __syncthreads();

  const int tiles = (b.nc + KT - 1) / KT;
  // Piece u of a thread: of the keys in the first half of the pieces, of the values in the second (a thread's one piece, where it
  // has one, by its wave).
  const int half = NPC == 1 ? tid >> 7 : 0;
  constexpr int HALF = NPC == 1 ? 1 : NPC / 2;
  uint32_t off[HALF], soff[HALF];            // in a tile of consecutive rows
  int prow[HALF], to[HALF];
#pragma unroll
  for (int u = 0; u < HALF; ++u) {
    int c;
    piece_place<X, PR>(NPC == 1 ? tid & 127 : u * 256 + tid, prow[u], c);
    off[u] = prow[u] * RB + 16 * c;
    soff[u] = prow[u] * (D / 32) + E * c / 32;
    to[u] = prow[u] * (2 * D) + ((c * X ^ piece_xor(prow[u])) << 4) + (NPC == 1 ? half * (KT * D * 2) : 0);
  }
  u32x4 raw[NPC];
  uint32_t rs[NPC];
  // Tiles from `even` to `even_end` are of consecutive rows; those from `high` on, and from `low` to `low_end`, are not seen whole by some row.
  const int even = max(0, (b.even - b.c0 + KT - 1) / KT), even_end = (b.even_end - b.c0) / KT;
  const int high = max(0, (b.first_high + 1 - b.c0) / KT);   // first_high >= −1
  const int low = max(0, (min(a.first, b.last_low) - b.c0) / KT), low_end = b.last_low > b.c0 ? (b.last_low - b.c0 + KT - 1) / KT : 0;
  const int row0 = b.even_row + b.c0 - b.even;
  auto fetch = [&](int t) {
    int64_t at[HALF], sat[HALF];             // one load for both ways to its address, so that none waits where they meet
    const int64_t r0 = row0 + t * KT;
#pragma unroll
    for (int h = 0; h < HALF; ++h) at[h] = r0 * RB + off[h], sat[h] = r0 * (D / 32) + soff[h];
    if (t < even || t >= even_end) {
#pragma unroll
      for (int h = 0; h < HALF; ++h) {
        const int64_t r = key_row(b, b.c0 + t * KT + prow[h]) - prow[h];
        at[h] = r * RB + off[h], sat[h] = r * (D / 32) + soff[h];
      }
    }
#pragma unroll
    for (int u = 0; u < NPC; ++u) {
      const bool v = NPC == 1 ? half != 0 : u >= HALF;
      raw[u] = load_global<u32x4>((v ? b.v_ : b.k) + at[u % HALF]);
      if constexpr (T::MX) rs[u] = load_global<uint8_t>((v ? b.vs : b.ks) + sat[u % HALF]);
    }
  };
  auto is_part = [&](int t) { return t >= high || (t >= low && t < low_end); };
  auto place = [&](int t, auto slot) {
    const bool part = is_part(t);
#pragma unroll
    for (int u = 0; u < NPC; ++u) {
      u32x4 o[X];
      uint32_t x[4] = {raw[u][0], raw[u][1], raw[u][2], raw[u][3]};
      widen<FMT, 16>(x, T::MX ? rs[u] : 0, o);
      if (part && (NPC == 1 || u >= HALF)) {
        if (NPC > 1 || half) {
          bool odd = false;
#pragma unroll
          for (int i = 0; i < X; ++i) odd |= take_odd<T::BF>(o[i]);
          if (odd) s_odd = 1;
        }
      }
#pragma unroll
      for (int i = 0; i < X; ++i)
        *(u32x4 *)(s_mem + slot * STAGE + (NPC > 1 && u >= HALF ? KT * D * 2 : 0) + (to[u % HALF] ^ (i << 4))) = o[i];
    }
  };
  float R = kNone, L = 0.f;
  const SplitConst kSplit;
  bool far = false;
  f32x16 acc[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) acc[n] = f32x16{};
  const int j16 = lane & 15;
  const int vrow = 4 * hh + (j16 >> 2), vpiece = (2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1)) ^ piece_xor(vrow);
  int kat[D / 16], vat[NB];                  // this lane's places in a tile of keys and of values
#pragma unroll
  for (int f = 0; f < D / 16; ++f) kat[f] = l32 * (2 * D) + (((2 * f + hh) ^ piece_xor(l32)) << 4);
#pragma unroll
  for (int n = 0; n < NB; ++n) vat[n] = vrow * (2 * D) + (j16 & 1) * 8 + ((vpiece ^ (4 * n)) << 4);
  auto compute = [&](int t, auto slot) {
    if (idle) return;
    const bool part = is_part(t);
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) {
      const int j = b.c0 + t * KT + 32 * k;
      if (part && (j > whigh || (j >= a.first && j + 32 <= wlow))) continue;
      const uint8_t *keys = s_mem + slot * STAGE + 64 * D * k, *values = keys + KT * D * 2;
      f32x16 S = f32x16{};
#pragma unroll
      for (int f = 0; f < D / 16; ++f) {
        const u32x4 kf = *(const u32x4 *)(keys + kat[f]);
#pragma unroll
        for (int n = 0; n < T::NQ; ++n) S = mfma32<T::BF>(kf, q[f][n], S);
      }
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = S[i];
      if (part) {
        // Element i is key 8 (i / 4) + 4 hh + i % 4 of the 32.
        const uint32_t hidden = ~((~first_keys(row.low - j) | first_keys(a.first - j)) & first_keys(row.high + 1 - j)) >> (4 * hh);
        hide<4, 8>(y, hidden, none, std::make_integer_sequence<int, 16>{});
      }
      const float corr = to_probabilities<T::BF, 16>(y, scale, R, L, far, [](float v) { return max_halves(v); });
      if (__any(corr != 1.f))
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[n] *= corr;
      // V^T: lane (l32, hh) takes dimension 32 n + l32 of keys 16 kc + 8 x + 4 hh .. + 3, the order of P^T.
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        u32x4 p[T::NP];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t x[T::NP];
          split_terms<T::BF, T::NP>(y[8 * kc + 2 * e], y[8 * kc + 2 * e + 1], kSplit, x);
#pragma unroll
          for (int n = 0; n < T::NP; ++n) p[n][e] = x[n];
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const u32x2 v0 = read_columns(values + vat[n] + 16 * kc * 2 * D), v1 = read_columns(values + vat[n] + (16 * kc + 8) * 2 * D);
          const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
          for (int k2 = 0; k2 < T::NP; ++k2) acc[n] = mfma32<T::BF>(vf, p[k2], acc[n]);
        }
      }
    }
  };
  typedef std::integral_constant<int, 0> zero_t;
  typedef std::integral_constant<int, 1> one_t;
  auto step = [&](int t, auto slot, auto next) {
    compute(t, slot);
    if (t + 1 < tiles) {
      place(t + 1, next);
      if (t + 2 < tiles) fetch(t + 2);
    }
    __syncthreads();
  };
  if (tiles > 0) fetch(0);
#pragma unroll
  for (int f = 0; f < D / 16; ++f) arrived(q[f]);
  if (tiles > 0) {
    place(0, zero_t{});
    if (tiles > 1) fetch(1);
  }
  __syncthreads();
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    step(t, zero_t{}, one_t{});
    if (++t >= tiles) break;
    step(t, one_t{}, zero_t{});
  }

  // What a lane's row leaves besides its sums: its state, or its denominator with the sink's share, lse, and the sums' factor.
  L += other_half(L);
  int64_t to_row = -1;                       // where its sums go
  float by = 1.f;
  if (row.in) {
    const int64_t out = ((int64_t)row.s * a.N + row.i) * a.qh + row.head;
    if (a.chunks > 1) {
      to_row = out * a.chunks + (shared ? 0 : a.pre.chunks) + b.chunk;
      if (hh == 0) a.pm[to_row] = R, a.pl[to_row] = L;
    } else {
      to_row = out;
      float m = R, den = L;
      by = sink_share(a, row.head, m, den);
      by *= den == 0.f ? 0.f : 1.f / den;
      if (hh == 0 && a.lse) a.lse[out] = lse_of(m, den);
    }
  }
  // Rows to their columns' order through LDS: a wave's own 32 rows.
  float *so = (float *)s_mem + (size_t)(wave * 32) * D;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *(f32x4 *)(so + l32 * D + 4 * ((8 * n + 2 * e + hh) ^ (l32 & 7))) =
          f32x4{acc[n][4 * e], acc[n][4 * e + 1], acc[n][4 * e + 2], acc[n][4 * e + 3]};
  asm volatile("" ::: "memory");
#pragma unroll 1
  for (int e = lane; e < 32 * (D / 4); e += 64) {
    const int r = e / (D / 4), q4 = e % (D / 4);
    f32x4 o = *(const f32x4 *)(so + r * D + 4 * (q4 ^ (r & 7)));
    const int64_t at = (int64_t)(((uint64_t)(uint32_t)__shfl((int)(to_row >> 32), r) << 32) | (uint32_t)__shfl((int)to_row, r));
    const float f = __shfl(by, r);
    const float all = o[0] + o[1] + (o[2] + o[3]);
    if (__any(s_odd || all != all)) {
      const int rlow = __shfl(row.low, r), rhigh = __shfl(row.high, r);
      put_odd<FMT, D, KT>(b, a.first, rlow, rhigh, tiles, s_odd, is_part, __shfl(L, r), q4, o);
    }
    if (at < 0) continue;
    if (a.chunks > 1) *(f32x4 *)(a.po + at * D + 4 * q4) = o;
    else store_out<QT>(a, at * D + 4 * q4, o * f);
  }
}

template <int QT, int FMT, int D, int RT, int OCC> __global__ __launch_bounds__(256, OCC) void history_few_kernel(HistAttnArgs a) {
  __shared__ __align__(1024) uint8_t s_mem[few_lds<D, RT, 4>()];
  warm_kernargs<sizeof(HistAttnArgs)>();
  history_few<QT, FMT, D, RT, 4>(a, false, (int)blockIdx.x, s_mem);
}
template <int QT, int FMT, int D, int OCC> __global__ __launch_bounds__(256, OCC) void history_many_kernel(HistAttnArgs a) {
  __shared__ __align__(1024) uint8_t s_mem[many_lds<D>()];
  warm_kernargs<sizeof(HistAttnArgs)>();
  history_many<QT, FMT, D>(a, false, blockIdx.x, s_mem);
}
// The prefix's pass and behind it the own histories', which fill the chip under its last workgroups: 64 streams of 500 over 24576 shared keys
// 56 us (fp32 85); four streams of 50 over 1000, fp32 in fp16, 10.4 (latencies). The prefix's rows of all streams are in one workgroup's tiles, so
// that its keys are read once for 128 rows.
template <int QT, int FMT, int D, int OCC> __global__ __launch_bounds__(256, OCC) void history_prefix_kernel(HistAttnArgs a) {
  constexpr int few = few_lds<D, 1, 4>();
  __shared__ __align__(1024) uint8_t s_mem[many_lds<D>() > few ? many_lds<D>() : few];
  warm_kernargs<sizeof(HistAttnArgs)>();
  const bool shared = blockIdx.x < (uint32_t)a.pre.blocks;
  const uint32_t block = shared ? blockIdx.x : blockIdx.x - a.pre.blocks;
  if ((shared ? a.pre.block_rows : a.own.block_rows) == 16) history_few<QT, FMT, D, 1, 4>(a, shared, (int)block, s_mem);
  else history_many<QT, FMT, D>(a, shared, block, s_mem);
}

// The chunks that a row has states of: of the prefix, then its own; none for a token that is not there.
struct RowChunks {
  int head, pre, own;
  __device__ __forceinline__ int64_t slot(const HistAttnArgs &a, int64_t row, int c) const { return row * a.chunks + (c < pre ? c : a.pre.chunks + c - pre); }
};
__device__ __forceinline__ RowChunks row_chunks(const HistAttnArgs &a, int64_t row) {
  RowChunks x{};
  x.head = (int)(row % a.qh);
  const int i = (int)(row / a.qh % a.N), s = (int)(row / ((int64_t)a.qh * a.N)), count = step_count(a.counts, s, a.N);
  if (i >= count) return x;
  const int r0 = (i * a.qm + x.head % a.qm) / a.own.block_rows * a.own.block_rows;
  const Visible v = visible_of(a, s, r0 / a.qm, min(count, (r0 + a.own.block_rows - 1) / a.qm + 1) - 1);
  x.own = used_chunks(v.n, chunk_keys(a.own, v.n));
  if (a.p.k) {
    const int n = visible_prefix(a).n;
    x.pre = used_chunks(n, chunk_keys(a.pre, n));
  }
  return x;
}

// Joins a row's chunks, in order: a wave per row, D / 4 lanes a chunk. 4096 rows of 25 chunks of 64: 7.7 us (3.5 TB/s); 512 of up to 12: 5.
template <int QT, int D> __global__ __launch_bounds__(256) void history_merge_kernel(HistAttnArgs a) {
  warm_kernargs<sizeof(HistAttnArgs)>();
  constexpr int LR = D / 4, GR = 64 / LR;    // lanes per chunk, chunks at a time
  const int lane = threadIdx.x & 63, q4 = lane % LR, cg = lane / LR;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.S * a.N * a.qh) return;
  const RowChunks rc = row_chunks(a, row);
  const int used = rc.pre + rc.own;
  float m = kNone;
  for (int c = lane; c < used; c += 64) m = fmaxf(m, a.pm[rc.slot(a, row, c)]);
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  float den = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = cg; c < used; c += GR) {
    const int64_t at = rc.slot(a, row, c);
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
  if (cg == 0 && used) finish_history_row<QT, D>(a, row, rc.head, q4, m, den, sum);
}

// The same for few rows, of many chunks: a workgroup for 64 of a row's columns. Every chunk's factor into LDS first; then sixteen lanes a chunk and sixteen
// chunks at a time, whose sums meet in LDS, in order. (16 rows of 256 chunks of 256: 6.0 us, a wave a row 30; 4096 rows
// of 25 chunks of 64 13, a wave a row 7.7.)
constexpr int kMergeChunks = 2 * kHistChunks, kWideRows = 256;
template <int QT, int D> __global__ __launch_bounds__(256) void history_merge_wide_kernel(HistAttnArgs a) {
  __shared__ float s_f[kMergeChunks], s_red[8];
  __shared__ __align__(16) f32x4 s_o[16][16];
  warm_kernargs<sizeof(HistAttnArgs)>();
  constexpr int PARTS = D / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = (int64_t)(blockIdx.x / PARTS);
  const int part = blockIdx.x % PARTS;
  const RowChunks rc = row_chunks(a, row);
  const int used = rc.pre + rc.own;          // at most kMergeChunks
  if (!used) return;
  float m2[2] = {kNone, kNone}, l2[2] = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (tid + 256 * k < used) m2[k] = a.pm[rc.slot(a, row, tid + 256 * k)], l2[k] = a.pl[rc.slot(a, row, tid + 256 * k)];
  float m = fmaxf(m2[0], m2[1]);
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) s_red[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  float den = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (tid + 256 * k < used) {
      const float f = exp2_(m2[k] - m);
      s_f[tid + 256 * k] = f;
      den = fmaf(l2[k], f, den);
    }
  for (int o = 32; o; o >>= 1) den += __shfl_xor(den, o);
  if (lane == 0) s_red[4 + wave] = den;
  __syncthreads();
  den = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  const int q4 = tid & 15, cg = tid >> 4;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = cg; c < used; c += 16) {
    const f32x4 w = *(const f32x4 *)(a.po + rc.slot(a, row, c) * D + 64 * part + 4 * q4);
    const float f = s_f[c];
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = fmaf(w[k], f, sum[k]);
  }
  s_o[cg][q4] = sum;
  __syncthreads();
  if (tid >= 16) return;
  sum = s_o[0][tid];
  for (int c = 1; c < min(used, 16); ++c) {
    const f32x4 w = s_o[c][tid];
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] += w[k];
  }
  finish_history_row<QT, D>(a, row, rc.head, 16 * part + tid, m, den, sum);
}

// Waves a SIMD of the kernels of few rows, by the registers that a tile's bytes, the queries' terms and the sums take.
template <int QT, int FMT, int D> constexpr int few_waves() {
  if (D == 256) return HistTypes<QT, FMT>::E == 8 || (FMT == H_MXFP8 && HistTypes<QT, FMT>::NQ == 3) ? 1 : 2;
  return D == 64 ? 4 : 3;
}
template <int QT, int FMT, int D> static hipError_t launch_types(HistAttnArgs a, hipStream_t s, int *launches) {
  constexpr int OCC = few_waves<QT, FMT, D>(), OCC_MANY = D == 256 ? 1 : D == 128 ? 2 : HistTypes<QT, FMT>::NQ == 1 && HistTypes<QT, FMT>::MX ? 4 : 3;
  const dim3 grid((uint32_t)(a.pre.blocks + a.own.blocks)), block(256);
  if (a.p.k) hipLaunchKernelGGL((history_prefix_kernel<QT, FMT, D, OCC_MANY>), grid, block, 0, s, a);
  else if (a.own.block_rows == 16) hipLaunchKernelGGL((history_few_kernel<QT, FMT, D, 1, OCC>), grid, block, 0, s, a);
  else if (a.own.block_rows == 32) hipLaunchKernelGGL((history_few_kernel<QT, FMT, D, 2, (OCC > 1 ? OCC - 1 : 1)>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((history_many_kernel<QT, FMT, D, OCC_MANY>), grid, block, 0, s, a);
  *launches = 1;
  if (a.chunks > 1) {
    const int64_t rows = (int64_t)a.S * a.N * a.qh;
    if (rows < kWideRows) hipLaunchKernelGGL((history_merge_wide_kernel<QT, D>), dim3((uint32_t)(rows * (D / 64))), block, 0, s, a);
    else hipLaunchKernelGGL((history_merge_kernel<QT, D>), dim3((uint32_t)((rows + 3) / 4)), block, 0, s, a);
    *launches = 2;
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
