// hh_tree.hip — attention of a tree of drafted tokens over the history, and the accumulation of
// the accepted tokens' attention weights.
//
// Attention. A kv head's rows are the (node, query head) pairs of its group, r = node·qm + head; a
// workgroup takes 32·RT of them and a chunk of the keys (the history's visible rows, behind the last of
// them the drafted ones), a wave 32 rows and every KS-th run of 32 keys. Keys and values go straight to
// an LDS ring, NST − 1 tiles of 32·KS keys ahead. One pass with the running maximum M and sum L of
// each row, everything in the exponent base 2 (y = logit·log2 e):
//   S^T [32 keys × 32 rows] = K · q^T, keys as the A operand, the rows' queries in registers;
//   O^T [D × 32 rows] += V^T · P^T, the value tile read by columns (transposing LDS reads), P^T from S^T's own
//   registers: a lane holds one row's probabilities at 16 keys, and the products' order over the keys is the
//   lane's. So a row's maximum and sum stay in its two lanes, and rescaling needs no exchange.
// Probabilities enter as pairs hi + lo of the values' type, two products each (a single rounding of them would be as large
// as that of the outputs; eight BF16 sequences of up to 8191 keys: 60 us, 58.6 with a single one), and so do the queries of
// F32 activations, of fp16.
// A chunk's state (M, L, O) goes to the workspace and tree_merge_kernel joins a row's chunks in order; a call of
// one chunk writes its outputs at once. The sink enters where the states are joined.
#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 16 bytes per lane from global memory straight into LDS byte `l` + 16·lane; the kernels wait with wait_vm. In
// assembly, so that the compiler does not order the wave's LDS reads after its loads in flight.
__device__ __forceinline__ void dma16(const void *p, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(p) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N < 63 ? N : 63) : "memory"); }
// Barrier after the wave's own LDS reads have returned: the next tile may overwrite what they read.
__device__ __forceinline__ void step_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
typedef __attribute__((address_space(3))) void *lds_ptr_t;
__device__ __forceinline__ uint32_t lds_addr(const void *l) { return (uint32_t)(uintptr_t)(lds_ptr_t)l; }

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

// The ancestors-or-self of every node as bit masks, lane i node i with parent `up`; a parent that is not
// an earlier node counts as none.
__device__ __forceinline__ uint64_t ancestors(int up, int lane) {
  if (up < 0 || up >= lane) up = -1;
  uint64_t mask = 1ull << lane;
  for (int r = 0; r < 6; ++r) {   // lines of up to 64 nodes, by doubling
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
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int at) {
  return ((uint64_t)__shfl((uint32_t)(v >> 32), at) << 32) | __shfl((uint32_t)v, at);
}

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
// Waits for the first of the tiles that were asked for ahead of the loop.
template <int NL, int NST> __device__ __forceinline__ void wait_first(int tiles) {
  if (tiles >= NST - 1) wait_vm<(NST - 2) * NL>();
  else wait_vm<0>();
}

// A sequence's visible history: positions first .. first + keys − 1 (those that its roots see), in chunks of
// `per` keys; chunk c is in use if c·per < keys, or c = 0. A launch sized for shorter histories has
// chunks of more keys.
struct Span {
  int length, first, keys, per;
};
__device__ __forceinline__ Span span_of(const TreeArgs &a, int s) {
  Span p;
  p.length = max(a.lengths[s], 0);
  if (!a.ring) p.length = min(p.length, a.rows);
  p.first = a.ring ? max(0, p.length - a.rows) : 0;
  if (a.window) p.first = max(p.first, (int)max((int64_t)0, (int64_t)p.length - a.window + 1));
  p.keys = p.length - p.first;
  p.per = a.per_chunk;
  if ((int64_t)p.per * a.chunks < p.keys) {
    const int need = (int)((uint32_t)p.keys / (uint32_t)a.chunks) + 1;
    p.per = (int)(((uint32_t)need + a.tile - 1) / (uint32_t)a.tile * (uint32_t)a.tile);
  }
  return p;
}

// A row's four outputs from its joined state: the sink's share of the denominator, the quotient, its rounding.
template <int QT, int D>
__device__ __forceinline__ void finish_row(const TreeArgs &a, int64_t row, int head, int q4, float m, float den, f32x4 o) {
  if (a.sinks) {
    const float y = bf16_bits_to_f32(a.sinks[head]) * kLog2e, mn = fmaxf(m, y), f = exp2_(m - mn);
    den = fmaf(den, f, exp2_(y - mn));
    o *= f;
    m = mn;
  }
  const float inv = 1.f / den;
  if constexpr (QT == E_F32) {
    *(f32x4 *)((float *)a.out + row * D + 4 * q4) = o * inv;
  } else if constexpr (QT == E_F16) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    *(f16x4 *)((_Float16 *)a.out + row * D + 4 * q4) = f16x4{(_Float16)(o[0] * inv), (_Float16)(o[1] * inv), (_Float16)(o[2] * inv), (_Float16)(o[3] * inv)};
  } else {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    *(bf16x4 *)((__bf16 *)a.out + row * D + 4 * q4) = bf16x4{(__bf16)(o[0] * inv), (__bf16)(o[1] * inv), (__bf16)(o[2] * inv), (__bf16)(o[3] * inv)};
  }
  if (q4 == 0 && a.lse) a.lse[row] = (m + __builtin_amdgcn_logf(den)) * kLn2;
}

// QT: hh_elem of q. RT row tiles of 32, KS key splits, a ring of NST tiles, OCC waves per SIMD.
template <int QT, int D, int RT, int KS, int NST, int OCC>
__global__ __launch_bounds__(64 * RT * KS, OCC) void tree_split_kernel(TreeArgs a) {
  constexpr int NW = RT * KS, NT = 64 * NW, KT = 32 * KS, CH = D / 8, NL = D / (8 * RT), STAGE = KT * D * 4;
  constexpr int ROWS = 32 * RT, NB = D / 32;
  constexpr bool BF = QT == E_BF16, PAIR = QT == E_F32;
  constexpr int OUTS = KS * ROWS * D * 4, LDS = NST * STAGE > OUTS ? NST * STAGE : OUTS;
  __shared__ __align__(1024) uint8_t s_mem[LDS];
  __shared__ float s_m[KS][ROWS], s_l[KS][ROWS];
  __shared__ uint64_t s_vis[ROWS];
  __shared__ int s_lo[ROWS], s_odd;
  warm_kernargs<sizeof(TreeArgs)>();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rt = wave % RT, ks = wave / RT, l32 = lane & 31, hh = lane >> 5;
  // Row blocks of one (sequence, kv head, chunk) on one XCD, one after the other: they read the same keys.
  const uint32_t grp = blockIdx.y * 8 + (blockIdx.x & 7), own = a.S * a.kvh;
  const int rb = blockIdx.x >> 3;
  // The last chunks first: theirs are the drafted nodes.
  const uint32_t at_chunk = grp / own;
  const int chunk = a.chunks - 1 - (int)at_chunk;
  if (chunk < 0) return;
  const int sg = (int)(grp - at_chunk * own), s = sg / a.kvh, g = sg - s * a.kvh, qm = a.qm;

  // The lane's row: its node and queries, asked for before anything else (a wait for them behind the tiles' loads
  // would be one for those too).
  const int r = rb * ROWS + rt * 32 + l32, rn = (int)(((float)r + 0.5f) * a.inv_qm);   // r / qm: exact below 2^20
  const bool in = rn < a.N;
  const int node = in ? rn : 0, head = g * qm + (in ? r - rn * qm : 0);
  const int up = lane < a.N ? a.parents[(int64_t)s * a.N + lane] : -1;
  u32x4 qf[D / 16], ql[PAIR ? D / 16 : 1];
  {
    const int64_t at = ((int64_t)s * a.N + node) * a.q_stride + (int64_t)head * D + 8 * hh;
#pragma unroll
    for (int dc = 0; dc < D / 16; ++dc) {
      if constexpr (PAIR) {
        const u32x4 *qp = (const u32x4 *)((const float *)a.q + at + 16 * dc);
        qf[dc] = qp[0];
        ql[dc] = qp[1];
      } else {
        qf[dc] = *(const u32x4 *)((const uint16_t *)a.q + at + 16 * dc);
      }
    }
  }
  const int count = min(max(a.counts[s], 0), a.N);
  if (rb * ROWS >= count * qm) return;
  const Span sp = span_of(a, s);
  const int64_t c064 = (int64_t)chunk * sp.per;
  if (chunk && c064 >= sp.keys) return;
  const int c0 = (int)c064, nc = min(sp.per, sp.keys - c0);   // cached keys of the chunk
  const bool last = c064 + sp.per >= sp.keys;
  const int tiles = (nc + (last ? count : 0) + KT - 1) / KT;
  const float scale = PAIR ? 1.f : fabsf(a.scale) * kLog2e;   // S -> y
#pragma unroll
  for (int dc = 0; dc < D / 16; ++dc) {
    if constexpr (PAIR) {
      f16x8 h, l;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = __uint_as_float(e < 4 ? qf[dc][e & 3] : ql[dc][e & 3]) * (a.scale * kLog2e);
        // Rounded to fp32 before it is split: hi must not come from the product by one mixed-precision
        // instruction, whose single rounding differs near ties from that of the hi that lo is the rest of.
        asm volatile("" : "+v"(v));
        h[e] = (_Float16)v;
        l[e] = (_Float16)(v - (float)h[e]);
      }
      qf[dc] = __builtin_bit_cast(u32x4, h);
      ql[dc] = __builtin_bit_cast(u32x4, l);
    } else {
      if (a.scale < 0.f) qf[dc] ^= 0x80008000u;
    }
  }
  uint64_t vis = 0;
  int lo = 0, lo_max = 0;   // the first cached key of the chunk that the node sees, and that every node sees
  if (last || a.window) {
    const uint64_t mask = ancestors(up, lane);
    vis = shfl64(mask, node);
    if (a.window) {
      auto low = [&](int depth) { return (int)max((int64_t)0, (int64_t)sp.length + depth - a.window + 1 - sp.first) - c0; };
      lo = low(__popcll(vis) - 1);
      int deepest = lane < count ? __popcll(mask) : 1;
      for (int o = 32; o; o >>= 1) deepest = max(deepest, __shfl_xor(deepest, o));
      lo_max = __builtin_amdgcn_readfirstlane(low(deepest - 1));
      while (__popcll(vis) > a.window) vis &= vis - 1;   // the oldest ancestors
    }
  }

  // Loads: 16-byte pieces of a row in consecutive lanes, XORed by the row (sw) so that both ways of reading
  // are free of bank conflicts. Tiles of cached keys that do not pass a ring's end step one address per lane.
  const uint32_t r0 = a.ring ? (uint32_t)(sp.first + c0) % (uint32_t)a.rows : sp.first + c0;
  const uint64_t kb = (uint64_t)(a.k + (int64_t)s * a.seq_stride + (int64_t)g * D);
  const uint64_t vb = (uint64_t)(a.v + (int64_t)s * a.seq_stride + (int64_t)g * D);
  const int64_t dbase = (int64_t)s * a.N * a.kv_stride + (int64_t)g * D;
  const uint64_t dkb = (uint64_t)((const uint16_t *)a.dk + dbase), dvb = (uint64_t)((const uint16_t *)a.dv + dbase);
  const uint32_t lds0 = lds_addr(s_mem), rstride = 2 * a.kvh * D, dstride = 2 * (uint32_t)a.kv_stride;
  auto sw = [](int row) { return ((row & 3) << 1) | ((row >> 2) & 1); };
  constexpr int RPL = NW * 64 / CH;                    // rows that one load of every wave covers
  constexpr int NPT = RPL < 8 ? 8 / RPL : 1;           // addresses per lane: rows not 8 apart differ in their XOR
  uint64_t step[NPT];
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const int p = (i * NW + wave) * 64 + lane, row = p / CH;
    step[i] = (uint64_t)(r0 + row) * rstride + 16 * ((p % CH) ^ sw(row));
  }
  const int plain = min(nc / KT, (int)(((uint32_t)a.rows - r0) / KT));   // tiles 0 .. plain − 1 step so
  auto load_tile = [&](int t, int slot) {
    const uint32_t l0 = lds0 + slot * STAGE + wave * 1024;
    if (t < plain) {
#pragma unroll
      for (int v = 0; v < 2; ++v)                      // keys, values
#pragma unroll
        for (int u = 0; u < NL / 2; ++u)
          dma16((const void *)(step[u % NPT] + ((v ? vb : kb) + (uint64_t)(u / NPT * NPT * RPL) * rstride)),
                __builtin_amdgcn_readfirstlane(l0 + v * (KT * D * 2) + u * NW * 1024));
#pragma unroll
      for (int i = 0; i < NPT; ++i) step[i] += (uint64_t)KT * rstride;
      return;
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const uint64_t cached = v ? vb : kb, drafted = v ? dvb : dkb;
#pragma unroll 4
      for (int u = 0; u < NL / 2; ++u) {
        const int p = (u * NW + wave) * 64 + lane, row = p / CH, c = (p % CH) ^ sw(row);
        const int idx = t * KT + row, m = idx - nc;
        uint32_t rw = r0 + idx;
        rw = rw >= (uint32_t)a.rows ? rw - a.rows : rw;    // a ring's end
        // Behind the cached keys the nodes; rows past the last node are masked: they read node 0's.
        const uint32_t at = m < 0 ? rw : m < count ? m : 0, stride = m < 0 ? rstride : dstride;
        const uint64_t base = (m < 0 ? cached : drafted) + 16 * c;
        dma16((const void *)(base + (uint64_t)at * stride),
              __builtin_amdgcn_readfirstlane(l0 + v * (KT * D * 2) + u * NW * 1024));
      }
    }
  };
  // Not unrolled, as little here is: the first workgroup of a compute unit waits for its instructions (about 0.1 us
  // a 64-byte line).
#pragma unroll 1
  for (int t = 0; t < min(NST - 1, tiles); ++t) load_tile(t, t);

  if (ks == 0 && hh == 0) {
    s_vis[rt * 32 + l32] = vis;
    s_lo[rt * 32 + l32] = lo;
  }
  if (tid == 0) s_odd = 0;
  // A tile that some row does not see whole: infinities and NaN among its values are taken out (0 · NaN would
  // carry them to rows that do not see them) and put back into the rows that do behind the loop.
  auto is_part = [&](int t) { return t * KT < lo_max || (t + 1) * KT > nc; };
  auto clean = [&](int t) {
    uint8_t *vt = s_mem + (t % NST) * STAGE + KT * D * 2;
#pragma unroll
    for (int u = 0; u < D / (16 * RT); ++u) {
      u32x4 *w = (u32x4 *)vt + u * NT + tid;
      u32x4 x = *w;
      bool odd = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t em = BF ? 0x7F80u : 0x7C00u;
        const bool l = (x[e] & em) == em, h = (x[e] >> 16 & em) == em;
        x[e] &= (l ? 0u : 0xFFFFu) | (h ? 0u : 0xFFFF0000u);
        odd |= l || h;
      }
      if (odd) {
        *w = x;
        s_odd = 1;
      }
    }
    step_barrier();
  };
  float M = kNone, L = 0.f, minus1 = -1.f;
  asm volatile("" : "+s"(minus1));
  f32x16 acc[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) acc[n] = f32x16{};
  const int j16 = lane & 15;
  const int vrow = 4 * hh + (j16 >> 2), vpiece = (2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1)) ^ sw(vrow), vhalf = (j16 & 1) * 8;
  // S^T of the wave's 32 keys of tile t.
  auto scores = [&](int t) {
    const uint8_t *krow = s_mem + (t % NST) * STAGE + (32 * ks + l32) * (2 * D);
    f32x16 S = f32x16{};
#pragma unroll
    for (int dc = 0; dc < D / 16; ++dc) {
      const u32x4 kf = *(const u32x4 *)(krow + (((2 * dc + hh) ^ sw(l32)) << 4));
      S = mfma32<BF>(kf, qf[dc], S);
      if constexpr (PAIR) S = mfma32<BF>(kf, ql[dc], S);
    }
    return S;
  };
  // Keys that the row does not see, and the row's maximum. Element i is key 8 (i / 4) + 4 hh + i % 4 of the 32.
  auto masked_top = [&](f32x16 &S, int t, bool part) {
    // Rounded to y here, once: an fma of S behind the maximum would see the product's lost bits, which for logits far from zero are
    // more than the exponent's range. (Only where the maximum is far from zero, by a branch: 64.4 us against 62.2, eight
    // ragged BF16 sequences of up to 8191 keys.)
    if constexpr (!PAIR) S *= scale;
    if (part) {
      // Bit j: the row sees key base + j. Cached keys from lo to nc, then the nodes.
      const int base = t * KT + 32 * ks, from = min(max(lo - base, 0), 32), to = min(max(nc - base, 0), 32), m = base - nc;
      uint32_t sees = (uint32_t)(((1ull << to) - 1) & ~((1ull << from) - 1));
      sees |= m >= 0 ? (m < 64 ? (uint32_t)(vis >> m) : 0u) : m > -32 ? (uint32_t)(vis << -m) : 0u;
      sees >>= 4 * hh;
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = sees >> (8 * (i >> 2) + (i & 3)) & 1 ? S[i] : -INFINITY;
    }
    float top = fmaxf(S[0], S[1]);
#pragma unroll
    for (int i = 2; i < 16; ++i) top = fmaxf(top, S[i]);
    return max_halves(top);
  };
  wait_first<NL, NST>(tiles);
  step_barrier();
  bool part = is_part(0);
  if (part) clean(0);
  f32x16 S = scores(0);
  float top = masked_top(S, 0, part);
  auto step_tile = [&](f32x16 &S, f32x16 &Sn, int t) {
    if (__any(top - M > kLag)) {   // (M + kLag could round past the next logit)
      const float mn = fmaxf(M, top), corr = exp2_(M - mn);
      M = mn;
      L *= corr;
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[n] *= corr;
    }
    // The next tile's scores are formed with this one's probabilities and values: the matrix unit works under the
    // exponentials. Its keys must be there; the slot that the tile before this one left is loaded again.
    const bool more = t + 1 < tiles;
    part = false;
    if (more) {
      if (t + NST - 2 < tiles) wait_vm<(NST - 3) * NL>();
      else wait_vm<0>();
      step_barrier();
      if (t + NST - 1 < tiles) load_tile(t + NST - 1, (t + NST - 1) % NST);
      part = is_part(t + 1);
      if (part) clean(t + 1);
    }
    // Behind the last tile its own scores once more: not used.
    Sn = scores(more ? t + 1 : t);
    const float sub = kOff - M;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      S[i] = exp2_(S[i] + sub);
      sum[i & 3] += S[i];
    }
    L += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    // V^T: lane (l32, hh) takes dimension 32 n + l32 of keys 16 kc + 8 x + 4 hh .. + 3, the order of P^T.
    const uint8_t *vcol = s_mem + (t % NST) * STAGE + KT * D * 2 + (32 * ks + vrow) * (2 * D) + vhalf;
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      u32x4 ph, pl;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = S[8 * kc + 2 * e], p1 = S[8 * kc + 2 * e + 1];
        const u32x2 w = BF ? split_pair_bf16(p0, p1) : split_pair(p0, p1, minus1);
        ph[e] = w[0];
        pl[e] = w[1];
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
        acc[n] = mfma32<BF>(vf, ph, acc[n]);
        acc[n] = mfma32<BF>(vf, pl, acc[n]);
      }
    }
    top = masked_top(Sn, t + 1, part);
  };
  // Two tiles a round: the scores of one and of the next in registers of their own, with no copies between.
  f32x16 Sn;
  for (int t = 0;;) {
    step_tile(S, Sn, t);
    if (++t >= tiles) break;
    step_tile(Sn, S, t);
    if (++t >= tiles) break;
  }

  // The splits' states meet in LDS, the sums of a row in 16-byte pieces XORed by the row.
  L += other_half(L);
  step_barrier();
  float *so = (float *)s_mem + (size_t)(ks * ROWS + rt * 32 + l32) * D;
  if (hh == 0) {
    s_m[ks][rt * 32 + l32] = M - kOff;   // the exponent that L and O are relative to
    s_l[ks][rt * 32 + l32] = L;
  }
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x4 w = {acc[n][4 * e], acc[n][4 * e + 1], acc[n][4 * e + 2], acc[n][4 * e + 3]};
      *(f32x4 *)(so + 4 * ((8 * n + 2 * e + hh) ^ (l32 & 7))) = w;
    }
  __syncthreads();
#pragma unroll 1
  for (int e = tid; e < ROWS * (D / 4); e += NT) {
    const int row = e / (D / 4), q4 = e % (D / 4), rr = rb * ROWS + row, n = (int)(((float)rr + 0.5f) * a.inv_qm);
    if (n >= count) break;               // rows are in the order of their nodes
    float m = s_m[0][row];
#pragma unroll
    for (int k = 1; k < KS; ++k) m = fmaxf(m, s_m[k][row]);
    float den = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const float f = exp2_(s_m[k][row] - m);
      den = fmaf(s_l[k][row], f, den);
      const f32x4 w = *(const f32x4 *)((const float *)s_mem + (size_t)(k * ROWS + row) * D + 4 * (q4 ^ (row & 7)));
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(w[i], f, o[i]);
    }
    if (s_odd) {
      // The infinities and NaN of the tiles that were seen in part, from memory.
      const uint64_t sees = s_vis[row];
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) {
        if (!is_part(t)) continue;
#pragma unroll 1
        for (int k = t * KT; k < min(t * KT + KT, nc + count); ++k) {
          const int m2 = k - nc;
          if (m2 < 0 ? k < s_lo[row] : !(sees >> m2 & 1)) continue;
          uint32_t at = r0 + k;
          at = at >= (uint32_t)a.rows ? at - a.rows : at;
          const uint64_t src = (m2 < 0 ? vb + (uint64_t)at * rstride : dvb + (uint64_t)m2 * dstride) + 8 * q4;
          const u32x2 w = *(const u32x2 *)src;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t h = w[i >> 1] >> 16 * (i & 1) & 0xFFFFu, em = BF ? 0x7F80u : 0x7C00u;
            if ((h & em) == em) o[i] += BF ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
          }
        }
      }
    }
    const int hd = g * qm + rr - n * qm;
    const int64_t out = ((int64_t)s * a.N + n) * a.qh + hd;
    if (a.chunks > 1) {
      const int64_t slot = out * a.chunks + chunk;
      *(f32x4 *)(a.po + slot * D + 4 * q4) = o;
      if (q4 == 0) {
        a.pm[slot] = m;
        a.pl[slot] = den;
      }
    } else {
      finish_row<QT, D>(a, out, hd, q4, m, den, o);
    }
  }
}

// Joins a row's chunks, in order: a wave per row, D / 4 lanes a chunk.
template <int QT, int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
  warm_kernargs<sizeof(TreeArgs)>();
  constexpr int LR = D / 4, GR = 64 / LR;    // lanes per chunk, chunks at a time
  const int lane = threadIdx.x & 63, q4 = lane % LR, cg = lane / LR;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.S * a.N * a.qh) return;
  const int hd = (int)(row % a.qh), n = (int)(row / a.qh % a.N), s = (int)(row / ((int64_t)a.qh * a.N));
  if (n >= a.counts[s]) return;
  const Span sp = span_of(a, s);
  const int used = sp.keys <= sp.per ? 1 : (int)(((uint32_t)sp.keys + sp.per - 1) / (uint32_t)sp.per);
  const float *pm = a.pm + row * a.chunks, *pl = a.pl + row * a.chunks, *po = a.po + row * a.chunks * D;
  float m = kNone;
  for (int c = lane; c < used; c += 64) m = fmaxf(m, pm[c]);
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  float den = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = cg; c < used; c += GR) {
    const float f = exp2_(pm[c] - m);
    den = fmaf(pl[c], f, den);
    const f32x4 w = *(const f32x4 *)(po + (int64_t)c * D + 4 * q4);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = fmaf(w[i], f, sum[i]);
  }
#pragma unroll
  for (int o = LR; o < 64; o <<= 1) {
    den += __shfl_xor(den, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += __shfl_xor(sum[i], o);
  }
  if (cg == 0) finish_row<QT, D>(a, row, hd, q4, m, den, sum);
}

// Accumulated weights. A wave takes 32 keys of a kv head and holds them as the B operand; the accepted tokens'
// queries pass as A tiles of 32 rows, S [32 rows × 32 keys], and a lane adds up one key's column. Every weight is
// read and written once by one lane, in a fixed order. The queries of a (sequence, kv head), scaled and as pairs for
// F32, are laid out in LDS once per workgroup of four waves, with the rows' lse; a row that does not see a key
// (rows of the path behind it) adds nothing. Bound by the keys' bytes; a workgroup walks several runs of keys so that
// the queries' layout is paid for.
constexpr int kWTiles = 4;    // row tiles of 32 that LDS holds at a time
template <int QT, int D>
__global__ __launch_bounds__(256) void weights_kernel(TreeArgs a) {
  constexpr bool BF = QT == E_BF16, PAIR = QT == E_F32;
  constexpr int TERMS = PAIR ? 2 : 1, FR = D / 16;                    // fragments of 16 dimensions
  __shared__ __align__(16) u32x4 s_q[kWTiles][TERMS][FR][64];         // A operand: lane (l32, hh) of each fragment
  __shared__ float s_lse[kWTiles * 32];
  __shared__ int s_row[kWTiles * 32];                                 // the last key that the row sees, −1: none
  warm_kernargs<sizeof(TreeArgs)>();
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, hh = lane >> 5;
  const int first = blockIdx.x % a.chunks, sg = blockIdx.x / a.chunks, s = sg / a.kvh, g = sg - s * a.kvh, qm = a.qm;
  const int length = min(max(a.lengths[s], 0), a.rows);
  const int acc = min(max(a.accepted[s], 0), min(a.N, length));
  const int runs = (length + 127) / 128;                              // of 128 keys, 32 a wave
  if (acc == 0 || first >= runs) return;
  const int rows = acc * qm, tiles = (rows + 31) / 32;
  const int rstride = a.kvh * D;
  const uint16_t *kb = a.k + (int64_t)s * a.seq_stride + (int64_t)g * D;
  float *w = a.weights + (int64_t)sg * a.rows;
  for (int t0 = 0; t0 < tiles; t0 += kWTiles) {
    const int nt = min(kWTiles, tiles - t0);
    if (t0) __syncthreads();
    for (int e = tid; e < nt * FR * 64; e += 256) {
      const int t = e / (FR * 64), dc = e / 64 % FR, l = e & 63;
      const int r = (t0 + t) * 32 + (l & 31), i = (int)(((float)r + 0.5f) * a.inv_qm);
      const int n = i < acc ? a.path[(int64_t)s * a.N + i] : -1;
      const bool ok = n >= 0 && n < a.N;
      const int64_t row = (int64_t)s * a.N + (ok ? n : 0), head = g * qm + (ok ? r - i * qm : 0);
      const int64_t at = row * a.q_stride + head * D + 16 * dc + 8 * (l >> 5);
      if constexpr (PAIR) {
        const f32x4 *qp = (const f32x4 *)((const float *)a.q + at);
        const f32x4 q0 = qp[0], q1 = qp[1];
        f16x8 h, lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float v = (k < 4 ? q0[k & 3] : q1[k & 3]) * (a.scale * kLog2e);
          asm volatile("" : "+v"(v));                                 // rounded before it is split, as above
          h[k] = (_Float16)v;
          lo[k] = (_Float16)(v - (float)h[k]);
        }
        s_q[t][0][dc][l] = __builtin_bit_cast(u32x4, h);
        s_q[t][TERMS - 1][dc][l] = __builtin_bit_cast(u32x4, lo);
      } else {
        s_q[t][0][dc][l] = *(const u32x4 *)((const uint16_t *)a.q + at);
      }
      if (dc == 0 && l < 32) {
        s_lse[t * 32 + l] = ok ? a.lse_in[row * a.qh + head] * kLog2e : 0.f;
        s_row[t * 32 + l] = ok ? length - acc + i : -1;
      }
    }
    __syncthreads();
    const float scale = PAIR ? 1.f : a.scale * kLog2e;
    for (int run = first; run < runs; run += a.chunks) {
      const int key = run * 128 + wave * 32 + l32;
      if (run * 128 + wave * 32 >= length) continue;
      const u32x4 *kp = (const u32x4 *)(kb + (int64_t)min(key, length - 1) * rstride) + hh;
      u32x4 kf[FR];
#pragma unroll
      for (int dc = 0; dc < FR; ++dc) kf[dc] = kp[2 * dc];
      float sum = 0.f;
      for (int t = 0; t < nt; ++t) {
        f32x16 S = f32x16{};
#pragma unroll
        for (int dc = 0; dc < FR; ++dc) {
          S = mfma32<BF>(s_q[t][0][dc][lane], kf[dc], S);
          if constexpr (PAIR) S = mfma32<BF>(s_q[t][TERMS - 1][dc][lane], kf[dc], S);
        }
        // Element i is row 8 (i / 4) + 4 hh + i % 4 of the tile.
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = 32 * t + 8 * (i >> 2) + 4 * hh + (i & 3);
          const float p = exp2_(fmaf(S[i], scale, -s_lse[r]));
          part[i & 3] += key <= s_row[r] ? p : 0.f;
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
      }
      sum += other_half(sum);
      if (hh == 0 && key < length) w[key] += sum;
    }
  }
}

// The launch: RT by the rows of a kv head; KS so that a workgroup fills its compute unit's LDS and registers by itself
// (two waves per SIMD, heads of 256 one) with four tiles, 64 KB or more, in flight or in use. Whole call, 16 nodes of
// 64 / 8 heads of 64 at 32768 keys (F32, RT 4): KS 2 with a ring of four tiles 31.6 us, of six 32.9, KS 3 (twelve waves) 31.3;
// before the next tile's scores were formed under the exponentials: two workgroups of KS 2 per unit 36.5, one of KS 4 41.
// RT 4 is at the matrix unit's and the VALU's time one after the other (16 products of 32 cycles and about 100
// instructions a tile and wave; eight ragged sequences with heads of 128: 39 and 45 percent of the busy cycles at 3.3 TB/s), smaller RT at HBM.
struct TreeShape { int rt, ks; };
static TreeShape tree_shape(int d, int rows) {
  const int rt = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  if (d == 64) return {rt, rt == 4 ? 2 : 4};
  return {rt, d == 128 ? 2 : 1};
}

// Fills in how the call's keys are split, for histories of up to `length` keys.
void tree_plan(TreeArgs &a, int64_t length) {
  const int rows = a.N * a.qm;
  const TreeShape t = tree_shape(a.d, rows);
  a.tile = 32 * t.ks;
  a.row_blocks = (rows + 32 * t.rt - 1) / (32 * t.rt);
  int64_t keys = length < a.rows ? length : a.rows;
  if (a.window && keys > a.window) keys = a.window;
  const int64_t own = (int64_t)a.S * a.kvh * a.row_blocks;
  int64_t chunks = kTreeGroups / own, most = (keys + a.tile - 1) / a.tile;
  // A few tiles one after the other take less than a second launch that joins them (4 to 6 us).
  if (chunks > most || most <= kTreeTiles) chunks = most <= kTreeTiles ? 1 : most;
  if (chunks > kTreeChunks) chunks = kTreeChunks;
  if (chunks < 1) chunks = 1;
  int64_t per = ((keys + chunks - 1) / chunks + a.tile - 1) / a.tile * a.tile;
  if (per < a.tile) per = a.tile;
  a.per_chunk = (int)per;
  a.chunks = (int)((keys + per - 1) / per);
  if (a.chunks < 1) a.chunks = 1;
}

size_t tree_workspace(const TreeArgs &a) {
  return a.chunks > 1 ? sizeof(float) * (size_t)a.S * a.N * a.qh * a.chunks * (a.d + 2) : 0;
}

// The most that tree_workspace asks for with up to a.S sequences, a.N nodes and `length` keys, whatever the windows. Fewer keys or
// nodes may take more chunks: chunks are whole tiles, and wider ones where a head has few rows.
size_t tree_reserve(const TreeArgs &a, int64_t length) {
  const int64_t keys = length < a.rows ? length : a.rows;
  size_t most = 0;
  for (int n = 1; n <= a.N; ++n) {
    const int rows = n * a.qm;
    const TreeShape t = tree_shape(a.d, rows);
    const int64_t own = (int64_t)a.kvh * ((rows + 32 * t.rt - 1) / (32 * t.rt)), tiles = (keys + 32 * t.ks - 1) / (32 * t.ks);
    int64_t chunks = kTreeGroups / own;                       // of all sequences
    if (chunks < 2 || tiles <= kTreeTiles) continue;          // one a sequence
    if (chunks > a.S * tiles) chunks = a.S * tiles;
    const size_t b = sizeof(float) * (size_t)n * a.qh * chunks * (a.d + 2);
    if (b > most) most = b;
  }
  return most;
}

template <int QT, int D> static hipError_t launch_tree_d(const TreeArgs &a, hipStream_t s) {
  const TreeShape t = tree_shape(D, a.N * (a.qh / a.kvh));
  const int64_t groups = (int64_t)a.S * a.kvh * a.chunks;
  const dim3 grid(8 * a.row_blocks, (uint32_t)((groups + 7) / 8)), block(64 * t.rt * t.ks);
  constexpr int K4 = D == 256 ? 1 : 2, K2 = D == 64 ? 4 : K4, NST = 4;
  if (t.rt == 1) hipLaunchKernelGGL((tree_split_kernel<QT, D, 1, K2, NST, 1>), grid, block, 0, s, a);
  else if (t.rt == 2) hipLaunchKernelGGL((tree_split_kernel<QT, D, 2, K2, NST, D == 64 ? 2 : 1>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((tree_split_kernel<QT, D, 4, K4, NST, D == 256 ? 1 : 2>), grid, block, 0, s, a);
  if (a.chunks > 1) {
    const int64_t rows = (int64_t)a.S * a.N * a.qh;
    hipLaunchKernelGGL((tree_merge_kernel<QT, D>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <int QT> static hipError_t launch_tree_q(const TreeArgs &a, hipStream_t s) {
  if (a.d == 64) return launch_tree_d<QT, 64>(a, s);
  return a.d == 128 ? launch_tree_d<QT, 128>(a, s) : launch_tree_d<QT, 256>(a, s);
}

hipError_t launch_tree(const TreeArgs &a, int type, hipStream_t s) {
  if (type == E_F32) return launch_tree_q<E_F32>(a, s);
  return type == E_F16 ? launch_tree_q<E_F16>(a, s) : launch_tree_q<E_BF16>(a, s);
}

template <int QT> static void launch_weights_q(const TreeArgs &a, dim3 grid, hipStream_t s) {
  if (a.d == 64) hipLaunchKernelGGL((weights_kernel<QT, 64>), grid, dim3(256), 0, s, a);
  else if (a.d == 128) hipLaunchKernelGGL((weights_kernel<QT, 128>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((weights_kernel<QT, 256>), grid, dim3(256), 0, s, a);
}

hipError_t launch_weights(TreeArgs a, int type, hipStream_t s) {
  const int64_t own = (int64_t)a.S * a.kvh, runs = ((int64_t)a.rows + 127) / 128;
  int64_t x = kWeightGroups / own;
  if (x > runs) x = runs;
  if (x < 1) x = 1;
  a.chunks = (int)x;   // workgroups of a (sequence, kv head)
  const dim3 grid((uint32_t)(x * own));
  if (type == E_F32) launch_weights_q<E_F32>(a, grid, s);
  else if (type == E_F16) launch_weights_q<E_F16>(a, grid, s);
  else launch_weights_q<E_BF16>(a, grid, s);
  return hipGetLastError();
}

}  // namespace hh
