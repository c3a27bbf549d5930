// hh_cache.hip — the accepted rows of a drafted tree into the histories of many layers, and the
// eviction of the rows of least accumulated weight.
#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

// Rows that a sequence's histories take: `accepted`, bounded by the path and the room left.
__device__ __forceinline__ int committed(const RowsLayer &y, const RowsArgs &a, int s) {
  const int acc = min(max(a.accepted[s], 0), a.N);
  return min(acc, max(0, y.limit - max(y.lengths[s], 0)));
}

// One workgroup per (layer, sequence, up to eight places on the path: 16 KB of rows). With `arrivals` (a launch of all
// layers), the last one of a sequence also does what advance_kernel does: the others have read the lengths by then. Bound
// by the launch and the chain length, node, row: 12 layers of eight sequences, 16 nodes, 10.9 us a call, 6.4 of it on the
// GPU; a workgroup a place (4.1) and a second launch for the lengths (1.9) took 13.9. 36 layers of one sequence, 28 nodes of
// 8 KB: 14 us by eight places a workgroup, 10 by two.
constexpr int kPlaces = 8;
__host__ __device__ inline int places(int kvh, int d) {   // 16 KB of a sequence's rows
  const int p = 16384 / (4 * kvh * d);
  return p < 1 ? 1 : p > kPlaces ? kPlaces : p;
}
__device__ __forceinline__ void advance(const RowsLayer &y, const RowsArgs &a, int s) {
  if (!y.last) return;
  const int c = committed(y, a, s);
  y.lengths[s] = max(y.lengths[s], 0) + c;
  if (y.next) y.next[s] += c;
}
__global__ __launch_bounds__(256) void commit_kernel(RowsArgs a) {
  __shared__ int64_t s_src[kPlaces], s_dst[kPlaces];   // elements; s_src −1: nothing to do
  __shared__ int s_last;
  const int each = places(a.kvh, a.d), parts = (a.N + each - 1) / each, i0 = blockIdx.x % parts * each, s = blockIdx.x / parts % a.S;
  const RowsLayer &y = a.layer[blockIdx.x / (parts * a.S)];
  const int tid = threadIdx.x, c = committed(y, a, s), n = min(each, c - i0), start = max(y.lengths[s], 0);
  if (n > 0) {
    if (tid < n) {
      const int i = i0 + tid, node = a.path[(int64_t)s * a.N + i];
      const int64_t pos = (int64_t)start + i, row = y.ring ? pos % y.rows : pos;
      // A ring takes the last rows of a path longer than itself.
      const bool in = node >= 0 && node < a.N && i >= c - y.rows && row < y.rows;
      s_src[tid] = in ? ((int64_t)s * a.N + node) * a.kv_stride : -1;
      s_dst[tid] = row;
    }
    __syncthreads();
    const int vecs = a.kvh * a.d / 8, all = n * 2 * vecs;
    for (int e0 = tid; e0 < all; e0 += 4 * 256) {
      u32x4 r[4];
      uint16_t *to[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + 256 * u, i = e / (2 * vecs), o = e - i * 2 * vecs;
        to[u] = nullptr;
        if (e >= all || s_src[i] < 0) continue;
        const bool v = o >= vecs;
        const int at = 8 * (v ? o - vecs : o);
        r[u] = *(const u32x4 *)((v ? y.dv : y.dk) + s_src[i] + at);
        to[u] = (v ? y.v : y.k) + (int64_t)s * y.seq_stride + s_dst[i] * a.kvh * a.d + at;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (to[u]) *(u32x4 *)to[u] = r[u];
    }
    if (y.weights || y.positions)
      for (int e = tid; e < n * a.kvh; e += 256) {
        const int i = e / a.kvh, g = e - i * a.kvh;
        if (s_src[i] < 0) continue;
        const int64_t at = ((int64_t)s * a.kvh + g) * y.rows + s_dst[i];
        if (y.weights) y.weights[at] = 0.f;
        if (y.positions) y.positions[at] = y.next[s] + i0 + i;
      }
  }
  if (!a.arrivals) return;
  __syncthreads();   // every wave has its lengths and next position
  if (tid == 0) s_last = atomicAdd(a.arrivals + s, 1u) == (uint32_t)(a.layers * parts) - 1;
  __syncthreads();
  if (!s_last) return;
  if (tid < a.layers) advance(a.layer[tid], a, s);
  if (tid == 0) atomicExch(a.arrivals + s, 0u);
}

// The lengths and next positions, once for the layers that share them.
__global__ __launch_bounds__(64) void advance_kernel(RowsArgs a) {
  for (int s = threadIdx.x; s < a.S; s += 64) advance(a.layer[blockIdx.x], a, s);
}

// Eviction's order as an unsigned key: recent rows above every weight, NaN as minus infinity, the two
// zeros equal.
__device__ __forceinline__ uint32_t rank_key(float w, int pos, int64_t oldest) {
  if (pos >= oldest) return 0xFFFFFFFFu;
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w == 0.f ? 0.f : w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup per (layer, sequence, kv head) finds the key of the keep-th row and lists the rows that move.
// A wave owns runs of 64 consecutive rows, a lane per row of a run, their keys in LDS (CAP = 0: more rows than that, read
// again from memory at each step). The key is built from its highest bit, eleven bits a step, by a histogram of the rows
// that share what is known of it; the bits that all keys share are skipped, which spreads the rest over many bins (LDS
// adds to one address go one after the other); a step whose bin is taken whole ends it. Then a lane holds the
// masks of a run's rows above and at the key, ranks the rows that go from below `keep` and those that stay from
// `keep` on by scans over the runs, and the rows are listed in order.
// 96 heads of 4112 rows: 13.6 us; the key two bits a step by counting, then the lists by two walks over the rows, 24; by
// histograms of eight bits with a serial scan 46 (both with 1024 threads).
template <int CAP, int T>
__global__ __launch_bounds__(T) void select_kernel(RowsArgs a) {
  constexpr int W = T / 64, kBits = T == 1024 ? 11 : T == 512 ? 10 : 9;   // 2·T bins
  static_assert(1 << kBits == 2 * T, "two bins a thread");
  __shared__ uint32_t s_key[CAP ? CAP : 1];
  __shared__ int s_hist[1 << kBits], s_sum[W], s_n[W][2], s_found[3];
  __shared__ uint32_t s_and[W], s_or[W];
  const int head = blockIdx.x, g = head % a.kvh, s = head / a.kvh % a.S;
  const RowsLayer &y = a.layer[head / (a.kvh * a.S)];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = min(max(y.lengths[s], 0), y.rows);
  if (n <= a.keep) {
    if (tid == 0) a.moves[head] = 0;
    return;
  }
  const int64_t oldest = (int64_t)y.next[s] - a.recent;
  const int64_t base = ((int64_t)s * a.kvh + g) * y.rows;
  const float *w = y.weights + base;
  const int *pos = y.positions + base;
  // Rows first .. first + 64 · runs − 1; four runs at a time (rows past n have key 0, which no row has).
  const int runs = ((n + T - 1) / T + 3) & ~3, first = wave * runs * 64;
  uint32_t all = 0xFFFFFFFFu, any = 0;
  for (int i0 = 0; i0 < runs; i0 += 4) {
    float wv[4];
    int pv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = min(first + 64 * (i0 + u) + lane, n - 1);
      wv[u] = w[at];
      pv[u] = pos[at];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = first + 64 * (i0 + u) + lane;
      const uint32_t k = rank_key(wv[u], pv[u], oldest);
      if (r < n) all &= k, any |= k;
      if constexpr (CAP > 0) s_key[r] = r < n ? k : 0;   // r < T · runs <= CAP
    }
  }
  auto key_of = [&](int i) -> uint32_t {
    const int r = first + 64 * i + lane;
    if constexpr (CAP > 0) return s_key[r];
    return r < n ? rank_key(w[r], pos[r], oldest) : 0;
  };
  for (int o = 32; o; o >>= 1) all &= __shfl_xor(all, o), any |= __shfl_xor(any, o);
  if (lane == 0) s_and[wave] = all, s_or[wave] = any;
  s_hist[2 * tid] = s_hist[2 * tid + 1] = 0;
  __syncthreads();
  for (int i = 0; i < W; ++i) all &= s_and[i], any |= s_or[i];
  // Of the rows that agree with t above `bit`, the `need` first in the order are among those that stay, as are all rows
  // above them. At the end t is the key of the last that stays.
  int bit = 32 - __builtin_clz((all ^ any) | 1), need = a.keep;
  uint32_t t = bit == 32 ? 0u : all >> bit << bit;
  while (bit > 0) {
    const int shift = max(bit - kBits, 0), bins = 1 << (bit - shift);
    const uint32_t known = bit == 32 ? 0u : ~0u << bit;
    for (int i0 = 0; i0 < runs; i0 += 4) {
      uint32_t k[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) k[u] = key_of(i0 + u);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k[u] && (k[u] & known) == t) atomicAdd(&s_hist[(k[u] & ~known) >> shift], 1);
    }
    __syncthreads();
    // Rows in this thread's two bins and in all above them.
    const int h0 = s_hist[2 * tid], h1 = s_hist[2 * tid + 1];
    int sum = h0 + h1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_down(sum, o);
      if (lane + o < 64) sum += v;
    }
    if (lane == 0) s_sum[wave] = sum;
    __syncthreads();
    for (int i = wave + 1; i < W; ++i) sum += s_sum[i];
    s_hist[2 * tid] = s_hist[2 * tid + 1] = 0;
    // The bin in which the count from the top reaches `need`.
    const int over = sum - h0 - h1;
    if (over < need && sum >= need) {
      const bool upper = over + h1 >= need;
      s_found[0] = 2 * tid + upper;
      s_found[1] = need - (upper ? over : over + h1);
      s_found[2] = upper ? h1 : h0;
    }
    __syncthreads();
    t |= (uint32_t)s_found[0] << shift;
    need = s_found[1];
    bit = shift;
    if (need == s_found[2]) break;   // the whole bin stays: every row of at least t
  }
  // Rows above t stay, and of those equal to it the first: as many as are left (all of them, if t splits exactly).
  const uint64_t below = (1ull << lane) - 1;
  uint64_t above = 0, equal = 0;     // of the rows of run `from` + lane
  auto masks = [&](int from) {
    above = equal = 0;
    for (int i0 = from; i0 < min(runs, from + 64); i0 += 4) {
      uint32_t k[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) k[u] = key_of(i0 + u);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint64_t m = __ballot(k[u] > t), e = __ballot(k[u] == t);
        if (lane == i0 + u - from) above = m, equal = e;
      }
    }
  };
  auto wave_total = [](int v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
  };
  auto before_lane = [&](int v) {    // exclusive prefix over the lanes
    int p = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int q = __shfl_up(p, o);
      if (lane >= o) p += q;
    }
    return p - v;
  };
  int n_above = 0, n_equal = 0;
  for (int from = 0; from < runs; from += 64) {
    masks(from);
    n_above += wave_total(__popcll(above));
    n_equal += wave_total(__popcll(equal));
  }
  if (lane == 0) s_n[wave][0] = n_above, s_n[wave][1] = n_equal;
  __syncthreads();
  int rank = 0, left = a.keep;       // equal rows of the waves before this one, and those that stay of all
  for (int i = 0; i < W; ++i) {
    left -= s_n[i][0];
    if (i < wave) rank += s_n[i][1];
  }
  __syncthreads();
  int32_t *src = a.from + (int64_t)head * a.max_moves, *dst = a.to + (int64_t)head * a.max_moves;
  int hole_at = 0, move_at = 0, total = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int eq_rank = rank, holes = 0, moves = 0;
    for (int from = 0; from < runs; from += 64) {
      if (runs > 64) masks(from);
      // This lane's run: its rows that stay, then those that leave a hole below `keep` and those that fill one.
      const int mine = __popcll(equal), had = eq_rank + before_lane(mine);
      uint64_t stay = equal;
      for (int drop = mine - max(0, min(mine, left - had)); drop > 0; --drop) stay &= ~(1ull << (63 - __clzll((long long)stay)));
      stay |= above;
      const int64_t r0 = first + 64 * (int64_t)(from + lane);
      const bool run = from + lane < runs;
      auto rows_below = [&](int64_t end) { return end <= r0 ? 0ull : end - r0 >= 64 ? ~0ull : (1ull << (end - r0)) - 1; };
      const uint64_t h = run ? rows_below(min(a.keep, n)) & ~stay : 0, m = run ? stay & ~rows_below(a.keep) : 0;
      const int nh = __popcll(h), nm = __popcll(m);
      if (pass) {
        int hi = hole_at + holes + before_lane(nh), mi = move_at + moves + before_lane(nm);
        for (uint64_t left_h = h; left_h; left_h &= left_h - 1, ++hi)
          if (hi < a.max_moves) dst[hi] = (int)r0 + __ffsll((unsigned long long)left_h) - 1;
        for (uint64_t left_m = m; left_m; left_m &= left_m - 1, ++mi)
          if (mi < a.max_moves) src[mi] = (int)r0 + __ffsll((unsigned long long)left_m) - 1;
      }
      eq_rank += wave_total(mine);
      holes += wave_total(nh);
      moves += wave_total(nm);
    }
    if (pass) break;
    if (lane == 0) s_n[wave][0] = holes, s_n[wave][1] = moves;
    __syncthreads();
    for (int i = 0; i < W; ++i) {
      if (i < wave) hole_at += s_n[i][0], move_at += s_n[i][1];
      total += s_n[i][1];
    }
  }
  if (tid == 0) a.moves[head] = min(total, a.max_moves);
}

// Moves the rows of a head, a group of lanes per row and four rows in flight; the sources, at `keep` and above,
// and the destinations, below it, do not overlap. One workgroup of the last layer that shares them shortens the
// lengths.
__global__ __launch_bounds__(256) void move_kernel(RowsArgs a, int parts) {
  const int head = blockIdx.x / parts, part = blockIdx.x % parts;
  const int g = head % a.kvh, s = head / a.kvh % a.S;
  const RowsLayer &y = a.layer[head / (a.kvh * a.S)];
  if (y.last && g == 0 && part == 0 && threadIdx.x == 0) y.lengths[s] = min(y.lengths[s], a.keep);
  const int moves = a.moves[head];
  const int32_t *src = a.from + (int64_t)head * a.max_moves, *dst = a.to + (int64_t)head * a.max_moves;
  const int lanes = a.d / 8, per = 256 / lanes, lane = threadIdx.x % lanes;
  const int64_t base = (int64_t)s * y.seq_stride + (int64_t)g * a.d + 8 * lane, meta = ((int64_t)s * a.kvh + g) * y.rows;
  const int64_t row = (int64_t)a.kvh * a.d;
  for (int i0 = part * 4 * per + threadIdx.x / lanes; i0 < moves; i0 += parts * 4 * per) {
    int f[4], t[4];
    u32x4 k[4], v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(i0 + u * per, moves - 1);
      f[u] = src[i];
      t[u] = dst[i];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      k[u] = *(const u32x4 *)(y.k + base + f[u] * row);
      v[u] = *(const u32x4 *)(y.v + base + f[u] * row);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + u * per >= moves) break;
      *(u32x4 *)(y.k + base + t[u] * row) = k[u];
      *(u32x4 *)(y.v + base + t[u] * row) = v[u];
      if (lane == 0) {
        y.weights[meta + t[u]] = y.weights[meta + f[u]];
        y.positions[meta + t[u]] = y.positions[meta + f[u]];
      }
    }
  }
}

hipError_t launch_commit(const RowsArgs &a, bool last, hipStream_t s) {
  const int each = places(a.kvh, a.d);
  if (last) hipLaunchKernelGGL(advance_kernel, dim3(a.layers), dim3(64), 0, s, a);
  else hipLaunchKernelGGL(commit_kernel, dim3(a.layers * a.S * ((a.N + each - 1) / each)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_evict(const RowsArgs &a, hipStream_t s) {
  const int heads = a.layers * a.S * a.kvh;
  int rows = 0;
  for (int i = 0; i < a.layers; ++i) rows = a.layer[i].rows > rows ? a.layer[i].rows : rows;
  // Waves by the rows: barriers cost more the more of them wait, and workgroups share a compute unit. 288 heads of 156
  // rows 20.4 us with 1024 threads, 12.5 with 256; 96 of 4112 15.8 with 1024, 13.6 with 512; a whole cycle with 384 heads
  // of 7016 34.8 and 27.8.
  if (rows <= 2048) hipLaunchKernelGGL((select_kernel<2048, 256>), dim3(heads), dim3(256), 0, s, a);
  else if (rows <= 8192) hipLaunchKernelGGL((select_kernel<8192, 512>), dim3(heads), dim3(512), 0, s, a);
  else if (rows <= 36864) hipLaunchKernelGGL((select_kernel<36864, 1024>), dim3(heads), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((select_kernel<0, 1024>), dim3(heads), dim3(1024), 0, s, a);
  // Workgroups enough to fill the chip with rows in flight, of at least four rounds' rows each.
  const int per = 4 * 256 / (a.d / 8);
  int parts = 4096 / heads, most = (a.max_moves + per - 1) / per;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  hipLaunchKernelGGL(move_kernel, dim3(heads * parts), dim3(256), 0, s, a, parts);
  return hipGetLastError();
}

}  // namespace hh
