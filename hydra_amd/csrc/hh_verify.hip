// hh_verify.hip — verification of drafted tokens against the target's probabilities.
//
// With p and q the target's and the draft's probabilities at a node, the residual after its first j
// children were rejected is, before it is normalised, r_j(v) = max(p(v) − c_j q_j(v), 0) off the tokens
// tried, of mass W_j: r_0 = p, c_0 = 0, W_0 = 1. Rejecting a child subtracts its distribution q_j from
// r_j / W_j. For independent draws q_j = q and c_{j+1} = c_j + W_j; where the tried tokens are not put back q_j is
// q off them, normalised, and c_{j+1} = (c_j + W_j) R_j, R_j the mass of q_j off the j-th; c = 0 for given tokens. A
// child with token x is accepted if r_j(x) > u W_j q_j(x). That needs no normalised copy of a row, and does
// not depend on what happens at other nodes: every node's tests are made at once, and the walk follows.
// q_j goes by the maximum and the sum of the tokens off those tried, which the chunks keep from round to round: what is
// left of a sharp draft may be any number of times smaller than what was tried.
//
// A row of logits is cut into chunks, a workgroup each, so that one sequence's rows fill the chip:
//   stats    every row's maximum and sum of exponentials by chunk (greedy: its largest entry);
//   round j  of the nodes with at least j children that a path may still end at: the j-th child's test, then W_j and
//            the draft's maxima and sums off it by chunk (given tokens: all tests and the last residual in one round);
//   leaf     (where leaves' logits are many) the statistics of the leaf that a path ends at;
//   walk     a workgroup per sequence follows the accepted children and finds the next token: its chunk by the
//            chunks' sums, its place by a scan of that chunk.
// Bound by the launches' dependent chain for a few rows, and by the exponentials in 64 bits for many: the next token
// is where a sum of up to V terms passes a random bound, and with errors of 1e-7 in it one in twenty draws from
// the tail of 250000 tokens would differ. exp goes by a table of 2^(i / 256) and four terms of a series behind the 1 (relative
// error below 1e-15 beside the argument's), thirteen instructions in fp64.
#include <climits>

#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

constexpr int kVT = 256;              // threads of stats and rounds
constexpr int kWalkT = 1024;
// Leaves' statistics are left for behind the rounds, when one a sequence is left, from this many bytes of logits on (a launch more). Four
// trees of V 248320, four children a node, both ways in turn on three sets of inputs: 31 nodes (119 MB) 97 to 99 us and without 110 to 113,
// 21 nodes (79 MB) 82 to 87 and 89 to 95, 16 (60 MB) 77 to 79 and 80 to 83, 11 (40 MB) 62 to 65 and 63 to 66; 21 given nodes 40 and 45.
constexpr size_t kLateLeaves = (size_t)64 << 20;

__device__ __forceinline__ float finite_or_less(float x) { return x != x ? -INFINITY : x; }

// exp((x − top) / temperature) = 2^(y / 256), y = (x − top)·k <= 0, with tab[i] = 2^(i / 256) in LDS and k = 256 log2(e) /
// temperature. (The difference first: x·k − top·k is wrong for rows of a type's lowest value.) y is split by adding
// 1.5·2^52, whose low word is then the nearest integer, and the power of two goes into the exponent's bits. Below
// 2^−1000: 0.
__device__ __forceinline__ double exp_of(float x, double top, double k, const double *tab) {
  constexpr double magic = 6755399441055744.0, c = 0.0027076061740622863;   // ln 2 / 256
  const double y = fmax(((double)x - top) * k, -256.0 * 1001), m = y + magic, f = y - (m - magic);
  const int i = (int)(uint32_t)__builtin_bit_cast(uint64_t, m);
  double s = fma(f, c * c * c * c / 24, c * c * c / 6);
  s = fma(f, s, c * c / 2);
  s = fma(f, s, c);
  s = fma(f, s, 1.0);
  const uint64_t v = __builtin_bit_cast(uint64_t, s * tab[i & 255]);
  const uint32_t hi = (uint32_t)(v >> 32) + ((uint32_t)(i >> 8) << 20);
  return i >= -256 * 1000 ? __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)v) : 0.0;
}
// The same for a row whose largest entry is infinite: its +inf entries share the probability, a row of −inf has none.
__device__ __forceinline__ double exp_any(float x, float top, double k, const double *tab) {
  if (fabsf(top) == INFINITY) return top > 0.f && x == top ? 1.0 : 0.0;
  return exp_of(x, top, k, tab);
}
// exp_any as a call: where each of a kernel's few uses is run once, its instructions are fetched once (a cold
// 64-byte line of instructions costs about 0.1 us).
__device__ __noinline__ double exp_call(float x, float top, double k, const double *tab) {
  return exp_any(x, top, k, tab);
}
__device__ __forceinline__ void fill_table(double *tab) {
  if (threadIdx.x < 256) tab[threadIdx.x] = exp2((double)threadIdx.x / 256);
}

// Sum and maximum over a workgroup, in a fixed order, in every thread. s_d: T / 64 doubles of its own per call site.
template <int T> __device__ __forceinline__ double block_sum(double v, double *s_d) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) s_d[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = s_d[0];
  for (int w = 1; w < T / 64; ++w) t += s_d[w];
  return t;
}
template <int T> __device__ __forceinline__ float block_max(float v, float *s_f) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) s_f[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = s_f[0];
  for (int w = 1; w < T / 64; ++w) t = fmaxf(t, s_f[w]);
  return t;
}

// Chunks begin at a multiple of four elements in memory, up to three before the row's first: rows of any length load whole
// vectors (16 trees of five rows of 131071 bf16, greedy: 13.2 us, single elements 15.4).
template <class T> __device__ __forceinline__ int first_of(const T *row, int chunk, int size) {
  return chunk * size - (int)((uintptr_t)row / sizeof(T) & 3);
}
// Logits v0 + 4 (256 i + thread) + e of a row, −inf outside it and for NaN.
template <class T, int EPT> __device__ __forceinline__ void load_chunk(const T *row, int v0, int V, float (&x)[EPT]) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const bool aligned = (((uintptr_t)row + v0 * (intptr_t)sizeof(T)) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < EPT / 4; ++i) {
    const int v = v0 + 4 * (kVT * i + (int)threadIdx.x);
    if (aligned && v >= 0 && v + 4 <= V) {
      const vec4 w = *(const vec4 *)(row + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = finite_or_less((float)w[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = v + e >= 0 && v + e < V ? finite_or_less((float)row[v + e]) : -INFINITY;
    }
  }
}

// What rounds leave of a node: reciprocals of its rows' sums, their maxima (the draft's off the tokens tried before), and the
// factor of the draft in the round's residual.
struct NodeState {
  double ip, iq, c;
  float mp, mq;
};

// The workspace. Chunk arrays are [row][chunks], row = s·N + n; part, state: of odd and even rounds; max_of, sum_of: of the
// target, and of the draft behind even (0: no token tried yet) and odd rounds.
// accept: the round in which a node was accepted, 0 if in none.
struct VerifyPlan {
  int chunk, chunks;
  size_t max_of[3], sum_of[3], part[2], state[2], accept, best, total;
};
constexpr size_t kWideChunks = (size_t)512 * 4096;   // logits from which on chunks are of 4096
__host__ __device__ inline void place_arrays(VerifyPlan &p, size_t rows, size_t n);
__host__ __device__ inline VerifyPlan verify_plan(int S, int N, int V, bool aligned) {
  VerifyPlan p{};
  const size_t rows = (size_t)S * N;
  // 4096 logits a workgroup where that makes 512 of them, else 1024 (16 or 4 a thread). Six nodes of 32000 fp32 logits:
  // 21 us with 1024, 28 with 4096; four trees of 21 nodes of 248320, up to four children a node: 100 to 103 and 82 to 87; 16 trees of
  // five nodes of 131071 bf16 logits, greedy: 16.5 and 13.5.
  p.chunk = rows * V >= kWideChunks ? 4096 : 1024;
  p.chunks = (V + (aligned ? 0 : 3) + p.chunk - 1) / p.chunk;
  place_arrays(p, rows, rows * p.chunks);
  return p;
}
// Where the arrays of `rows` rows and `n` chunks lie.
__host__ __device__ inline void place_arrays(VerifyPlan &p, size_t rows, size_t n) {
  size_t c = 0;
  auto take = [&](size_t bytes) {
    const size_t o = c;
    c += (bytes + 255) / 256 * 256;
    return o;
  };
  for (int i = 0; i < 3; ++i) {
    p.max_of[i] = take(4 * n);
    p.sum_of[i] = take(8 * n);
  }
  for (int i = 0; i < 2; ++i) {
    p.part[i] = take(8 * n);
    p.state[i] = take(sizeof(NodeState) * rows);
  }
  p.accept = take(4 * rows);
  p.best = take(4 * n);
  p.total = c;
}

// The children of node n as a mask, the first `most`, from every node's parent in its lane of the wave.
__device__ __forceinline__ uint64_t children_in(int parent, int n, int count, int most) {
  const int lane = threadIdx.x & 63;
  uint64_t m = __ballot(lane > n && lane < count && parent == n);
  if (__popcll(m) > most) {
    uint64_t left = m;
    for (int i = 0; i < most; ++i) left &= left - 1;
    m &= ~left;
  }
  return m;
}

__device__ __forceinline__ uint64_t children_of(const VerifyArgs &a, int s, int n, int count, int most) {
  return children_in(a.parents[(int64_t)s * a.N + min((int)threadIdx.x & 63, a.N - 1)], n, count, most);
}

// Flags of `accept` in a launch that also writes them: only what earlier rounds wrote may count, so that what a workgroup does
// is the same for all its waves, whenever they look.
__device__ __forceinline__ bool accepted_before(const int32_t *flag, int round) {
  const int at = __hip_atomic_load(flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return at != 0 && at < round;
}
__device__ __forceinline__ void accept_in(int32_t *flag, int round) {
  __hip_atomic_store(flag, round, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The node that a path ends at, in every lane of the wave: yes, up: a node accepted at its parent, in its lane. len: nodes of
// the path; place: the path's entry of this lane.
__device__ __forceinline__ int path_end(bool yes, int up, int count, int &len, int &place) {
  const int lane = threadIdx.x & 63;
  int cur = 0;
  len = count > 0 ? 1 : 0, place = lane == 0 && len ? 0 : -1;
  if (count > 0)
    for (;;) {   // a child comes behind its parent: at most N steps
      const uint64_t m = __ballot(yes && up == cur);
      if (!m) break;
      cur = __ffsll((unsigned long long)m) - 1;
      if (lane == len) place = cur;
      ++len;
    }
  return cur;
}

// Sum of a chunk's exponentials below its largest entry, in every thread of the workgroup.
template <int EPT>
__device__ __forceinline__ double chunk_sum(const float (&x)[EPT], float all, double k, const double *tab, double *s_d) {
  double sum = 0.0;
  if (fabsf(all) == INFINITY) {
    const bool one = all > 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) sum += one && x[i] == all ? 1.0 : 0.0;
  } else {
    const double top = all;
#pragma unroll
    for (int i = 0; i < EPT; ++i) sum += exp_of(x[i], top, k, tab);   // −inf: 0
  }
  return block_sum<kVT>(sum, s_d);
}

template <class T, int EPT, bool GREEDY>
__global__ __launch_bounds__(kVT) void stats_kernel(VerifyArgs a, VerifyPlan w) {
  __shared__ double s_tab[256], s_d[kVT / 64];
  __shared__ float s_f[kVT / 64];
  __shared__ int s_i[kVT / 64];
  const int chunk = blockIdx.x % w.chunks, row = blockIdx.x / w.chunks, s = row / a.N, n = row - s * a.N, tid = threadIdx.x;
  const int count = min(max(a.counts[s], 0), a.N), of = blockIdx.y;
  if (n >= count) return;
  if (!GREEDY && !of && chunk == 0 && tid == 0) ((int32_t *)(a.ws + w.accept))[row] = 0;
  // The draft's row of a node that has no children is not used; of the target's one of a sequence's at most.
  if ((of || (!GREEDY && a.late_leaves)) && children_of(a, s, n, count, a.children) == 0) return;
  if (!GREEDY) fill_table(s_tab);
  const T *base = (const T *)(of ? a.draft : a.target) + (int64_t)row * (of ? a.d_stride : a.t_stride);
  float x[EPT];
  // Both rows in the target's chunks, as the rounds: equal rows have equal sums.
  const int v0 = first_of((const T *)a.target + (int64_t)row * a.t_stride, chunk, w.chunk);
  load_chunk<T, EPT>(base, v0, a.V, x);
  float top = x[0];
#pragma unroll
  for (int i = 1; i < EPT; ++i) top = fmaxf(top, x[i]);
  const float all = block_max<kVT>(top, s_f);
  const size_t at = (size_t)row * w.chunks + chunk;
  if (GREEDY) {
    int best = a.V;
#pragma unroll
    for (int i = EPT - 1; i >= 0; --i)
      if (x[i] == all) best = v0 + 4 * (kVT * (i / 4) + tid) + i % 4;
    for (int o = 32; o; o >>= 1) best = min(best, __shfl_xor(best, o));
    if ((tid & 63) == 0) s_i[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
      for (int k = 1; k < kVT / 64; ++k) best = min(best, s_i[k]);
      ((float *)(a.ws + w.max_of[0]))[at] = all;
      ((int32_t *)(a.ws + w.best))[at] = best;
    }
    return;
  }
  const double sum = chunk_sum<EPT>(x, all, a.k, s_tab, s_d);
  if (tid == 0) {
    ((float *)(a.ws + w.max_of[of]))[at] = all;
    ((double *)(a.ws + w.sum_of[of]))[at] = sum;
  }
}

// With late_leaves: the statistics of the one leaf that a sequence's path ends at, if it ends at one.
template <class T, int EPT>
__global__ __launch_bounds__(kVT) void leaf_kernel(VerifyArgs a, VerifyPlan w) {
  __shared__ double s_tab[256], s_d[kVT / 64];
  __shared__ float s_f[kVT / 64];
  const int chunk = blockIdx.x % w.chunks, s = blockIdx.x / w.chunks, tid = threadIdx.x, lane = tid & 63;
  const int count = min(max(a.counts[s], 0), a.N);
  if (count == 0) return;
  const int64_t node = (int64_t)s * a.N + min(lane, a.N - 1);
  const int up = a.parents[node], took = ((const int32_t *)(a.ws + w.accept))[node];
  int len, place;
  const int n = path_end(lane < count && up >= 0 && up < lane && took, up, count, len, place);
  if (children_in(up, n, count, a.children)) return;
  fill_table(s_tab);
  const int64_t row = (int64_t)s * a.N + n;
  float x[EPT];
  const T *base = (const T *)a.target + row * a.t_stride;
  load_chunk<T, EPT>(base, first_of(base, chunk, w.chunk), a.V, x);
  float top = x[0];
#pragma unroll
  for (int i = 1; i < EPT; ++i) top = fmaxf(top, x[i]);
  const float all = block_max<kVT>(top, s_f);
  const double sum = chunk_sum<EPT>(x, all, a.k, s_tab, s_d);
  if (tid == 0) {
    ((float *)(a.ws + w.max_of[0]))[(size_t)row * w.chunks + chunk] = all;
    ((double *)(a.ws + w.sum_of[0]))[(size_t)row * w.chunks + chunk] = sum;
  }
}

// A row's maximum and sum from its chunks'.
template <int T>
__device__ __forceinline__ double joined(const float *mx, const double *sm, int chunks, double k, const double *tab, float *s_f,
                                         double *s_d, float &top) {
  float m = -INFINITY;
  for (int c = threadIdx.x; c < chunks; c += T) m = fmaxf(m, mx[c]);
  top = block_max<T>(m, s_f);
  double z = 0.0;
#pragma unroll 1
  for (int c = threadIdx.x; c < chunks; c += T) z += sm[c] * exp_call(mx[c], top, k, tab);
  return block_sum<T>(z, s_d);
}

template <class T, int EPT, int MODE>
__global__ __launch_bounds__(kVT) void round_kernel(VerifyArgs a, VerifyPlan w, int round) {
  __shared__ double s_tab[256], s_d[5][kVT / 64];
  __shared__ float s_f[3][kVT / 64];
  __shared__ int s_tok[kTreeNodes];
  constexpr bool DRAWN = MODE != 0;
  const int chunk = blockIdx.x % w.chunks, row = blockIdx.x / w.chunks, s = row / a.N, n = row - s * a.N, tid = threadIdx.x;
  const int lane = tid & 63;
  const int count = min(max(a.counts[s], 0), a.N);
  if (n >= count) return;
  const int parent = a.parents[(int64_t)s * a.N + min(lane, a.N - 1)];
  const uint64_t kids = children_in(parent, n, count, a.children);
  const int k = __popcll(kids);
  if (k < round) return;
  if (DRAWN && round > 1) {
    // Rows that no path ends at any more by the rounds before: with a child accepted, or rejected themselves, or with a
    // sibling accepted.
    const int32_t *flag = (const int32_t *)(a.ws + w.accept) + (int64_t)s * a.N + min(lane, a.N - 1);
    const uint64_t taken = __ballot(lane < count && accepted_before(flag, round));
    if (kids & taken) return;
    if (n > 0) {
      const uint64_t sib = children_in(parent, __shfl(parent, n), count, a.children), me = 1ull << n;
      const bool told = __popcll(sib & (me - 1)) < round - 1;
      if (!(sib & me) || (sib & taken & ~me) || (told && !(taken & me))) return;
    }
  }
  const int tried = DRAWN ? round : k;       // given tokens: what is left when all are rejected
  const T *tr = (const T *)a.target + (int64_t)row * a.t_stride;
  const T *dr = (const T *)a.draft + (int64_t)row * a.d_stride;
  const int v0 = first_of(tr, chunk, w.chunk);
  float x[EPT], y[DRAWN ? EPT : 1];
  load_chunk<T, EPT>(tr, v0, a.V, x);
  if constexpr (DRAWN) load_chunk<T, EPT>(dr, v0, a.V, y);
  fill_table(s_tab);
  if (tid < 64 && (kids >> lane & 1)) {      // the tokens in the order of their trial
    const int at = __popcll(kids & ((1ull << lane) - 1));
    s_tok[at] = a.tokens[(int64_t)s * a.N + lane];
  }
  __syncthreads();
  const size_t at = (size_t)row * w.chunks;
  NodeState st{};
  double mass = 1.0;
  if (round == 1) {
    float m;
    const double zp = joined<kVT>((const float *)(a.ws + w.max_of[0]) + at, (const double *)(a.ws + w.sum_of[0]) + at, w.chunks,
                                  a.k, s_tab, s_f[0], s_d[0], m);
    st.mp = m;
    st.ip = zp > 0 ? 1.0 / zp : 0.0;
  } else {
    st = ((const NodeState *)(a.ws + w.state[(round - 1) & 1]))[row];
    const double *pw = (const double *)(a.ws + w.part[(round - 1) & 1]) + at;
    double sw = 0.0;
    for (int c = tid; c < w.chunks; c += kVT) sw += pw[c];
    mass = block_sum<kVT>(sw, s_d[2]);
  }
  const int before = 1 + ((round - 1) & 1);   // the draft's maxima and sums off the tokens tried before this round
  const float *mx_q = (const float *)(a.ws + w.max_of[before]) + at;
  const double *sm_q = (const double *)(a.ws + w.sum_of[before]) + at;
  if (DRAWN && (round == 1 || MODE == 2)) {
    float m;
    const double zq = joined<kVT>(mx_q, sm_q, w.chunks, a.k, s_tab, s_f[1], s_d[1], m);
    if (round > 1) st.c *= zq * exp_call(m, st.mq, a.k, s_tab) * st.iq;   // the mass off the last token
    st.mq = m;
    st.iq = zq > 0 ? 1.0 / zq : 0.0;
  }
  if (chunk == 0 && tid < 64) {
    int32_t *accept = (int32_t *)(a.ws + w.accept) + (int64_t)s * a.N;
    if constexpr (DRAWN) {
      uint64_t m = kids;
      for (int i = 1; i < round; ++i) m &= m - 1;
      const int child = __ffsll((unsigned long long)m) - 1, t = s_tok[round - 1];
      bool again = false;
      for (int i = 0; i < round - 1; ++i) again |= s_tok[i] == t;
      if (lane == 0 && mass > 0 && t >= 0 && t < a.V && !again) {
        const double p = exp_call(finite_or_less((float)tr[t]), st.mp, a.k, s_tab) * st.ip;
        const double q = exp_call(finite_or_less((float)dr[t]), st.mq, a.k, s_tab) * st.iq;
        if (fmax(p - st.c * q, 0.0) > (double)a.u[(int64_t)s * a.N + child] * mass * q) accept_in(accept + child, round);
      }
    } else if (kids >> lane & 1) {
      // Every child at once, in its own lane: the mass left at its turn is what the distinct tokens before it have not.
      const int mine = __popcll(kids & ((1ull << lane) - 1)), t = s_tok[mine];
      double before = 0.0;
      bool again = false;
      for (int i = 0; i < mine; ++i) {
        const int o = s_tok[i];
        again |= o == t;
        bool first = o >= 0 && o < a.V;
        for (int e = 0; e < i; ++e) first &= s_tok[e] != o;
        if (first) before += exp_call(finite_or_less((float)tr[o]), st.mp, a.k, s_tab) * st.ip;
      }
      if (t >= 0 && t < a.V && !again &&
          exp_call(finite_or_less((float)tr[t]), st.mp, a.k, s_tab) * st.ip > (double)a.u[(int64_t)s * a.N + lane] * fmax(1.0 - before, 0.0))
        accept_in(accept + lane, round);
    }
  }
  st.c = DRAWN ? st.c + mass : 0.0;
  if (chunk == 0 && tid == 0) ((NodeState *)(a.ws + w.state[round & 1]))[row] = st;
  // The residual off the tokens tried, of which few chunks hold one.
  bool here = false;
  for (int i = 0; i < tried; ++i) here |= s_tok[i] >= v0 && s_tok[i] < v0 + w.chunk;
  if (here) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int v = v0 + 4 * (kVT * (i / 4) + tid) + i % 4;
      for (int e = 0; e < tried; ++e)
        if (s_tok[e] == v) {
          x[i] = -INFINITY;
          if constexpr (DRAWN) y[i] = -INFINITY;
        }
    }
  }
  double sw = 0.0;
  if (!(mass > 0)) {
    // Nothing was left before: p and the draft normalised anew would differ by a rounding.
  } else if (fabsf(st.mp) == INFINITY || (DRAWN && fabsf(st.mq) == INFINITY)) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const double p = exp_call(x[i], st.mp, a.k, s_tab) * st.ip;
      double q = 0.0;
      if constexpr (DRAWN) q = exp_call(y[i], st.mq, a.k, s_tab) * st.iq;
      sw += fmax(p - st.c * q, 0.0);
    }
  } else {
    const double mp = st.mp, mq = st.mq, cq = st.c * st.iq;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const double p = exp_of(x[i], mp, a.k, s_tab);
      if constexpr (DRAWN) {
        const double q = exp_of(y[i], mq, a.k, s_tab);
        sw += fmax(p * st.ip - cq * q, 0.0);
      } else {
        sw += p * st.ip;
      }
    }
  }
  sw = block_sum<kVT>(sw, s_d[4]);
  if (tid == 0) ((double *)(a.ws + w.part[round & 1]))[at + chunk] = sw;
  if constexpr (MODE == 2) {
    // The draft off this round's token too: new where it is this chunk's.
    float top = mx_q[chunk];
    double sum = sm_q[chunk];
    if (s_tok[round - 1] >= v0 && s_tok[round - 1] < v0 + w.chunk) {
      float most = y[0];
#pragma unroll
      for (int i = 1; i < EPT; ++i) most = fmaxf(most, y[i]);
      top = block_max<kVT>(most, s_f[2]);
      sum = chunk_sum<EPT>(y, top, a.k, s_tab, s_d[3]);
    }
    if (tid == 0) {
      ((float *)(a.ws + w.max_of[1 + (round & 1)]))[at + chunk] = top;
      ((double *)(a.ws + w.sum_of[1 + (round & 1)]))[at + chunk] = sum;
    }
  }
}

template <class T>
__global__ __launch_bounds__(kWalkT) void walk_kernel(VerifyArgs a, VerifyPlan w) {
  __shared__ double s_tab[256], s_d[kWalkT / 64], s_scan[kWalkT / 64], s_goal;
  __shared__ float s_f[kWalkT / 64];
  __shared__ int s_best[kTreeNodes], s_tok[kTreeNodes], s_cur, s_hit[2];
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int count = min(max(a.counts[s], 0), a.N);
  const bool greedy = a.inv_t == 0.0;
  if (greedy) {
    for (int n = wave; n < count; n += kWalkT / 64) {   // the rows' largest entries, the lowest of equals
      const size_t at = ((size_t)s * a.N + n) * w.chunks;
      const float *mx = (const float *)(a.ws + w.max_of[0]) + at;
      const int32_t *bx = (const int32_t *)(a.ws + w.best) + at;
      float m = -INFINITY;
      int b = a.V;
      for (int c = lane; c < w.chunks; c += 64)
        if (mx[c] > m) m = mx[c], b = bx[c];
      for (int o = 32; o; o >>= 1) {
        const float om = __shfl_xor(m, o);
        const int ob = __shfl_xor(b, o);
        if (om > m || (om == m && ob < b)) m = om, b = ob;
      }
      if (lane == 0) s_best[n] = m > -INFINITY ? b : -1;
    }
    __syncthreads();
  } else {
    fill_table(s_tab);
  }
  if (wave == 0) {
    const int64_t at = (int64_t)s * a.N;
    const bool real = lane < count;
    const int up = real ? a.parents[at + lane] : -1, token = real ? a.tokens[at + lane] : -1;
    bool yes = real && up >= 0 && up < lane;
    if (greedy) {
      yes = yes && token >= 0 && token == s_best[yes ? up : 0];
      // Children past the most that are tried.
      int before = 0;
      for (int i = 0; i < 64; ++i) {
        const int other = __shfl(up, i);   // by every lane: lane i among them
        before += i < lane && other == up;
      }
      yes = yes && before < a.children;
    } else if (yes) {
      yes = ((const int32_t *)(a.ws + w.accept))[at + lane] != 0;
    }
    int len, place;
    const int cur = path_end(yes, up, count, len, place);
    if (lane < a.N) a.path[at + lane] = place;
    if (lane == 0) {
      a.accepted[s] = len;
      s_cur = cur;
    }
  }
  __syncthreads();
  const int n = s_cur, row = s * a.N + n;
  if (count == 0 || greedy) {
    if (tid == 0) a.next[s] = count == 0 ? -1 : s_best[n];
    return;
  }
  const size_t at = (size_t)row * w.chunks;
  const uint64_t kids = children_of(a, s, n, count, a.children);
  const int k = __popcll(kids);
  if (tid < 64 && (kids >> lane & 1)) s_tok[__popcll(kids & ((1ull << lane) - 1))] = a.tokens[(int64_t)s * a.N + lane];
  const float *mx = (const float *)(a.ws + w.max_of[0]) + at;
  const double *sm = (const double *)(a.ws + w.sum_of[0]) + at;
  const int parity = a.mode ? k & 1 : 1;
  const double *pw = (const double *)(a.ws + w.part[parity]) + at;
  // Runs of chunks per thread; the running sum over them, first of the residual.
  const int per = (w.chunks + kWalkT - 1) / kWalkT, c0 = min(tid * per, w.chunks), c1 = min(c0 + per, w.chunks);
  auto scan = [&](double v, double &whole) {   // exclusive prefix over the threads
    double p = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double q = __shfl_up(p, o);
      if (lane >= o) p += q;
    }
    __syncthreads();
    if (lane == 63) s_scan[wave] = p;
    __syncthreads();
    double before = 0.0;
    whole = 0.0;
    for (int i = 0; i < kWalkT / 64; ++i) {
      if (i < wave) before += s_scan[i];
      whole += s_scan[i];
    }
    const double e = __shfl_up(p, 1);
    return before + (lane ? e : 0.0);
  };
  NodeState st{};
  double own = 0.0, whole = 0.0, run = 0.0;
  if (k) {
    st = ((const NodeState *)(a.ws + w.state[parity]))[row];
    for (int c = c0; c < c1; ++c) own += pw[c];
    run = scan(own, whole);
  }
  // A leaf, or a residual without mass: the target's own probabilities.
  const bool resid = whole > 0;
  if (!resid) {
    const double zp = joined<kWalkT>(mx, sm, w.chunks, a.k, s_tab, s_f, s_d, st.mp);
    if (!(zp > 0)) {
      if (tid == 0) a.next[s] = -1;
      return;
    }
    st.ip = 1.0 / zp;
    own = 0.0;
#pragma unroll 1
    for (int c = c0; c < c1; ++c) own += sm[c] * exp_call(mx[c], st.mp, a.k, s_tab) * st.ip;
    run = scan(own, whole);
  }
  // s_hit[0]: the first chunk past the goal, s_hit[1]: the last with any mass (for a goal that rounding puts at the whole).
  const double goal = (double)fmaxf(a.u_final[s], 0.f) * whole;
  if (tid < 2) s_hit[tid] = tid ? -1 : w.chunks;
  __syncthreads();
  // (One atomic a wave: the same address from every lane would be 64 of them in turn.)
  auto meet = [&](int first, int last) {
    const uint64_t f = __ballot(first < INT_MAX), l = __ballot(last >= 0);
    if (f && lane == __ffsll((unsigned long long)f) - 1) atomicMin(&s_hit[0], first);
    if (l && lane == 63 - __clzll((long long)l)) atomicMax(&s_hit[1], last);
  };
  double upto = run;
  int first = INT_MAX, last = -1;
#pragma unroll 1
  for (int c = c0; c < c1; ++c) {
    const double v = resid ? pw[c] : sm[c] * exp_call(mx[c], st.mp, a.k, s_tab) * st.ip;
    if (v > 0) {
      last = c;
      if (upto + v > goal) first = min(first, c);
    }
    upto += v;
  }
  meet(first, last);
  __syncthreads();
  const int chunk = s_hit[0] < w.chunks ? s_hit[0] : s_hit[1];
  __syncthreads();
  if (chunk >= c0 && chunk < c1) {   // the thread that holds it: what is left of the goal there
    upto = run;
#pragma unroll 1
    for (int c = c0; c < chunk; ++c) upto += resid ? pw[c] : sm[c] * exp_call(mx[c], st.mp, a.k, s_tab) * st.ip;
    s_goal = goal - upto;
  }
  if (tid < 2) s_hit[tid] = tid ? -1 : a.V;
  __syncthreads();
  // The place in the chunk: one or four logits a thread.
  const T *tr = (const T *)a.target + (int64_t)row * a.t_stride;
  const T *dr = (const T *)a.draft + (int64_t)row * a.d_stride;
  const int ept = w.chunk / kWalkT, v0 = first_of(tr, chunk, w.chunk) + tid * ept;
  float x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = i < ept && v0 + i >= 0 && v0 + i < a.V;
    x[i] = in ? finite_or_less((float)tr[v0 + i]) : -INFINITY;
    y[i] = in && resid && a.mode ? finite_or_less((float)dr[v0 + i]) : -INFINITY;
  }
  bool here = false;
  if (resid)
    for (int e = 0; e < k; ++e) here |= s_tok[e] >= v0 && s_tok[e] < v0 + ept;
  double r[4], mine = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = 0.0;
    if (i >= ept) break;
    r[i] = exp_call(x[i], st.mp, a.k, s_tab) * st.ip;
    if (resid && a.mode) r[i] = fmax(r[i] - st.c * st.iq * exp_call(y[i], st.mq, a.k, s_tab), 0.0);
    if (here)
      for (int e = 0; e < k; ++e) r[i] = s_tok[e] == v0 + i ? 0.0 : r[i];
    mine += r[i];
  }
  const double want = s_goal;
  double end, sum = scan(mine, end);
  first = INT_MAX, last = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r[i] > 0) {
      last = v0 + i;
      if (sum + r[i] > want) first = min(first, v0 + i);
    }
    sum += r[i];
  }
  meet(first, last);
  __syncthreads();
  if (tid == 0) a.next[s] = s_hit[0] < a.V ? s_hit[0] : s_hit[1];
}

bool verify_fits(int S, int N, int V) {
  const VerifyPlan p = verify_plan(S, N, V, false);
  return (size_t)S * N * p.chunks <= (size_t)1 << 22;
}

size_t verify_workspace(int S, int N, int V) { return verify_plan(S, N, V, false).total; }

// Fewer logits may make more chunks, of 1024: each begun one of a row, and all of fewer than kWideChunks logits.
size_t verify_reserve(int S, int N, int V) {
  VerifyPlan p = verify_plan(S, N, V, false);
  const size_t rows = (size_t)S * N;
  size_t n = rows * p.chunks;
  if (p.chunk == 4096) {
    const size_t some = kWideChunks / 1024 + rows * (1024 + 2) / 1024 + 1, all = rows * ((V + 3 + 1023) / 1024);
    const size_t narrow = some < all ? some : all;
    if (narrow > n) n = narrow;
  }
  place_arrays(p, rows, n);
  return p.total;
}

template <class T, int EPT> static int launch_verify_t(const VerifyArgs &a, const VerifyPlan &w, hipStream_t s) {
  const uint32_t blocks = (uint32_t)((size_t)a.S * a.N * w.chunks);
  int launches = 2;
  if (a.inv_t == 0.0) {
    hipLaunchKernelGGL((stats_kernel<T, EPT, true>), dim3(blocks), dim3(kVT), 0, s, a, w);
  } else {
    hipLaunchKernelGGL((stats_kernel<T, EPT, false>), dim3(blocks, a.mode && a.children ? 2 : 1), dim3(kVT), 0, s, a, w);
    const int rounds = a.mode ? a.children : a.children ? 1 : 0;
    for (int j = 1; j <= rounds; ++j) {
      if (a.mode == 0) hipLaunchKernelGGL((round_kernel<T, EPT, 0>), dim3(blocks), dim3(kVT), 0, s, a, w, j);
      else if (a.mode == 1) hipLaunchKernelGGL((round_kernel<T, EPT, 1>), dim3(blocks), dim3(kVT), 0, s, a, w, j);
      else hipLaunchKernelGGL((round_kernel<T, EPT, 2>), dim3(blocks), dim3(kVT), 0, s, a, w, j);
    }
    launches += rounds;
    if (a.late_leaves) {
      hipLaunchKernelGGL((leaf_kernel<T, EPT>), dim3((uint32_t)(a.S * w.chunks)), dim3(kVT), 0, s, a, w);
      ++launches;
    }
  }
  hipLaunchKernelGGL((walk_kernel<T>), dim3(a.S), dim3(kWalkT), 0, s, a, w);
  return launches;
}

hipError_t launch_verify(VerifyArgs a, hipStream_t s, int *launches) {
  const size_t vec = a.type == E_F32 ? 16 : 8;
  const bool drafted = a.mode != 0;
  const VerifyPlan w = verify_plan(a.S, a.N, a.V, ((uintptr_t)a.target | (drafted ? (uintptr_t)a.draft : 0)) % vec == 0 &&
                                                      (a.t_stride | (drafted ? a.d_stride : 0)) % 4 == 0);
  a.late_leaves = a.inv_t != 0.0 && (size_t)a.S * (a.N - 1) * a.V * (a.type == E_F32 ? 4 : 2) >= kLateLeaves;
  auto go = [&](auto t) {
    using T = decltype(t);
    return w.chunk == 4096 ? launch_verify_t<T, 16>(a, w, s) : launch_verify_t<T, 4>(a, w, s);
  };
  *launches = a.type == E_F32 ? go(float{}) : a.type == E_F16 ? go(_Float16{}) : go(__bf16{});
  return hipGetLastError();
}

}  // namespace hh
