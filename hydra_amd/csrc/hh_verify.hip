// hh_verify.hip — verification of drafted tokens against the target's probabilities.
//
// With p and q the target's and the draft's probabilities at a node, the residual after its first j
// children were rejected is, before it is normalised, r_j(v) = max(p(v) − c_j q(v), 0) off the tokens
// tried, of mass W_j: r_0 = p, c_0 = 0, W_0 = 1. Rejecting a child subtracts its distribution q_j from
// r_j / W_j, so c_{j+1} = c_j + W_j for independent draws (q_j = q), c_j + W_j / R_j where the tried
// tokens are not put back (q_j = q / R_j, R_j the mass of q off them), and c = 0 for given tokens. A
// child with token x is accepted if r_j(x) > u W_j q_j(x). That needs no normalised copy of a row, and does
// not depend on what happens at other nodes: every node's tests are made at once, and the walk follows.
#include "hh_common.hpp"
#include "hh_draft.hpp"

namespace hh {

template <class T> __device__ __forceinline__ float logit(const void *row, int v) {
  const float x = (float)((const T *)row)[v];
  return x != x ? -INFINITY : x;
}

// exp((x − top) / temperature): entries equal to the largest are 1 also where that is infinite.
__device__ __forceinline__ double scaled_exp(float x, float top, double inv_t) {
  if (x == -INFINITY) return 0.0;
  return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t);
}

constexpr int kVT = 1024;

template <class F> __device__ __forceinline__ double block_sum(double v, double *s_d) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_d[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < kVT / 64; ++w) t += s_d[w];
  return t;
}
__device__ __forceinline__ float block_max(float v, double *s_d) {
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_d[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = -INFINITY;
  for (int w = 0; w < kVT / 64; ++w) t = fmaxf(t, (float)s_d[w]);
  return t;
}

struct NodeState {
  double zp, zq, c, w, rest;
  float mp, mq;
  int tried;
};

__device__ __forceinline__ bool is_tried(const int *s_tok, int n, int v) {
  for (int i = 0; i < n; ++i)
    if (s_tok[i] == v) return true;
  return false;
}

// Children of a node in order, at most `most`: their indices into s_child; returns how many.
__device__ __forceinline__ int children_of(const VerifyArgs &a, int s, int n, int count, int most, int *s_child) {
  int k = 0;
  for (int m = n + 1; m < count && k < most; ++m)
    if (a.parents[(int64_t)s * a.N + m] == n) s_child[k++] = m;
  return k;
}

template <class T>
__global__ __launch_bounds__(kVT) void node_kernel(VerifyArgs a) {
  __shared__ double s_d[kVT / 64];
  __shared__ int s_child[kTreeNodes], s_tok[kTreeNodes], s_k;
  const int n = blockIdx.x % a.N, s = blockIdx.x / a.N, tid = threadIdx.x;
  const int count = min(max(a.counts[s], 0), a.N);
  if (n >= count) return;
  NodeState *st = (NodeState *)a.ws + blockIdx.x;
  int *accept = (int *)((NodeState *)a.ws + a.S * a.N) + s * a.N;
  if (tid == 0) s_k = children_of(a, s, n, count, a.children, s_child);
  __syncthreads();
  const int k = s_k;
  const T *tr = (const T *)a.target + ((int64_t)s * a.N + n) * a.t_stride;
  const T *dr = (const T *)a.draft + ((int64_t)s * a.N + n) * a.d_stride;
  const bool q_on = a.mode != 0 && k > 0;
  float mp = -INFINITY, mq = -INFINITY;
  for (int v = tid; v < a.V; v += kVT) {
    mp = fmaxf(mp, logit<T>(tr, v));
    if (q_on) mq = fmaxf(mq, logit<T>(dr, v));
  }
  mp = block_max(mp, s_d);
  mq = block_max(mq, s_d);
  if (a.inv_t == 0.0) {   // greedy: the lowest of the largest
    int best = a.V;
    for (int v = tid; v < a.V; v += kVT)
      if (logit<T>(tr, v) == mp) { best = v; break; }
    for (int o = 32; o; o >>= 1) best = min(best, __shfl_xor(best, o));
    __shared__ int s_best[kVT / 64];
    if ((tid & 63) == 0) s_best[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < kVT / 64; ++w) best = min(best, s_best[w]);
      if (mp == -INFINITY) best = -1;
      st->tried = best;
      for (int j = 0; j < k; ++j) {
        const int x = a.tokens[(int64_t)s * a.N + s_child[j]];
        accept[s_child[j]] = x >= 0 && x == best;
      }
    }
    return;
  }
  double zp = 0.0, zq = 0.0;
  for (int v = tid; v < a.V; v += kVT) {
    zp += scaled_exp(logit<T>(tr, v), mp, a.inv_t);
    if (q_on) zq += scaled_exp(logit<T>(dr, v), mq, a.inv_t);
  }
  zp = block_sum<T>(zp, s_d);
  zq = block_sum<T>(zq, s_d);
  const double ip = zp > 0 ? 1.0 / zp : 0.0, iq = zq > 0 ? 1.0 / zq : 0.0;
  double c = 0.0, w = 1.0, rest = 1.0;
  int tried = 0;
  for (int j = 0; j < k; ++j) {
    const int m = s_child[j], x = a.tokens[(int64_t)s * a.N + m];
    const bool in = x >= 0 && x < a.V, again = in && is_tried(s_tok, tried, x);
    if (tid == 0) {
      int yes = 0;
      if (in && !again) {
        const double p = scaled_exp(logit<T>(tr, x), mp, a.inv_t) * ip;
        const double q0 = q_on ? scaled_exp(logit<T>(dr, x), mq, a.inv_t) * iq : 1.0;
        const double q = a.mode == 2 ? q0 / fmax(rest, 0x1p-52) : q0;
        const double r = q_on ? fmax(p - c * q0, 0.0) : p;
        yes = r > (double)a.u[(int64_t)s * a.N + m] * w * q;
      }
      accept[m] = yes;
    }
    __syncthreads();
    if (in && !again) {
      if (tid == 0) s_tok[tried] = x;
      ++tried;
    }
    __syncthreads();
    if (q_on) c += a.mode == 2 ? w / fmax(rest, 0x1p-52) : w;
    double ws = 0.0, rs = 0.0;
    for (int v = tid; v < a.V; v += kVT) {
      if (is_tried(s_tok, tried, v)) continue;
      const double p = scaled_exp(logit<T>(tr, v), mp, a.inv_t) * ip;
      if (!q_on) { ws += p; continue; }
      const double q = scaled_exp(logit<T>(dr, v), mq, a.inv_t) * iq;
      ws += fmax(p - c * q, 0.0);
      rs += q;
    }
    w = block_sum<T>(ws, s_d);
    rest = block_sum<T>(rs, s_d);
  }
  if (tid == 0) *st = NodeState{zp, zq, c, w, rest, mp, mq, tried};
}

template <class T>
__global__ __launch_bounds__(kVT) void walk_kernel(VerifyArgs a) {
  __shared__ int s_cur, s_k, s_child[kTreeNodes], s_tok[kTreeNodes], s_hit, s_last;
  __shared__ double s_sum[kVT];
  const int s = blockIdx.x, tid = threadIdx.x;
  const int count = min(max(a.counts[s], 0), a.N);
  const int *accept = (const int *)((NodeState *)a.ws + a.S * a.N) + s * a.N;
  if (tid == 0) {
    int cur = 0, len = count > 0 ? 1 : 0;
    if (len) a.path[(int64_t)s * a.N] = 0;
    // Children come behind their parent, in the order of their trial.
    for (int m = 1; m < count; ++m) {
      const int up = a.parents[(int64_t)s * a.N + m];
      if (up != cur) continue;
      int before = 0;   // children past the most that are tried carry no flag
      for (int i = up + 1; i < m; ++i) before += a.parents[(int64_t)s * a.N + i] == up;
      if (before < a.children && accept[m]) {
        cur = m;
        a.path[(int64_t)s * a.N + len++] = m;
      }
    }
    for (int i = len; i < a.N; ++i) a.path[(int64_t)s * a.N + i] = -1;
    a.accepted[s] = len;
    s_cur = cur;
    s_hit = a.V;
    s_last = -1;
    s_k = children_of(a, s, cur, count, a.children, s_child);
  }
  __syncthreads();
  const int n = s_cur;
  if (count == 0) {
    if (tid == 0) a.next[s] = -1;
    return;
  }
  const NodeState st = ((NodeState *)a.ws)[s * a.N + n];
  if (a.inv_t == 0.0) {
    if (tid == 0) a.next[s] = st.tried;
    return;
  }
  if (!(st.zp > 0)) {
    if (tid == 0) a.next[s] = -1;
    return;
  }
  // A residual without mass: the target's own probabilities.
  const bool left = s_k == 0 || st.w > 0;
  const bool q_on = a.mode != 0 && s_k > 0 && left;
  if (tid < s_k) s_tok[tid] = a.tokens[(int64_t)s * a.N + s_child[tid]];
  __syncthreads();
  const int tried = left ? s_k : 0;
  const T *tr = (const T *)a.target + ((int64_t)s * a.N + n) * a.t_stride;
  const T *dr = (const T *)a.draft + ((int64_t)s * a.N + n) * a.d_stride;
  const double ip = 1.0 / st.zp, iq = st.zq > 0 ? 1.0 / st.zq : 0.0;
  auto r = [&](int v) -> double {
    if (is_tried(s_tok, tried, v)) return 0.0;
    const double p = scaled_exp(logit<T>(tr, v), st.mp, a.inv_t) * ip;
    return q_on ? fmax(p - st.c * (scaled_exp(logit<T>(dr, v), st.mq, a.inv_t) * iq), 0.0) : p;
  };
  const int per = (a.V + kVT - 1) / kVT, v0 = min(tid * per, a.V), v1 = min(v0 + per, a.V);
  double own = 0.0;
  for (int v = v0; v < v1; ++v) own += r(v);
  s_sum[tid] = own;
  __syncthreads();
  if (tid == 0) {
    double run = 0.0;
    for (int i = 0; i < kVT; ++i) {
      const double t = run + s_sum[i];
      s_sum[i] = run;
      run = t;
    }
    const double goal = (double)fmaxf(a.u_final[s], 0.f) * run;
    int at = -1, last = -1;
    for (int i = 0; i < kVT; ++i) {
      const double end = i + 1 < kVT ? s_sum[i + 1] : run;
      if (end > s_sum[i]) {
        last = i;
        if (at < 0 && end > goal) at = i;
      }
    }
    if (at < 0) at = last;
    double sum = s_sum[at < 0 ? 0 : at];
    int token = -1;
    for (int v = at * per; at >= 0 && v < min(at * per + per, a.V); ++v) {
      const double x = r(v);
      if (x <= 0.0) continue;
      token = v;
      sum += x;
      if (sum > goal) break;
    }
    a.next[s] = token;
  }
}

size_t verify_workspace(int S, int N, int V, int mode, int children, bool greedy) {
  return (sizeof(NodeState) + sizeof(int)) * (size_t)S * N;
}

hipError_t launch_verify(const VerifyArgs &a, hipStream_t s) {
  auto go = [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(node_kernel<T>, dim3(a.S * a.N), dim3(kVT), 0, s, a);
    hipLaunchKernelGGL(walk_kernel<T>, dim3(a.S), dim3(kVT), 0, s, a);
  };
  if (a.type == E_F32) go(float{});
  else if (a.type == E_F16) go(_Float16{});
  else go(__bf16{});
  return hipGetLastError();
}

}  // namespace hh
