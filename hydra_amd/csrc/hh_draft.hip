// hh_draft.hip — C entries of decoding with drafted tokens: their checks, workspace and launches.
#include <climits>
#include <cmath>

#include "hh_ctx.hpp"
#include "hh_draft.hpp"

namespace {

using hh::fail;

constexpr int kMaxSequences = 4096, kMaxLayers = 256;

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The workspace grows in eager calls; recorded graphs hold its address.
int ensure_draft(hh_ctx *ctx, size_t bytes) {
  if (ctx->draft_bytes >= bytes) return HH_OK;
  if (ctx->capturing || ctx->live_graphs > 0)
    return fail(HH_EINVAL, "the call needs a larger draft workspace, which may not grow while a graph of this context is "
                           "recorded or lives (hh_draft_reserve before capture)");
  if (ctx->draft) {
    HH_HIP(hipStreamSynchronize(ctx->stream));
    HH_HIP(hipFree(ctx->draft));
    ctx->draft = nullptr;
    ctx->draft_bytes = 0;
  }
  void *p = nullptr;
  if (hipMalloc(&p, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return fail(HH_ENOMEM, "draft workspace allocation failed");
  }
  ctx->draft = (uint8_t *)p;
  ctx->draft_bytes = bytes;
  return HH_OK;
}

// The commit's counters, if they are there or can be made now (not while a graph is recorded).
int ensure_arrivals(hh_ctx *ctx) {
  if (ctx->arrivals || ctx->capturing) return HH_OK;
  void *p = nullptr;
  if (hipMalloc(&p, sizeof(uint32_t) * kMaxSequences) != hipSuccess) {
    (void)hipGetLastError();
    return fail(HH_ENOMEM, "commit counters allocation failed");
  }
  const hipError_t e = hipMemsetAsync(p, 0, sizeof(uint32_t) * kMaxSequences, ctx->stream);
  if (e != hipSuccess) {
    (void)hipFree(p);
    return hh::hip_fail(e, "hipMemsetAsync");
  }
  ctx->arrivals = (uint32_t *)p;
  return HH_OK;
}

// Sizes that every call with a tree description goes by.
int check_rows(const hh_tree_desc *d) {
  if (!d) return fail(HH_EINVAL, "desc is NULL");
  if (d->sequences < 1 || d->sequences > kMaxSequences) return fail(HH_EINVAL, "sequences outside 1..4096");
  if (d->kv_heads < 1 || d->kv_heads > 256) return fail(HH_ESHAPE, "kv_heads outside 1..256");
  if ((int64_t)d->sequences * d->kv_heads > 1 << 18) return fail(HH_EINVAL, "sequences x kv_heads above 2^18");
  if (d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256)
    return fail(HH_ESHAPE, "head_dim must be 64, 128 or 256");
  return HH_OK;
}

int check_nodes(const hh_tree_desc *d) {
  if (int rc = check_rows(d)) return rc;
  if (d->nodes < 1 || d->nodes > HH_TREE_MAX_NODES) return fail(HH_EINVAL, "nodes outside 1..64");
  if (d->cache_type != HH_F16 && d->cache_type != HH_BF16) return fail(HH_EINVAL, "cache_type must be F16 or BF16");
  const int64_t row = (int64_t)d->kv_heads * d->head_dim;
  if (d->kv_stride > 1 << 30) return fail(HH_ESHAPE, "kv_stride above 2^30");
  if (d->kv_stride && d->kv_stride < row) return fail(HH_ESHAPE, "kv_stride is smaller than a node's rows");
  if (d->kv_stride % 8) return fail(HH_EALIGN, "kv_stride must be a multiple of 16 bytes");
  return HH_OK;
}

int check_tree(const hh_tree_desc *d) {
  if (int rc = check_nodes(d)) return rc;
  if (d->q_heads < 1 || d->q_heads % d->kv_heads || d->q_heads / d->kv_heads > hh::kTreeQM)
    return fail(HH_ESHAPE, "q_heads must be kv_heads x 1..16");
  if (!((d->type == HH_F32 && d->cache_type == HH_F16) || (d->type != HH_F32 && d->type == d->cache_type)))
    return fail(HH_EINVAL, "types must be F32 over F16, F16 over F16 or BF16 over BF16");
  if (d->window < 0 || d->max_length < 0) return fail(HH_EINVAL, "window and max_length must be >= 0");
  if (!std::isfinite(d->sm_scale) || d->sm_scale == 0.f) return fail(HH_EINVAL, "sm_scale must be finite and not 0");
  const int64_t row = (int64_t)d->q_heads * d->head_dim;
  if (d->q_stride && d->q_stride < row) return fail(HH_ESHAPE, "q_stride is smaller than a node's heads");
  if (d->q_stride % (d->type == HH_F32 ? 4 : 8)) return fail(HH_EALIGN, "q_stride must be a multiple of 16 bytes");
  return HH_OK;
}

int check_cache(const hh_tree_desc *d, const hh_kv_cache *c) {
  if (!c) return fail(HH_EINVAL, "cache is NULL");
  if (!c->k || !c->v || !c->lengths) return fail(HH_EINVAL, "a cache needs k, v and lengths");
  if (c->rows < 1 || c->rows > 1 << 30) return fail(HH_EINVAL, "a cache's rows outside 1..2^30");
  if (!aligned16(c->k) || !aligned16(c->v)) return fail(HH_EALIGN, "the caches must be 16-byte aligned");
  const int64_t all = (int64_t)c->rows * d->kv_heads * d->head_dim;
  if (c->sequence_stride && c->sequence_stride < all) return fail(HH_ESHAPE, "sequence_stride is smaller than a sequence's rows");
  if (c->sequence_stride % 8) return fail(HH_EALIGN, "sequence_stride must be a multiple of 16 bytes");
  if (c->ring && (c->weights || c->positions)) return fail(HH_EINVAL, "a ring has no weights or positions");
  if ((c->positions != nullptr) != (c->next_position != nullptr))
    return fail(HH_EINVAL, "positions and next_position come together");
  return HH_OK;
}

int64_t seq_stride(const hh_tree_desc *d, const hh_kv_cache *c) {
  return c->sequence_stride ? c->sequence_stride : (int64_t)c->rows * d->kv_heads * d->head_dim;
}

hh::TreeArgs tree_args(const hh_tree_desc *d, const hh_kv_cache *c, const void *q) {
  hh::TreeArgs a{};
  a.q = q;
  a.k = c->k;
  a.v = c->v;
  a.lengths = c->lengths;
  a.S = d->sequences;
  a.N = d->nodes;
  a.qh = d->q_heads;
  a.kvh = d->kv_heads;
  a.d = d->head_dim;
  a.rows = c->rows;
  a.ring = c->ring != 0;
  a.window = d->window;
  a.scale = d->sm_scale;
  a.q_stride = d->q_stride ? d->q_stride : (int64_t)d->q_heads * d->head_dim;
  a.kv_stride = d->kv_stride ? d->kv_stride : (int64_t)d->kv_heads * d->head_dim;
  a.seq_stride = seq_stride(d, c);
  a.qm = d->q_heads / d->kv_heads;
  a.inv_qm = 1.f / (float)a.qm;
  return a;
}

// The layers of a commit or an eviction, checked: caches that share lengths share what advances with them.
int check_layers(const hh_tree_desc *d, const hh_kv_cache *caches, int32_t count) {
  if (count < 1 || count > kMaxLayers) return fail(HH_EINVAL, "count outside 1..256");
  if (!caches) return fail(HH_EINVAL, "caches is NULL");
  if ((int64_t)(count < hh::kRowsLayers ? count : hh::kRowsLayers) * d->sequences * d->kv_heads > 1 << 21)
    return fail(HH_EINVAL, "more than 2^21 heads a launch: split the batch");
  for (int i = 0; i < count; ++i) {
    if (int rc = check_cache(d, caches + i)) return rc;
    const hh_kv_cache &x = caches[i];
    if (x.k == x.v) return fail(HH_EINVAL, "k and v are the same memory");
    for (int j = 0; j <= i; ++j) {
      const hh_kv_cache &y = caches[j];
      if (x.next_position == y.lengths || y.next_position == x.lengths)   // lengths are never NULL
        return fail(HH_EINVAL, "lengths and next_position are the same memory");
      if (j == i) break;
      if (x.k == y.k || x.v == y.v || x.k == y.v || x.v == y.k) return fail(HH_EINVAL, "two layers share a cache");
      if ((x.weights && x.weights == y.weights) || (x.positions && x.positions == y.positions))
        return fail(HH_EINVAL, "two layers share weights or positions");
      if (x.next_position && y.next_position && (x.lengths == y.lengths) != (x.next_position == y.next_position))
        return fail(HH_EINVAL, "caches share both lengths and next_position, or neither");
    }
  }
  return HH_OK;
}

hh::RowsLayer rows_layer(const hh_tree_desc *d, const hh_kv_cache *caches, int32_t count, int i) {
  const hh_kv_cache &c = caches[i];
  hh::RowsLayer y{};
  y.k = c.k;
  y.v = c.v;
  y.lengths = c.lengths;
  y.weights = c.weights;
  y.positions = c.positions;
  y.next = c.next_position;
  y.seq_stride = seq_stride(d, &c);
  y.rows = c.rows;
  y.ring = c.ring != 0;
  y.limit = INT_MAX;
  y.last = 1;
  for (int j = 0; j < count; ++j) {
    if (caches[j].lengths != c.lengths) continue;
    if (!caches[j].ring && caches[j].rows < y.limit) y.limit = caches[j].rows;
    if (!y.next) y.next = caches[j].next_position;   // advanced by whichever layer comes last
    if (j > i) y.last = 0;
  }
  return y;
}

// Moves of an eviction's launch: [layers][S][kvh] counts, then sources and destinations.
size_t evict_bytes(const hh_tree_desc *d, int layers, int rows) {
  const size_t heads = (size_t)layers * d->sequences * d->kv_heads;
  return sizeof(int32_t) * heads * (1 + 2 * (size_t)(rows / 2));   // min(keep, rows − keep) <= rows / 2
}

int check_verify(const hh_verify_desc *d) {
  if (!d) return fail(HH_EINVAL, "desc is NULL");
  if (d->sequences < 1 || d->sequences > kMaxSequences) return fail(HH_EINVAL, "sequences outside 1..4096");
  if (d->nodes < 1 || d->nodes > HH_TREE_MAX_NODES) return fail(HH_EINVAL, "nodes outside 1..64");
  if (d->vocab < 1 || d->vocab > 1 << 24) return fail(HH_EINVAL, "vocab outside 1..2^24");
  if (d->type < HH_F32 || d->type > HH_BF16) return fail(HH_EINVAL, "unknown type");
  if (d->draft < HH_DRAFT_GIVEN || d->draft > HH_DRAFT_DISTINCT) return fail(HH_EINVAL, "unknown draft mode");
  if (d->max_children < 0 || d->max_children >= HH_TREE_MAX_NODES) return fail(HH_EINVAL, "max_children outside 0..63");
  if (!hh::verify_fits(d->sequences, d->nodes, d->vocab)) return fail(HH_EINVAL, "more than 2^22 chunks of logits: split the batch");
  if (!(d->temperature >= 0.f) || !std::isfinite(d->temperature)) return fail(HH_EINVAL, "temperature must be finite and >= 0");
  if (d->temperature != 0.f && d->temperature < 1e-6f)
    return fail(HH_EINVAL, "temperature below 1e-6: 0 is greedy");
  if ((d->target_stride && d->target_stride < d->vocab) || (d->draft_stride && d->draft_stride < d->vocab))
    return fail(HH_ESHAPE, "a row stride is smaller than the vocabulary");
  return HH_OK;
}

int verify_children(const hh_verify_desc *d) {
  const int most = d->nodes - 1;
  return d->max_children && d->max_children < most ? d->max_children : most;
}

}  // namespace

extern "C" {

int hh_attention_tree(hh_ctx *ctx, const hh_tree_desc *d, const hh_kv_cache *cache, const void *q, const void *draft_k,
                      const void *draft_v, const int32_t *parents, const int32_t *node_counts, const uint16_t *sinks,
                      void *out, float *lse) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_tree(d)) return rc;
  if (int rc = check_cache(d, cache)) return rc;
  if (d->window && cache->positions) return fail(HH_EINVAL, "a window goes by the rows' order, which eviction does not keep: none with positions");
  if (!q || !draft_k || !draft_v || !parents || !node_counts || !out) return fail(HH_EINVAL, "NULL argument");
  if (!aligned16(q) || !aligned16(draft_k) || !aligned16(draft_v) || !aligned16(out))
    return fail(HH_EALIGN, "q, draft_k, draft_v and out must be 16-byte aligned");
  HH_HIP(hipSetDevice(ctx->device));
  hh::TreeArgs a = tree_args(d, cache, q);
  a.dk = draft_k;
  a.dv = draft_v;
  a.parents = parents;
  a.counts = node_counts;
  a.sinks = sinks;
  a.out = out;
  a.lse = lse;
  hh::tree_plan(a, d->max_length ? d->max_length : cache->rows);
  if (int rc = ensure_draft(ctx, hh::tree_workspace(a))) return rc;
  const size_t slots = (size_t)a.S * a.N * a.qh * a.chunks;
  a.po = (float *)ctx->draft;
  a.pm = a.po + slots * a.d;
  a.pl = a.pm + slots;
  HH_HIP(hh::launch_tree(a, d->type, ctx->stream));
  ctx->dispatches += a.chunks > 1 ? 2 : 1;
  return HH_OK;
}

int hh_attention_weights(hh_ctx *ctx, const hh_tree_desc *d, const hh_kv_cache *cache, const void *q, const float *lse,
                         const int32_t *path, const int32_t *accepted) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_tree(d)) return rc;
  if (int rc = check_cache(d, cache)) return rc;
  if (cache->ring || d->window) return fail(HH_EINVAL, "weights are not accumulated for rings or windows");
  if (!cache->weights) return fail(HH_EINVAL, "the cache has no weights");
  if (!q || !lse || !path || !accepted) return fail(HH_EINVAL, "NULL argument");
  if (!aligned16(q)) return fail(HH_EALIGN, "q must be 16-byte aligned");
  HH_HIP(hipSetDevice(ctx->device));
  hh::TreeArgs a = tree_args(d, cache, q);
  a.lse_in = lse;
  a.path = path;
  a.accepted = accepted;
  a.weights = cache->weights;
  HH_HIP(hh::launch_weights(a, d->type, ctx->stream));
  ctx->dispatches += 1;
  return HH_OK;
}

int hh_draft_verify(hh_ctx *ctx, const hh_verify_desc *d, const void *target, const void *draft, const int32_t *tokens,
                    const int32_t *parents, const int32_t *node_counts, const float *uniforms,
                    const float *final_uniforms, int32_t *path, int32_t *accepted, int32_t *next_token) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_verify(d)) return rc;
  const bool greedy = d->temperature == 0.f;
  const int mode = greedy ? HH_DRAFT_GIVEN : d->draft;
  if (!target || !tokens || !parents || !node_counts || !path || !accepted || !next_token)
    return fail(HH_EINVAL, "NULL argument");
  if (!greedy && (!uniforms || !final_uniforms)) return fail(HH_EINVAL, "sampling needs uniforms and final_uniforms");
  if (mode != HH_DRAFT_GIVEN && !draft) return fail(HH_EINVAL, "draws from a distribution need the draft's logits");
  HH_HIP(hipSetDevice(ctx->device));
  if (int rc = ensure_draft(ctx, hh::verify_workspace(d->sequences, d->nodes, d->vocab))) return rc;
  hh::VerifyArgs a{};
  a.target = target;
  a.draft = draft;
  a.t_stride = d->target_stride ? d->target_stride : d->vocab;
  a.d_stride = d->draft_stride ? d->draft_stride : d->vocab;
  a.tokens = tokens;
  a.parents = parents;
  a.counts = node_counts;
  a.u = uniforms;
  a.u_final = final_uniforms;
  a.path = path;
  a.accepted = accepted;
  a.next = next_token;
  a.S = d->sequences;
  a.N = d->nodes;
  a.V = d->vocab;
  a.type = d->type;
  a.mode = mode;
  a.children = verify_children(d);
  a.inv_t = greedy ? 0.0 : 1.0 / (double)d->temperature;
  a.ws = ctx->draft;
  a.k = 256 * 1.4426950408889634074 * a.inv_t;
  int launches = 0;
  HH_HIP(hh::launch_verify(a, ctx->stream, &launches));
  ctx->dispatches += launches;
  return HH_OK;
}

int hh_cache_commit(hh_ctx *ctx, const hh_tree_desc *d, const hh_kv_cache *caches, int32_t count,
                    const void *const *draft_k, const void *const *draft_v, const int32_t *path,
                    const int32_t *accepted) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_nodes(d)) return rc;
  if (int rc = check_layers(d, caches, count)) return rc;
  if (!draft_k || !draft_v || !path || !accepted) return fail(HH_EINVAL, "NULL argument");
  for (int i = 0; i < count; ++i) {
    if (!draft_k[i] || !draft_v[i]) return fail(HH_EINVAL, "a layer's drafted rows are NULL");
    if (!aligned16(draft_k[i]) || !aligned16(draft_v[i])) return fail(HH_EALIGN, "drafted rows must be 16-byte aligned");
  }
  HH_HIP(hipSetDevice(ctx->device));
  hh::RowsArgs a{};
  a.path = path;
  a.accepted = accepted;
  a.S = d->sequences;
  a.N = d->nodes;
  a.kvh = d->kv_heads;
  a.d = d->head_dim;
  a.kv_stride = d->kv_stride ? d->kv_stride : (int64_t)d->kv_heads * d->head_dim;
  if (int rc = ensure_arrivals(ctx)) return rc;
  if (count <= hh::kRowsLayers) a.arrivals = ctx->arrivals;
  // Otherwise the rows of every layer first: they go by the lengths that the second round advances.
  for (int round = 0; round < (a.arrivals ? 1 : 2); ++round)
    for (int l = 0; l < count; l += hh::kRowsLayers) {
      a.layers = count - l < hh::kRowsLayers ? count - l : hh::kRowsLayers;
      for (int i = 0; i < a.layers; ++i) {
        a.layer[i] = rows_layer(d, caches, count, l + i);
        a.layer[i].dk = (const uint16_t *)draft_k[l + i];
        a.layer[i].dv = (const uint16_t *)draft_v[l + i];
      }
      HH_HIP(hh::launch_commit(a, round == 1, ctx->stream));
      ctx->dispatches += 1;
    }
  return HH_OK;
}

int hh_cache_evict(hh_ctx *ctx, const hh_tree_desc *d, const hh_kv_cache *caches, int32_t count, int32_t keep,
                   int32_t recent) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_rows(d)) return rc;
  if (int rc = check_layers(d, caches, count)) return rc;
  if (keep < 1 || recent < 0 || recent > keep) return fail(HH_EINVAL, "keep must be positive and recent within 0..keep");
  int most = 0;
  for (int i = 0; i < count; ++i) {
    const hh_kv_cache &c = caches[i];
    if (c.ring || !c.weights || !c.positions) return fail(HH_EINVAL, "eviction needs weights and positions, and no rings");
    if (keep > c.rows) return fail(HH_EINVAL, "keep is above a cache's rows");
    const int moves = keep < c.rows - keep ? keep : c.rows - keep;
    if (moves > most) most = moves;
  }
  HH_HIP(hipSetDevice(ctx->device));
  const int per = count < hh::kRowsLayers ? count : hh::kRowsLayers;
  const size_t heads = (size_t)per * d->sequences * d->kv_heads;
  if (int rc = ensure_draft(ctx, sizeof(int32_t) * heads * (1 + 2 * (size_t)most))) return rc;
  hh::RowsArgs a{};
  a.S = d->sequences;
  a.kvh = d->kv_heads;
  a.d = d->head_dim;
  a.keep = keep;
  a.recent = recent;
  a.max_moves = most;
  a.moves = (int32_t *)ctx->draft;
  a.from = a.moves + heads;
  a.to = a.from + heads * most;
  for (int l = 0; l < count; l += hh::kRowsLayers) {
    a.layers = count - l < hh::kRowsLayers ? count - l : hh::kRowsLayers;
    for (int i = 0; i < a.layers; ++i) a.layer[i] = rows_layer(d, caches, count, l + i);
    HH_HIP(hh::launch_evict(a, ctx->stream));
    ctx->dispatches += 2;
  }
  return HH_OK;
}

int hh_draft_reserve(hh_ctx *ctx, const hh_tree_desc *tree, const hh_kv_cache *cache, int32_t layers,
                     const hh_verify_desc *verify) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (layers < 0 || layers > kMaxLayers) return fail(HH_EINVAL, "layers outside 0..256");
  if ((layers > 0 || cache) && (!tree || !cache)) return fail(HH_EINVAL, "a cache needs its tree description, and layers a cache");
  // Where the workspace may not grow, the calls of these sizes themselves.
  const bool fixed = ctx->capturing || ctx->live_graphs > 0;
  size_t need = 0;
  if (cache) {
    if (int rc = check_rows(tree)) return rc;
    if (int rc = check_cache(tree, cache)) return rc;
    const int per = layers < hh::kRowsLayers ? layers : hh::kRowsLayers;
    if (layers) need = evict_bytes(tree, per, cache->rows);
    if (tree->nodes) {
      if (int rc = check_tree(tree)) return rc;
      hh::TreeArgs a = tree_args(tree, cache, nullptr);
      const int64_t length = tree->max_length ? tree->max_length : cache->rows;
      hh::tree_plan(a, length);
      const size_t b = fixed ? hh::tree_workspace(a) : hh::tree_reserve(a, length);
      if (b > need) need = b;
    }
  }
  if (verify) {
    if (int rc = check_verify(verify)) return rc;
    const size_t b = (fixed ? hh::verify_workspace : hh::verify_reserve)(verify->sequences, verify->nodes, verify->vocab);
    if (b > need) need = b;
  }
  HH_HIP(hipSetDevice(ctx->device));
  if (cache)
    if (int rc = ensure_arrivals(ctx)) return rc;
  return ensure_draft(ctx, need);
}

}  // extern "C"
