// hh_history.hip — C entries of rotary positions and of histories in 16, 8 and 4 bits: their checks, workspace and launches.
#include <cmath>

#include "hh_ctx.hpp"
#include "hh_hist.hpp"

namespace {

using hh::fail;

constexpr int kMaxSequences = 4096, kMaxTokens = 65536, kMaxRows = 1 << 28, kMaxStep = 1 << 22, kMaxHeadRows = 1 << 25;

bool aligned(const void *p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
bool elem(int32_t type) { return type >= HH_F32 && type <= HH_BF16; }

// n rows of `bytes`, `step` (at least that) apart.
struct Rows {
  const void *at;
  int64_t step, bytes, n;
};
// Whether some byte is in rows of both.
bool meet(const Rows &a, const Rows &b) {
  const int64_t d = (int64_t)((intptr_t)b.at - (intptr_t)a.at);
  if (d >= (a.n - 1) * a.step + a.bytes || -d >= (b.n - 1) * b.step + b.bytes) return false;
  // Row j of b meets row i of a where d + j·b.step − i·a.step is above −b.bytes and below a.bytes: the first j above, for each i.
  auto above = [](int64_t x, int64_t step) { return x < 0 ? -((-x + step - 1) / step) + 1 : x / step + 1; };   // least k: k·step > x
  if (a.step == b.step) {                  // k = j − i
    const int64_t k = above(-b.bytes - d, a.step), least = 1 - a.n;
    const int64_t from = k > least ? k : least;
    return from < b.n && d + from * a.step < a.bytes;
  }
  for (int64_t i = 0; i < a.n; ++i) {
    const int64_t e = d - i * a.step, k = above(-b.bytes - e, b.step), j = k > 0 ? k : 0;
    if (j < b.n && e + j * b.step < a.bytes) return true;
  }
  return false;
}

// The workspace grows in eager calls; recorded graphs hold its address.
int ensure_history(hh_ctx *ctx, size_t bytes) {
  if (ctx->hist_bytes >= bytes) return HH_OK;
  if (ctx->capturing || ctx->live_graphs > 0)
    return fail(HH_EINVAL, "the call needs a larger history workspace, which may not grow while a graph of this context is recorded "
                           "or lives (hh_history_reserve before capture)");
  if (ctx->hist) {
    HH_HIP(hipStreamSynchronize(ctx->stream));
    HH_HIP(hipFree(ctx->hist));
    ctx->hist = nullptr;
    ctx->hist_bytes = 0;
  }
  void *p = nullptr;
  if (hipMalloc(&p, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return fail(HH_ENOMEM, "history workspace allocation failed");
  }
  ctx->hist = (uint8_t *)p;
  ctx->hist_bytes = bytes;
  return HH_OK;
}

int check_rotary(const hh_rotary_desc *d) {
  if (!d) return fail(HH_EINVAL, "desc is NULL");
  if (d->head_dim < 8 || d->head_dim > 1024 || d->head_dim % 8) return fail(HH_ESHAPE, "head_dim must be a multiple of 8, 8..1024");
  const int span = d->span ? d->span : d->rotated;
  if (d->rotated < 2 || d->rotated % 2 || span < d->rotated || span % 2 || span > d->head_dim)
    return fail(HH_ESHAPE, "rotated and span must be even, 2 <= rotated <= span <= head_dim");
  if (d->scaling < HH_ROTARY_PLAIN || d->scaling > HH_ROTARY_YARN) return fail(HH_EINVAL, "unknown scaling");
  if (!std::isfinite(d->base) || !(d->base > 1.0)) return fail(HH_EINVAL, "base must be finite and above 1");
  if (d->scaling != HH_ROTARY_PLAIN && !(std::isfinite(d->factor) && d->factor >= 1.f)) return fail(HH_EINVAL, "factor must be 1 or more");
  if (d->scaling == HH_ROTARY_YARN) {
    if (d->original_length < 1) return fail(HH_EINVAL, "YARN needs original_length");
    if (!(std::isfinite(d->beta_fast) && d->beta_slow > 0.f && d->beta_fast > d->beta_slow))
      return fail(HH_EINVAL, "beta_fast must be above beta_slow, and both positive");
  }
  return HH_OK;
}

int check_history(const hh_history *h) {
  if (!h) return fail(HH_EINVAL, "history is NULL");
  if (h->sequences < 1 || h->sequences > kMaxSequences) return fail(HH_EINVAL, "sequences outside 1..4096");
  if (h->kv_heads < 1 || h->kv_heads > 256) return fail(HH_ESHAPE, "kv_heads outside 1..256");
  if ((int64_t)h->sequences * h->kv_heads > 1 << 18) return fail(HH_EINVAL, "sequences x kv_heads above 2^18");
  if (h->head_dim != 64 && h->head_dim != 128 && h->head_dim != 256) return fail(HH_ESHAPE, "head_dim must be 64, 128 or 256");
  if (h->format < HH_HISTORY_F16 || h->format > HH_HISTORY_MXFP4) return fail(HH_EINVAL, "unknown history format");
  if (h->rows < 1 || h->rows > kMaxRows) return fail(HH_EINVAL, "a history's rows outside 1..2^28");
  if (h->pinned < 0 || h->pinned >= h->rows || (h->pinned && !h->ring)) return fail(HH_EINVAL, "pinned rows are a ring's, fewer than its rows");
  if (!h->k || !h->v || !h->lengths) return fail(HH_EINVAL, "a history needs k, v and lengths");
  if (h->k == h->v) return fail(HH_EINVAL, "k and v are the same memory");
  if (!aligned(h->k, 16) || !aligned(h->v, 16)) return fail(HH_EALIGN, "a history's k and v must be 16-byte aligned");
  if (h->format >= HH_HISTORY_MXFP8) {
    if (!h->k_scales || !h->v_scales) return fail(HH_EINVAL, "MXFP8 and MXFP4 histories need scales");
    if (h->k_scales == h->v_scales) return fail(HH_EINVAL, "k_scales and v_scales are the same memory");
    if (!aligned(h->k_scales, 8) || !aligned(h->v_scales, 8)) return fail(HH_EALIGN, "scales must be 8-byte aligned");
  }
  return HH_OK;
}

int check_step(const hh_history *h, int32_t tokens) {
  if (tokens < 1 || tokens > kMaxTokens) return fail(HH_EINVAL, "tokens outside 1..65536");
  if ((int64_t)h->sequences * tokens > kMaxStep) return fail(HH_EINVAL, "more than 2^22 tokens: split the batch");
  return HH_OK;
}

hh::HistView view(const hh_history *h) {
  hh::HistView v{};
  v.k = (uint8_t *)h->k;
  v.v = (uint8_t *)h->v;
  v.ks = h->k_scales;
  v.vs = h->v_scales;
  v.lengths = h->lengths;
  v.rows = h->rows;
  v.ring = h->ring != 0;
  v.pinned = h->pinned;
  return v;
}

hh::HistRowsArgs rows_args(const hh_history *h, int32_t type, int32_t tokens, const int32_t *counts) {
  hh::HistRowsArgs a{};
  a.h = view(h);
  a.counts = counts;
  a.S = h->sequences;
  a.N = tokens;
  a.kvh = h->kv_heads;
  a.d = h->head_dim;
  a.format = h->format;
  a.type = type;
  return a;
}

// The sizes of an attention call, without its pointers.
int check_attention(const hh_history_desc *d, const hh_history *h, const hh_history *prefix) {
  if (!d) return fail(HH_EINVAL, "desc is NULL");
  if (int rc = check_history(h)) return rc;
  if (int rc = check_step(h, d->tokens)) return rc;
  if (d->q_heads < 1 || d->q_heads % h->kv_heads || d->q_heads / h->kv_heads > hh::kTreeQM)
    return fail(HH_ESHAPE, "q_heads must be kv_heads x 1..16");
  if ((int64_t)h->sequences * d->tokens * d->q_heads > kMaxHeadRows) return fail(HH_EINVAL, "more than 2^25 heads of tokens: split the batch");
  const bool mx = h->format >= HH_HISTORY_MXFP8;
  if (!elem(d->type) || !(mx || h->format == (d->type == HH_BF16 ? HH_HISTORY_BF16 : HH_HISTORY_F16)))
    return fail(HH_EINVAL, "types must be F32 or F16 over F16, BF16 over BF16, or any over MXFP8 or MXFP4");
  if (d->window < 0 || d->first < 0 || d->max_length < 0) return fail(HH_EINVAL, "window, first and max_length must be >= 0");
  if (d->first && !d->window) return fail(HH_EINVAL, "first tokens are a window's");
  if (!std::isfinite(1.5f * d->sm_scale) || d->sm_scale == 0.f) return fail(HH_EINVAL, "sm_scale must be finite, log2(e) times too, and not 0");
  if (h->ring) {
    if (!d->window || (int64_t)d->window + d->tokens - 1 > h->rows - h->pinned)
      return fail(HH_EINVAL, "a ring needs a window, and rows for window + tokens - 1 positions besides the pinned ones");
    if (d->first > h->pinned) return fail(HH_EINVAL, "a ring keeps its pinned first positions only");
  }
  if (d->q_stride && d->q_stride < (int64_t)d->q_heads * h->head_dim) return fail(HH_ESHAPE, "q_stride is smaller than a token's heads");
  if (d->q_stride % (d->type == HH_F32 ? 4 : 8)) return fail(HH_EALIGN, "q_stride must be a multiple of 16 bytes");
  if (d->q_stride > 1 << 30) return fail(HH_ESHAPE, "q_stride above 2^30");
  if (prefix) {
    if (int rc = check_history(prefix)) return rc;
    if (prefix->sequences != 1 || prefix->ring) return fail(HH_EINVAL, "a prefix is a history of one sequence, and no ring");
    if (prefix->kv_heads != h->kv_heads || prefix->head_dim != h->head_dim || prefix->format != h->format)
      return fail(HH_ESHAPE, "the prefix must agree with the history in kv_heads, head_dim and format");
    if (d->window) return fail(HH_EINVAL, "a prefix is seen whole: no window");
  }
  return HH_OK;
}

hh::HistAttnArgs attention_args(const hh_history_desc *d, const hh_history *h, const hh_history *prefix) {
  hh::HistAttnArgs a{};
  a.h = view(h);
  if (prefix) a.p = view(prefix);
  a.S = h->sequences;
  a.N = d->tokens;
  a.qh = d->q_heads;
  a.kvh = h->kv_heads;
  a.d = h->head_dim;
  a.qm = d->q_heads / h->kv_heads;
  a.window = d->window;
  a.first = d->first;
  a.format = h->format;
  a.scale = d->sm_scale;
  a.q_stride = d->q_stride ? d->q_stride : (int64_t)d->q_heads * h->head_dim;
  return a;
}

}  // namespace

extern "C" {

int hh_rotary_table(const hh_rotary_desc *d, double *turns, float *magnitude) {
  if (int rc = check_rotary(d)) return rc;
  if (!turns || !magnitude) return fail(HH_EINVAL, "NULL argument");
  constexpr double kTurn = 6.283185307179586477;
  const int span = d->span ? d->span : d->rotated, pairs = d->rotated / 2;
  const double factor = d->scaling == HH_ROTARY_PLAIN ? 1.0 : (double)d->factor;
  double low = 0, high = 0;
  if (d->scaling == HH_ROTARY_YARN) {
    // The pair that turns b times in the original length L: base^(2i / span) = L / (2 pi b).
    auto pair = [&](double b) { return span * std::log(d->original_length / (kTurn * b)) / (2 * std::log(d->base)); };
    low = pair(d->beta_fast);
    high = pair(d->beta_slow);
    if (d->truncate) low = std::floor(low), high = std::ceil(high);
    low = std::fmax(low, 0.0);
    high = std::fmin(high, span - 1.0);
    if (!(high - low >= 0.001)) high = low + 0.001;
  }
  for (int i = 0; i < pairs; ++i) {
    const double f = std::pow(d->base, -2.0 * i / span);
    double ramp = 1;   // of the divided frequency
    if (d->scaling == HH_ROTARY_YARN) ramp = std::fmin(std::fmax((i - low) / (high - low), 0.0), 1.0);
    turns[i] = (f / factor * ramp + f * (1 - ramp)) / kTurn;
  }
  *magnitude = d->scaling == HH_ROTARY_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.f;
  return HH_OK;
}

int hh_rotary(hh_ctx *ctx, const hh_rotary_desc *d, const double *turns, float magnitude, int32_t type, int32_t tokens,
              const int32_t *positions, const hh_rotary_rows *rows, int32_t count) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_rotary(d)) return rc;
  if (!elem(type)) return fail(HH_EINVAL, "unknown type");
  if (tokens < 0 || tokens > kMaxStep) return fail(HH_EINVAL, "tokens outside 0..2^22");
  if (!turns || !positions || !rows) return fail(HH_EINVAL, "NULL argument");
  if (!aligned(turns, 8)) return fail(HH_EALIGN, "turns must be 8-byte aligned");
  if (count < 1 || count > 2) return fail(HH_EINVAL, "count must be 1 or 2");
  if (!std::isfinite(magnitude)) return fail(HH_EINVAL, "magnitude must be finite");
  hh::RotaryArgs a{};
  for (int i = 0; i < count; ++i) {
    const hh_rotary_rows &r = rows[i];
    if (!r.x || !r.y) return fail(HH_EINVAL, "NULL argument");
    if (!aligned(r.x, 16) || !aligned(r.y, 16)) return fail(HH_EALIGN, "x and y must be 16-byte aligned");
    if (r.heads < 1 || r.heads > 1024) return fail(HH_ESHAPE, "heads outside 1..1024");
    const int64_t row = (int64_t)r.heads * d->head_dim, xs = r.x_stride ? r.x_stride : row, ys = r.y_stride ? r.y_stride : row;
    if (xs < row || ys < row) return fail(HH_ESHAPE, "a stride is smaller than a token's heads");
    if (xs > 1 << 30 || ys > 1 << 30) return fail(HH_ESHAPE, "a stride above 2^30");
    if (xs % (type == HH_F32 ? 4 : 8) || ys % (type == HH_F32 ? 4 : 8)) return fail(HH_EALIGN, "strides must be multiples of 16 bytes");
    if (r.x == r.y && xs != ys) return fail(HH_EINVAL, "in place, x and y are spaced alike");
    a.r[i] = {r.x, r.y, r.heads, xs, ys};
  }
  if (count == 2 && a.r[0].y == a.r[1].y) return fail(HH_EINVAL, "both outputs are the same memory");
  if (count == 2 && (a.r[0].y == a.r[1].x || a.r[1].y == a.r[0].x)) return fail(HH_EINVAL, "an output is the other's input");
  if (tokens == 0) return HH_OK;
  const int64_t size = type == HH_F32 ? 4 : 2;
  auto rows_of = [&](const void *p, int64_t stride, int heads) { return Rows{p, size * stride, size * heads * d->head_dim, tokens}; };
  for (int i = 0; i < count; ++i)
    for (int j = 0; j < count; ++j) {
      const Rows y = rows_of(a.r[i].y, a.r[i].y_stride, a.r[i].heads);
      if ((i != j || a.r[i].x != a.r[i].y) && meet(y, rows_of(a.r[j].x, a.r[j].x_stride, a.r[j].heads)))
        return fail(HH_EINVAL, "an output overlaps an input: y is its x, with the same stride, or apart from every x");
      if (i < j && meet(y, rows_of(a.r[j].y, a.r[j].y_stride, a.r[j].heads))) return fail(HH_EINVAL, "the outputs overlap");
    }
  a.turns = turns;
  a.positions = positions;
  a.magnitude = magnitude;
  a.tokens = tokens;
  a.count = count;
  a.d = d->head_dim;
  a.rotated = d->rotated;
  a.span = d->span ? d->span : d->rotated;
  a.interleaved = d->interleaved != 0;
  a.type = type;
  HH_HIP(hipSetDevice(ctx->device));
  HH_HIP(hh::launch_rotary(a, ctx->stream));
  ctx->dispatches += 1;
  return HH_OK;
}

int hh_history_write(hh_ctx *ctx, const hh_history *h, int32_t type, const void *k, const void *v, int64_t kv_stride,
                     int32_t tokens, const int32_t *counts) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_history(h)) return rc;
  if (int rc = check_step(h, tokens)) return rc;
  if (!elem(type)) return fail(HH_EINVAL, "unknown type");
  if (!k || !v || !counts) return fail(HH_EINVAL, "NULL argument");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(HH_EALIGN, "k and v must be 16-byte aligned");
  const int64_t row = (int64_t)h->kv_heads * h->head_dim;
  if (kv_stride && kv_stride < row) return fail(HH_ESHAPE, "kv_stride is smaller than a token's rows");
  if (kv_stride > 1 << 30) return fail(HH_ESHAPE, "kv_stride above 2^30");
  if (kv_stride % (type == HH_F32 ? 4 : 8)) return fail(HH_EALIGN, "kv_stride must be a multiple of 16 bytes");
  const int64_t held = (int64_t)h->sequences * h->kv_heads * h->rows, codes = held * hh::hist_row_bytes(h->format, h->head_dim);
  const int64_t scales = h->format >= HH_HISTORY_MXFP8 ? held * (h->head_dim / 32) : 0;
  const Rows own[5] = {{h->k, codes, codes, 1}, {h->v, codes, codes, 1}, {h->lengths, 4 * h->sequences, 4 * h->sequences, 1},
                       {h->k_scales, scales, scales, 1}, {h->v_scales, scales, scales, 1}};
  for (int i = 0; i < (scales ? 5 : 3); ++i)
    for (int j = 0; j < i; ++j)
      if (meet(own[i], own[j])) return fail(HH_EINVAL, "tensors of the history overlap");
  hh::HistRowsArgs a = rows_args(h, type, tokens, counts);
  a.k = k;
  a.v = v;
  a.kv_stride = kv_stride ? kv_stride : row;
  HH_HIP(hipSetDevice(ctx->device));
  HH_HIP(hh::launch_history_write(a, ctx->stream));
  ctx->dispatches += 1;
  return HH_OK;
}

int hh_history_read(hh_ctx *ctx, const hh_history *h, int32_t type, const int32_t *starts, int32_t tokens,
                    const int32_t *counts, void *k, void *v) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_history(h)) return rc;
  if (int rc = check_step(h, tokens)) return rc;
  if (!elem(type)) return fail(HH_EINVAL, "unknown type");
  if (!starts || !counts || !k || !v) return fail(HH_EINVAL, "NULL argument");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(HH_EALIGN, "k and v must be 16-byte aligned");
  const int64_t out = (int64_t)h->sequences * tokens * h->kv_heads * h->head_dim * (type == HH_F32 ? 4 : 2);
  if (meet({k, out, out, 1}, {v, out, out, 1})) return fail(HH_EINVAL, "k and v overlap");
  hh::HistRowsArgs a = rows_args(h, type, tokens, counts);
  a.ko = k;
  a.vo = v;
  a.starts = starts;
  HH_HIP(hipSetDevice(ctx->device));
  HH_HIP(hh::launch_history_read(a, ctx->stream));
  ctx->dispatches += 1;
  return HH_OK;
}

int hh_history_advance(hh_ctx *ctx, const hh_history *h, int32_t tokens, const int32_t *counts) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_history(h)) return rc;
  if (int rc = check_step(h, tokens)) return rc;
  if (!counts) return fail(HH_EINVAL, "NULL argument");
  const int64_t bytes = 4 * h->sequences;
  if (meet({h->lengths, bytes, bytes, 1}, {counts, bytes, bytes, 1})) return fail(HH_EINVAL, "lengths and counts overlap");
  HH_HIP(hipSetDevice(ctx->device));
  HH_HIP(hh::launch_history_advance(const_cast<int32_t *>(h->lengths), counts, h->sequences, tokens, ctx->stream));
  ctx->dispatches += 1;
  return HH_OK;
}

int hh_history_attention(hh_ctx *ctx, const hh_history_desc *d, const hh_history *h, const hh_history *prefix, const void *q,
                         const int32_t *counts, const uint16_t *sinks, void *out, float *lse) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_attention(d, h, prefix)) return rc;
  if (!q || !counts || !out) return fail(HH_EINVAL, "NULL argument");
  if (!aligned(q, 16) || !aligned(out, 16)) return fail(HH_EALIGN, "q and out must be 16-byte aligned");
  hh::HistAttnArgs a = attention_args(d, h, prefix);
  a.q = q;
  a.counts = counts;
  a.sinks = sinks;
  a.out = out;
  a.lse = lse;
  const int64_t n = (int64_t)a.S * a.N, size = d->type == HH_F32 ? 4 : 2, row = (int64_t)a.qh * a.d;
  const Rows to = {out, size * row, size * row, n}, from = {q, size * a.q_stride, size * row, n}, sums = {lse, 4 * a.qh, 4 * a.qh, n};
  // In place a workgroup reads its rows' queries before it writes them, and reads no others'.
  if ((out != q || (a.q_stride != row && n > 1)) && meet(to, from)) return fail(HH_EINVAL, "out overlaps q: it is q, packed, or apart from it");
  if (lse && (meet(sums, to) || meet(sums, from))) return fail(HH_EINVAL, "lse overlaps q or out");
  HH_HIP(hipSetDevice(ctx->device));
  hh::history_plan(a, d->max_length ? d->max_length : h->rows, prefix ? prefix->rows : 0);
  if (int rc = ensure_history(ctx, hh::history_workspace(a))) return rc;
  const size_t slots = (size_t)a.S * a.N * a.qh * a.chunks;
  a.po = (float *)ctx->hist;
  a.pm = a.po + slots * a.d;
  a.pl = a.pm + slots;
  int launches = 0;
  HH_HIP(hh::launch_history_attention(a, d->type, ctx->stream, &launches));
  ctx->dispatches += launches;
  return HH_OK;
}

int hh_history_reserve(hh_ctx *ctx, const hh_history_desc *d, const hh_history *h, const hh_history *prefix) {
  if (!ctx) return fail(HH_EINVAL, "ctx is NULL");
  if (int rc = check_attention(d, h, prefix)) return rc;
  hh::HistAttnArgs a = attention_args(d, h, prefix);
  const int64_t length = d->max_length ? d->max_length : h->rows;
  size_t need;
  if (ctx->capturing || ctx->live_graphs > 0) {   // where the workspace may not grow, a call of these sizes itself
    hh::history_plan(a, length, prefix ? prefix->rows : 0);
    need = hh::history_workspace(a);
  } else {
    need = hh::history_reserve(a, length, prefix ? prefix->rows : 0);
  }
  HH_HIP(hipSetDevice(ctx->device));
  return ensure_history(ctx, need);
}

}  // extern "C"
