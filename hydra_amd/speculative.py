"""Decoding with drafted tokens over the HydraHIP C ABI: attention of a drafted tree over the history
(`hh_attention_tree`), verification (`hh_draft_verify`), the accepted rows into the histories
(`hh_cache_commit`), and histories of bounded size (`hh_attention_weights`, `hh_cache_evict`).

The layers themselves run the S·N drafted tokens as one batch (`MoELayer`, `Runner`); a step is

    per layer   attention_tree_into(ctx, cache, q, draft_k, draft_v, parents, counts, out, lse=lse)
    then        draft_verify_into(ctx, logits, tokens, parents, counts, u, u_final, path, accepted, next)
                cache_commit(ctx, caches, draft_k, draft_v, path, accepted)
    per layer   attention_weights_into(ctx, cache, q, lse, path, accepted)
    at times    cache_evict(ctx, caches, keep, recent)

Every function enqueues on the context's stream and returns at once; tensors that another stream
wrote must be complete, and must live until the call has run. Nothing of a call is kept: lengths,
counts and paths are read on the device, so a call recorded with `Context.capture` follows them.
The conventions of trees, types and shapes are include/hydra_hip.h's.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import KVCacheC, TreeDescC, VerifyDescC, check, lib
from .layer import Context

GIVEN, IID, DISTINCT = 0, 1, 2
ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_I32, _F32 = torch.int32, torch.float32


def _same(t, name, shape, dtype, device):
    """Raises unless `t` is a packed tensor of this shape and type on this device."""
    if t.shape != shape or t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a packed {dtype} tensor {tuple(shape)} on {device}, "
                         f"not {t.dtype} {tuple(t.shape)} on {t.device} with strides {t.stride()}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _step(name, s, shape, row):
    """The elements between nodes of [S][N] nodes of `row` elements, which may not overlap (0 is the C entries' packed)."""
    step = s[1] if shape[1] > 1 else s[0] if shape[0] > 1 else row
    if step < row:
        raise ValueError(f"{name}: nodes {step} elements apart overlap")
    return step


def _spaced(t, name, got, s, shape, dtype, device):
    """The elements between nodes of a [S][N][heads][d] tensor (shape `got`, strides `s`) whose heads are packed and
    whose nodes are equally spaced: a slice of a wider product's output, or the packed tensor."""
    if got != shape or t.dtype is not dtype or t.device != device or s[3] != 1 or \
            (s[2] != shape[3] and shape[2] > 1) or (s[0] != shape[1] * s[1] and shape[0] > 1 and shape[1] > 1):
        raise ValueError(f"{name} must be a {dtype} tensor {tuple(shape)} on {device} with packed heads and equally spaced "
                         f"nodes, not {t.dtype} {tuple(got)} on {t.device} with strides {s}")
    return _step(name, s, shape, shape[2] * shape[3])


def _node_stride(t, name, shape, dtype, device):
    return _spaced(t, name, t.shape, t.stride(), shape, dtype, device)


class KVCache:
    """One layer's history (hh_kv_cache): k, v fp16 or bf16 [S][rows][kv_heads][d] (a sequence's rows
    packed), lengths int32 [S]. `ring`: position p is row p % rows, lengths count every token. weights fp32 and
    positions int32 [S][kv_heads][rows] with next_position int32 [S] are what eviction goes by. The
    tensors are the caller's and are updated in place."""

    def __init__(self, k, v, lengths, ring=False, weights=None, positions=None, next_position=None):
        S, rows, heads, d = k.shape
        dev = k.device
        if k.dtype not in (torch.float16, torch.bfloat16) or v.dtype is not k.dtype or v.shape != k.shape or \
                v.device != dev or v.stride() != k.stride() or k.stride()[1:] != (heads * d, d, 1):
            raise ValueError("k and v must be alike, fp16 or bf16 [S][rows][kv_heads][d] with a sequence's rows packed")
        if S > 1 and k.stride(0) < rows * heads * d:
            raise ValueError("the sequences' histories overlap")
        _same(lengths, "lengths", (S,), _I32, dev)
        if weights is not None:
            _same(weights, "weights", (S, heads, rows), _F32, dev)
        if positions is not None:
            _same(positions, "positions", (S, heads, rows), _I32, dev)
        if next_position is not None:
            _same(next_position, "next_position", (S,), _I32, dev)
        self.k, self.v, self.lengths, self.ring = k, v, lengths, bool(ring)
        self.weights, self.positions, self.next_position = weights, positions, next_position
        self.shape, self.dtype, self.device = tuple(k.shape), k.dtype, dev
        self.c = KVCacheC(k.data_ptr(), v.data_ptr(), k.stride(0) if S > 1 else 0, rows, int(self.ring), lengths.data_ptr(),
                          _ptr(weights), _ptr(positions), _ptr(next_position))


class CacheSet:
    """The histories of the layers that one commit or eviction takes: alike in sequences, heads, head_dim, type."""

    def __init__(self, caches):
        self.caches = list(caches)
        if not self.caches:
            raise ValueError("a CacheSet needs a cache")
        a = self.caches[0]
        for b in self.caches:
            if (b.shape[0], b.shape[2:], b.dtype, b.device) != (a.shape[0], a.shape[2:], a.dtype, a.device):
                raise ValueError("the caches of a set must agree in sequences, kv_heads, head_dim, type and device")
        self.c = (KVCacheC * len(self.caches))(*[x.c for x in self.caches])
        self.pointers = C.c_void_p * len(self.caches)

    def __len__(self):
        return len(self.caches)


def _cuda(ctx, device):
    if device.type != "cuda" or device.index != ctx.device:
        raise ValueError(f"the tensors are on {device}, the context on cuda:{ctx.device}")


def attention_tree_into(ctx: Context, cache: KVCache, q, draft_k, draft_v, parents, node_counts, out, lse=None,
                        sinks=None, window: int = 0, sm_scale: float | None = None, max_length: int = 0):
    """Attention of the drafted nodes (hh_attention_tree). q, out [S][N][q_heads][d]; draft_k, draft_v
    [S][N][kv_heads][d] of the cache's type; parents int32 [S][N], node_counts int32 [S]; sinks bf16
    (or int16 bits) [q_heads]; lse fp32 [S][N][q_heads]. q and the drafted rows may be slices with equally
    spaced nodes. No window over a cache with positions. Returns `out`."""
    S, N, H, D = q.shape
    dev = cache.device
    _cuda(ctx, dev)
    if cache.shape[0] != S or cache.shape[3] != D:
        raise ValueError(f"the cache {cache.shape} does not fit q {tuple(q.shape)}")
    if q.dtype not in ELEM:
        raise ValueError(f"q must be fp32, fp16 or bf16, not {q.dtype}")
    G = cache.shape[2]
    qs = _node_stride(q, "q", q.shape, q.dtype, dev)
    ks = _node_stride(draft_k, "draft_k", (S, N, G, D), cache.dtype, dev)
    if _node_stride(draft_v, "draft_v", (S, N, G, D), cache.dtype, dev) != ks:
        raise ValueError("draft_k and draft_v must be spaced alike")
    _same(out, "out", q.shape, q.dtype, dev)
    _same(parents, "parents", (S, N), _I32, dev)
    _same(node_counts, "node_counts", (S,), _I32, dev)
    if lse is not None:
        _same(lse, "lse", (S, N, H), _F32, dev)
    if sinks is not None:
        _same(sinks, "sinks", (H,), sinks.dtype if sinks.dtype is torch.int16 else torch.bfloat16, dev)
    d = TreeDescC(S, N, H, G, D, ELEM[q.dtype], ELEM[cache.dtype], window, max_length,
                  D ** -0.5 if sm_scale is None else sm_scale, qs, ks)
    check(lib().hh_attention_tree(ctx.handle, C.byref(d), C.byref(cache.c), q.data_ptr(), draft_k.data_ptr(),
                                  draft_v.data_ptr(), parents.data_ptr(), node_counts.data_ptr(), _ptr(sinks),
                                  out.data_ptr(), _ptr(lse)))
    return out


def attention_weights_into(ctx: Context, cache: KVCache, q, lse, path, accepted, sm_scale: float | None = None):
    """Adds the accepted nodes' attention to cache.weights (hh_attention_weights), after the commit, which must have found
    room for all of them (rows for N nodes behind the longest length): q and lse as attention_tree_into had and gave
    them, path int32 [S][N], accepted int32 [S]. Returns cache.weights."""
    S, N, H, D = q.shape
    dev = cache.device
    _cuda(ctx, dev)
    if cache.shape[0] != S or cache.shape[3] != D:
        raise ValueError(f"the cache {cache.shape} does not fit q {tuple(q.shape)}")
    if q.dtype not in ELEM:
        raise ValueError(f"q must be fp32, fp16 or bf16, not {q.dtype}")
    qs = _node_stride(q, "q", q.shape, q.dtype, dev)
    _same(lse, "lse", (S, N, H), _F32, dev)
    _same(path, "path", (S, N), _I32, dev)
    _same(accepted, "accepted", (S,), _I32, dev)
    d = TreeDescC(S, N, H, cache.shape[2], D, ELEM[q.dtype], ELEM[cache.dtype], 0, 0,
                  D ** -0.5 if sm_scale is None else sm_scale, qs, 0)
    check(lib().hh_attention_weights(ctx.handle, C.byref(d), C.byref(cache.c), q.data_ptr(), lse.data_ptr(),
                                     path.data_ptr(), accepted.data_ptr()))
    return cache.weights


def _layers(t, name, caches, shape, dtype, device):
    """(host array of the layers' addresses, node stride) of one tensor [layers][S][N][heads][d] or a list."""
    layers = len(caches)
    if torch.is_tensor(t):
        if t.dim() != 5 or t.shape[0] != layers:
            raise ValueError(f"{name} must hold {layers} layers, not {tuple(t.shape)}")
        s = t.stride()
        stride = _spaced(t, name, t.shape[1:], s[1:], shape, dtype, device)
        p, step = t.data_ptr(), s[0] * t.element_size()
        return caches.pointers(*range(p, p + layers * step, step) if step else [p] * layers), stride
    if len(t) != layers:
        raise ValueError(f"{name} must hold {layers} layers, not {len(t)}")
    strides = {_node_stride(x, name, shape, dtype, device) for x in t}
    if len(strides) != 1:
        raise ValueError(f"{name}: the layers' nodes must be spaced alike")
    return caches.pointers(*[x.data_ptr() for x in t]), strides.pop()


def cache_commit(ctx: Context, caches: CacheSet, draft_k, draft_v, path, accepted):
    """The accepted nodes' rows into every layer's history, and the lengths on (hh_cache_commit). draft_k and
    draft_v: a list of [S][N][kv_heads][d], one per layer, or one tensor with the layers in front."""
    S, _, G, D = caches.caches[0].shape
    dev, dtype, N, L = caches.caches[0].device, caches.caches[0].dtype, path.shape[-1], len(caches)
    _cuda(ctx, dev)
    _same(path, "path", (S, N), _I32, dev)
    _same(accepted, "accepted", (S,), _I32, dev)
    kp, ks = _layers(draft_k, "draft_k", caches, (S, N, G, D), dtype, dev)
    vp, vs = _layers(draft_v, "draft_v", caches, (S, N, G, D), dtype, dev)
    if ks != vs:
        raise ValueError("draft_k and draft_v must be spaced alike")
    d = TreeDescC(S, N, G, G, D, ELEM[dtype], ELEM[dtype], 0, 0, 1.0, 0, ks)
    check(lib().hh_cache_commit(ctx.handle, C.byref(d), caches.c, L, kp, vp, path.data_ptr(), accepted.data_ptr()))


def cache_evict(ctx: Context, caches: CacheSet, keep: int, recent: int):
    """Histories longer than `keep` back to `keep` rows a head: the `recent` newest stay, then the largest
    weights (hh_cache_evict)."""
    S, _, G, D = caches.caches[0].shape
    _cuda(ctx, caches.caches[0].device)
    e = ELEM[caches.caches[0].dtype]
    d = TreeDescC(S, 1, G, G, D, e, e, 0, 0, 1.0, 0, 0)
    check(lib().hh_cache_evict(ctx.handle, C.byref(d), caches.c, len(caches), keep, recent))


def _row_stride(t, name, shape, dtype, device):
    s = t.stride()
    if t.shape != shape or t.dtype is not dtype or t.device != device or (s[2] != 1 and shape[2] > 1) or \
            (s[0] != shape[1] * s[1] and shape[0] > 1 and shape[1] > 1):
        raise ValueError(f"{name} must be a {dtype} tensor {tuple(shape)} on {device} with equally spaced rows, not "
                         f"{t.dtype} {tuple(t.shape)} on {t.device} with strides {s}")
    return _step(name, s, shape, shape[2])


def draft_verify_into(ctx: Context, target, tokens, parents, node_counts, uniforms, final_uniforms, path, accepted,
                      next_token, draft=None, distinct: bool = False, temperature: float = 1.0, max_children: int = 0):
    """Verification of the drafted tokens (hh_draft_verify). target, draft: logits [S][N][V], fp32, fp16 or
    bf16, row i the distribution behind node i; tokens, parents, path int32 [S][N]; node_counts, accepted,
    next_token int32 [S]; uniforms fp32 [S][N], final_uniforms fp32 [S] in [0, 1). `draft` None: the tokens were
    chosen, not drawn; otherwise a node's children were drawn independently, or with `distinct` without
    putting back. temperature 0 is greedy (the random numbers may then be None)."""
    S, N, V = target.shape
    dev = target.device
    _cuda(ctx, dev)
    if target.dtype not in ELEM:
        raise ValueError(f"target must be fp32, fp16 or bf16, not {target.dtype}")
    if distinct and draft is None:
        raise ValueError("tokens drawn without putting back need the draft's logits")
    ts = _row_stride(target, "target", target.shape, target.dtype, dev)
    ds = 0 if draft is None else _row_stride(draft, "draft", target.shape, target.dtype, dev)
    for t, name in ((tokens, "tokens"), (parents, "parents"), (path, "path")):
        _same(t, name, (S, N), _I32, dev)
    for t, name in ((node_counts, "node_counts"), (accepted, "accepted"), (next_token, "next_token")):
        _same(t, name, (S,), _I32, dev)
    if temperature != 0 or uniforms is not None:
        if uniforms is None or final_uniforms is None:
            raise ValueError("sampling needs uniforms and final_uniforms")
        _same(uniforms, "uniforms", (S, N), _F32, dev)
        _same(final_uniforms, "final_uniforms", (S,), _F32, dev)
    d = VerifyDescC(S, N, V, ELEM[target.dtype], GIVEN if draft is None else DISTINCT if distinct else IID, max_children,
                    temperature, ts, ds)
    check(lib().hh_draft_verify(ctx.handle, C.byref(d), target.data_ptr(), _ptr(draft), tokens.data_ptr(),
                                parents.data_ptr(), node_counts.data_ptr(), _ptr(uniforms), _ptr(final_uniforms),
                                path.data_ptr(), accepted.data_ptr(), next_token.data_ptr()))


def reserve(ctx: Context, cache: KVCache | None = None, nodes: int = 1, q_heads: int = 0, q_dtype=None, layers: int = 0,
            max_length: int = 0, verify: tuple | None = None, verify_dtype=torch.float32, distinct: bool = False,
            drawn: bool = True, temperature: float = 1.0, max_children: int = 0):
    """Pre-sizes the context's workspace (hh_draft_reserve), for calls that a graph will record: tree attention
    of up to `nodes` nodes and q_heads heads on `cache` (histories up to max_length, 0: its rows; any window), eviction of
    `layers` layers like it, and verification of logits up to the shape `verify` = (S, N, V)."""
    t, v = None, None
    if cache is not None:
        S, _, G, D = cache.shape
        t = TreeDescC(S, nodes, q_heads or G, G, D, ELEM[q_dtype or cache.dtype], ELEM[cache.dtype], 0, max_length, D ** -0.5, 0, 0)
    if verify is not None:
        v = VerifyDescC(*verify, ELEM[verify_dtype], (DISTINCT if distinct else IID) if drawn else GIVEN, max_children,
                        temperature, 0, 0)
    check(lib().hh_draft_reserve(ctx.handle, None if t is None else C.byref(t), None if cache is None else C.byref(cache.c),
                                 layers, None if v is None else C.byref(v)))
