"""Decoding with drafted tokens over key/value histories of bounded size: the operators that a
speculative decoding step adds around the layers, as cases that can be timed and compared.

A case is one pass of one operator through `hydra_amd.speculative`:

  attention  the drafted tokens of each sequence's tree against its history and their ancestors;
  verify     the tree's tokens against the target's probabilities, with given random numbers;
  weights    what the accepted tokens' attention adds to each key's accumulated weight;
  commit     the accepted tokens' keys and values into every layer's history;
  evict      the histories back to their budget: the rows of least accumulated weight go. `cycle`: a
             decoding loop's commit with the eviction behind it; otherwise once, after a prompt.

With `own` false, `run` computes the same in elementary torch operations. All states share one
context, as a program has one.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _attention(**kw):
    return {"kind": "attention", "sequences": 1, "nodes": 8, "q_heads": 64, "kv_heads": 8, "head_dim": 64,
            "type": "f32", "length": 4096, "window": 0, "sinks": True, **kw}


def _verify(**kw):
    return {"kind": "verify", "sequences": 1, "nodes": 8, "vocab": 32000, "type": "f32", "mode": "iid",
            "branch": 1, "temperature": 1.0, **kw}


def listed():
    return [
        # The first drafted tokens of one stream, the history just begun: the smallest call.
        _attention(name="tree_5_first", nodes=5, length=1),
        # One stream at a long history, a tree of usual size, the heads of the decode attention.
        _attention(name="tree_16_at_32768", nodes=16, length=32768),
        # Eight streams of ragged lengths and trees, 16-bit activations, heads of 128.
        _attention(name="tree_batch_ragged", sequences=8, nodes=25, q_heads=32, head_dim=128, type="bf16",
                   length=8191, sinks=False),
        # The sliding-window layers of four streams: their rings' 128 newest keys.
        _attention(name="tree_window_128", sequences=4, nodes=12, type="f16", length=5000, window=128),
        # One stream's chain of drafted tokens, sampled.
        _verify(name="verify_chain_6", nodes=6),
        # Trees of four streams over a large vocabulary, four independent draws a node.
        _verify(name="verify_tree_248320", sequences=4, nodes=21, vocab=248320, branch=4, temperature=0.8),
        # Sixteen streams decoded greedily, 16-bit logits.
        _verify(name="verify_greedy_16", sequences=16, nodes=5, vocab=131071, type="bf16", mode="given",
                temperature=0.0),
        # The accepted tokens of one stream against its budget of keys.
        {"name": "weights_4096", "kind": "weights", "sequences": 1, "nodes": 8, "q_heads": 64, "kv_heads": 8,
         "head_dim": 64, "type": "f32", "length": 4096},
        # The same for four streams at long histories with 16-bit activations.
        {"name": "weights_batch_32768", "kind": "weights", "sequences": 4, "nodes": 16, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "type": "bf16", "length": 32768},
        # Accepted rows into the rings of the twelve sliding-window layers of eight streams.
        {"name": "commit_rings", "kind": "commit", "layers": 12, "sequences": 8, "nodes": 16, "kv_heads": 8,
         "head_dim": 64, "type": "f16", "rows": 192},
        # The decoding loop of one stream: twelve full-attention layers held at 4096 keys a head.
        {"name": "evict_cycle_4096", "kind": "evict", "cycle": True, "layers": 12, "sequences": 1, "nodes": 16,
         "kv_heads": 8, "head_dim": 64, "type": "f16", "keep": 4096, "more": 0},
        # After a long prompt: half of its keys go, in two layers of two streams.
        {"name": "evict_half_of_32768", "kind": "evict", "cycle": False, "layers": 2, "sequences": 2, "nodes": 1,
         "kv_heads": 8, "head_dim": 128, "type": "bf16", "keep": 16384, "more": 16384},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


HEADS = [(64, 8), (32, 8), (16, 2), (24, 4), (8, 8), (5, 1), (16, 1)]


def draw(rng):
    kind = rng.choice(["attention"] * 4 + ["verify"] * 3 + ["weights", "commit", "evict", "evict"])
    if kind == "verify":
        mode = rng.choice(["iid", "iid", "distinct", "given"])
        sequences, vocab = _spread(rng, 1, 16), _spread(rng, 100, 248320)
        nodes = min(_spread(rng, 1, 64), max(1, 9_000_000 // (sequences * vocab)))
        return _verify(sequences=sequences, nodes=nodes, vocab=vocab, type=rng.choice(["f32", "f32", "f16", "bf16"]),
                       mode=mode, branch=rng.randint(1, 4),
                       temperature=0.0 if mode == "given" and rng.random() < 0.5 else round(rng.uniform(0.5, 1.5), 2))
    if kind == "commit":
        layers, nodes = _spread(rng, 1, 36), _spread(rng, 1, 64)
        kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        most = max(1, min(16, 4_000_000 // (layers * nodes * kv_heads * head_dim)))
        return {"kind": kind, "layers": layers, "sequences": _spread(rng, 1, most), "nodes": nodes,
                "kv_heads": kv_heads, "head_dim": head_dim,
                "type": rng.choice(["f16", "bf16"]), "rows": _spread(rng, 64, 1024)}
    if kind == "evict":
        cycle = rng.random() < 0.5
        keep = _spread(rng, 64, 16384)
        kv_heads, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256])
        most = max(1, 67_108_864 // (keep * 2 * kv_heads * head_dim))
        layers = _spread(rng, 1, min(36, most))
        return {"kind": kind, "cycle": cycle, "layers": layers, "sequences": _spread(rng, 1, max(1, min(8, most // layers))),
                "nodes": min(keep, _spread(rng, 1, 64)), "kv_heads": kv_heads, "head_dim": head_dim,
                "type": rng.choice(["f16", "bf16"]), "keep": keep, "more": 0 if cycle else _spread(rng, 1, keep)}
    q_heads, kv_heads = rng.choice(HEADS)
    head_dim = rng.choice([64, 64, 128, 256])
    type_ = rng.choice(["f32", "f16", "bf16"])
    length = min(_spread(rng, 1, 65536), 40_000_000 // (kv_heads * head_dim))
    sequences = _spread(rng, 1, max(1, min(16, 32_000_000 // (length * kv_heads * head_dim))))
    nodes = min(_spread(rng, 1, 64), max(1, 3_600_000_000 // (sequences * q_heads * head_dim * length)))
    if kind == "weights":
        return {"kind": kind, "sequences": sequences, "nodes": min(nodes, length), "q_heads": q_heads, "kv_heads": kv_heads,
                "head_dim": head_dim, "type": type_, "length": length}
    return _attention(sequences=sequences, nodes=nodes, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, type=type_,
                      length=length, window=_spread(rng, 32, 2048) if rng.random() < 0.3 else 0, sinks=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + part) & 0x7FFFFFFFFFFF)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _whole(g, low, high, shape):
    """Whole numbers low..high."""
    return torch.randint(low, high + 1, shape, dtype=torch.int32, device=DEV, generator=g)


def _counts(g, sequences, nodes):
    if sequences == 1:
        return torch.full((1,), nodes, dtype=torch.int32, device=DEV)
    return _whole(g, (nodes + 1) // 2, nodes, (sequences,))


def _lengths(g, sequences, length):
    if sequences == 1:
        return torch.full((1,), length, dtype=torch.int32, device=DEV)
    return _whole(g, (length + 1) // 2, length, (sequences,))


def _cache_type(case):
    return torch.bfloat16 if case["type"] == "bf16" else torch.float16


def _attention_inputs(case, seed):
    g = _generator(seed, 1)
    S, N, D, G = case["sequences"], case["nodes"], case["head_dim"], case["kv_heads"]
    act, kept = TYPES[case["type"]], _cache_type(case)
    # A windowed layer keeps a ring a little larger than its window.
    rows = case["window"] + 64 if case["window"] else case["length"] + 64
    first = torch.arange(N, device=DEV, dtype=torch.int32)
    # Each node hangs under one of the four before it.
    parents = torch.maximum(first - _whole(g, 1, 4, (S, N)), torch.zeros_like(first))
    parents[:, 0] = -1
    return {"q": _normal(g, (S, N, case["q_heads"], D), act), "draft_k": _normal(g, (S, N, G, D), kept),
            "draft_v": _normal(g, (S, N, G, D), kept), "k": _normal(g, (S, rows, G, D), kept),
            "v": _normal(g, (S, rows, G, D), kept), "parents": parents, "counts": _counts(g, S, N),
            "lengths": _lengths(g, S, case["length"]),
            "sinks": _normal(g, (case["q_heads"],), torch.bfloat16) if case["sinks"] else None}


def _verify_inputs(case, seed):
    g = _generator(seed, 2)
    S, N, V, b = case["sequences"], case["nodes"], case["vocab"], case["branch"]
    # Probabilities that fall off as a power of the rank; the draft's are near the target's.
    target = torch.empty((S, N, V), device=DEV).exponential_(1.0, generator=g) * 1.3
    draft = (target + _normal(g, (S, N, V), std=0.5)).to(TYPES[case["type"]])
    target = target.to(TYPES[case["type"]])
    parents = torch.div(torch.arange(N, device=DEV) - 1, b, rounding_mode="floor").clamp_(min=-1).int()
    up, child = parents.long().clamp(min=0), ((torch.arange(N, device=DEV) - 1) % b).clamp_(min=0)
    scaled = draft.float() / (case["temperature"] or 1.0)
    if case["mode"] == "iid":       # a node's children are drawn independently
        noise = -torch.empty((S, N, V), device=DEV).exponential_(1.0, generator=g).log_()
        tokens = (scaled[:, up] + noise).argmax(-1)
    else:                           # drawn without putting back, or the draft's most probable ones
        if case["mode"] == "distinct":
            scaled = scaled - torch.empty((S, N, V), device=DEV).exponential_(1.0, generator=g).log_()
        top = scaled.topk(min(b, V), dim=-1).indices
        tokens = top[:, up, child]
    return {"target": target, "draft": None if case["mode"] == "given" else draft, "tokens": tokens.int().contiguous(),
            "parents": parents.expand(S, N).contiguous(), "counts": _counts(g, S, N),
            "uniforms": torch.rand((S, N), device=DEV, generator=g), "final": torch.rand((S,), device=DEV, generator=g)}


def _path(g, S, N):
    """Accepted paths: increasing nodes from 0 on, -1 behind the last."""
    accepted = _whole(g, 1, N, (S,))
    order = torch.rand((S, N), device=DEV, generator=g)
    order[:, 0] = 2.0
    chosen = torch.zeros((S, N), dtype=torch.bool, device=DEV)
    chosen.scatter_(1, order.argsort(dim=1, descending=True), torch.arange(N, device=DEV) < accepted.unsqueeze(1))
    at = torch.where(chosen, torch.arange(N, device=DEV), N).sort(dim=1).values
    return torch.where(at < N, at, -1).int(), accepted


def _weights_inputs(case, seed):
    g = _generator(seed, 3)
    S, N, D, G, H = case["sequences"], case["nodes"], case["head_dim"], case["kv_heads"], case["q_heads"]
    rows, kept = case["length"] + 64, _cache_type(case)
    q, k = _normal(g, (S, N, H, D), TYPES[case["type"]]), _normal(g, (S, rows, G, D), kept)
    path, accepted = _path(g, S, N)
    # Logits of unit variance: their exponentials' sum over the keys is near the key count times e^(1/2).
    lse = math.log(case["length"]) + 0.5 + 0.1 * _normal(g, (S, N, H))
    return {"q": q, "k": k, "v": torch.zeros_like(k), "lse": lse, "path": path, "accepted": accepted,
            "lengths": _lengths(g, S, case["length"]).clamp(min=N),
            "weights": torch.rand((S, G, rows), device=DEV, generator=g)}


def _rows_inputs(case, seed):
    """Histories, drafted rows and paths of the commit and evict cases; a layer's tensors are [layer]."""
    g = _generator(seed, 4)
    L, S, N, G, D = (case[k] for k in ("layers", "sequences", "nodes", "kv_heads", "head_dim"))
    evict = case["kind"] == "evict"
    rows = case["keep"] + max(case["more"], 64) if evict else case["rows"]
    kept = TYPES[case["type"]]
    path, accepted = _path(g, S, N)
    s = {"k": _normal(g, (L, S, rows, G, D), kept), "v": _normal(g, (L, S, rows, G, D), kept),
         "draft_k": _normal(g, (L, S, N, G, D), kept), "draft_v": _normal(g, (L, S, N, G, D), kept),
         "path": path, "accepted": accepted}
    if not evict:
        s["lengths"] = _whole(g, 0, 100000, (S,))
        return s
    s["lengths"] = torch.full((S,), case["keep"], dtype=torch.int32, device=DEV)
    if not case["cycle"]:
        s["lengths"] += _whole(g, (case["more"] + 1) // 2, case["more"], (S,))
    # Accumulated weights fall off as a power, as attention's do; the oldest rows have gathered longest.
    s["weights"] = torch.rand((L, S, G, rows), device=DEV, generator=g).pow_(-0.7)
    s["positions"] = torch.arange(rows, dtype=torch.int32, device=DEV).expand(L, S, G, rows).contiguous()
    s["next"] = s["lengths"].clone()
    return s


def prepare(case, seed):
    s = {"attention": _attention_inputs, "verify": _verify_inputs, "weights": _weights_inputs,
         "commit": _rows_inputs, "evict": _rows_inputs}[case["kind"]](case, seed)
    s["case"] = case
    if case["kind"] == "attention":
        s["out"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros(s["q"].shape[:3], device=DEV)
    elif case["kind"] == "verify":
        S, N = s["tokens"].shape
        s["path"] = torch.zeros((S, N), dtype=torch.int32, device=DEV)
        s["accepted"], s["next"] = (torch.zeros((S,), dtype=torch.int32, device=DEV) for _ in range(2))
    elif case["kind"] == "evict" and not case["cycle"]:
        s["before"] = [s[k].clone() for k in ("lengths", "weights", "positions")]
    torch.cuda.synchronize()
    return s


def _recent(case):
    """Rows that eviction leaves alone whatever their weight: the newest."""
    return max(case["nodes"], case["keep"] // 8)


# ---- the framework's operators -------------------------------------------------------------------

_context = None


def _run_own(s):
    global _context
    from hydra_amd import speculative as sp
    if _context is None:
        from hydra_amd.layer import Context
        _context = Context(0)
    ctx, case, kind = _context, s["case"], s["case"]["kind"]
    if kind == "verify":
        sp.draft_verify_into(ctx, s["target"], s["tokens"], s["parents"], s["counts"], s["uniforms"], s["final"], s["path"],
                             s["accepted"], s["next"], draft=s["draft"], distinct=case["mode"] == "distinct",
                             temperature=case["temperature"], max_children=case["branch"])
        return s["path"], s["accepted"], s["next"]
    if kind in ("attention", "weights"):
        if "cache" not in s:        # the handle that a program keeps for a layer's history
            s["cache"] = sp.KVCache(s["k"], s["v"], s["lengths"], ring=bool(case.get("window")), weights=s.get("weights"))
        if kind == "weights":
            sp.attention_weights_into(ctx, s["cache"], s["q"], s["lse"], s["path"], s["accepted"])
            return s["weights"]
        sp.attention_tree_into(ctx, s["cache"], s["q"], s["draft_k"], s["draft_v"], s["parents"], s["counts"], s["out"],
                               lse=s["lse"], sinks=s["sinks"], window=case["window"], max_length=case["length"])
        return s["out"], s["lse"]
    if "caches" not in s:
        bounded = kind == "evict"
        s["caches"] = sp.CacheSet([sp.KVCache(s["k"][i], s["v"][i], s["lengths"], ring=not bounded,
                                              weights=s["weights"][i] if bounded else None,
                                              positions=s["positions"][i] if bounded else None,
                                              next_position=s["next"] if bounded else None)
                                   for i in range(case["layers"])])
    if kind == "commit" or case["cycle"]:
        sp.cache_commit(ctx, s["caches"], s["draft_k"], s["draft_v"], s["path"], s["accepted"])
    else:
        with torch.cuda.stream(ctx.stream):
            _restore(s)
    if kind == "evict":
        sp.cache_evict(ctx, s["caches"], case["keep"], _recent(case))
    return _rows_outputs(s)


def _rows_outputs(s):
    return tuple(s[k] for k in ("k", "v", "lengths", "weights", "positions", "next") if k in s)


def _restore(s):
    """What the prompt left of the counters that eviction changes."""
    for k, t in zip(("lengths", "weights", "positions"), s["before"]):
        s[k].copy_(t)


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "attention":
        return _attention_plain(s)
    if kind == "verify":
        return _verify_plain(s)
    if kind == "weights":
        return _weights_plain(s)
    if kind == "commit" or s["case"]["cycle"]:
        _commit_plain(s)
    else:
        _restore(s)
    if kind == "evict":
        _evict_plain(s)
    return _rows_outputs(s)


# ---- plain forms -----------------------------------------------------------------------------------

def _grouped(q, kv_heads):
    """[S][N][H][D] -> fp32 [S][G][N * H/G][D]."""
    S, N, H, D = q.shape
    return q.float().view(S, N, kv_heads, H // kv_heads, D).transpose(1, 2).reshape(S, kv_heads, -1, D)


def _attention_plain(s):
    case = s["case"]
    S, N, H, D = s["q"].shape
    G, rows, window = case["kv_heads"], s["k"].shape[1], case["window"]
    length = s["lengths"].long().view(S, 1)
    # The history's keys: positions first .. first + n - 1, the last `rows` of a ring.
    n = min(case["length"], rows) if window else case["length"]
    first = (length - rows).clamp(min=0) if window else torch.zeros_like(length)
    position = first + torch.arange(n, device=DEV)
    if window:
        at = (position % rows).view(S, n, 1, 1).expand(S, n, G, D)
        k, v = s["k"].gather(1, at), s["v"].gather(1, at)
    else:
        k, v = s["k"][:, :n], s["v"][:, :n]
    k = torch.cat([k, s["draft_k"]], 1).float().permute(0, 2, 3, 1).contiguous()
    v = torch.cat([v, s["draft_v"]], 1).float().transpose(1, 2).contiguous()
    # Ancestors: the parent relation's closure, by doubling.
    node = torch.arange(N, device=DEV)
    sees = (node.view(1, N, 1) == node) | (s["parents"].long().view(S, N, 1) == node)
    for _ in range(max(1, (N - 1).bit_length())):
        sees = torch.matmul(sees.float(), sees.float()) > 0
    depth = sees.sum(-1) - 1
    drafted = length.view(S, 1, 1) + depth.view(S, 1, N)
    position = torch.cat([position.view(S, 1, n).expand(S, N, n), drafted.expand(S, N, N)], 2)
    visible = torch.cat([(position[:, :, :n] < length.view(S, 1, 1)), sees], 2)
    if window:
        visible = visible & (position > drafted.view(S, N, 1) - window)
    scores = torch.matmul(_grouped(s["q"], G), k) * (1.0 / math.sqrt(D))
    scores = scores.view(S, G, N, H // G, n + N).masked_fill(~visible.view(S, 1, N, 1, n + N), -math.inf)
    sink = torch.full((H,), -math.inf, device=DEV) if s["sinks"] is None else s["sinks"].float()
    sink = sink.view(1, G, 1, H // G, 1)
    top = torch.maximum(scores.amax(-1, keepdim=True), sink)
    p = torch.exp(scores - top)
    den = p.sum(-1, keepdim=True) + torch.exp(sink - top)
    out = torch.matmul((p / den).view(S, G, -1, n + N), v).view(S, G, N, H // G, D)
    lse = (top + torch.log(den)).squeeze(-1)
    real = node < s["counts"].view(S, 1)
    out, lse = out.transpose(1, 2).reshape(S, N, H, D), lse.transpose(1, 2).reshape(S, N, H)
    s["out"].copy_(torch.where(real.view(S, N, 1, 1), out, s["out"].float()))
    s["lse"].copy_(torch.where(real.view(S, N, 1), lse, s["lse"]))
    return s["out"], s["lse"]


def _probabilities(logits, temperature):
    """softmax(logits / temperature) in 64 bits; NaN counts as minus infinity, a row of those is all zero."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    e = torch.where(x == top, 1.0, torch.exp((x - top) / temperature))
    e = torch.where(x == -math.inf, 0.0, e)
    return e / e.sum(-1, keepdim=True).clamp(min=1.0)


def _walk(s, accept, cur):
    """Follows accepted children from node 0: a node's children come behind it, in the order of their trial."""
    S, N = accept.shape
    path = torch.full((S, N), -1, dtype=torch.int32, device=DEV)
    count = (s["counts"] > 0).int()
    path[:, 0] = count - 1
    one = torch.arange(N, device=DEV)
    for n in range(1, N):
        yes = accept[:, n] & (s["parents"][:, n] == cur)
        path = torch.where(yes.unsqueeze(1) & (one == count.unsqueeze(1)), n, path)
        count = count + yes.int()
        cur = torch.where(yes, n, cur)
    return path.int(), count.int(), cur


def _verify_plain(s):
    case = s["case"]
    S, N = s["tokens"].shape
    V = s["target"].shape[-1]
    node = torch.arange(N, device=DEV)
    zero = torch.zeros((S,), dtype=torch.int32, device=DEV)
    real = node < s["counts"].view(S, 1)
    if case["temperature"] == 0:
        x = s["target"].float()
        x = torch.where(x.isnan(), -math.inf, x)
        top = x.amax(-1, keepdim=True)
        best = torch.where((x == top) & (x > -math.inf), torch.arange(V, device=DEV), V).amin(-1)
        best = torch.where(best == V, -1, best)
        above = best.gather(1, s["parents"].long().clamp(min=0))
        accept = real & (s["tokens"] == above) & (s["tokens"] >= 0)
        path, count, cur = _walk(s, accept, zero)
        after = best.gather(1, cur.long().unsqueeze(1)).squeeze(1).int()
        return path, count, torch.where(count > 0, after, -1)
    p = _probabilities(s["target"], case["temperature"])
    q = None if s["draft"] is None else _probabilities(s["draft"], case["temperature"])
    tried = torch.zeros((S, N, V), dtype=torch.bool, device=DEV)
    mass = torch.ones((S, N, 1), dtype=torch.float64, device=DEV)     # of the residual
    rest = torch.ones_like(mass)                                      # of the draft, off the tokens tried
    lowered = torch.zeros_like(mass)
    residual = p
    accept = torch.zeros((S, N), dtype=torch.bool, device=DEV)
    parents = torch.where(real, s["parents"].long(), -1)
    is_child = parents.view(S, 1, N) == node.view(1, N, 1)            # [parent][child]
    order = is_child.int().cumsum(-1)
    for j in range(case["branch"]):
        this = is_child & (order == j + 1)
        has, child = this.any(-1), this.int().argmax(-1)
        token = s["tokens"].long().gather(1, child)
        has_token = has & (token >= 0) & (token < V)
        at = token.clamp(0, V - 1).unsqueeze(-1)
        drawn = mass.new_ones((S, N, 1)) if q is None else q.gather(-1, at)
        if case["mode"] == "distinct":
            drawn = torch.where(tried.gather(-1, at), 0.0, drawn / rest.clamp(min=2.0 ** -52))
        u = s["uniforms"].double().gather(1, child).unsqueeze(-1)
        yes = (residual.gather(-1, at) > u * mass * drawn).squeeze(-1) & has_token
        accept = accept | (this & yes.unsqueeze(-1)).any(1)
        # What is left of every node that has this child, should it be rejected.
        more = has.unsqueeze(-1)
        tried = tried | (has_token.unsqueeze(-1) & (torch.arange(V, device=DEV) == at))
        if q is not None:
            by = mass / rest.clamp(min=2.0 ** -52) if case["mode"] == "distinct" else mass
            lowered = torch.where(more, lowered + by, lowered)
            residual = torch.where(more, (p - lowered * q).clamp(min=0), residual)
            rest = torch.where(more, q.masked_fill(tried, 0.0).sum(-1, keepdim=True), rest)
        residual = residual.masked_fill(tried, 0.0)
        mass = torch.where(more, residual.sum(-1, keepdim=True), mass)
    path, count, cur = _walk(s, accept, zero)
    at = cur.long().view(S, 1, 1).expand(S, 1, V)
    r, plain = residual.gather(1, at).squeeze(1), p.gather(1, at).squeeze(1)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, plain)
    sums = r.cumsum(-1)
    up_to = s["final"].double().unsqueeze(1) * sums[:, -1:]
    last = torch.where(r > 0, torch.arange(V, device=DEV), -1).amax(-1)
    after = torch.minimum((sums <= up_to).sum(-1), last)
    return path, count, torch.where(count > 0, after, -1).int()


def _weights_plain(s):
    S, N, H, D = s["q"].shape
    G, n = s["case"]["kv_heads"], max(s["case"]["length"], N)
    at = s["path"].long().clamp(min=0)
    q = s["q"].gather(1, at.view(S, N, 1, 1).expand(S, N, H, D))
    lse = s["lse"].gather(1, at.view(S, N, 1).expand(S, N, H)).view(S, N, G, H // G).transpose(1, 2).reshape(S, G, -1, 1)
    k = s["k"][:, :n].float().permute(0, 2, 3, 1).contiguous()
    p = torch.exp(torch.matmul(_grouped(q, G), k) * (1.0 / math.sqrt(D)) - lse).view(S, G, N, H // G, n)
    order = torch.arange(N, device=DEV)
    row = (s["lengths"] - s["accepted"]).view(S, 1) + order
    seen = (order < s["accepted"].view(S, 1)).unsqueeze(-1) & (torch.arange(n, device=DEV) <= row.unsqueeze(-1))
    s["weights"][:, :, :n] += p.masked_fill(~seen.view(S, 1, N, 1, n), 0.0).sum((2, 3))
    return s["weights"]


def _commit_plain(s):
    L, S, rows, G, D = s["k"].shape
    N = s["path"].shape[1]
    ring = "positions" not in s
    order = torch.arange(N, device=DEV)
    accepted = s["accepted"].view(S, 1)
    position = s["lengths"].long().view(S, 1) + order
    there = order < accepted
    # A ring takes the last rows of a path longer than itself; a history of fixed rows ends at its last.
    there = there & (order >= accepted - rows) if ring else there & (position < rows)
    row = position % rows
    node = s["path"].long().clamp(min=0)
    for name in ("k", "v"):
        new = s["draft_" + name].gather(2, node.view(1, S, N, 1, 1).expand(L, S, N, G, D))
        at = torch.where(there, row, 0).view(1, S, N, 1, 1).expand(L, S, N, G, D)
        moved = torch.zeros((L, S, rows + 1, G, D), dtype=s[name].dtype, device=DEV)
        slot = torch.where(there, row, rows)
        moved.scatter_(2, slot.view(1, S, N, 1, 1).expand(L, S, N, G, D), new)
        hit = torch.zeros((S, rows + 1), dtype=torch.bool, device=DEV).scatter_(1, slot, True)[:, :rows]
        s[name].copy_(torch.where(hit.view(1, S, rows, 1, 1), moved[:, :, :rows], s[name]))
    s["lengths"] += s["accepted"]
    if ring:
        return
    s["weights"].masked_fill_(hit.view(1, S, 1, rows), 0.0)
    place = s["next"].long().view(S, 1) + order
    place = torch.zeros((S, rows + 1), dtype=torch.long, device=DEV).scatter_(1, slot, place)[:, :rows].int()
    s["positions"].copy_(torch.where(hit.view(1, S, 1, rows), place.view(1, S, 1, rows), s["positions"]))
    s["next"] += s["accepted"]
    s["lengths"].clamp_(max=rows)


def _evict_plain(s):
    case = s["case"]
    L, S, rows, G, D = s["k"].shape
    keep = case["keep"]
    n = s["lengths"].view(1, S, 1, 1)
    row = torch.arange(rows, device=DEV)
    w = torch.where(s["weights"].isnan(), -math.inf, s["weights"])
    recent = s["positions"] >= (s["next"] - _recent(case)).view(1, S, 1, 1)
    group = torch.where(row < n, torch.where(recent, 2, 1), 0)
    # By group, then by weight, then by row.
    order = w.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, group.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices)
    rank = torch.empty_like(order).scatter_(-1, order, row.expand_as(order))
    stays = rank < keep
    full = n > keep
    hole, moves = full & ~stays & (row < keep), full & stays & (row >= keep)
    # The i-th hole takes the i-th of the rows to move.
    slot = torch.where(moves, moves.cumsum(-1) - 1, rows)
    source = torch.zeros((L, S, G, rows + 1), dtype=torch.long, device=DEV).scatter_(-1, slot, row.expand_as(slot))[..., :rows]
    source = torch.where(hole, source.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), row)[..., :keep]
    for name in ("weights", "positions"):
        s[name][..., :keep] = s[name].gather(-1, source)
    at = source.transpose(2, 3).unsqueeze(-1).expand(L, S, keep, G, D)
    for name in ("k", "v"):
        s[name][:, :, :keep] = s[name].gather(2, at)
    s["lengths"].clamp_(max=keep)


# ---- what a pass cannot do without ---------------------------------------------------------------

def _mean(most):
    """Of a whole number from half of `most` to `most`."""
    return (most + (most + 1) // 2) / 2


def work(case):
    S, N = case["sequences"], case["nodes"]
    if case["kind"] == "verify":
        size = 4 if case["type"] == "f32" else 2
        nodes = S * (N if S == 1 else _mean(N))
        inner = max(1.0, (nodes / S - 1) / case["branch"]) * S
        rows = nodes + (inner if case["mode"] != "given" else 0)
        return {"bytes": rows * case["vocab"] * size, "flops": rows * case["vocab"] * 2.0}
    G, D = case["kv_heads"], case["head_dim"]
    if case["kind"] in ("attention", "weights"):
        H, size = case["q_heads"], 4 if case["type"] == "f32" else 2
        keys = case["length"] if S == 1 else _mean(case["length"])
        if case["kind"] == "weights":
            some = (N + 1) / 2
            return {"bytes": S * (keys * G * (2 * D + 8) + some * H * (D * size + 4)), "flops": 2.0 * S * some * H * keys * D}
        keys = min(keys, case["window"] + N) if case["window"] else keys
        nodes = N if S == 1 else _mean(N)
        return {"bytes": S * (4 * (keys + nodes) * G * D + nodes * H * (2 * D * size + 4)),
                "flops": 4.0 * S * nodes * H * (keys + nodes / 2) * D}
    L, some = case["layers"], (N + 1) / 2
    committed = L * S * some * G * D * 8.0
    if case["kind"] == "commit":
        return {"bytes": committed, "flops": 0}
    more = some if case["cycle"] else _mean(case["more"])
    n = case["keep"] + more
    moved = case["keep"] * more / n
    return {"bytes": (committed if case["cycle"] else 0) + L * S * G * (n * 8 + moved * (D * 8 + 16)), "flops": 0}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------

def _exact_attention(case, seed):
    s = _attention_inputs(case, seed)
    S, N, H, D = s["q"].shape
    G, window, rows = case["kv_heads"], case["window"], s["k"].shape[1]
    out = torch.zeros((S, N, H, D), dtype=torch.float64, device=DEV)
    lse = torch.zeros((S, N, H), dtype=torch.float64, device=DEV)
    for i in range(S):
        length, count, parents = int(s["lengths"][i]), int(s["counts"][i]), s["parents"][i].tolist()
        low = max(0, length - rows) if window else 0
        at = torch.arange(low, length, device=DEV)
        keys = torch.cat([s["k"][i, at % rows], s["draft_k"][i, :count]]).double()
        values = torch.cat([s["v"][i, at % rows], s["draft_v"][i, :count]]).double()
        mask = torch.zeros((count, length - low + count), dtype=torch.bool)
        for m in range(count):
            line = [m]
            while parents[line[-1]] >= 0:
                line.append(parents[line[-1]])
            oldest = length + len(line) - 1 - window + 1 if window else 0
            mask[m, max(0, oldest - low):length - low] = True
            for up, a in enumerate(line):
                if not window or up < window:
                    mask[m, length - low + a] = True
        mask = mask.to(DEV)
        for h in range(H):
            g = h // (H // G)
            x = (s["q"][i, :count, h].double() @ keys[:, g].T) / math.sqrt(D)
            x = torch.where(mask, x, -math.inf)
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(count, 1)], 1)
            lse[i, :count, h] = torch.logsumexp(x, 1)
            out[i, :count, h] = torch.softmax(x, 1)[:, :keys.shape[0]] @ values[:, g]
    return out, lse


def _exact_verify(case, seed):
    """One sequence after the other, by the rule as it is stated: the residual is normalised after each rejection."""
    s = _verify_inputs(case, seed)
    S, N = s["tokens"].shape
    path, accepted, after = torch.full((S, N), -1), torch.zeros((S,)), torch.full((S,), -1)
    for i in range(S):
        count, parents, tokens = int(s["counts"][i]), s["parents"][i].tolist(), s["tokens"][i].tolist()
        cur, line = 0, [0]
        while True:
            x = s["target"][i, cur].double()
            children = [n for n in range(1, count) if parents[n] == cur][:case["branch"]]
            if case["temperature"] == 0:
                best = int((x == x.max()).nonzero()[0])
                match = [n for n in children if tokens[n] == best]
                if not match:
                    after[i] = best
                    break
                cur = match[0]
                line.append(cur)
                continue
            p = torch.softmax(x / case["temperature"], 0)
            q = None if s["draft"] is None else torch.softmax(s["draft"][i, cur].double() / case["temperature"], 0)
            found = None
            for n in children:
                t = tokens[n]
                if float(s["uniforms"][i, n]) * (1.0 if q is None else float(q[t])) < float(p[t]):
                    found = n
                    break
                p = p.clone() if q is None else (p - q).clamp(min=0)
                p[t] = 0.0
                p = p / p.sum()
                if case["mode"] == "distinct":
                    q = q.clone()
                    q[t] = 0.0
                    q = q / q.sum()
            if found is None:
                u = float(s["final"][i])
                after[i] = min(int((p.cumsum(0) <= u * p.sum()).sum()), int(p.nonzero()[-1]))
                break
            cur = found
            line.append(cur)
        path[i, :len(line)] = torch.tensor(line)
        accepted[i] = len(line)
    return path, accepted, after


def _exact_weights(case, seed):
    s = _weights_inputs(case, seed)
    S, _, H, D = s["q"].shape
    G = case["kv_heads"]
    w = s["weights"].double()
    for i in range(S):
        length, count = int(s["lengths"][i]), int(s["accepted"][i])
        for j, n in enumerate(s["path"][i, :count].tolist()):
            last = length - count + j + 1
            for g in range(G):
                heads = slice(g * (H // G), (g + 1) * (H // G))
                x = s["q"][i, n, heads].double() @ s["k"][i, :last, g].double().T / math.sqrt(D)
                w[i, g, :last] += torch.exp(x - s["lse"][i, n, heads].double().unsqueeze(1)).sum(0)
    return w


def _exact_rows(case, seed):
    """Row by row on the host: what is held at the end, as numbers."""
    s = {k: v.cpu() for k, v in _rows_inputs(case, seed).items()}
    L, S, rows, G, _ = s["k"].shape
    k, v = s["k"].double(), s["v"].double()
    lengths = s["lengths"].tolist()
    evict = case["kind"] == "evict"
    w, pos, nxt = (s["weights"].double(), s["positions"].long(), s["next"].tolist()) if evict else (None, None, None)
    if not evict or case["cycle"]:
        for i in range(S):
            for j, n in enumerate(s["path"][i, :int(s["accepted"][i])].tolist()):
                r = lengths[i] if evict else lengths[i] % rows
                k[:, i, r], v[:, i, r] = s["draft_k"][:, i, n].double(), s["draft_v"][:, i, n].double()
                if evict:
                    w[:, i, :, r], pos[:, i, :, r] = 0.0, nxt[i]
                    nxt[i] += 1
                lengths[i] += 1
    if not evict:
        return k, v, None
    keep = case["keep"]
    for i in range(S):
        for l in range(L):
            for g in range(G):
                ranked = torch.where(pos[l, i, g, :lengths[i]] >= nxt[i] - _recent(case), math.inf, w[l, i, g, :lengths[i]])
                best = torch.sort(ranked, descending=True, stable=True).indices[:keep]
                left = torch.ones(lengths[i], dtype=torch.bool)
                left[best] = False
                hole = left[:keep].nonzero().flatten()
                take = keep + (~left[keep:]).nonzero().flatten()
                k[l, i, hole, g], v[l, i, hole, g] = k[l, i, take, g], v[l, i, take, g]
                w[l, i, g, hole], pos[l, i, g, hole] = w[l, i, g, take], pos[l, i, g, take]
    return k, v, None, w, None, None


def exact(case, seed):
    if case["kind"] == "attention":
        return _exact_attention(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(case, seed)
    if case["kind"] == "weights":
        return _exact_weights(case, seed)
    return _exact_rows(case, seed)
