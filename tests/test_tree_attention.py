"""Attention of a drafted tree (hh_attention_tree) and the accumulated weights (hh_attention_weights)
against a plain implementation in 64 bits on inputs of the kernels' types.

Tolerances, rel-L2 of all outputs. F32: the queries as fp16 pairs (2^-22 of a value), fp32 sums of up to 256
products of unit normals (terms of a logit sum to ~10 in magnitude: sqrt(256)·10·2^-24 = 1e-5 of a
probability), sums over the keys alike: 2e-5. F16 and BF16: one rounding of each probability and one of each
output, half a step each: 2·2^-11 and 2·2^-8. lse, absolute: 1e-5 of a logit's error, its sum's and its logarithm's
with it 4e-5."""
import ctypes as C
import math

import numpy as np
import pytest

TOL = {"f32": 2e-5, "f16": 2 * 2.0 ** -11, "bf16": 2 * 2.0 ** -8}
LSE = 4e-5


def line_of(parents, m):
    """Node m and its ancestors; a parent that is not an earlier node counts as none."""
    line = [m]
    while 0 <= parents[line[-1]] < line[-1]:
        line.append(int(parents[line[-1]]))
    return line


def reference(q, k, v, dk, dv, lengths, parents, counts, sinks, window, ring, scale):
    """fp64 outputs and lse per (sequence, real node, head), from only the keys each node sees."""
    S, N, H, D = q.shape
    rows, G = k.shape[1], k.shape[2]
    out, lse = {}, {}
    for s in range(S):
        length = max(0, int(lengths[s]))
        if not ring:
            length = min(length, rows)
        for m in range(min(N, max(0, int(counts[s])))):
            line = line_of(parents[s], m)
            pos = length + len(line) - 1
            low = max(0, length - rows) if ring else 0
            if window:
                low = max(low, pos - window + 1)
            at = np.arange(low, length) % rows
            sees = [a for up, a in enumerate(line) if not window or up < window]
            kk = np.concatenate([k[s, at], dk[s, sees]]).astype(np.float64)
            vv = np.concatenate([v[s, at], dv[s, sees]]).astype(np.float64)
            for h in range(H):
                g = h // (H // G)
                x = scale * (kk[:, g] @ q[s, m, h].astype(np.float64))
                top = max(x.max(), sinks[h]) if sinks is not None else x.max()
                e = np.exp(x - top)
                den = e.sum() + (math.exp(sinks[h] - top) if sinks is not None else 0.0)
                out[s, m, h] = (e / den) @ vv[:, g]
                lse[s, m, h] = top + math.log(den)
    return out, lse


def make(torch, S, N, H, G, D, kind, rows, lengths, counts=None, parents=None, seed=0, sinks=True):
    act = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    kept = torch.bfloat16 if kind == "bf16" else torch.float16
    g = torch.Generator().manual_seed(seed)
    n = lambda shape, t: torch.randn(shape, generator=g).to(t)
    p = np.asarray(parents if parents is not None else
                   [[int(torch.randint(max(0, i - 5), i, (1,), generator=g)) if i else -1 for i in range(N)] for _ in range(S)])
    return dict(q=n((S, N, H, D), act), k=n((S, rows, G, D), kept), v=n((S, rows, G, D), kept), dk=n((S, N, G, D), kept),
                dv=n((S, N, G, D), kept), parents=torch.tensor(np.broadcast_to(p, (S, N)).copy(), dtype=torch.int32),
                counts=torch.tensor([N] * S if counts is None else counts, dtype=torch.int32),
                lengths=torch.tensor(lengths, dtype=torch.int32), sinks=n((H,), torch.bfloat16) if sinks else None)


def call(torch, ctx, t, ring=False, window=0, scale=None, max_length=0, lse=True, cache=None):
    from hydra_amd import speculative as sp
    d = {k: None if x is None else x.to("cuda:0") for k, x in t.items()}
    cache = cache or sp.KVCache(d["k"], d["v"], d["lengths"], ring=ring)
    out = torch.full(t["q"].shape, 7.0, dtype=t["q"].dtype, device="cuda:0")
    ls = torch.full(t["q"].shape[:3], 7.0, device="cuda:0") if lse else None
    torch.cuda.synchronize()
    sp.attention_tree_into(ctx, cache, d["q"], d["dk"], d["dv"], d["parents"], d["counts"], out, lse=ls, sinks=d["sinks"],
                           window=window, sm_scale=scale, max_length=max_length)
    ctx.synchronize()
    return out, ls


def check(torch, t, kind, out, lse, ring=False, window=0, scale=None):
    num = lambda x: None if x is None else x.to(torch.float64).numpy()
    S, N, H, D = t["q"].shape
    ro, rl = reference(num(t["q"]), num(t["k"]), num(t["v"]), num(t["dk"]), num(t["dv"]), t["lengths"].numpy(),
                       t["parents"].numpy(), t["counts"].numpy(), num(t["sinks"]), window, ring,
                       D ** -0.5 if scale is None else scale)
    got, gl = out.double().cpu().numpy(), None if lse is None else lse.double().cpu().numpy()
    real = np.zeros((S, N), bool)
    for (s, m, h) in ro:
        real[s, m] = True
    assert np.all(got[~real] == 7.0) and (gl is None or np.all(gl[~real] == 7.0)), "padded nodes were written"
    if not ro:
        return
    a = np.stack([got[i] for i in ro])
    b = np.stack([ro[i] for i in ro])
    assert np.isfinite(a).all()
    assert np.linalg.norm(a - b) / np.linalg.norm(b) < TOL[kind]
    if gl is not None:
        assert max(abs(gl[i] - rl[i]) for i in rl) < LSE


CHAIN = [[i - 1 for i in range(64)]]
STAR = [[-1] + [0] * 63]
CASES = [
    # S, N, H, G, D, type, rows, lengths, window, ring, parents
    (1, 1, 64, 8, 64, "f32", 8, [0], 0, False, None),            # no history: the node itself
    (1, 1, 64, 8, 64, "f32", 8, [1], 0, False, None),
    (1, 5, 64, 8, 64, "f16", 70, [63], 0, False, None),          # tiles end at and around the history's end
    (1, 5, 64, 8, 64, "bf16", 70, [64], 0, False, None),
    (1, 5, 64, 8, 64, "f32", 70, [65], 0, False, None),
    (2, 64, 8, 8, 64, "f32", 200, [130, 200], 0, False, CHAIN),  # 64 nodes in one line; a full history
    (2, 64, 16, 2, 64, "f16", 300, [257, 3], 0, False, STAR),    # 63 children of one node
    (3, 33, 6, 6, 128, "f32", 600, [511, 0, 600], 0, False, None),
    (2, 17, 5, 1, 128, "bf16", 400, [389, 128], 0, False, None),     # five heads a group
    (2, 9, 16, 1, 256, "f16", 300, [290, 31], 0, False, None),       # sixteen heads a group
    (1, 12, 24, 4, 256, "f32", 900, [880], 0, False, None),
    (1, 7, 8, 4, 256, "bf16", 130, [97], 0, False, None),
    (4, 12, 16, 4, 64, "f32", 40, [1000, 39, 41, 5], 24, True, None),   # rings, wrapped and not yet full
    (2, 64, 8, 2, 64, "f16", 70, [300, 69], 10, True, CHAIN),    # most of the line is out of the window
    (2, 20, 8, 2, 128, "bf16", 500, [480, 100], 60, False, None),       # a window without a ring
    (1, 6, 8, 2, 64, "f32", 33, [100], 0, True, None),           # a ring without a window: its rows
    (2, 3, 8, 2, 64, "f32", 300, [290, 290], 1, False, CHAIN),   # a window of one: every node alone
    (1, 16, 64, 8, 64, "f32", 5000, [4987], 0, False, None),     # many chunks
    (1, 2, 2, 1, 64, "f32", 70000, [69990], 0, False, None),     # the most chunks of a sequence
    (2, 40, 16, 1, 64, "bf16", 700, [650, 699], 0, False, None), # five blocks of rows
    (1, 33, 4, 1, 256, "f32", 1500, [1500], 0, False, None),
    (9, 4, 8, 2, 64, "f16", 2500, [2400, 1, 0, 77, 2500, 1024, 1025, 640, 2000], 0, False, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("S,N,H,G,D,kind,rows,lengths,window,ring,parents", CASES)
def test_tree_attention(S, N, H, G, D, kind, rows, lengths, window, ring, parents):
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] tree attention S={S} N={N} H={H} G={G} D={D} {kind} {lengths} w={window} ring={ring}", flush=True)
    par = None if parents is None else [p[:N] for p in parents]
    ctx = Context(0)
    try:
        for sinks in (True, False):
            t = make(torch, S, N, H, G, D, kind, rows, lengths, parents=par, seed=N * 100 + H, sinks=sinks)
            out, lse = call(torch, ctx, t, ring, window)
            check(torch, t, kind, out, lse, ring, window)
    finally:
        ctx.close()


@pytest.mark.gpu
def test_padding_odd_parents_and_lengths_out_of_range():
    """Counts from none to all, parents that are no earlier nodes, lengths above the rows and below zero."""
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        parents = [[5, 0, 7, -9, 3, 5, 4, 4], [-1, 0, 1, 2, 3, 4, 5, 6], [-1] * 8, [-1, 0, 0, 1, 1, 2, 2, 3]]
        t = make(torch, 4, 8, 8, 2, 64, "f32", 100, [250, -3, 100, 40], counts=[8, 5, 0, 70], parents=parents, seed=5)
        out, lse = call(torch, ctx, t)
        check(torch, t, "f32", out, lse)
        # The launch is sized for shorter histories than there are, and without lse.
        out2, _ = call(torch, ctx, t, max_length=10, lse=False)
        check(torch, t, "f32", out2, None)
        # Another scale, and a negative one.
        outn, lsen = call(torch, ctx, t, scale=-0.2)
        check(torch, t, "f32", outn, lsen, scale=-0.2)
        b = make(torch, 2, 5, 8, 2, 64, "bf16", 100, [90, 3], seed=6)
        outb, lseb = call(torch, ctx, b, scale=-0.2)
        check(torch, b, "bf16", outb, lseb, scale=-0.2)
        out3, lse3 = call(torch, ctx, t, scale=0.5)
        check(torch, t, "f32", out3, lse3, scale=0.5)
    finally:
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,D,H,G,N", [("f32", 64, 16, 2, 21), ("f16", 128, 4, 4, 13), ("bf16", 256, 8, 1, 6), ("f16", 64, 8, 1, 3)])
@pytest.mark.parametrize("ring", [False, True])
def test_keys_that_a_node_does_not_see_have_no_part(kind, D, H, G, N, ring):
    """NaN and infinities in rows past the length, in padded nodes, in rows that left every window, in rows that
    left some nodes' windows only, and in nodes that are no ancestors."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] masked NaN {kind} D={D} ring={ring}", flush=True)
    ctx = Context(0)
    try:
        rows, length, window = (90, 200, 70) if ring else (300, 280, 70)
        t = make(torch, 2, N, H, G, D, kind, rows, [length, 30], counts=[N - 1, N - 1], seed=3)
        nan, inf = float("nan"), float("inf")
        for x in (t["k"], t["v"]):
            x[1, 30:] = nan
            if ring:
                x[0, torch.arange(110, 131) % rows] = nan
            else:
                x[0, 280:] = -inf
                x[0, :280 - 70 + 1] = nan         # out of every window (the root's begins at 211)
        for x in (t["dk"], t["dv"]):
            x[:, N - 1:] = inf
        out, lse = call(torch, ctx, t, ring, window)
        check(torch, t, kind, out, lse, ring, window)
        # A key that only the shallow nodes see, and a drafted node's value: the nodes that see it are lost, no others.
        depth = np.array([len(line_of(t["parents"][0].tolist(), m)) - 1 for m in range(N - 1)])
        bad = length - window + 1     # the oldest key in the root's window, in nobody else's
        t["v"][0, bad % rows] = inf
        t["k"][0, bad % rows] = nan
        t["dv"][0, 2] = nan
        out2, _ = call(torch, ctx, t, ring, window)
        hit = np.array([depth[m] == 0 or 2 in line_of(t["parents"][0].tolist(), m) for m in range(N - 1)])
        assert hit.any() and not hit.all()
        assert not torch.isfinite(out2[0, :N - 1][torch.tensor(hit)]).any()
        # The tile that holds such values is added key by key, in other roundings: both results are within TOL of the
        # exact one, so within twice TOL of each other (plus a second-order term, below TOL^2).
        a, b = (x[0, :N - 1][torch.tensor(~hit)].double() for x in (out2, out))
        assert torch.isfinite(a).all() and (a - b).norm() < 2 * TOL[kind] * (1 + TOL[kind]) * b.norm()
        assert torch.equal(out2[1], out[1])
    finally:
        ctx.close()


@pytest.mark.gpu
def test_slices_of_a_fused_projection():
    """q and the drafted rows as slices of one product's output; the histories with a stride between sequences."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        S, N, H, G, D = 3, 6, 8, 2, 64
        t = make(torch, S, N, H, G, D, "bf16", 120, [100, 7, 120], seed=9)
        want, _ = call(torch, ctx, t)
        wide = torch.cat([t["q"], t["dk"], t["dv"]], dim=2).to("cuda:0")
        big = torch.full((S, 2, 130, G, D), float("nan"), dtype=torch.bfloat16, device="cuda:0")
        big[:, 0, :120], big[:, 1, :120] = t["k"].to("cuda:0"), t["v"].to("cuda:0")
        cache = sp.KVCache(big[:, 0, :120], big[:, 1, :120], t["lengths"].to("cuda:0"))
        out = torch.empty_like(want)
        torch.cuda.synchronize()
        sp.attention_tree_into(ctx, cache, wide[:, :, :H], wide[:, :, H:H + G], wide[:, :, H + G:], t["parents"].to("cuda:0"),
                               t["counts"].to("cuda:0"), out, sinks=t["sinks"].to("cuda:0"))
        ctx.synchronize()
        assert torch.equal(out, want)
    finally:
        ctx.close()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Sequences more than 2^32 elements apart, and rows past 2^32 bytes within one."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    S, N, H, G, D = 2, 5, 4, 2, 64
    rows = (1 << 32) // (G * D) + 64          # a sequence: 2^32 elements and a little
    ctx = Context(0)
    try:
        t = make(torch, S, N, H, G, D, "f16", 80, [80, 75], seed=1)
        want, wl = call(torch, ctx, t, ring=True, window=60)
        # The same keys at positions that end a ring of all those rows: 2 * rows + 40.
        k, v = (torch.empty((S, rows, G, D), dtype=torch.float16, device="cuda:0") for _ in range(2))
        lengths = torch.tensor([2 * rows + 40, rows], dtype=torch.int64).to(torch.int32).to("cuda:0")
        for s, (length, old) in enumerate(((2 * rows + 40, 80), (rows, 75))):
            pos = torch.arange(length - old, length)
            k[s, (pos % rows).to("cuda:0")] = t["k"][s, :old].to("cuda:0")
            v[s, (pos % rows).to("cuda:0")] = t["v"][s, :old].to("cuda:0")
        cache = sp.KVCache(k, v, lengths, ring=True)
        out, lse = call(torch, ctx, t, window=60, cache=cache)
        assert (out - want).abs().max() < 4 * 2.0 ** -11 and (lse - wl).abs().max() < LSE
    finally:
        ctx.close()


@pytest.mark.gpu
def test_recorded_calls_follow_the_device_and_share_the_workspace():
    """Two graphs of one context, of other shapes, replayed in turn while lengths and inputs change."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        parts, graphs = [], []
        for i, (S, N, H, G, D, kind) in enumerate([(1, 16, 16, 2, 64, "f32"), (3, 7, 8, 4, 128, "bf16")]):
            t = make(torch, S, N, H, G, D, kind, 3000, [3000] * S, seed=i)
            d = {k: x.to("cuda:0") for k, x in t.items()}
            cache = sp.KVCache(d["k"], d["v"], d["lengths"])
            sp.reserve(ctx, cache, nodes=N, q_heads=H, q_dtype=t["q"].dtype)
            parts.append((t, d, cache, torch.empty_like(d["q"]), torch.empty(t["q"].shape[:3], device="cuda:0")))
        torch.cuda.synchronize()
        for t, d, cache, out, lse in parts:
            graphs.append(ctx.capture(lambda: sp.attention_tree_into(ctx, cache, d["q"], d["dk"], d["dv"], d["parents"],
                                                                     d["counts"], out, lse=lse, sinks=d["sinks"])))
        for rep in range(4):
            want = []
            for t, d, cache, out, lse in parts:
                d["lengths"].copy_(torch.randint(0, 3000, d["lengths"].shape, dtype=torch.int32))
                d["q"].normal_()
                d["parents"][:, 3:] = rep % 3
                out.fill_(3.0)
                torch.cuda.synchronize()
                o, l = torch.empty_like(out), torch.empty_like(lse)
                sp.attention_tree_into(ctx, cache, d["q"], d["dk"], d["dv"], d["parents"], d["counts"], o, lse=l, sinks=d["sinks"])
                ctx.synchronize()
                want.append((o, l))
            for g in graphs + graphs[::-1]:
                g.launch()
            ctx.synchronize()
            for (t, d, cache, out, lse), (o, l) in zip(parts, want):
                assert torch.equal(out, o) and torch.equal(lse, l), rep
        for g in graphs:
            g.close()
    finally:
        ctx.close()


# ---- accumulated weights ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("S,N,H,G,D,kind,rows,lengths,accepted", [
    (1, 1, 8, 2, 64, "f32", 10, [1], [1]),
    (1, 8, 64, 8, 64, "f32", 300, [300], [8]),
    (3, 5, 6, 6, 128, "f16", 200, [64, 5, 199], [3, 5, 0]),
    (2, 64, 5, 1, 128, "bf16", 150, [129, 64], [64, 63]),
    (2, 9, 32, 2, 256, "f32", 1100, [1027, 400], [9, 2]),
    (2, 3, 8, 4, 256, "bf16", 70, [70, 33], [1, 3]),
    (1, 16, 16, 2, 64, "f16", 5000, [4999], [11]),
])
def test_accumulated_weights(S, N, H, G, D, kind, rows, lengths, accepted):
    """Tolerance: the exponent's error as above, 1e-5, and fp32 sums of up to 1024 terms: 2e-5 relative."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    print(f"[gpu] weights S={S} N={N} H={H} D={D} {kind}", flush=True)
    t = make(torch, S, N, H, G, D, kind, rows, lengths, seed=N)
    g = torch.Generator().manual_seed(4)
    path = torch.full((S, N), -1, dtype=torch.int32)
    for s in range(S):
        path[s, :accepted[s]] = torch.sort(torch.randperm(N, generator=g)[:accepted[s]]).values.int()
    lse = math.log(max(lengths)) + 0.5 + 0.1 * torch.randn((S, N, H), generator=g)
    w0 = torch.rand((S, G, rows), generator=g)
    t["k"][0, lengths[0]:] = float("nan")
    ctx = Context(0)
    try:
        d = {k: x.to("cuda:0") for k, x in t.items()}
        w = w0.to("cuda:0")
        cache = sp.KVCache(d["k"], d["v"], d["lengths"], weights=w)
        pd, ad, ld = path.to("cuda:0"), torch.tensor(accepted, dtype=torch.int32, device="cuda:0"), lse.to("cuda:0")
        torch.cuda.synchronize()
        sp.attention_weights_into(ctx, cache, d["q"], ld, pd, ad)
        ctx.synchronize()
    finally:
        ctx.close()
    want = w0.double().numpy()
    for s in range(S):
        for i in range(accepted[s]):
            n, last = int(path[s, i]), lengths[s] - accepted[s] + i + 1
            for h in range(H):
                x = t["k"][s, :last, h // (H // G)].double().numpy() @ t["q"][s, n, h].double().numpy() * D ** -0.5
                want[s, h // (H // G), :last] += np.exp(x - float(lse[s, n, h]))
    got = w.double().cpu().numpy()
    for s in range(S):
        assert np.array_equal(got[s, :, lengths[s]:], w0.double().numpy()[s, :, lengths[s]:])
    assert np.max(np.abs(got - want) / np.maximum(want, 1e-3)) < 2e-5


@pytest.mark.gpu
def test_weights_of_one_token_sum_to_one():
    """The weights that attention's own lse gives: every head's probabilities, without a sink."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        t = make(torch, 2, 1, 16, 4, 64, "f32", 500, [400, 31], seed=2, sinks=False)
        d = {k: None if x is None else x.to("cuda:0") for k, x in t.items()}
        w = torch.zeros((2, 4, 500), device="cuda:0")
        nxt = torch.tensor([400, 31], dtype=torch.int32, device="cuda:0")
        pos = torch.zeros((2, 4, 500), dtype=torch.int32, device="cuda:0")
        cache = sp.KVCache(d["k"], d["v"], d["lengths"], weights=w, positions=pos, next_position=nxt)
        out, lse = torch.empty_like(d["q"]), torch.empty((2, 1, 16), device="cuda:0")
        path, one = torch.zeros((2, 1), dtype=torch.int32, device="cuda:0"), torch.ones(2, dtype=torch.int32, device="cuda:0")
        torch.cuda.synchronize()
        sp.attention_tree_into(ctx, cache, d["q"], d["dk"], d["dv"], d["parents"], d["counts"], out, lse=lse)
        sp.cache_commit(ctx, sp.CacheSet([cache]), [d["dk"]], [d["dv"]], path, one)
        sp.attention_weights_into(ctx, cache, d["q"], lse, path, one)
        ctx.synchronize()
        # Four heads a group: 4, each probability's error below 2e-5 of it.
        assert (w.double().sum(-1) - 4).abs().max() < 4 * 4e-5
    finally:
        ctx.close()


# ---- refusals (no GPU) ------------------------------------------------------------------------------

def _call(fn="hh_attention_tree", desc=None, cache=None, **kw):
    """The entry with sound arguments but those named; a context that is never reached must not be needed."""
    from hydra_amd import _lib
    L = _lib.lib()
    d = dict(sequences=1, nodes=4, q_heads=8, kv_heads=2, head_dim=64, type=0, cache_type=1, window=0, max_length=0, sm_scale=0.125,
             q_stride=0, kv_stride=0)
    d.update(desc or {})
    c = dict(k=4096, v=8192, sequence_stride=0, rows=16, ring=0, lengths=64, weights=64, positions=None, next_position=None)
    c.update(cache or {})
    dc, cc = _lib.TreeDescC(**d), _lib.KVCacheC(**c)
    ctx = C.create_string_buffer(4096)      # zeros: never used, the checks come first
    if fn == "hh_attention_tree":
        a = dict(q=16, dk=16, dv=16, parents=16, counts=16, sinks=None, out=16, lse=None)
    else:
        a = dict(q=16, lse=16, path=16, accepted=16)
    a.update(kw)
    return getattr(L, fn)(ctx, C.byref(dc), C.byref(cc), *a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(desc=dict(sequences=0)), -1), (dict(desc=dict(nodes=0)), -1), (dict(desc=dict(nodes=65)), -1),
    (dict(desc=dict(head_dim=96)), -6), (dict(desc=dict(q_heads=7)), -6), (dict(desc=dict(q_heads=34)), -6),
    (dict(desc=dict(kv_heads=0)), -6), (dict(desc=dict(type=1, cache_type=2)), -1), (dict(desc=dict(type=0, cache_type=2)), -1),
    (dict(desc=dict(cache_type=0)), -1), (dict(desc=dict(type=3)), -1), (dict(desc=dict(window=-1)), -1),
    (dict(desc=dict(max_length=-1)), -1), (dict(desc=dict(sm_scale=float("nan"))), -1), (dict(desc=dict(sm_scale=0.0)), -1),
    (dict(desc=dict(sequences=4096, kv_heads=128, q_heads=128)), -1), (dict(cache=dict(rows=(1 << 30) + 1)), -1), (dict(desc=dict(q_stride=100)), -6),
    (dict(desc=dict(q_stride=514)), -2), (dict(desc=dict(kv_stride=64)), -6), (dict(desc=dict(kv_stride=132)), -2),
    (dict(cache=dict(k=None)), -1), (dict(cache=dict(v=8200)), -2), (dict(cache=dict(rows=0)), -1),
    (dict(cache=dict(sequence_stride=100)), -6), (dict(cache=dict(sequence_stride=2052)), -2), (dict(cache=dict(lengths=None)), -1),
    (dict(cache=dict(ring=1)), -1), (dict(cache=dict(positions=64)), -1), (dict(q=None), -1), (dict(q=20), -2), (dict(out=24), -2),
    (dict(parents=None), -1), (dict(counts=None), -1), (dict(dk=18), -2),
])
def test_tree_refusals(kw, code):
    assert _call(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(desc=dict(window=8)), -1), (dict(cache=dict(weights=None)), -1), (dict(cache=dict(ring=1, weights=None)), -1),
    (dict(lse=None), -1), (dict(path=None), -1), (dict(q=8), -2), (dict(desc=dict(nodes=65)), -1),
])
def test_weights_refusals(kw, code):
    assert _call("hh_attention_weights", **kw) == code


def test_null_arguments():
    from hydra_amd._lib import lib
    assert lib().hh_attention_tree(None, None, None, *[None] * 8) == -1
    assert lib().hh_attention_weights(None, None, None, *[None] * 4) == -1


def test_python_refuses_tensors_that_do_not_fit():
    import torch
    from hydra_amd import speculative as sp
    k = torch.zeros((2, 8, 2, 64), dtype=torch.float16)
    lengths = torch.zeros(2, dtype=torch.int32)
    for bad in (lambda: sp.KVCache(k, k[:, :4], lengths), lambda: sp.KVCache(k.float(), k.float(), lengths),
                lambda: sp.KVCache(k, k, lengths.long()), lambda: sp.KVCache(k.transpose(1, 2), k.transpose(1, 2), lengths),
                lambda: sp.KVCache(k, k.clone(), lengths, weights=torch.zeros((2, 2, 7)))):
        with pytest.raises(ValueError):
            bad()

    class Ctx:
        device, handle = 0, None
    with pytest.raises(ValueError):        # another device than the context's
        sp.attention_tree_into(Ctx, sp.KVCache(k, k.clone(), lengths), torch.zeros((2, 3, 4, 64)), None, None, None, None, None)


def test_python_refuses_expanded_tensors():
    """A step of 0 between nodes or sequences would be taken for the packed one, and memory behind the tensor read."""
    import torch
    from hydra_amd import speculative as sp
    f16 = torch.float16
    for shape, base in (((2, 3, 4, 64), (1, 1, 4, 64)), ((2, 1, 4, 64), (1, 1, 4, 64)), ((1, 3, 4, 64), (1, 1, 4, 64))):
        t = torch.zeros(base, dtype=f16).expand(shape)
        with pytest.raises(ValueError):
            sp._node_stride(t, "q", shape, f16, t.device)
        row = torch.zeros((1, 1, 64)).expand(shape[:2] + (64,))
        with pytest.raises(ValueError):
            sp._row_stride(row, "target", row.shape, row.dtype, row.device)
    one = torch.zeros((1, 1, 4, 64), dtype=f16)
    assert sp._node_stride(one, "q", one.shape, f16, one.device) == 256
    wide = torch.zeros((2, 3, 12, 64), dtype=f16)[:, :, 4:8]
    assert sp._node_stride(wide, "q", wide.shape, f16, wide.device) == 768
    k = torch.zeros((1, 8, 2, 64), dtype=f16)
    lengths = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        sp.KVCache(k.expand(2, 8, 2, 64), k.expand(2, 8, 2, 64), lengths)
    sp.KVCache(k, k.clone(), lengths[:1])
