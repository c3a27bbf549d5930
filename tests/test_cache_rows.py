"""Accepted rows into the histories (hh_cache_commit) and eviction (hh_cache_evict), against row-by-row
restatements. Values are moved, not computed: results are equal bit for bit."""
import ctypes as C

import numpy as np
import pytest


def commit_ref(c, path, accepted, dk, dv, limit):
    """One layer of the commit on numpy arrays; the lengths are advanced by the caller."""
    rows = c["k"].shape[1]
    for s in range(len(path)):
        n = min(max(int(accepted[s]), 0), len(path[s]), max(0, limit - max(int(c["lengths"][s]), 0)))
        for i in range(n):
            node = int(path[s][i])
            if not 0 <= node < len(path[s]) or i < n - rows:
                continue
            pos = max(int(c["lengths"][s]), 0) + i
            r = pos % rows if c["ring"] else pos
            c["k"][s, r], c["v"][s, r] = dk[s, node], dv[s, node]
            if c["weights"] is not None:
                c["weights"][s, :, r] = 0
            if c["positions"] is not None:
                c["positions"][s, :, r] = c["next"][s] + i


def evict_ref(c, keep, recent):
    S, rows, G, _ = c["k"].shape
    for s in range(S):
        n = min(max(int(c["lengths"][s]), 0), rows)
        if n <= keep:
            continue
        for g in range(G):
            w = c["weights"][s, g, :n].astype(np.float64)
            w[np.isnan(w)] = -np.inf
            new = c["positions"][s, g, :n] >= int(c["next"][s]) - recent
            order = sorted(range(n), key=lambda r: (not new[r], 0 if new[r] else -w[r], r))
            stay = set(order[:keep])
            holes = [r for r in range(keep) if r not in stay]
            for t, f in zip(holes, [r for r in range(keep, n) if r in stay]):
                for name in ("k", "v"):
                    c[name][s, t, g] = c[name][s, f, g]
                for name in ("weights", "positions"):
                    c[name][s, g, t] = c[name][s, g, f]


def layer(rng, S, rows, G, D, dtype, ring, bounded):
    f = lambda: rng.integers(0, 1 << 15, (S, rows, G, D)).astype(np.int16)
    return dict(k=f(), v=f(), ring=ring, weights=rng.random((S, G, rows)).astype(np.float32) if bounded else None,
                positions=np.broadcast_to(np.arange(rows, dtype=np.int32), (S, G, rows)).copy() if bounded else None, dtype=dtype)


def to_gpu(torch, c, lengths, nxt):
    from hydra_amd import speculative as sp
    up = lambda a: None if a is None else torch.from_numpy(a.copy()).to("cuda:0")
    return sp.KVCache(up(c["k"]).view(c["dtype"]), up(c["v"]).view(c["dtype"]), lengths, ring=c["ring"], weights=up(c["weights"]),
                      positions=up(c["positions"]), next_position=nxt if c["positions"] is not None else None)


def same(torch, got, want):
    for name in ("k", "v", "weights", "positions"):
        if want[name] is not None:
            g = getattr(got, name)
            g = (g.view(torch.int16) if name in "kv" else g).cpu().numpy()
            assert np.array_equal(g, want[name], equal_nan=name == "weights"), name


@pytest.mark.gpu
@pytest.mark.parametrize("S,N,G,D,dtype,kinds,lengths", [
    # per layer (rows, ring, bounded)
    (1, 1, 1, 64, "float16", [(4, False, False)], [0]),
    (3, 8, 2, 64, "float16", [(40, False, True)] * 3, [0, 31, 36]),        # the last fills up
    (2, 16, 4, 128, "bfloat16", [(10, True, False), (24, True, False)], [1000, 5]),   # rings shorter than a path
    (2, 7, 2, 256, "bfloat16", [(64, False, False), (30, True, False)] * 2, [58, 20]),   # full layers and rings share lengths
    (2, 64, 8, 64, "float16", [(200, False, True)] * 70, [100, 0]),        # more layers than one launch
    (5, 3, 3, 64, "float16", [(9, True, False)], [-2, 0, 9, 2**30, 8]),
])
def test_commit(S, N, G, D, dtype, kinds, lengths):
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    print(f"[gpu] commit S={S} N={N} G={G} D={D} layers={len(kinds)}", flush=True)
    rng = np.random.default_rng(S * N)
    dt = getattr(torch, dtype)
    ctx = Context(0)
    try:
        host = [layer(rng, S, rows, G, D, dt, ring, bounded) for rows, ring, bounded in kinds]
        ln = torch.tensor(lengths, dtype=torch.int32, device="cuda:0")
        nx = ln + 1000
        dev = [to_gpu(torch, c, ln, nx) for c in host]
        dk, dv = (rng.integers(0, 1 << 15, (len(kinds), S, N, G, D)).astype(np.int16) for _ in range(2))
        accepted = rng.integers(0, N + 1, S)
        accepted[0] = N
        path = np.full((S, N), -1, np.int32)
        for s in range(S):
            path[s, :accepted[s]] = np.sort(rng.permutation(N)[:accepted[s]])
        limit = min([rows for rows, ring, _ in kinds if not ring], default=2**31 - 1)
        l0, n0 = np.array(lengths), nx.cpu().numpy()
        for c, a, b in zip(host, dk, dv):
            c["lengths"], c["next"] = l0, n0
            commit_ref(c, path, accepted, a, b, limit)
        torch.cuda.synchronize()
        k, v = (torch.from_numpy(x).to("cuda:0").view(dt) for x in (dk, dv))
        torch.cuda.synchronize()
        sp.cache_commit(ctx, sp.CacheSet(dev), k, v, torch.from_numpy(path).to("cuda:0"),
                        torch.from_numpy(accepted.astype(np.int32)).to("cuda:0"))
        ctx.synchronize()
        torch.cuda.synchronize()
        for a, b in zip(dev, host):
            same(torch, a, b)
        taken = np.minimum(np.minimum(accepted, N), np.maximum(0, limit - np.maximum(l0, 0)))
        assert np.array_equal(ln.cpu().numpy(), np.maximum(l0, 0) + taken)
        bounded = any(b for *_, b in kinds)
        assert np.array_equal(nx.cpu().numpy(), n0 + (taken if bounded else 0))
    finally:
        ctx.close()


@pytest.mark.gpu
def test_commit_of_paths_that_name_no_node():
    """Entries outside the tree write nothing; counts out of range are bounded; the draft may be strided."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    rng = np.random.default_rng(3)
    S, N, G, D = 3, 4, 2, 64
    ctx = Context(0)
    try:
        host = layer(rng, S, 20, G, D, torch.float16, False, True)
        ln, nx = (torch.tensor([3, 0, 9], dtype=torch.int32, device="cuda:0") for _ in range(2))
        dev = to_gpu(torch, host, ln, nx)
        path = np.array([[0, -1, 4, 2], [2**31 - 1, -2**31, 1, 1], [0, 1, 2, 3]], np.int32)
        acc = np.array([4, 100, -3], np.int32)
        wide = rng.integers(0, 1 << 15, (S, N, 3 * G, D)).astype(np.int16)
        host["lengths"], host["next"] = np.array([3, 0, 9]), np.array([3, 0, 9])
        commit_ref(host, path, acc, wide[:, :, G:2 * G], wide[:, :, 2 * G:], 20)
        w = torch.from_numpy(wide).to("cuda:0").view(torch.float16)
        p, a = torch.from_numpy(path).to("cuda:0"), torch.from_numpy(acc).to("cuda:0")
        torch.cuda.synchronize()
        sp.cache_commit(ctx, sp.CacheSet([dev]), [w[:, :, G:2 * G]], [w[:, :, 2 * G:]], p, a)
        ctx.synchronize()
        same(torch, dev, host)
        assert ln.tolist() == [7, 4, 9] and nx.tolist() == [7, 4, 9]
    finally:
        ctx.close()


def weights_of(rng, kind, shape):
    if kind == "ties":
        return rng.integers(0, 4, shape).astype(np.float32)
    if kind == "odd":
        return rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0, 1e-40, -1.0, 3e38], np.float32), shape)
    if kind == "close":       # differ in the last bits only
        return (np.float32(1.0).view(np.int32) + rng.integers(0, 50, shape)).astype(np.int32).view(np.float32)
    return (rng.random(shape) ** -0.7).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("S,G,D,rows,lengths,keep,recent,kind,layers", [
    (1, 1, 64, 2, [2], 1, 0, "power", 1),
    (1, 1, 64, 2, [2], 1, 1, "power", 1),
    (4, 2, 64, 100, [100, 64, 65, 3], 64, 8, "power", 2),           # at, above and below the budget
    (3, 4, 128, 300, [300, 299, 1], 1, 0, "ties", 1),
    (2, 2, 256, 300, [300, 250], 249, 249, "ties", 1),              # all that stays is recent
    (2, 3, 64, 1500, [1500, 1025], 700, 16, "odd", 2),
    (2, 2, 64, 2100, [2100, 2047], 1024, 0, "close", 1),
    (1, 8, 64, 4112, [4112], 4096, 512, "power", 40),               # more layers than one launch
    (1, 2, 64, 70000, [69999], 40000, 100, "power", 1),
    (1, 1, 128, 33000, [33000], 5, 5, "ties", 1),
])
def test_evict(S, G, D, rows, lengths, keep, recent, kind, layers):
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    print(f"[gpu] evict S={S} G={G} D={D} rows={rows} keep={keep} {kind} layers={layers}", flush=True)
    rng = np.random.default_rng(rows + keep)
    ctx = Context(0)
    try:
        host = [layer(rng, S, rows, G, D, torch.float16, False, True) for _ in range(layers)]
        for c in host:
            c["weights"] = weights_of(rng, kind, (S, G, rows))
            # Rows in no order of position, as earlier evictions leave them.
            for s in range(S):
                for g in range(G):
                    c["positions"][s, g, :lengths[s]] = rng.permutation(lengths[s]) + 50
            c["lengths"], c["next"] = np.array(lengths), np.array(lengths) + 50
        ln = torch.tensor(lengths, dtype=torch.int32, device="cuda:0")
        nx = ln + 50
        dev = [to_gpu(torch, c, ln, nx) for c in host]
        for c in host:
            evict_ref(c, keep, recent)
        group = sp.CacheSet(dev)
        torch.cuda.synchronize()
        sp.cache_evict(ctx, group, keep, recent)
        sp.cache_evict(ctx, group, keep, recent)      # nothing is left to evict
        ctx.synchronize()
        for a, b in zip(dev, host):
            same(torch, a, b)
        assert ln.tolist() == [min(n, keep) for n in lengths]
        assert nx.tolist() == [n + 50 for n in lengths]
    finally:
        ctx.close()


@pytest.mark.gpu
def test_recorded_cycles():
    """A commit and an eviction as one graph, replayed: each replay continues from where the last one ended."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    rng = np.random.default_rng(8)
    S, N, G, D, keep, recent, rows = 2, 6, 2, 64, 100, 10, 110
    ctx = Context(0)
    try:
        host = [layer(rng, S, rows, G, D, torch.float16, False, True) for _ in range(3)]
        l0 = np.array([98, 40])
        ln, nx = (torch.tensor(l0, dtype=torch.int32, device="cuda:0") for _ in range(2))
        for c in host:
            c["lengths"], c["next"] = l0, l0.copy()
        dev = sp.CacheSet([to_gpu(torch, c, ln, nx) for c in host])
        dk, dv = (torch.zeros((3, S, N, G, D), dtype=torch.float16, device="cuda:0") for _ in range(2))
        path, acc = torch.zeros((S, N), dtype=torch.int32, device="cuda:0"), torch.zeros(S, dtype=torch.int32, device="cuda:0")
        sp.reserve(ctx, dev.caches[0], nodes=N, layers=3)
        torch.cuda.synchronize()

        def both():
            sp.cache_commit(ctx, dev, dk, dv, path, acc)
            sp.cache_evict(ctx, dev, keep, recent)
        graph = ctx.capture(both)
        lengths, nxt = l0.copy(), l0.copy()
        for rep in range(12):
            a, b = (rng.integers(0, 1 << 15, (3, S, N, G, D)).astype(np.int16) for _ in range(2))
            n = rng.integers(1, N + 1, S)
            p = np.full((S, N), -1, np.int32)
            for s in range(S):
                p[s, :n[s]] = np.sort(rng.permutation(N)[:n[s]])
            dk.copy_(torch.from_numpy(a).view(torch.float16))
            dv.copy_(torch.from_numpy(b).view(torch.float16))
            path.copy_(torch.from_numpy(p))
            acc.copy_(torch.from_numpy(n.astype(np.int32)))
            torch.cuda.synchronize()
            graph.launch()
            ctx.synchronize()
            for c, x, y in zip(host, a, b):
                c["lengths"], c["next"] = lengths, nxt
                commit_ref(c, p, n, x, y, rows)
            lengths, nxt = lengths + n, nxt + n
            for c in host:
                c["lengths"], c["next"] = lengths, nxt
                evict_ref(c, keep, recent)
            lengths = np.minimum(lengths, keep)
            for x, y in zip(dev.caches, host):
                same(torch, x, y)
            assert ln.tolist() == lengths.tolist() and nx.tolist() == nxt.tolist()
        graph.close()
    finally:
        ctx.close()


@pytest.mark.gpu
def test_commits_one_after_the_other():
    """Many sequences, layers with two sets of lengths, four commits in a row: eager, and recorded by a context that has
    run nothing before."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    rng = np.random.default_rng(12)
    S, N, G, D, rows, L = 150, 20, 1, 64, 60, 5
    for captured in (False, True):
        print(f"[gpu] commits in a row, captured={captured}", flush=True)
        ctx = Context(0)
        try:
            host = [layer(rng, S, rows, G, D, torch.float16, False, i % 2 == 0) for i in range(L)]
            l0 = [rng.integers(0, 30, S), rng.integers(0, 30, S)]
            ln = [torch.tensor(x, dtype=torch.int32, device="cuda:0") for x in l0]
            nx = ln[0] + 7
            n0 = l0[0] + 7
            for i, c in enumerate(host):
                c["lengths"], c["next"] = l0[i % 2], n0
            dev = [to_gpu(torch, c, ln[i % 2], nx) for i, c in enumerate(host)]
            dk, dv = (rng.integers(0, 1 << 15, (L, S, N, G, D)).astype(np.int16) for _ in range(2))
            k, v = (torch.from_numpy(x).to("cuda:0").view(torch.float16) for x in (dk, dv))
            path = np.tile(np.arange(N, dtype=np.int32), (S, 1))
            acc = rng.integers(0, N + 1, S).astype(np.int32)
            p, a = torch.from_numpy(path).to("cuda:0"), torch.from_numpy(acc).to("cuda:0")
            caches = sp.CacheSet(dev)
            torch.cuda.synchronize()
            call = lambda: sp.cache_commit(ctx, caches, k, v, p, a)
            graph = ctx.capture(call) if captured else None
            for rep in range(4):
                graph.launch() if captured and rep != 2 else call()
                for i, c in enumerate(host):
                    c["lengths"], c["next"] = l0[i % 2], n0
                    commit_ref(c, path, acc, dk[i], dv[i], rows)
                taken = [np.minimum(acc, rows - x) for x in l0]
                l0, n0 = [x + t for x, t in zip(l0, taken)], n0 + taken[0]
            ctx.synchronize()
            for x, y in zip(dev, host):
                same(torch, x, y)
            assert [x.tolist() for x in ln] == [x.tolist() for x in l0] and nx.tolist() == n0.tolist()
            if captured:
                graph.close()
        finally:
            ctx.close()


# ---- refusals (no GPU) ------------------------------------------------------------------------------

def _call(fn, desc=None, caches=None, count=2, **kw):
    from hydra_amd import _lib
    L = _lib.lib()
    d = dict(sequences=1, nodes=4, q_heads=8, kv_heads=2, head_dim=64, type=1, cache_type=1, window=0, max_length=0, sm_scale=0.1,
             q_stride=0, kv_stride=0)
    d.update(desc or {})
    base = dict(sequence_stride=0, rows=16, ring=0, lengths=64, next_position=128)
    layers = [dict(base, k=4096 << 2 * i, v=8192 << 2 * i, weights=1024 + 16 * i, positions=2048 + 16 * i) for i in range(9)]
    for i, c in (caches or {}).items():
        layers[i].update(c)
    arr = (_lib.KVCacheC * 9)(*[_lib.KVCacheC(**c) for c in layers])
    ctx = C.create_string_buffer(4096)      # zeros: never used, the checks come first
    dc = _lib.TreeDescC(**d)
    if fn == "evict":
        a = dict(keep=8, recent=2)
        a.update(kw)
        return L.hh_cache_evict(ctx, C.byref(dc), arr, count, a["keep"], a["recent"])
    p = (C.c_void_p * 9)(kw.get("dk", 16), *[16] * 8)
    return L.hh_cache_commit(ctx, C.byref(dc), arr, count, p, kw.get("dv", p), kw.get("path", 16), 16)


@pytest.mark.parametrize("kw,code", [
    (dict(keep=0), -1), (dict(keep=17), -1), (dict(recent=9), -1), (dict(recent=-1), -1), (dict(count=0), -1), (dict(count=257), -1),
    (dict(caches={1: dict(ring=1, weights=None, positions=None, next_position=None)}), -1), (dict(caches={1: dict(weights=None)}), -1),
    (dict(caches={0: dict(positions=None, next_position=None)}), -1), (dict(caches={1: dict(next_position=None)}), -1),
    (dict(caches={1: dict(next_position=256)}), -1), (dict(caches={1: dict(lengths=256)}), -1), (dict(caches={1: dict(k=4096)}), -1),
    (dict(caches={1: dict(rows=4)}), -1), (dict(desc=dict(head_dim=32)), -6), (dict(desc=dict(sequences=0)), -1),
    (dict(caches={1: dict(weights=1024)}), -1), (dict(caches={1: dict(positions=2048)}), -1),
    (dict(desc=dict(sequences=4096, kv_heads=64), count=9), -1),
])
def test_evict_refusals(kw, code):
    assert _call("evict", **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(desc=dict(nodes=0)), -1), (dict(desc=dict(cache_type=0)), -1), (dict(desc=dict(kv_stride=64)), -6), (dict(dk=None), -1),
    (dict(dk=8), -2), (dict(dv=None), -1), (dict(path=None), -1), (dict(caches={0: dict(v=8194)}), -2), (dict(caches={1: dict(v=4096)}), -1),
    (dict(count=0), -1), (dict(caches={0: dict(v=4096)}), -1), (dict(caches={0: dict(next_position=64)}), -1),
    (dict(caches={1: dict(lengths=128, next_position=256)}), -1), (dict(caches={1: dict(lengths=256, next_position=64)}), -1),
    (dict(caches={1: dict(lengths=128, weights=None, positions=None, next_position=None)}), -1),
])
def test_commit_refusals(kw, code):
    assert _call("commit", **kw) == code


def test_reserve_refusals():
    from hydra_amd import _lib
    L, ctx = _lib.lib(), C.create_string_buffer(4096)
    d = _lib.TreeDescC(1, 4, 8, 2, 64, 1, 1, 0, 0, 0.1, 0, 0)
    assert L.hh_draft_reserve(ctx, C.byref(d), None, 3, None) == -1      # layers of no cache
    assert L.hh_draft_reserve(ctx, None, None, -1, None) == -1
    v = _lib.VerifyDescC(1, 4, 0, 0, 1, 0, 1.0, 0, 0)
    assert L.hh_draft_reserve(ctx, None, None, 0, C.byref(v)) == -1
