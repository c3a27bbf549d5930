"""Attention over histories where its launches change: every way that rows and keys are cut, reservations and recorded graphs,
logits far from zero, rows past 4 GB."""
import numpy as np
import pytest

import history_ref as R
from test_history_attention import TOL, call, check, histories, make, torch_type

pytestmark = pytest.mark.gpu

CASES = [
    # S, N, H, G, D, type, format, rows, lengths, counts, window, first, ring, pinned, shared, sinks
    (1, 1, 8, 2, 64, "bf16", "mxfp8", 9000, [8990], None, 0, 0, False, 0, None, True),       # 16 rows, chunks
    (2, 4, 12, 2, 64, "f32", "mxfp4", 5000, [4990, 100], None, 0, 0, False, 0, None, False),  # 24 rows, chunks
    (2, 5, 8, 2, 128, "f16", "mxfp8", 5000, [4990, 700], [5, 2], 0, 0, False, 0, None, True),
    (1, 2, 32, 2, 256, "f32", "mxfp8", 3000, [2990], None, 0, 0, False, 0, None, False),
    (1, 2, 32, 2, 256, "bf16", "bf16", 3000, [2990], None, 0, 0, False, 0, None, False),
    (1, 33, 8, 2, 64, "bf16", "mxfp4", 5000, [4900], None, 0, 0, False, 0, None, True),      # 128 rows, chunks
    (1, 33, 8, 2, 256, "f32", "mxfp4", 3000, [2900], None, 0, 0, False, 0, None, True),
    (1, 40, 8, 1, 128, "f32", "mxfp8", 3000, [2900], None, 0, 0, False, 0, None, True),
    (2, 1, 8, 2, 64, "f32", "mxfp8", 500, [490, 3], None, 0, 0, False, 0, 3000, True),       # prefix: 16 rows, both passes cut
    (2, 1, 8, 2, 64, "bf16", "mxfp8", 5000, [4990, 3], None, 0, 0, False, 0, 3000, False),
    (4, 1, 16, 2, 128, "f16", "mxfp4", 700, [690, 3, 5, 200], [1, 0, 1, 1], 0, 0, False, 0, 2000, True),   # 128 rows, 16 of their own
    (2, 40, 8, 2, 64, "f16", "f16", 500, [300, 3], [40, 17], 0, 0, False, 0, 1500, True),     # 128 and 128
    (2, 20, 8, 2, 256, "f32", "f16", 300, [200, 3], None, 0, 0, False, 0, 700, False),
    (1, 700, 2, 2, 64, "bf16", "mxfp8", 800, [90], None, 0, 0, False, 0, None, False),        # one head a group: a block of 128 tokens
    (1, 600, 2, 2, 64, "f32", "mxfp8", 900, [250], None, 200, 3, False, 0, None, True),
    (2, 300, 4, 1, 128, "bf16", "mxfp8", 600, [1000, 40], [300, 211], 250, 4, True, 4, None, False),
    (3, 12, 16, 2, 64, "f16", "mxfp8", 90, [1000, 40, 0], None, 60, 8, True, 9, None, True),  # 96 rows over rings
    (1, 16, 3, 1, 64, "f32", "mxfp8", 5000, [4900], None, 4000, 70, False, 0, None, True),    # first tokens over a tile's end
    (2, 2, 8, 1, 64, "bf16", "mxfp4", 300, [280, 64], None, 5, 63, False, 0, None, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_cuts(case):
    import torch
    from hydra_amd.layer import Context
    S, N, H, G, D, kind, fmt, rows, lengths, counts, window, first, ring, pinned, shared, sinks = case
    print(f"[gpu] history cut {case}", flush=True)
    t = make(torch, S, N, H, G, D, kind, fmt, rows, lengths, counts, sinks, shared, seed=5)
    kw = dict(window=window, first=first, ring=ring, pinned=pinned)
    check(torch, t, *call(torch, Context(0), t, **kw), **kw)


@pytest.mark.parametrize("S,N,H,G,D,kind,fmt,rows,lengths,shared,most", [
    (1, 1, 64, 8, 64, "f32", "mxfp8", 9000, [8990], None, dict(S=3, N=9, rows=12000)),
    (2, 7, 16, 2, 128, "bf16", "mxfp4", 3000, [2990, 5], None, dict(S=2, N=8, rows=3000)),
    (3, 1, 8, 1, 64, "f16", "f16", 400, [390, 0, 77], 1999, dict(S=40, N=2, rows=500, shared=6000)),
    (1, 60, 8, 2, 256, "bf16", "mxfp8", 1500, [1400], None, dict(S=1, N=100, rows=1600)),
])
def test_reservations_cover_smaller_calls(S, N, H, G, D, kind, fmt, rows, lengths, shared, most):
    """A context that has reserved, and run nothing, records calls up to those sizes; replays give the eager bits."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    print(f"[gpu] history reserve S={S} N={N} of {most}", flush=True)
    t = make(torch, S, N, H, G, D, kind, fmt, rows, lengths, sinks=True, shared=shared, seed=6)
    eager, ctx = Context(0), Context(0)
    want, wl = call(torch, eager, t)
    big = hi.History.empty(most["S"], G, most["rows"], D, format=fmt)
    prefix = None if shared is None else hi.History.empty(1, G, most["shared"], D, format=fmt)
    hi.history_reserve(ctx, big, most["N"], H, torch_type(torch, kind), prefix=prefix)
    h, p = histories(torch, t)
    q, c, s = t["q"].cuda(), t["counts"].cuda(), t["sinks"].cuda()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device="cuda:0")
    torch.cuda.synchronize()
    graph = ctx.capture(lambda: hi.history_attention_into(ctx, h, q, c, out, lse=lse, sinks=s, prefix=p))
    for _ in range(3):
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wl)
    graph.close()


def test_workspaces_do_not_grow_under_a_graph():
    import torch
    from hydra_amd import history as hi
    from hydra_amd._lib import HydraHIPError
    from hydra_amd.layer import Context
    ctx = Context(0)
    t = make(torch, 1, 1, 8, 2, 64, "f32", "mxfp8", 3000, [2990])
    want, _ = call(torch, ctx, t)            # sizes the workspace
    h, _ = histories(torch, t)
    q, c = t["q"].cuda(), t["counts"].cuda()
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    graph = ctx.capture(lambda: hi.history_attention_into(ctx, h, q, c, out))
    larger = make(torch, 3, 2, 8, 2, 64, "f32", "mxfp8", 9000, [8990, 8000, 10])
    hb, _ = histories(torch, larger)
    with pytest.raises(HydraHIPError) as e:
        hi.history_reserve(ctx, hb, 2, 8, torch.float32)
    assert e.value.code == -1 and "graph" in str(e.value)
    with pytest.raises(HydraHIPError):
        call(torch, ctx, larger)
    hi.history_reserve(ctx, h, 1, 8, torch.float32)      # what it has covers just this
    graph.launch()
    ctx.synchronize()
    assert torch.equal(out, want)
    graph.close()
    check(torch, larger, *call(torch, ctx, larger))      # and grows again behind the graph


def test_two_graphs_of_one_context_and_lengths_that_move():
    """Both use the context's workspace; the stream keeps them apart. Lengths are read at every replay."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    a = make(torch, 2, 1, 8, 2, 64, "f32", "mxfp8", 4000, [3000, 10], seed=1)
    b = make(torch, 1, 3, 8, 2, 64, "f32", "mxfp8", 4000, [2000], seed=2, shared=700)
    for t in (a, b):
        call(torch, ctx, t)
    runs = []
    for t in (a, b):
        h, p = histories(torch, t)
        q, c = t["q"].cuda(), t["counts"].cuda()
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device="cuda:0")
        torch.cuda.synchronize()
        runs.append((t, h, out, lse, ctx.capture(lambda: hi.history_attention_into(ctx, h, q, c, out, lse=lse, prefix=p))))
    for step in range(3):
        for t, h, out, lse, _ in runs:
            t["lengths"] = (t["lengths"] * 0 + torch.tensor([3990 - 1500 * step, 5 + 997 * step])[:len(t["lengths"])]).int()
            h.lengths.copy_(t["lengths"])
            out.fill_(7.0)
            lse.fill_(7.0)
        torch.cuda.synchronize()
        for *_, graph in runs:
            graph.launch()
        ctx.synchronize()
        for t, h, out, lse, _ in runs:
            check(torch, t, out, lse)
    for *_, graph in runs:
        graph.close()


@pytest.mark.parametrize("kind,fmt", [("f32", "mxfp8"), ("bf16", "mxfp4"), ("f16", "f16")])
@pytest.mark.parametrize("N", [1, 60])
@pytest.mark.parametrize("scale", [2.0 ** 18, -2.0 ** 22, 2.0 ** 60])
def test_logits_far_from_zero(kind, fmt, N, scale):
    """Whole-number products, so that logits are equal or far apart: the largest share the probability evenly. The value's rounding and the
    quotient's, and of 16-bit outputs their own."""
    import torch
    from hydra_amd.layer import Context
    t = make(torch, 1, N, 8, 2, 64, kind, fmt, 300, [200], seed=8)
    g = np.random.default_rng(9)
    t["q"] = torch.from_numpy(g.integers(-1, 2, t["q"].shape)).to(t["q"].dtype)
    t["kn"] = g.integers(-1, 2, t["kn"].shape).astype(np.float64)
    if fmt == "f16":
        t["k"] = torch.from_numpy(t["kn"]).to(torch.float16)
    else:
        from test_history_attention import fast_encode
        x = t["kn"].copy()
        x[..., ::32] = np.where(x[..., ::32] == 0, 1, x[..., ::32])      # no group of zeros
        t["kn"] = x
        codes, scales, values = fast_encode(x, fmt)
        assert np.array_equal(values, x)
        t["k"], t["ks"] = torch.from_numpy(codes), torch.from_numpy(scales)
    out, _ = call(torch, Context(0), t, scale=scale)
    ro, _ = R.attention(t["q"].double().numpy(), t["kn"], t["vn"], [200], [N], None, scale)
    for at, want in ro.items():
        assert np.linalg.norm(out[at].double().cpu().numpy() - want) <= TOL[kind] * np.linalg.norm(want), at


@pytest.mark.parametrize("fmt,N", [("mxfp8", 1), ("mxfp8", 40), ("bf16", 1)])
def test_rows_past_4_gb(fmt, N):
    """Written, read and attended at the end of a history of more than 2^32 bytes."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    D = 256
    rows = (1 << 32) // (D if fmt == "mxfp8" else 2 * D) + 4000
    print(f"[gpu] history of {rows} rows", flush=True)
    ctx = Context(0)
    h = hi.History.empty(1, 1, rows, D, format=fmt, lengths=torch.tensor([rows - 300], dtype=torch.int32, device="cuda:0"))
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn((1, 300, 1, D), generator=g).bfloat16() for _ in range(2))
    c = torch.tensor([300], dtype=torch.int32, device="cuda:0")
    ko, vo = (torch.zeros((1, 300, 1, D), device="cuda:0") for _ in range(2))
    q = torch.randn((1, N, 4, D), generator=g).bfloat16()
    out = torch.zeros((1, N, 4, D), dtype=torch.bfloat16, device="cuda:0")
    kd, vd, qd = k.cuda(), v.cuda(), q.cuda()
    torch.cuda.synchronize()
    hi.history_write(ctx, h, kd, vd, c)
    hi.history_read_into(ctx, h, h.lengths, c, ko, vo)
    h2 = hi.History(h.k, h.v, torch.tensor([rows - N], dtype=torch.int32, device="cuda:0"), h.k_scales, h.v_scales)
    n = torch.tensor([N], dtype=torch.int32, device="cuda:0")
    torch.cuda.synchronize()
    hi.history_attention_into(ctx, h2, qd, n, out, window=200)
    ctx.synchronize()
    if fmt == "bf16":
        assert torch.equal(ko.cpu(), k.float()) and torch.equal(vo.cpu(), v.float())
    else:
        assert np.array_equal(ko.double().cpu().numpy(), R.encode(k.double().numpy(), fmt)[2])
    kn, vn = (x.double().cpu().numpy().transpose(0, 2, 1, 3) for x in (ko, vo))
    # The last 300 positions as a history of their own.
    ro, _ = R.attention(q.double().numpy(), kn, vn, [300 - N], [N], None, D ** -0.5, window=200)
    for at, want in ro.items():
        assert np.linalg.norm(out[at].double().cpu().numpy() - want) <= TOL["bf16"] * np.linalg.norm(want), at


def test_another_context_and_torch_streams_beside_it():
    """Two contexts at once, and torch's own work on the default stream between."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    a, b = Context(0), Context(0)
    t = make(torch, 2, 2, 8, 2, 64, "bf16", "mxfp8", 4000, [3990, 1000], seed=4)
    want, wl = call(torch, a, t)
    h, _ = histories(torch, t)
    q, c = t["q"].cuda(), t["counts"].cuda()
    outs = [torch.zeros_like(q) for _ in range(8)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        hi.history_attention_into((a, b)[i % 2], h, q, c, o)
        torch.ones((64, 64), device="cuda:0") @ torch.ones((64, 64), device="cuda:0")
    a.synchronize()
    b.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("kind,fmt", [("bf16", "mxfp8"), ("f16", "f16"), ("f32", "mxfp4")])
@pytest.mark.parametrize("S,N,rows,shared", [(2, 3, 900, None), (2, 50, 300, None), (3, 40, 80, 500)])
def test_outputs_in_place_strided_queries_and_no_lse(kind, fmt, S, N, rows, shared):
    """The same bits as into memory of their own with lse, whatever few or many rows, chunks or a prefix do with them."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    H, G, D = 8, 2, 64
    t = make(torch, S, N, H, G, D, kind, fmt, rows, [rows - N, 5, 0][:S], sinks=True, shared=shared, seed=3)
    want, _ = call(torch, ctx, t)
    h, p = histories(torch, t)
    q, c, sinks = t["q"].cuda(), t["counts"].cuda(), t["sinks"].cuda()
    wide = torch.full((S, N, (H + 2 * G) * D), float("nan"), dtype=q.dtype, device="cuda:0")
    wide[..., :H * D] = q.reshape(S, N, -1)
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    hi.history_attention_into(ctx, h, wide[..., :H * D].unflatten(-1, (H, D)), c, out, sinks=sinks, prefix=p)
    hi.history_attention_into(ctx, h, q, c, q, sinks=sinks, prefix=p)
    ctx.synchronize()
    assert torch.equal(out, want) and torch.equal(q, want)


@pytest.mark.parametrize("kind,fmt", [("bf16", "mxfp8"), ("f16", "f16"), ("f32", "mxfp8")])
@pytest.mark.parametrize("N,shared", [(2, None), (40, None), (40, 300)])
def test_a_query_of_nan_or_infinities_stays_alone(kind, fmt, N, shared):
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    t = make(torch, 2, N, 8, 2, 64, kind, fmt, 400, [300, 7], shared=shared, seed=4)
    want, wl = call(torch, ctx, t)
    t["q"][0, 1, 3, 5] = float("nan")
    t["q"][1, 0, 2] = float("inf")
    out, lse = call(torch, ctx, t)
    touched = torch.zeros(out.shape[:3], dtype=torch.bool, device="cuda:0")
    touched[0, 1, 3] = touched[1, 0, 2] = True
    assert torch.equal(out[~touched], want[~touched]) and torch.equal(lse[~touched], wl[~touched])
    assert torch.isnan(out[touched]).all()
