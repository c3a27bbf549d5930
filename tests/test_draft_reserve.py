"""hh_draft_reserve: a context that has reserved for some sizes records every call up to them, those among them that need more
workspace than the largest (fewer keys or nodes may be cut into more chunks)."""
import pytest

from test_draft_verify import call as verify_call
from test_draft_verify import inputs
from test_tree_attention import call as tree_call
from test_tree_attention import make


def attention(torch, sp, ctx, t, ring, window, max_length, reserve):
    """The attention of `t` as a recorded call of a context that has reserved, and run nothing."""
    d = {k: None if x is None else x.to("cuda:0") for k, x in t.items()}
    cache = sp.KVCache(d["k"], d["v"], d["lengths"], ring=ring)
    out = torch.full_like(d["q"], 7.0)
    reserve(cache)
    torch.cuda.synchronize()
    graph = ctx.capture(lambda: sp.attention_tree_into(ctx, cache, d["q"], d["dk"], d["dv"], d["parents"], d["counts"], out,
                                                       sinks=d["sinks"], window=window, max_length=max_length))
    for _ in range(2):
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
    graph.close()
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("S,nodes,N,H,G,D,kind,rows,lengths,window,max_length", [
    (1, 8, 8, 64, 8, 64, "f32", 4160, [9000], 4096, 0),             # a window: chunks of fewer keys
    (1, 17, 16, 64, 8, 64, "f16", 5000, [5000], 0, 0),              # fewer nodes: one block of rows
    (1, 40, 3, 16, 1, 128, "bf16", 9000, [8999], 0, 0),
    (3, 9, 9, 16, 2, 64, "f32", 20000, [20000, 700, 5000], 0, 8000),    # launches sized for shorter histories
    (2, 25, 1, 8, 4, 256, "bf16", 3000, [3000, 2999], 1500, 0),
])
def test_attention_up_to_the_reserved_sizes(S, nodes, N, H, G, D, kind, rows, lengths, window, max_length):
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    print(f"[gpu] tree reserve S={S} N={N} of {nodes} rows={rows} w={window}", flush=True)
    t = make(torch, S, N, H, G, D, kind, rows, lengths, seed=N)
    eager, ctx = Context(0), Context(0)
    try:
        want, _ = tree_call(torch, eager, t, bool(window), window, max_length=max_length)
        got = attention(torch, sp, ctx, t, bool(window), window, max_length,
                        lambda cache: sp.reserve(ctx, cache, nodes=nodes, q_heads=H, q_dtype=t["q"].dtype))
        assert torch.equal(got, want)
    finally:
        eager.close()
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("most,sizes", [
    ((16, 1, 131072), [(16, 1, 131000), (1, 1, 131072), (16, 1, 131072)]),       # chunks of 4096, then of 1024
    ((2, 21, 50000), [(2, 20, 50000), (1, 21, 50000), (2, 21, 49000)]),
    ((4, 5, 1000), [(4, 5, 999), (1, 1, 7)]),
])
def test_verification_up_to_the_reserved_sizes(most, sizes):
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    eager, ctx = Context(0), Context(0)
    try:
        sp.reserve(ctx, verify=most)
        hold = ctx.capture(lambda: None)          # no workspace may grow from here on
        for S, N, V in sizes:
            print(f"[gpu] verify reserve {S} {N} {V} of {most}", flush=True)
            t = inputs(torch, S, N, V, "f32", "iid", 2, V)
            assert all(torch.equal(a, b) for a, b in zip(verify_call(torch, ctx, t, "iid"), verify_call(torch, eager, t, "iid")))
        hold.close()
    finally:
        eager.close()
        ctx.close()


@pytest.mark.gpu
def test_reserving_again_while_a_graph_lives():
    """What eager calls have grown the workspace to is enough for the same calls, also where it may not grow any more."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd._lib import HydraHIPError
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        t, v = make(torch, 1, 8, 64, 8, 64, "f32", 4160, [4160], seed=1), inputs(torch, 2, 5, 900, "f32", "iid", 2, 3)
        tree_call(torch, ctx, t)
        verify_call(torch, ctx, v, "iid")
        hold = ctx.capture(lambda: None)
        cache = sp.KVCache(t["k"].to("cuda:0"), t["v"].to("cuda:0"), t["lengths"].to("cuda:0"))
        sp.reserve(ctx, cache, nodes=8, q_heads=64, q_dtype=torch.float32)
        sp.reserve(ctx, verify=(2, 5, 900))
        with pytest.raises(HydraHIPError):
            sp.reserve(ctx, cache, nodes=64, q_heads=64, q_dtype=torch.float32)
        hold.close()
        sp.reserve(ctx, cache, nodes=64, q_heads=64, q_dtype=torch.float32)
    finally:
        ctx.close()
