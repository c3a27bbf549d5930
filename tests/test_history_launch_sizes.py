"""Attention over histories whose launches were sized for other lengths (max_length), where a kv head has many rows: chunks grow past the
planned ones, and the join has to agree. The same tolerances as at the planned lengths."""
import pytest

from test_history_attention import call, check, make

pytestmark = pytest.mark.gpu

CASES = [
    # S, N, H, G, D, rows, lengths, counts, window, first, ring, pinned, shared, sinks
    (1, 33, 8, 2, 64, 5000, [4900], None, 0, 0, False, 0, None, True),
    (2, 40, 8, 2, 128, 4000, [3900, 3], [40, 11], 0, 0, False, 0, None, False),
    (1, 50, 4, 1, 256, 3000, [2900], None, 0, 0, False, 0, None, True),
    (1, 70, 8, 2, 64, 5000, [4800], None, 3000, 70, False, 0, None, True),        # a window and first tokens
    (1, 45, 4, 1, 128, 2100, [9000], None, 2000, 5, True, 5, None, False),        # a ring
    (3, 40, 8, 2, 64, 2500, [2400, 0, 777], [40, 0, 40], 0, 0, False, 0, 1900, True),     # behind a prefix
    (2, 1, 8, 2, 64, 4000, [3990, 20], None, 0, 0, False, 0, 3000, False),        # few rows behind one
    (20, 2, 8, 2, 128, 600, [590 - 20 * i for i in range(20)], None, 0, 0, False, 0, 900, False),
]


@pytest.mark.parametrize("kind,fmt", [("bf16", "mxfp8"), ("f16", "f16"), ("f32", "mxfp4")])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
@pytest.mark.parametrize("max_length", [1, 300, 700, 100000])
def test_launches_sized_for_other_lengths(kind, fmt, case, max_length):
    import torch
    from hydra_amd.layer import Context
    S, N, H, G, D, rows, lengths, counts, window, first, ring, pinned, shared, sinks = case
    print(f"[gpu] launch for {max_length}: {kind} {fmt} {case}", flush=True)
    t = make(torch, S, N, H, G, D, kind, fmt, rows, lengths, counts, sinks, shared, seed=11)
    kw = dict(window=window, first=first, ring=ring, pinned=pinned)
    check(torch, t, *call(torch, Context(0), t, max_length=max_length, **kw), **kw)


@pytest.mark.parametrize("shared", [None, 1900])
def test_graphs_sized_for_short_histories(shared):
    """Recorded for 300 positions and replayed as the histories grow past that: the eager call's bits of the same size."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    from test_history_attention import histories
    ctx = Context(0)
    t = make(torch, 2, 40, 8, 2, 64, "bf16", "mxfp8", 3000, [0, 0], shared=shared, seed=12)
    h, p = histories(torch, t)
    q, c = t["q"].cuda(), t["counts"].cuda()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device="cuda:0")
    torch.cuda.synchronize()
    hi.history_attention_into(ctx, h, q, c, out, lse=lse, prefix=p, max_length=300)      # sizes the workspace
    ctx.synchronize()
    graph = ctx.capture(lambda: hi.history_attention_into(ctx, h, q, c, out, lse=lse, prefix=p, max_length=300))
    for lengths in ([10, 250], [1000, 2959], [2900, 0]):
        t["lengths"] = torch.tensor(lengths, dtype=torch.int32)
        h.lengths.copy_(t["lengths"])
        out.fill_(7.0)
        lse.fill_(7.0)
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
        check(torch, t, out, lse)
        want, wl = call(torch, Context(0), t, max_length=300)
        assert torch.equal(out, want) and torch.equal(lse, wl)
    graph.close()
