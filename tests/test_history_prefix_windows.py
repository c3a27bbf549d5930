"""Streams behind a shared document in a model that mixes layers: those that see everything take the document as a prefix, those with a window
hold its last rows in rings of their own, whose lengths count it. Both the same as histories that hold all of it."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind,fmt", [("float32", "mxfp8"), ("bfloat16", "bf16"), ("float16", "f16")])
def test_rings_and_prefixes_behind_one_document(kind, fmt, captured):
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    S, G, H, D, P, T, N, window, first = 3, 2, 8, 64, 61, 9, 3, 24, 2
    g = torch.Generator().manual_seed(4)
    dtype = getattr(torch, kind)
    make = lambda *shape: torch.randn(shape, generator=g).to(dtype).to("cuda:0")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda:0")
    doc_k, doc_v = make(1, P, G, D), make(1, P, G, D)
    many_k, many_v = (x.expand(S, P, G, D).contiguous() for x in (doc_k, doc_v))
    k, v, q = make(S, N, G, D), make(S, N, G, D), make(S, N, H, D)
    ctx = Context(0)
    all_p, counts, one = i32(*[P] * S), i32(N, 2, 0), i32(P)
    prefix = hi.History.empty(1, G, P, D, format=fmt)
    own = hi.History.empty(S, G, T, D, format=fmt)                                              # lengths without the document
    ring = hi.History.empty(S, G, first + window + N - 1, D, format=fmt, ring=True, pinned=first)   # lengths with it
    whole = hi.History.empty(S, G, P + T, D, format=fmt)
    outs = [torch.zeros_like(q) for _ in range(4)]
    torch.cuda.synchronize()
    hi.history_write(ctx, prefix, doc_k, doc_v, one)
    hi.history_advance(ctx, prefix, one, P)
    for h in (ring, whole):
        hi.history_write(ctx, h, many_k, many_v, all_p)
        hi.history_advance(ctx, h, all_p, P)
    for h, kw in ((own, dict(prefix=prefix)), (ring, dict(window=window, first=first)), (whole, {}), (whole, dict(window=window, first=first))):
        hi.history_reserve(ctx, h, N, H, dtype, **kw)
    ctx.synchronize()

    def enqueue():
        for h in (own, ring, whole):
            hi.history_write(ctx, h, k, v, counts)
        hi.history_attention_into(ctx, own, q, counts, outs[0], prefix=prefix)
        hi.history_attention_into(ctx, whole, q, counts, outs[1])
        hi.history_attention_into(ctx, ring, q, counts, outs[2], window=window, first=first)
        hi.history_attention_into(ctx, whole, q, counts, outs[3], window=window, first=first)
        for h in (own, ring, whole):
            hi.history_advance(ctx, h, counts, N)

    graph = ctx.capture(enqueue) if captured else None
    # Two sums of the same products in fp32: 2e-5; a rounding of 16-bit outputs may go the other way, one step (twice half a step) at most.
    tol = {"float32": 2e-5, "bfloat16": 2 * 2.0 ** -8, "float16": 2 * 2.0 ** -11}[kind]
    for step in range(3):
        for x in outs:
            x.fill_(7.0)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g).to(dtype))
        torch.cuda.synchronize()
        graph.launch() if graph else enqueue()
        ctx.synchronize()
        for a, b in ((outs[0], outs[1]), (outs[2], outs[3])):
            for s, n in enumerate((N, 2, 0)):
                assert (a[s, n:] == 7.0).all() and (b[s, n:] == 7.0).all()
                assert (a[s, :n].float() - b[s, :n].float()).norm() <= tol * b[s, :n].float().norm()
    assert own.lengths.tolist() == [3 * N, 6, 0] and ring.lengths.tolist() == whole.lengths.tolist() == [P + 3 * N, P + 6, P]
    if graph:
        graph.close()
