"""One drafted node a sequence as a slice of a longer batch: attention, weights and commit read the rows that the
packed tensors give."""
import pytest


@pytest.mark.gpu
def test_one_node_of_a_longer_batch():
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    S, N, H, G, D, rows = 3, 5, 8, 2, 64, 40
    g = torch.Generator().manual_seed(2)
    n = lambda *shape: torch.randn(shape, generator=g).half().to("cuda:0")
    q, dk, dv, k, v = n(S, N, H, D), n(S, N, G, D), n(S, N, G, D), n(S, rows, G, D), n(S, rows, G, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda:0")
    ctx = Context(0)
    try:
        answers = []
        for view in (lambda x: x[:, 1:2], lambda x: x[:, 1:2].contiguous()):
            lengths, nxt, w = i32([20, 0, 7]), i32([20, 0, 7]), torch.zeros((S, G, rows), device="cuda:0")
            cache = sp.KVCache(k.clone(), v.clone(), lengths, weights=w, next_position=nxt,
                               positions=torch.zeros((S, G, rows), dtype=torch.int32, device="cuda:0"))
            out, lse = torch.empty((S, 1, H, D), dtype=torch.float16, device="cuda:0"), torch.empty((S, 1, H), device="cuda:0")
            path, one, parents = i32([[0]] * S), i32([1] * S), i32([[-1]] * S)
            torch.cuda.synchronize()
            sp.attention_tree_into(ctx, cache, view(q), view(dk), view(dv), parents, one, out, lse=lse)
            sp.cache_commit(ctx, sp.CacheSet([cache]), [view(dk)], [view(dv)], path, one)
            sp.attention_weights_into(ctx, cache, view(q), lse, path, one)
            ctx.synchronize()
            answers.append((out, lse, cache.k, cache.v, w, lengths))
        assert all(torch.equal(a, b) for a, b in zip(*answers))
        assert answers[0][5].tolist() == [21, 1, 8]
    finally:
        ctx.close()
