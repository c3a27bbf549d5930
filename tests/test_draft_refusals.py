"""Calls around drafted tokens that the C entries refuse."""
from test_tree_attention import _call


def test_a_window_over_rows_in_no_order():
    """Eviction leaves a history's rows in no order of position, so that a window cannot go by them."""
    kept = dict(positions=64, next_position=64)
    assert _call(desc=dict(window=8), cache=kept) == -1
    assert _call(desc=dict(window=8), cache=kept, q=None) == -1
    assert _call("hh_attention_weights", desc=dict(window=8), cache=kept) == -1


def test_python_takes_one_node_of_a_longer_batch():
    """x[:, :1] of [S][N] nodes: with one node a sequence, the step between nodes is the one between sequences."""
    import torch
    from hydra_amd import speculative as sp
    x = torch.zeros((3, 5, 4, 64), dtype=torch.float16)
    one = x[:, :1]
    assert sp._node_stride(one, "q", one.shape, torch.float16, x.device) == 5 * 4 * 64
    part = x[:, 2:3, 1:3]
    assert sp._node_stride(part, "draft_k", part.shape, torch.float16, x.device) == 5 * 4 * 64
    layers = torch.zeros((2, 3, 5, 4, 64), dtype=torch.float16)
    kv = torch.zeros((3, 8, 4, 64), dtype=torch.float16)
    caches = sp.CacheSet([sp.KVCache(kv, kv.clone(), torch.zeros(3, dtype=torch.int32)) for _ in range(2)])
    _, step = sp._layers(layers[:, :, :1], "draft_k", caches, (3, 1, 4, 64), torch.float16, kv.device)
    assert step == 5 * 4 * 64
