"""Calls around drafted tokens that the C entries refuse."""
from test_tree_attention import _call


def test_a_window_over_rows_in_no_order():
    """Eviction leaves a history's rows in no order of position, so that a window cannot go by them."""
    kept = dict(positions=64, next_position=64)
    assert _call(desc=dict(window=8), cache=kept) == -1
    assert _call(desc=dict(window=8), cache=kept, q=None) == -1
    assert _call("hh_attention_weights", desc=dict(window=8), cache=kept) == -1
