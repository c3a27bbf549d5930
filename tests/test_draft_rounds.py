"""Verification (hh_draft_verify): the rounds of a launch chain on trees whose paths go through children of every rank."""
import pytest

from test_draft_verify import call, check, inputs


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["iid", "distinct"])
def test_rounds_that_accept_and_drop_rows(mode):
    """Acceptances in every round of wide trees, next to rows that the same round still works on: every sequence by the
    rule, and the same answer from every run. Each round's decisions go by earlier rounds only."""
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    ranks = set()
    try:
        for S, N, V, branch in ((40, 31, 1100, 5), (3, 64, 9001, 7), (6, 43, 70001, 6)):
            print(f"[gpu] verify rounds {mode} S={S} N={N} V={V}", flush=True)
            t = inputs(torch, S, N, V, "f32", mode, branch, S)
            t["u"] = 1 - (1 - t["u"]) * 0.6                   # later children too are the accepted ones
            got = call(torch, ctx, t, mode, 0.8)
            check(t, mode, got, 0.8)
            ranks |= {(int(n) - 1) % branch for row in got[0] for n in row[1:] if n >= 0}
            for _ in range(4):
                assert all(torch.equal(x, y) for x, y in zip(call(torch, ctx, t, mode, 0.8), got))
    finally:
        ctx.close()
    assert len(ranks) > 2, "the paths go through children of few ranks"
