"""Attention over histories: a row's bits are its own. What other tokens' queries hold, however large, must not change them: a row's
running maximum steps by its own logits."""
import pytest

from test_history_attention import call, make

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "mxfp8"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "mxfp4"), ("f32", "mxfp8"), ("f32", "f16")]


def others(torch, want, out, touched):
    (a, la), (b, lb) = want, out
    assert torch.equal(a[~touched], b[~touched]) and torch.equal(la[~touched], lb[~touched])


@pytest.mark.parametrize("kind,fmt", TYPES)
@pytest.mark.parametrize("N,D,shared", [(2, 64, None), (7, 128, None), (40, 64, None), (33, 256, None), (40, 64, 300), (1, 64, 300)])
def test_an_infinity_in_one_column_stays_alone(kind, fmt, N, D, shared):
    """Its logits are infinities, not NaN: the row's maximum becomes one."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] infinity {kind} {fmt} N={N} D={D} shared={shared}", flush=True)
    ctx = Context(0)
    t = make(torch, 2, N, 8, 2, D, kind, fmt, 400, [300, 7], shared=shared, seed=4)
    want = call(torch, ctx, t)
    touched = torch.zeros(want[0].shape[:3], dtype=torch.bool, device="cuda:0")
    for at, x in (((0, 0, 2), float("inf")), ((1, N - 1, 7), float("-inf"))):
        t["q"][at][5] = x
        touched[at] = True
    out = call(torch, ctx, t)
    others(torch, want, out, touched)
    assert torch.isnan(out[0][touched]).all()


@pytest.mark.parametrize("kind,fmt", TYPES)
@pytest.mark.parametrize("N,D,shared", [(2, 64, None), (7, 128, None), (40, 64, None), (33, 256, None), (40, 64, 300), (1, 64, 300)])
@pytest.mark.parametrize("size", [8.0, 400.0])
def test_other_queries_do_not_change_a_row(kind, fmt, N, D, shared, size):
    """The rows beside it step at other tiles, or have references so far from zero that their products are rounded first."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] larger queries {kind} {fmt} N={N} D={D} shared={shared}", flush=True)
    ctx = Context(0)
    t = make(torch, 2, N, 8, 2, D, kind, fmt, 400, [300, 7], shared=shared, seed=5, std=3.0)
    want = call(torch, ctx, t, scale=8.0)
    touched = torch.zeros(want[0].shape[:3], dtype=torch.bool, device="cuda:0")
    touched[:, :, 1::2] = True
    t["q"][:, :, 1::2] *= size
    others(torch, want, call(torch, ctx, t, scale=8.0), touched)


@pytest.mark.parametrize("kind,fmt", TYPES)
@pytest.mark.parametrize("S,N,D,shared", [(3, 2, 64, 300), (9, 3, 128, 1300), (20, 5, 256, 40), (3, 40, 64, None), (3, 2, 64, None)])
def test_tokens_that_are_not_there_are_not_read(kind, fmt, S, N, D, shared):
    """Whatever stands behind counts[s], tokens of a sequence that has none among them."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] padding {kind} {fmt} S={S} N={N} D={D} shared={shared}", flush=True)
    ctx = Context(0)
    counts = [N, 0, 1] + [(i % (N + 1)) for i in range(S - 3)]
    t = make(torch, S, N, 8, 2, D, kind, fmt, 90, [50 - i for i in range(S)], counts=counts, shared=shared, seed=6)
    there = torch.arange(N)[None] < torch.tensor(counts)[:, None]
    t["q"][~there] = 0.0
    want, wl = call(torch, ctx, t)
    assert (want[~there] == 7.0).all() and (wl[~there] == 7.0).all()
    for x in (float("nan"), float("inf"), 60000.0):
        t["q"][~there] = x
        out, lse = call(torch, ctx, t)
        assert torch.equal(out, want) and torch.equal(lse, wl)
