"""Attention over histories: an infinity among the values that a token sees is its output's in that column, whether its tile is seen whole or
not and however little weight it has: the mean in 64 bits, where every weight is above zero, says the same. The other columns keep their
tolerance."""
import numpy as np
import pytest

import history_ref as R
from test_history_attention import TOL, call, make

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f16"), ("bf16", "mxfp8"), ("f32", "mxfp4"), ("f16", "mxfp8")]


def plant(t, which, s, row, column, value):
    """An infinity (or NaN) into a row of values; of codes the 32 columns with it: the largest code, or its negative, beside zeros at 2^127."""
    v, vs, vn = which
    if t[vs] is None:
        t[v][s, :, row, column] = value
        t[vn][s, :, row, column] = value
        return
    low = column // 32 * 32
    t[vn][s, :, row, low:low + 32] = 0.0
    t[vn][s, :, row, column] = value
    if t["fmt"] == "mxfp8":
        t[v][s, :, row, low:low + 32] = 0
        t[v][s, :, row, column] = 0x7F if np.isnan(value) else 0x7E if value > 0 else 0xFE
    else:
        assert not np.isnan(value)
        t[v][s, :, row, low // 2:low // 2 + 16] = 0
        t[v][s, :, row, column // 2] = (7 if value > 0 else 15) << 4 * (column % 2)
    t[vs][s, :, row, low // 32] = 254


def far_key(t, which, s, row, D):
    """A key whose logits are 40 less than its row's others: queries' first columns are 8, this key's -5·sqrt(D) (so that a format holds it
    nearly; what it holds is what counts)."""
    k, ks, kn = which
    x = np.zeros(D)
    x[0] = -5.0 * D ** 0.5
    if t[ks] is None:
        t[k][s, :, row] = 0
        t[k][s, :, row, 0] = float(x[0])
        t[kn][s, :, row] = 0
        t[kn][s, :, row, 0] = t[k][s, 0, row, 0].double().item()
        return
    import torch
    codes, scales, values = R.encode(x, t["fmt"])
    t[k][s, :, row], t[ks][s, :, row], t[kn][s, :, row] = torch.from_numpy(codes), torch.from_numpy(scales), values


CASES = [
    # N, D, rows, length, window, first, shared
    (2, 64, 400, 300, 0, 0, None),
    (40, 64, 400, 300, 0, 0, None),
    (2, 64, 5000, 4900, 0, 0, None),       # chunks
    (33, 128, 3000, 2900, 0, 0, None),
    (6, 128, 400, 300, 0, 0, None),
    (2, 256, 400, 300, 0, 0, None),
    (33, 256, 400, 300, 0, 0, None),
    (40, 64, 600, 500, 450, 4, None),      # some have it behind their window
    (1, 64, 200, 150, 0, 0, 500),          # in the prefix too
    (30, 64, 200, 150, 0, 0, 500),
]


@pytest.mark.parametrize("kind,fmt", TYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("far", [False, True])
def test_infinities_at_old_positions(kind, fmt, case, far):
    import torch
    from hydra_amd.layer import Context
    N, D, rows, length, window, first, shared = case
    print(f"[gpu] infinities {kind} {fmt} {case} far={far}", flush=True)
    t = make(torch, 2, N, 8, 2, D, kind, fmt, rows, [length, length // 2], shared=shared, seed=8)
    t["q"][..., 0] = 8.0
    own, prefix = ("v", "vs", "vn"), ("pv", "pvs", "pvn")
    at = length - window + 20 if window else 70
    plant(t, own, 0, at, 7, np.inf)
    plant(t, own, 0, at + 1, 33, -np.inf)
    plant(t, own, 1, 66, 40, np.inf)
    plant(t, own, 1, 130, 40, -np.inf)     # both: NaN
    if far:
        for s, r in ((0, at), (0, at + 1), (1, 66), (1, 130)):
            far_key(t, ("k", "ks", "kn"), s, r, D)
    if shared is not None:
        plant(t, prefix, 0, 100, 50, -np.inf)
        if far:
            far_key(t, ("pk", "pks", "pkn"), 0, 100, D)
    out, lse = call(torch, Context(0), t, window=window, first=first)
    with np.errstate(invalid="ignore"):
        want, _ = R.attention(t["q"].double().numpy(), t["kn"], t["vn"], t["lengths"].numpy(), [N, N], None, D ** -0.5, window, first,
                              prefix=None if shared is None else (t["pkn"][0], t["pvn"][0]), prefix_length=shared or 0)
    got, seen = out.double().cpu().numpy(), 0
    for i, w in want.items():
        odd = ~np.isfinite(w)
        seen += odd.any()
        assert np.array_equal(got[i][odd], w[odd], equal_nan=True), (i, got[i][odd], w[odd])
        assert np.isfinite(got[i][~odd]).all()
        assert np.linalg.norm(got[i][~odd] - w[~odd]) <= TOL[kind] * np.linalg.norm(w[~odd]), i
    assert seen
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("kind,fmt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "mxfp8")])
@pytest.mark.parametrize("N,length", [(2, 300), (40, 300), (2, 4900), (40, 4900)])
def test_nan_at_old_positions(kind, fmt, N, length):
    """In its column, of those who see it."""
    import torch
    from hydra_amd.layer import Context
    t = make(torch, 1, N, 8, 2, 64, kind, fmt, length + N, [length], seed=8)
    for row in (3, length - 2):
        plant(t, ("v", "vs", "vn"), 0, row, 9, np.nan)
    out, _ = call(torch, Context(0), t)
    nan = torch.isnan(out)
    assert nan[..., 9].all() and not nan[..., :9].any() and not nan[..., 10:].any()
