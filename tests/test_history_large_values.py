"""Attention over histories of values near the end of fp32: their weighted means are numbers, and so are the outputs.

Tolerance: that of outputs of ordinary size (fp32 sums and weights in terms, the output's own rounding), since nothing depends on the size."""
import numpy as np
import pytest

import history_ref as R
from test_history_attention import TOL, call, make, torch_type

pytestmark = pytest.mark.gpu


def filled(torch, t, value):
    """Every value of the history `value` with a sign by its column, as the format holds it."""
    fmt, shape = t["fmt"], t["vn"].shape
    x = np.broadcast_to(np.where(np.arange(shape[-1]) % 3 == 0, -value, value), shape[-1:]).astype(np.float64)
    if fmt == "bf16":
        v = torch.from_numpy(x).to(torch.bfloat16)
        t["v"], t["vn"] = v.expand(shape).contiguous(), np.broadcast_to(v.double().numpy(), shape)
        return
    codes, scales, values = R.encode(x, fmt)
    assert np.abs(values).max() < 3.4e38
    t["v"] = torch.from_numpy(np.broadcast_to(codes, shape[:-1] + codes.shape).copy())
    t["vs"] = torch.from_numpy(np.broadcast_to(scales, shape[:-1] + scales.shape).copy())
    t["vn"] = np.broadcast_to(values, shape)


@pytest.mark.parametrize("kind,fmt", [("bf16", "bf16"), ("bf16", "mxfp8"), ("bf16", "mxfp4"), ("f32", "mxfp8"), ("f32", "mxfp4")])
@pytest.mark.parametrize("N,D,length,window,shared", [(1, 64, 0, 0, None), (40, 64, 60, 1, None), (2, 128, 60, 1, None), (33, 256, 5, 1, None),
                                                      (2, 64, 3000, 0, None), (40, 64, 3000, 0, None), (3, 128, 7, 0, 0)])
def test_large_values(kind, fmt, N, D, length, window, shared):
    """One key seen, and as many as the values leave room for."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] large values {kind} {fmt} N={N} D={D} length={length}", flush=True)
    t = make(torch, 1, N, 8, 2, D, kind, fmt, length + N, [length], shared=shared, seed=2)
    seen = 1 if window else length + N
    filled(torch, t, (3.3e38 if fmt == "bf16" else 2.5e38) / seen)
    out, _ = call(torch, Context(0), t, window=window)
    want, _ = R.attention(t["q"].double().numpy(), t["kn"], t["vn"], [length], [N], None, D ** -0.5, window)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    for at, w in want.items():
        assert np.linalg.norm((got[at] - w) / 1e30) <= TOL[kind] * np.linalg.norm(w / 1e30), at
