"""Attention over histories: what its weights are held to does not depend on how many tokens or streams share a call.

Element by element, against 64 bits: the output's own rounding, half a step of it (bf16 2^-8, fp16 2^-11 of its size at most), and on top of it
errors of the weights p, which carry every |v| that they meet: 2e-5 of sums in fp32 over up to 256 products, as the rows' norms
are tested to, and 2^-15 (3e-5) of each weight where its terms are bf16: (2e-5 + 2^-15)·Σ p |v|. Weights rounded once to the output's type
would be off by up to 2^-9 (bf16) or 2^-12 (fp16) each: with two keys of much weight that is 10 times this bound."""
import numpy as np
import pytest

import history_ref as R
from test_history_attention import call, make

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}

CASES = [
    # S, N, H, G, D, type, format, rows, lengths, shared
    (1, 40, 8, 2, 64, "bf16", "mxfp8", 200, [100], None),
    (1, 40, 8, 2, 64, "f16", "f16", 200, [100], None),
    (1, 40, 8, 2, 64, "f16", "mxfp4", 200, [100], None),
    (2, 20, 16, 2, 128, "bf16", "bf16", 3000, [2900, 17], None),      # chunks
    (1, 35, 4, 1, 128, "f16", "f16", 90, [50], None),
    (1, 33, 4, 1, 256, "bf16", "mxfp4", 90, [50], None),
    (1, 33, 4, 1, 256, "f16", "f16", 90, [50], None),
    (20, 1, 8, 2, 64, "bf16", "mxfp8", 40, list(range(1, 40, 2)), 300),   # one token a stream behind a prefix
    (20, 1, 8, 2, 64, "f16", "f16", 40, list(range(1, 40, 2)), 300),
    (1, 2, 8, 2, 64, "bf16", "mxfp8", 200, [100], None),              # few rows
    (1, 2, 8, 2, 64, "f16", "f16", 200, [100], None),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_weights(case):
    import torch
    from hydra_amd.layer import Context
    S, N, H, G, D, kind, fmt, rows, lengths, shared = case
    print(f"[gpu] history weights {case}", flush=True)
    t = make(torch, S, N, H, G, D, kind, fmt, rows, lengths, shared=shared, seed=7)
    out, _ = call(torch, Context(0), t, scale=2.0 / D ** 0.5)        # a few keys have most of the weight
    args = [t["q"].double().numpy(), t["kn"], None, lengths, [N] * S, None, 2.0 / D ** 0.5, 0, 0, False, 0]
    both = []
    for f in (lambda x: x, np.abs):
        args[2] = f(t["vn"])
        both.append(R.attention(*args, None if shared is None else (t["pkn"][0], f(t["pvn"][0])), shared or 0)[0])
    got = out.double().cpu().numpy()
    worst = max(np.max(np.abs(got[at] - want) - HALF[kind] * np.abs(want) - (2e-5 + 2.0 ** -15) * both[1][at])
                for at, want in both[0].items())
    assert worst <= 0, worst
