"""Roundings of the tree attention (hh_attention_tree) with 16-bit activations, output by output against 64 bits on the
same inputs. An output is rounded once: half a step of its type, 2^-11 (fp16, 2^-25 below its normal range) and 2^-8 (bf16) of its
value. What comes before that is in fp32 or as good, and its errors go by sum(p |v|), not by the output, which may be
small beside it: a probability's two parts (2^-21 fp16, 2^-15 bf16), and 1e-5 twice for the logits' fp32 sums (at most 16 + 4
roundings of 2^-24 of partial sums below 8) in the exponential and in the denominator."""
import math

import numpy as np
import pytest

from test_tree_attention import call, make, reference

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
PARTS = {"f16": 2.0 ** -21, "bf16": 2.0 ** -15}
LEAST = {"f16": 2.0 ** -25, "bf16": 0.0}


def outputs_of(t, got, window=0, ring=False, scale=None):
    """(got, exact, sum of p |v|) of every real node's outputs, in 64 bits."""
    num = lambda x: None if x is None else x.double().numpy()
    scale = t["q"].shape[3] ** -0.5 if scale is None else scale
    args = lambda v, dv: (num(t["q"]), num(t["k"]), v, num(t["dk"]), dv, t["lengths"].numpy(), t["parents"].numpy(),
                          t["counts"].numpy(), num(t["sinks"]), window, ring, scale)
    want, _ = reference(*args(num(t["v"]), num(t["dv"])))
    size, _ = reference(*args(np.abs(num(t["v"])), np.abs(num(t["dv"]))))
    g = got.double().cpu().numpy()
    return np.stack([g[i] for i in want]), np.stack([want[i] for i in want]), np.stack([size[i] for i in want])


@pytest.mark.gpu
@pytest.mark.parametrize("S,N,H,G,D,kind,rows,lengths,window,ring", [
    (1, 1, 8, 2, 64, "f16", 40, [3], 0, False),               # few keys: large probabilities
    (1, 1, 8, 2, 64, "bf16", 40, [3], 0, False),
    (2, 5, 8, 2, 128, "bf16", 90, [9, 80], 0, False),
    (4, 12, 16, 2, 64, "f16", 192, [5000, 191, 3000, 40], 128, True),
    (2, 25, 8, 2, 128, "bf16", 700, [690, 351], 0, False),    # four tiles of rows, chunks
    (1, 40, 16, 2, 128, "f16", 1500, [1477], 0, False),
    (1, 7, 4, 1, 256, "bf16", 1200, [1111], 0, False),
    (2, 9, 16, 1, 256, "f16", 300, [290, 31], 60, False),
    (1, 33, 4, 4, 64, "bf16", 600, [577], 0, False),
])
def test_outputs_are_rounded_once(S, N, H, G, D, kind, rows, lengths, window, ring):
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] tree rounding S={S} N={N} H={H} G={G} D={D} {kind} {lengths} w={window}", flush=True)
    t = make(torch, S, N, H, G, D, kind, rows, lengths, seed=N + D)
    ctx = Context(0)
    try:
        out, _ = call(torch, ctx, t, ring, window)
    finally:
        ctx.close()
    got, want, size = outputs_of(t, out, window, ring)
    before = (PARTS[kind] + 2e-5) * size
    off = np.abs(got - want) / (HALF[kind] * (np.abs(want) + before) + LEAST[kind] + before)
    assert off.max() <= 1.0, (off.max(), (off > 1).mean())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,D,size", [("bf16", 64, 1e16), ("bf16", 128, 3e18), ("bf16", 256, 1e5), ("f16", 64, 4e4), ("f16", 128, 6e3),
                                         ("f16", 256, 1e4)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_logits_of_any_size(kind, D, size, sign):
    """Logits far from zero, all of one sign (to 10^36 in bf16, 10^8 in fp16). One dimension counts, so that every logit is a product:
    the keys that hold the largest tie, the others are lost by more than fp32 tells apart. The outputs are the winners' mean; lse is
    the largest logit to eight roundings of fp32."""
    import torch
    from hydra_amd.layer import Context
    S, N, H, G, n = 2, 6, 16, 2, 300
    t = make(torch, S, N, H, G, D, kind, n, [n, 37], seed=3, sinks=False)
    for x in ("q", "k", "dk"):
        t[x].zero_()
    t["q"][..., 0] = size * (1 + torch.arange(N * H).view(1, N, H) / (N * H)) / 2
    t["k"][..., 0], t["dk"][..., 0] = sign * size, sign * size
    loser = torch.arange(n) % 3 == 1
    t["k"][:, loser, :, 0] *= 0.5 if sign > 0 else 1.5
    print(f"[gpu] tree logits {kind} D={D} {sign * size}", flush=True)
    ctx = Context(0)
    try:
        for scale, most in ((None, 0), (None, 64), (0.3, 0)):
            out, lse = call(torch, ctx, t, scale=scale, max_length=most)
            got, want, mean = outputs_of(t, out, scale=scale)
            assert np.isfinite(got).all()
            before = (PARTS[kind] + 2e-5) * mean
            assert (np.abs(got - want) <= HALF[kind] * (np.abs(want) + before) + LEAST[kind] + before).all()
            top = (t["q"][..., 0].double() * sign * t["k"][0, 0, 0, 0].double().abs() * (D ** -0.5 if scale is None else scale)).numpy()
            assert (np.abs(lse.double().cpu().numpy() - top) <= 8 * 2.0 ** -24 * np.abs(top) + 7).all()
    finally:
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_a_long_tail_behind_one_key(kind):
    """One key takes nearly all, 32767 alike share the rest, each 2^-28.5 of the largest. A probability below fp16's normal
    range is held to 2^-32 of the row's largest, so the tail is off by at most that a key, and by 2e-5 of itself."""
    import torch
    from hydra_amd.layer import Context
    n, D = 32768, 256                          # heads of 256: one wave walks all the keys of a chunk
    t = make(torch, 1, 1, 1, 1, D, kind, n, [n], sinks=False)
    for x in ("q", "k", "dk", "dv"):
        t[x].zero_()
    t["v"].fill_(1.0)
    t["q"][..., 0], t["k"][0, 5, 0, 0], t["v"][0, 5] = 1.0, 28.5, 0.0
    print(f"[gpu] tree tail {kind}", flush=True)
    ctx = Context(0)
    try:
        out, _ = call(torch, ctx, t, scale=math.log(2.0), max_length=64)     # one chunk
    finally:
        ctx.close()
    tail = (n - 1) * 2.0 ** -28.5
    want = tail / (1 + tail + 2.0 ** -28.5)
    off = (out.double().cpu() - want).abs().max()
    assert off < n * 2.0 ** -32 + 2e-5 * want + (2.0 ** -11 * want if kind == "f16" else 0.0), (float(off), want)
