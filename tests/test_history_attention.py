"""Attention over a history (hh_history_attention) against a plain implementation in 64 bits on the numbers that the history holds.

Tolerances, rel-L2 of a row (one token's head). fp32 sums of up to 256 products (terms of a logit sum to ~10 in magnitude:
sqrt(256)·10·2^-24 = 1e-5 of a probability), probabilities and their sums alike: 2e-5. F16 and BF16 outputs are rounded once, half
a step of each number; probabilities of BF16's products are pairs, to 2^-15 each (3e-5). Of more than 32 rows of a kv head (16 of a
prefix's) probabilities of the output's own type are rounded once too, and normalised by their rounded sum: an error of Σ d_j p_j (v_j − o)
besides, |d_j| up to half a step, for independent d_j a fraction sqrt(Σ p_j^2) |v − o| / |o| of d's 0.42 half steps (rms), as the output's own 0.42:
0.6 of the half step with values as large as their spread. lse, absolute: 1e-5 of a logit's
error, its sum's and its logarithm's with it 4e-5."""
import math

import numpy as np
import pytest

import history_ref as R

TOL = {"f32": 2e-5, "f16": 2.0 ** -11 + 2e-5 + 3e-5, "bf16": 2.0 ** -8 + 2e-5 + 3e-5}
LSE = 4e-5


def torch_type(torch, kind):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def held(torch, shape, fmt, seed, std=1.0):
    """(tensor of codes, scales or None, the numbers in 64 bits) of a history [S][G][rows][D] with numbers in every row."""
    g = np.random.default_rng(seed)
    x = g.standard_normal(shape) * std * np.exp(0.3 * g.standard_normal(shape[-1]))
    if fmt in ("f16", "bf16"):
        t = torch.from_numpy(x).float().to(torch_type(torch, fmt))
        return t, None, t.double().numpy()
    codes, scales, values = fast_encode(x, fmt)
    return torch.from_numpy(codes), torch.from_numpy(scales), values


def fast_encode(x, fmt):
    """history_ref.encode without its loop, for finite numbers that are not all zero."""
    top = np.abs(x.reshape(*x.shape[:-1], -1, 32)).max(-1)
    largest = R.HELD[fmt][-1]
    e = np.ceil(np.log2(top / largest)).astype(np.int64)
    y = x.reshape(*x.shape[:-1], -1, 32) / 2.0 ** e[..., None].astype(np.float64)
    mids = (R.HELD[fmt][1:] + R.HELD[fmt][:-1]) / 2
    pick = np.searchsorted(mids, np.abs(y))
    values = (np.copysign(R.HELD[fmt][pick], y) * 2.0 ** e[..., None].astype(np.float64)).reshape(x.shape)
    codes = (pick + (128 if fmt == "mxfp8" else 8) * (y < 0)).reshape(x.shape).astype(np.uint8)
    return (codes[..., ::2] + 16 * codes[..., 1::2] if fmt == "mxfp4" else codes), (e + 127).astype(np.uint8), values


def make(torch, S, N, H, G, D, kind, fmt, rows, lengths, counts=None, sinks=False, shared=None, prefix_rows=None, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    t = dict(q=torch.randn((S, N, H, D), generator=g).to(torch_type(torch, kind)), lengths=torch.tensor(lengths, dtype=torch.int32),
             counts=torch.tensor([N] * S if counts is None else counts, dtype=torch.int32), kind=kind, fmt=fmt,
             sinks=torch.randn((H,), generator=g).to(torch.bfloat16) if sinks else None, shared=shared)
    t["k"], t["ks"], t["kn"] = held(torch, (S, G, rows, D), fmt, 10 * seed + 1, std)
    t["v"], t["vs"], t["vn"] = held(torch, (S, G, rows, D), fmt, 10 * seed + 2)
    if shared is not None:
        n = max(1, prefix_rows or shared)
        t["pk"], t["pks"], t["pkn"] = held(torch, (1, G, n, D), fmt, 10 * seed + 3, std)
        t["pv"], t["pvs"], t["pvn"] = held(torch, (1, G, n, D), fmt, 10 * seed + 4)
    return t


def histories(torch, t, ring=False, pinned=0):
    from hydra_amd import history as hi
    up = lambda x: None if x is None else x.to("cuda:0")
    h = hi.History(up(t["k"]), up(t["v"]), up(t["lengths"]), up(t["ks"]), up(t["vs"]), ring=ring, pinned=pinned)
    p = None
    if t["shared"] is not None:
        p = hi.History(up(t["pk"]), up(t["pv"]), torch.tensor([t["shared"]], dtype=torch.int32, device="cuda:0"), up(t["pks"]), up(t["pvs"]))
    return h, p


def call(torch, ctx, t, window=0, first=0, ring=False, pinned=0, scale=None, max_length=0):
    from hydra_amd import history as hi
    h, p = histories(torch, t, ring, pinned)
    q, c = t["q"].to("cuda:0"), t["counts"].to("cuda:0")
    s = None if t["sinks"] is None else t["sinks"].to("cuda:0")
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device="cuda:0")
    torch.cuda.synchronize()
    hi.history_attention_into(ctx, h, q, c, out, lse=lse, sinks=s, window=window, first=first, sm_scale=scale, max_length=max_length, prefix=p)
    ctx.synchronize()
    return out, lse


def check(torch, t, out, lse, window=0, first=0, ring=False, pinned=0, scale=None):
    S, N, H, D = t["q"].shape
    prefix = None if t["shared"] is None else (t["pkn"][0], t["pvn"][0])
    with np.errstate(invalid="ignore"):
        ro, rl = R.attention(t["q"].double().numpy(), t["kn"], t["vn"], t["lengths"].numpy(), t["counts"].numpy(),
                             None if t["sinks"] is None else t["sinks"].double().numpy(), D ** -0.5 if scale is None else scale,
                             window, first, ring, pinned, prefix, t["shared"] or 0)
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    real = np.zeros((S, N), bool)
    for (s, i, h) in ro:
        real[s, i] = True
    assert np.all(got[~real] == 7.0) and np.all(gl[~real] == 7.0), "tokens that are not there were written"
    for at, want in ro.items():
        a = got[at]
        if np.isneginf(rl[at]):
            assert np.all(a == 0) and np.isneginf(gl[at]), at
            continue
        assert np.array_equal(np.isnan(a), np.isnan(want)), at
        ok = ~np.isnan(want)
        assert np.linalg.norm(a[ok] - want[ok]) <= TOL[t["kind"]] * np.linalg.norm(want[ok]) + 1e-30, at
        if not np.isnan(rl[at]):
            assert abs(gl[at] - rl[at]) < LSE, at


CASES = [
    # S, N, H, G, D, type, format, rows, lengths, counts, window, first, ring, pinned, shared, sinks
    (1, 1, 64, 8, 64, "f32", "mxfp8", 4, [0], None, 0, 0, False, 0, None, True),        # the token itself
    (1, 1, 64, 8, 64, "bf16", "mxfp4", 70, [63], None, 0, 0, False, 0, None, False),    # keys end at and around a tile's end
    (1, 1, 64, 8, 64, "f16", "f16", 70, [64], None, 0, 0, False, 0, None, False),
    (2, 1, 16, 2, 256, "bf16", "bf16", 300, [31, 290], None, 0, 0, False, 0, None, False),
    (2, 1, 16, 1, 128, "f32", "f16", 700, [650, 0], None, 0, 0, False, 0, None, True),  # sixteen heads a group
    (3, 1, 5, 1, 64, "f32", "mxfp4", 3000, [2999, 1023, 511], None, 0, 0, False, 0, None, False),
    (1, 1, 8, 8, 256, "f16", "mxfp8", 900, [880], None, 0, 0, False, 0, None, True),
    (4, 3, 24, 4, 128, "bf16", "mxfp8", 400, [389, 0, 128, 7], [3, 2, 0, 1], 0, 0, False, 0, None, False),
    (2, 9, 8, 2, 64, "f32", "mxfp8", 200, [150, 20], [9, 5], 0, 0, False, 0, None, True),
    (1, 40, 64, 8, 64, "bf16", "mxfp8", 40, [0], None, 0, 0, False, 0, None, True),     # a prompt
    (2, 131, 6, 2, 128, "f16", "mxfp4", 420, [257, 3], [131, 77], 0, 0, False, 0, None, False),
    (1, 70, 16, 2, 256, "f32", "mxfp8", 333, [250], None, 0, 0, False, 0, None, False),
    (1, 300, 5, 1, 64, "f32", "f16", 310, [10], None, 0, 0, False, 0, None, True),
    (2, 1, 64, 8, 64, "f32", "mxfp8", 150, [1000, 130], None, 128, 4, True, 4, None, True),   # rings, wrapped and not yet full
    (3, 4, 16, 4, 64, "f16", "f16", 40, [1000, 39, 2], [4, 4, 3], 24, 3, True, 5, None, False),
    (2, 20, 8, 2, 128, "bf16", "mxfp4", 90, [500, 0], None, 33, 16, True, 16, None, True),
    (1, 150, 8, 1, 64, "bf16", "mxfp8", 400, [200], None, 40, 4, False, 0, None, False),      # windows without rings
    (1, 65, 16, 2, 256, "bf16", "bf16", 400, [300], None, 1, 2, False, 0, None, True),        # itself and the first two
    (2, 33, 8, 8, 128, "f32", "mxfp8", 600, [511, 0], [33, 12], 100, 1, False, 0, None, False),
    (1, 3, 8, 2, 64, "f32", "mxfp8", 60, [5], None, 50, 9, False, 0, None, False),            # first tokens that are not there yet
    (1, 6, 8, 2, 64, "f32", "mxfp8", 20, [18], None, 3, 1, False, 0, None, False),            # behind a full history: some see little,
    (1, 9, 8, 2, 64, "f32", "mxfp8", 20, [17], None, 3, 0, False, 0, None, False),            # some nothing
    (1, 9, 8, 2, 64, "f32", "mxfp8", 20, [17], None, 3, 0, False, 0, None, True),
    (2, 2, 8, 2, 64, "bf16", "mxfp8", 20, [40, 19], None, 0, 0, False, 0, None, False),
    (2, 1, 8, 2, 64, "f32", "mxfp8", 20, [-3, 5], [1, 7], 0, 0, False, 0, None, False),       # out of range
    (4, 1, 24, 4, 64, "f32", "f16", 60, [50, 0, 3, 59], None, 0, 0, False, 0, 1000, False),   # prefixes
    (9, 1, 64, 8, 64, "bf16", "mxfp8", 70, list(range(60, 69)), [1, 0, 1, 1, 1, 1, 1, 1, 1], 0, 0, False, 0, 515, True),
    (3, 7, 8, 2, 128, "f16", "mxfp4", 80, [0, 70, 33], [7, 5, 6], 0, 0, False, 0, 129, True),
    (2, 3, 16, 1, 256, "f32", "mxfp8", 80, [11, 50], None, 0, 0, False, 0, 77, False),
    (3, 2, 8, 2, 64, "bf16", "bf16", 30, [5, 0, 28], None, 0, 0, False, 0, 0, False),         # an empty prefix
    (33, 5, 4, 2, 64, "bf16", "mxfp8", 9, [3] * 33, None, 0, 0, False, 0, 300, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace(" ", ""))
def test_attention(case):
    import torch
    from hydra_amd.layer import Context
    S, N, H, G, D, kind, fmt, rows, lengths, counts, window, first, ring, pinned, shared, sinks = case
    t = make(torch, S, N, H, G, D, kind, fmt, rows, lengths, counts, sinks, shared)
    ctx = Context(0)
    kw = dict(window=window, first=first, ring=ring, pinned=pinned)
    check(torch, t, *call(torch, ctx, t, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,fmt,D", [("f32", "mxfp8", 64), ("bf16", "mxfp4", 128), ("bf16", "bf16", 64), ("f16", "f16", 256)])
@pytest.mark.parametrize("max_length", [1, 700, 100000])
def test_launches_sized_for_other_lengths(kind, fmt, D, max_length):
    """max_length only sizes the launch."""
    import torch
    from hydra_amd.layer import Context
    t = make(torch, 3, 2, 8, 2, D, kind, fmt, 5000, [4990, 0, 1234], shared=None)
    check(torch, t, *call(torch, Context(0), t, max_length=max_length))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [3.0, -0.25, 40.0])
@pytest.mark.parametrize("kind,fmt", [("f32", "mxfp8"), ("bf16", "mxfp8"), ("f16", "f16")])
def test_scales(kind, fmt, scale):
    """Sharp and turned-over distributions. A logit's error grows with it: 2^-24·sqrt(D) of its terms' size."""
    import torch
    from hydra_amd.layer import Context
    t = make(torch, 2, 3, 8, 2, 64, kind, fmt, 300, [250, 40])
    out, lse = call(torch, Context(0), t, scale=scale)
    ro, rl = R.attention(t["q"].double().numpy(), t["kn"], t["vn"], [250, 40], [3, 3], None, scale)
    terms = abs(scale) * 64 * 4.0
    tol = terms * 2.0 ** -24 * 8
    for at, want in ro.items():
        assert abs(float(lse[at]) - rl[at]) < tol + abs(rl[at]) * 2.0 ** -22 + LSE
        err = np.linalg.norm(out[at].double().cpu().numpy() - want) / np.linalg.norm(want)
        assert err < TOL[kind] + 2 * tol, at


@pytest.mark.gpu
@pytest.mark.parametrize("kind,fmt", [("f32", "mxfp8"), ("bf16", "mxfp4"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("ring", [False, True])
@pytest.mark.parametrize("N", [3, 40])
def test_what_a_token_does_not_see_has_no_part(kind, fmt, ring, N):
    """NaN and infinities in rows that no token sees, that only later tokens see, and that have left the window of some."""
    import torch
    from hydra_amd.layer import Context
    S, H, G, D, window, first = 2, 8, 2, 64, 30, 2
    rows = first + window + N + 5 if ring else 200
    lengths = [100, 61]
    t = make(torch, S, N, H, G, D, kind, fmt, rows, lengths, seed=3)
    bad = {0: [lengths[0] + N - 1, lengths[0] + N // 2, lengths[0] - window + N // 2], 1: [lengths[1] + N - 1, lengths[1] - window + 1]}
    for s, positions in bad.items():
        free = [p for p in range(lengths[s] + N, lengths[s] + N + 4)]   # rows that no position of the step has
        for j, p in enumerate(positions + free):
            r = R.row_of(p, rows, ring, first if ring else 0)
            if r < 0 or (ring and p in free and p - (rows - first) > lengths[s] - window):
                continue
            for c, sc, n in (("k", "ks", "kn"), ("v", "vs", "vn")):
                value = [np.nan, np.inf, -np.inf][(j + (c == "v")) % 3]
                if t[sc] is None:
                    t[c][s, :, r, 5 if c == "v" else 9] = float(value)
                    t[n][s, :, r, 5 if c == "v" else 9] = value
                else:
                    t[sc][s, :, r, 1] = 255
                    t[n][s, :, r, 32:] = np.nan
    kw = dict(window=window, first=first, ring=ring, pinned=first if ring else 0)
    out, lse = call(torch, Context(0), t, **kw)
    with np.errstate(invalid="ignore"):
        ro, _ = R.attention(t["q"].double().numpy(), t["kn"], t["vn"], lengths, [N, N], None, D ** -0.5, window, first, ring, kw["pinned"])
    clean = 0
    for at, want in ro.items():
        a = out[at].double().cpu().numpy()
        if np.isfinite(want).all():
            clean += 1
            assert np.linalg.norm(a - want) <= TOL[kind] * np.linalg.norm(want), at
        else:
            assert not np.isfinite(a).all(), at
    assert clean > 0 and clean < len(ro)


@pytest.mark.gpu
def test_infinite_values_reach_those_who_see_them():
    """An infinity among 16-bit values is one of the outputs' of the tokens that see it, in its column alone."""
    import torch
    from hydra_amd.layer import Context
    for N in (2, 40):
        t = make(torch, 1, N, 8, 2, 64, "bf16", "bf16", 100, [50], seed=4)
        t["v"][0, :, 50 + N - 1, 7] = float("inf")
        t["vn"][0, :, 50 + N - 1, 7] = np.inf
        out, lse = call(torch, Context(0), t)
        o = out.float().cpu()
        assert torch.isfinite(o[0, :N - 1]).all()
        assert (o[0, N - 1, :, 7] == float("inf")).all()
        rest = o[0, N - 1].clone()
        rest[:, 7] = 0
        assert torch.isfinite(rest).all()


@pytest.mark.gpu
def test_strided_queries_int16_sinks_and_no_lse():
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    S, N, H, G, D = 2, 3, 8, 2, 64
    t = make(torch, S, N, H, G, D, "bf16", "mxfp8", 80, [60, 9], sinks=True)
    wide = torch.zeros((S, N, (H + 2 * G) * D), dtype=torch.bfloat16)
    wide[..., :H * D] = t["q"].reshape(S, N, -1)
    h, _ = histories(torch, t)
    q = wide.cuda()[..., :H * D].unflatten(-1, (H, D))
    out = torch.zeros((S, N, H, D), dtype=torch.bfloat16, device="cuda:0")
    torch.cuda.synchronize()
    hi.history_attention_into(ctx, h, q, t["counts"].cuda(), out, sinks=t["sinks"].view(torch.int16).cuda())
    ctx.synchronize()
    want, lse = call(torch, ctx, t)
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_the_same_call_twice_gives_the_same_bits():
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    t = make(torch, 3, 2, 16, 2, 128, "f32", "mxfp8", 3000, [2990, 100, 1777], shared=900)
    a, la = call(torch, ctx, t)
    b, lb = call(torch, ctx, t)
    assert torch.equal(a, b) and torch.equal(la, lb)
