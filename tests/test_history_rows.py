"""A history's rows: written (hh_history_write), read back (hh_history_read), lengths moved on. Codes, scales and numbers equal
those of the formats' definitions, bit for bit; what no token reaches is left as it was."""
import numpy as np
import pytest

import history_ref as R

TYPES = ("f32", "f16", "bf16")


def torch_type(torch, kind):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]


def decode(torch, h):
    """The numbers that a history's tensors hold, on the host in 64 bits: k, v [S][G][rows][D]."""
    out = []
    for c, s in ((h.k, h.k_scales), (h.v, h.v_scales)):
        if s is None:
            out.append(c.double().cpu().numpy())
            continue
        c, s = c.cpu().numpy(), s.cpu().numpy().astype(np.int64)
        if h.format == 3:
            x = np.concatenate([R.HELD["mxfp8"], [np.nan], -R.HELD["mxfp8"], [np.nan]])[c]
        else:
            x = np.concatenate([R.HELD["mxfp4"], -R.HELD["mxfp4"]])[np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)]
        x = x.reshape(*s.shape, 32) * np.where(s == 255, np.nan, 2.0 ** (np.minimum(s, 254) - 127.0))[..., None]
        out.append(x.reshape(*x.shape[:-2], -1))
    return out


def fill(torch, h, seed=9):
    """Every byte of the history something."""
    g = torch.Generator().manual_seed(seed)
    for t in (h.k, h.v, h.k_scales, h.v_scales):
        if t is not None and t.dtype is torch.uint8:
            t.copy_(torch.randint(1, 120, t.shape, generator=g, dtype=torch.uint8))
        elif t is not None:
            t.copy_(torch.randn(t.shape, generator=g))


def numbers(torch, shape, kind, seed, wild=True):
    """Rows of very different sizes, zeros, ties, the type's extremes."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-12, 12, shape[:-1] + (1,), generator=g).float())
    if wild:
        flat = x.view(-1, 32)
        n = flat.shape[0]
        flat[0] = 0.0
        flat[1 % n] = torch.arange(32).float() * 0.25 - 4.0          # ties of e2m1
        flat[2 % n] = 448.0 - torch.arange(32).float()               # ties of e4m3, the largest number
        flat[3 % n] = torch.tensor([6.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -2.5, -5.0] + [0.1] * 20)
        flat[4 % n] = torch.tensor([449.0] + [17.0, 18.0, 19.0, -17.0, 0.0] + [2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10] + [1.0] * 23)
        flat[5 % n] = 6.001
        flat[6 % n] = {"f32": 3.0e38, "f16": 65504.0, "bf16": 3.0e38}[kind]
        flat[7 % n] = 2.0 ** -140 if kind == "f32" else 2.0 ** -24
    return x.to(torch_type(torch, kind))


CASES = [
    # S, N, G, D, format, type, rows, ring, pinned, lengths, counts
    (1, 1, 8, 64, "mxfp8", "f32", 10, False, 0, [0], [1]),
    (3, 5, 2, 64, "mxfp4", "f32", 9, False, 0, [0, 4, 7], [5, 0, 4]),          # past the rows; none
    (2, 33, 3, 128, "mxfp8", "bf16", 50, False, 0, [11, 17], [33, 20]),
    (2, 7, 1, 256, "mxfp4", "f16", 40, True, 5, [0, 1000], [7, 6]),             # a ring that fills, one that wraps
    (2, 50, 2, 64, "mxfp8", "f16", 24, True, 4, [0, 77], [50, 31]),             # steps longer than the ring
    (1, 9, 2, 128, "mxfp8", "f32", 8, True, 7, [3], [9]),                       # one row besides the pinned ones
    (2, 4, 4, 64, "f16", "f32", 12, True, 0, [10, 5], [4, 3]),
    (2, 4, 4, 128, "bf16", "bf16", 12, False, 0, [8, 9], [4, 4]),
    (1, 3, 1, 256, "bf16", "f16", 7, False, 0, [2], [3]),
    (2, 3, 1, 64, "f16", "bf16", 7, False, 0, [-5, 2], [9, -1]),                # lengths and counts out of range
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_written_and_read(case):
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    S, N, G, D, fmt, kind, rows, ring, pinned, lengths, counts = case
    ctx = Context(0)
    h = hi.History.empty(S, G, rows, D, format=fmt, ring=ring, pinned=pinned,
                         lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda:0"))
    fill(torch, h)
    k, v = numbers(torch, (S, N, G, D), kind, 1), numbers(torch, (S, N, G, D), kind, 2)
    c = torch.tensor(counts, dtype=torch.int32, device="cuda:0")
    held = [t.clone() for t in (h.k, h.v)], [None if t is None else t.clone() for t in (h.k_scales, h.v_scales)]
    torch.cuda.synchronize()
    hi.history_write(ctx, h, k.cuda(), v.cuda(), c)
    ctx.synchronize()
    for x, codes, scales, c0, s0 in ((k, h.k, h.k_scales, held[0][0], held[1][0]), (v, h.v, h.v_scales, held[0][1], held[1][1])):
        want, want_s = c0.cpu().clone(), None if s0 is None else s0.cpu().clone()
        for s in range(S):
            start = max(0, lengths[s])
            for i in range(min(N, max(0, counts[s]))):
                r = R.row_of(start + i, rows, ring, pinned)
                if r < 0:
                    continue
                if fmt in ("f16", "bf16"):
                    want[s, :, r] = x[s, i].float().to(want.dtype)
                else:
                    cc, ss, _ = R.encode(x[s, i].double().numpy(), fmt)
                    want[s, :, r], want_s[s, :, r] = torch.from_numpy(cc), torch.from_numpy(ss)
        if fmt in ("f16", "bf16"):
            assert torch.equal(codes.cpu().view(torch.int16), want.view(torch.int16))
        else:
            assert torch.equal(scales.cpu(), want_s)
            assert torch.equal(codes.cpu(), want)
    # Back as numbers of every type, from other places too.
    for out_kind in TYPES:
        starts = [max(0, n) for n in lengths] if out_kind != "f16" else [n - 2 for n in lengths]
        dtype = torch_type(torch, out_kind)
        ko, vo = (torch.full((S, N, G, D), 7.0, dtype=dtype, device="cuda:0") for _ in range(2))
        torch.cuda.synchronize()
        hi.history_read_into(ctx, h, torch.tensor(starts, dtype=torch.int32, device="cuda:0"), c, ko, vo)
        ctx.synchronize()
        for got, all_ in zip((ko, vo), decode(torch, h)):
            want = torch.full((S, N, G, D), 7.0, dtype=dtype)
            for s in range(S):
                for i in range(min(N, max(0, counts[s]))):
                    p = starts[s] + i
                    r = R.row_of(p, rows, ring, pinned) if p >= 0 else -1
                    if r >= 0:
                        want[s, i] = torch.from_numpy(all_[s, :, r]).to(torch.float32).to(dtype)   # held numbers are exact in fp32
            assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=-77.0), torch.nan_to_num(want.float(), nan=-77.0))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_infinities_and_nan_make_their_32_columns_nan(fmt):
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    h = hi.History.empty(1, 2, 6, 64, format=fmt)
    k = torch.randn((1, 4, 2, 64))
    k[0, 0, 0, 5], k[0, 1, 1, 40], k[0, 2, 0, 63] = float("inf"), float("nan"), float("-inf")
    c = torch.tensor([4], dtype=torch.int32, device="cuda:0")
    hi.history_write(ctx, h, k.cuda(), k.cuda(), c)
    ko, vo = torch.zeros((1, 4, 2, 64), device="cuda:0"), torch.zeros((1, 4, 2, 64), device="cuda:0")
    hi.history_read_into(ctx, h, h.lengths, c, ko, vo)
    ctx.synchronize()
    nan = torch.zeros((1, 4, 2, 2), dtype=torch.bool)
    nan[0, 0, 0, 0] = nan[0, 1, 1, 1] = nan[0, 2, 0, 1] = True
    assert torch.equal(ko.cpu().isnan(), nan.repeat_interleave(32, -1)) and torch.equal(vo.cpu().isnan(), nan.repeat_interleave(32, -1))


@pytest.mark.gpu
def test_slices_of_a_wider_product():
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    S, N, G, D = 2, 3, 2, 64
    wide = torch.randn((S, N, 5 * G * D)).cuda()
    k, v = wide[..., G * D:2 * G * D].unflatten(-1, (G, D)), wide[..., 3 * G * D:4 * G * D].unflatten(-1, (G, D))
    c = torch.full((S,), N, dtype=torch.int32, device="cuda:0")
    a, b = hi.History.empty(S, G, 8, D), hi.History.empty(S, G, 8, D)
    torch.cuda.synchronize()
    hi.history_write(ctx, a, k, v, c)
    hi.history_write(ctx, b, k.contiguous(), v.contiguous(), c)
    ctx.synchronize()
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.k_scales, b.k_scales)


@pytest.mark.gpu
def test_lengths_move_on():
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    n = 130
    lengths = torch.arange(n, dtype=torch.int32, device="cuda:0") - 3
    counts = torch.arange(n, dtype=torch.int32, device="cuda:0") % 7 - 1
    h = hi.History.empty(n, 1, 4, 64, lengths=lengths.clone())
    torch.cuda.synchronize()
    hi.history_advance(ctx, h, counts, 4)
    ctx.synchronize()
    assert torch.equal(h.lengths, lengths.clamp(min=0) + counts.clamp(0, 4))
