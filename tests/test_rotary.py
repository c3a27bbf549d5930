"""Rotary positions (hh_rotary, hh_rotary_table) against 64 bits.

Tolerance of an output, relative to m·(|x1| + |x2|): the angle, within half a turn, is rounded to fp32 once (pi·2^-25 = 9.4e-8 rad;
the fp64 product of position and frequency before it 2e5 turns·2^-53), sine and cosine are off by up to two of their last places
(2^-23 = 1.2e-7), m times them and the two products by half a last place each (3·2^-24 = 1.8e-7): together 4e-7; the output's own
rounding, half a step of its type, on top."""
import ctypes as C

import numpy as np
import pytest

import history_ref as R

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SIN = 4e-7

CASES = [
    # tokens, q_heads, k_heads, head_dim, rotated, span, interleaved, type, base, scaling, factor, far
    (1, 64, 8, 64, 64, 0, False, "f32", 150000.0, "yarn", 32.0, 131072),
    (3, 5, 1, 64, 64, 0, False, "f16", 10000.0, "none", 1.0, 10),
    (200, 24, 4, 128, 128, 0, True, "bf16", 10000.0, "linear", 7.5, 1 << 20),
    (65, 16, 2, 256, 64, 0, False, "bf16", 1e7, "none", 1.0, 262144),
    (33, 8, 8, 256, 64, 256, False, "f32", 1e6, "none", 1.0, 131072),      # a quarter of the pairs of the whole head
    (17, 3, 1, 128, 34, 0, False, "f32", 10000.0, "none", 1.0, 5000),      # halves at an odd distance
    (17, 3, 1, 128, 34, 0, True, "f16", 10000.0, "none", 1.0, 5000),
    (9, 2, 2, 72, 46, 54, False, "bf16", 10000.0, "yarn", 4.0, 30000),
    (2, 1, 1, 8, 2, 0, False, "f32", 100.0, "none", 1.0, 100),
    (1100, 7, 1, 64, 32, 0, False, "f16", 10000.0, "yarn", 16.0, 65536),
    (40, 2, 1, 1024, 1024, 0, True, "f32", 10000.0, "none", 1.0, 4096),
]


def inputs(torch, T, H, G, D, kind, far, seed=0):
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, far, (T,), generator=g, dtype=torch.int32)
    pos[0] = far - 1
    if T > 1:
        pos[1] = 0
    return torch.randn((T, H, D), generator=g).to(dtype), torch.randn((T, G, D), generator=g).to(dtype), pos


def compare(x, y, pos, rot, kind):
    f, m, span, interleaved = rot
    want, size = R.rotary(x.double().cpu().numpy(), pos.cpu().numpy(), f, m, span, interleaved)
    err = np.abs(y.double().cpu().numpy() - want)
    assert np.all(err <= SIN * size + HALF[kind] * np.abs(want))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rotary(case):
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    T, H, G, D, rotated, span, inter, kind, base, scaling, factor, far = case
    q, k, pos = inputs(torch, T, H, G, D, kind, far)
    ctx = Context(0)
    rot = hi.Rotary(D, rotated=rotated, span=span, interleaved=inter, base=base, scaling=scaling, factor=factor, original_length=4096)
    f, m = R.frequencies(rotated, span or rotated, base, scaling, factor, 4096, 32, 1, True)
    ref = (f, m, span or rotated, inter)
    qd, kd, pd = q.cuda(), k.cuda(), pos.cuda()
    qo, ko = torch.full_like(qd, 7.0), torch.full_like(kd, 7.0)
    torch.cuda.synchronize()
    hi.rotary_into(ctx, rot, pd, qd, qo, kd, ko)
    ctx.synchronize()
    compare(q, qo, pos, ref, kind)
    compare(k, ko, pos, ref, kind)
    # In place, the same bit for bit; the keys alone.
    hi.rotary_into(ctx, rot, pd, qd, qd, kd, kd)
    k2 = torch.full_like(kd, 7.0)
    hi.rotary_into(ctx, rot, pd, k.cuda(), k2)
    ctx.synchronize()
    assert torch.equal(qd, qo) and torch.equal(kd, ko) and torch.equal(k2, ko)


@pytest.mark.gpu
def test_slices_of_a_wider_product_and_several_leading_dimensions():
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    S, N, H, G, D = 3, 5, 4, 2, 64
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((S, N, (H + 2 * G) * D), generator=g)
    pos = torch.randint(0, 1000, (S, N), generator=g, dtype=torch.int32)
    ctx, rot = Context(0), hi.Rotary(D, base=10000.0)
    w, p = wide.cuda(), pos.cuda()
    before = w.clone()
    q = w[..., :H * D].unflatten(-1, (H, D))
    k = w[..., H * D:(H + G) * D].unflatten(-1, (G, D))
    torch.cuda.synchronize()
    hi.rotary_into(ctx, rot, p, q, q, k, k)
    ctx.synchronize()
    f, m = R.frequencies(D, D, 10000.0, "none", 1, 0, 32, 1, True)
    for part, lo, heads in ((q, 0, H), (k, H * D, G)):
        x = before[..., lo:lo + heads * D].reshape(S * N, heads, D)
        compare(x, part.reshape(S * N, heads, D), pos.reshape(-1), (f, m, D, False), "f32")
    assert torch.equal(w[..., (H + G) * D:], before[..., (H + G) * D:]), "the values were touched"
    # No tokens.
    e = torch.zeros((0, H, D), device="cuda:0")
    hi.rotary_into(ctx, rot, torch.zeros((0,), dtype=torch.int32, device="cuda:0"), e, e)


@pytest.mark.gpu
def test_recorded_and_replayed_with_new_positions():
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    q, k, pos = inputs(torch, 6, 8, 2, 128, "bf16", 100000)
    ctx, rot = Context(0), hi.Rotary(128, rotated=64, base=1e6)
    qd, kd, pd = q.cuda(), k.cuda(), pos.cuda()
    qo, ko = torch.zeros_like(qd), torch.zeros_like(kd)
    torch.cuda.synchronize()
    graph = ctx.capture(lambda: hi.rotary_into(ctx, rot, pd, qd, qo, kd, ko))
    f, m = R.frequencies(64, 64, 1e6, "none", 1, 0, 32, 1, True)
    for step in range(3):
        p = pos + 977 * step
        pd.copy_(p)
        torch.cuda.synchronize()
        graph.launch()
        ctx.synchronize()
        compare(q, qo, p, (f, m, 64, False), "bf16")
        compare(k, ko, p, (f, m, 64, False), "bf16")
    graph.close()


def table(**kw):
    from hydra_amd import _lib as L
    d = dict(head_dim=64, rotated=64, span=0, interleaved=0, scaling=0, original_length=4096, truncate=1, factor=1.0, beta_fast=32.0,
             beta_slow=1.0, base=10000.0)
    d.update(kw)
    out, m = (C.c_double * 512)(), C.c_float()
    rc = L.lib().hh_rotary_table(C.byref(L.RotaryDescC(**d)), out, C.byref(m))
    return rc, np.array(out[:d["rotated"] // 2]), m.value


@pytest.mark.parametrize("kw", [
    dict(), dict(rotated=16, span=64), dict(scaling=1, factor=8.0), dict(scaling=2, factor=32.0, base=150000.0),
    dict(scaling=2, factor=32.0, base=150000.0, truncate=0), dict(scaling=2, factor=4.0, original_length=16, rotated=24),
    dict(scaling=2, factor=2.5, base=1e7, head_dim=256, rotated=64), dict(scaling=2, factor=1.0),
])
def test_frequencies(kw):
    rc, got, m = table(**kw)
    assert rc == 0
    a = dict(rotated=64, span=0, base=10000.0, scaling=0, factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0, truncate=1)
    a.update({k: v for k, v in kw.items() if k in a})
    f, want = R.frequencies(a["rotated"], a["span"] or a["rotated"], a["base"], ["none", "linear", "yarn"][a["scaling"]], a["factor"],
                            a["original_length"], a["beta_fast"], a["beta_slow"], a["truncate"])
    np.testing.assert_allclose(got * 2 * np.pi, f, rtol=1e-13)
    assert abs(m - want) <= 2.0 ** -23 * want


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=60), -6), (dict(head_dim=0), -6), (dict(head_dim=2048), -6), (dict(rotated=3), -6), (dict(rotated=0), -6),
    (dict(rotated=66), -6), (dict(rotated=32, span=30), -6), (dict(span=66), -6), (dict(scaling=3), -1), (dict(base=1.0), -1),
    (dict(base=float("nan")), -1), (dict(scaling=1, factor=0.5), -1), (dict(scaling=1, factor=float("nan")), -1),
    (dict(scaling=2, factor=2.0, original_length=0), -1), (dict(scaling=2, factor=2.0, beta_fast=1.0), -1),
    (dict(scaling=2, factor=2.0, beta_slow=0.0), -1),
])
def test_descriptions_that_are_refused(kw, code):
    assert table(**kw)[0] == code


def call(rows=None, count=1, tokens=4, type_=0, ctx=1 << 20, positions=64, turns=64, magnitude=1.0, **kw):
    """The C entry's code; arguments that pass every check would reach the device, so none of these does."""
    from hydra_amd import _lib as L
    d = L.RotaryDescC(64, 64, 0, 0, 0, 0, 0, 1.0, 32.0, 1.0, 10000.0)
    for k, v in kw.items():
        setattr(d, k, v)
    r = [L.RotaryRowsC(64, 1024, 4, 0, 0), L.RotaryRowsC(4096, 8192, 2, 0, 0)]
    for i, change in (rows or {}).items():
        for k, v in change.items():
            setattr(r[i], k, v)
    return L.lib().hh_rotary(ctx, C.byref(d), turns, magnitude, type_, tokens, positions, (L.RotaryRowsC * 2)(*r), count)


@pytest.mark.parametrize("kw,code", [
    (dict(ctx=None), -1), (dict(type_=3), -1), (dict(tokens=-1), -1), (dict(tokens=(1 << 22) + 1), -1), (dict(count=0), -1),
    (dict(count=3), -1), (dict(positions=None), -1), (dict(turns=None), -1), (dict(turns=4), -2), (dict(magnitude=float("inf")), -1),
    (dict(rows={0: dict(x=None)}), -1), (dict(rows={0: dict(y=None)}), -1), (dict(rows={0: dict(x=8)}), -2),
    (dict(rows={0: dict(y=8)}), -2), (dict(rows={0: dict(heads=0)}), -6), (dict(rows={0: dict(heads=1025)}), -6),
    (dict(rows={0: dict(x_stride=128)}), -6), (dict(rows={0: dict(y_stride=255)}), -6), (dict(rows={0: dict(x_stride=257)}), -2),
    (dict(rows={0: dict(x_stride=260)}, type_=1), -2), (dict(rows={0: dict(y=64, y_stride=512)}), -1),
    (dict(rows={0: dict(x_stride=1 << 31)}), -6), (dict(rows={1: dict(y=1024)}, count=2), -1), (dict(rows={1: dict(x=None)}, count=2), -1),
    (dict(rotated=65), -6), (dict(rows={1: dict(y=64)}, count=2), -1), (dict(rows={0: dict(y=4096)}, count=2), -1),
])
def test_calls_that_are_refused(kw, code):
    assert call(**kw) == code
