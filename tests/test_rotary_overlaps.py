"""Outputs of rotary positions (hh_rotary) that overlap a tensor of the call, wherever they begin, are refused; tensors that lie in
each other's gaps are not."""
import ctypes as C
import random

import pytest

EHIP = -4
# Every byte −1: a context of no device, so that a call that passes the checks goes no further than choosing it.
NO_DEVICE = C.create_string_buffer(b"\xff" * 65536, 65536)
BASE = 1 << 30


def call(tokens, rows, type_=0, head_dim=8):
    from hydra_amd import _lib as L
    d = L.RotaryDescC(head_dim, head_dim, 0, 0, 0, 0, 0, 1.0, 32.0, 1.0, 10000.0)
    r = (L.RotaryRowsC * 2)(*[L.RotaryRowsC(BASE + x, BASE + y, h, xs, ys) for x, y, h, xs, ys in rows])
    return L.lib().hh_rotary(C.addressof(NO_DEVICE), C.byref(d), 64, 1.0, type_, tokens, 64, r, len(rows))


def held(at, stride, heads, tokens, size):
    return {at // 16 + t * stride * size // 16 + i for t in range(tokens) for i in range(heads * 8 * size // 16)}


def overlaps(tokens, rows, size):
    t = [(held(x, xs, h, tokens, size), held(y, ys, h, tokens, size), x == y) for x, y, h, xs, ys in rows]
    if any(t[i][1] & t[j][0] for i in range(len(t)) for j in range(len(t)) if i != j or not t[i][2]):
        return True
    return len(t) == 2 and bool(t[0][1] & t[1][1])


@pytest.mark.parametrize("seed", range(8))
def test_every_layout(seed):
    rng = random.Random(seed)
    seen = {True: 0, False: 0}
    for _ in range(400):
        type_ = rng.randrange(3)
        size, tokens = (4, 2, 2)[type_], rng.choice([1, 2, 3, 7])
        step = 4 if type_ == 0 else 8
        common = step * rng.randint(2, 24)
        rows = []
        for _ in range(rng.randint(1, 2)):
            h = rng.randint(1, 2)
            stride = lambda: max(h * 8, common if rng.random() < 0.7 else step * rng.randint(2, 24))
            xs, ys, x, y = stride(), stride(), 16 * rng.randint(0, 200), 16 * rng.randint(0, 200)
            rows.append((x, x, h, xs, xs) if rng.random() < 0.3 else (x, y, h, xs, ys))
        if any(x == y and xs != ys for x, y, _, xs, ys in rows):
            continue
        bad = overlaps(tokens, rows, size)
        seen[bad] += 1
        assert call(tokens, rows, type_) == (-1 if bad else EHIP), (tokens, rows, type_)
    assert min(seen.values()) > 20


def test_large_calls():
    n, row = 1 << 22, 64
    for rows, bad in (([(0, 0, 8, row, row)], False), ([(0, 4 * row * n, 8, row, row)], False), ([(0, 4 * row * n - 16, 8, row, row)], True),
                      ([(0, 4 * row, 8, 2 * row, 2 * row)], False), ([(0, 4 * row + 16, 8, 2 * row, 2 * row)], True),
                      ([(0, 4 * row, 8, 2 * row, 4 * row)], False), ([(0, 4 * row - 16, 8, 1 << 30, 1 << 29)], True)):
        assert call(n, rows) == (-1 if bad else EHIP), rows
    assert call(0, [(0, 16, 8, row, row)]) == 0      # no tokens, no bytes


@pytest.mark.gpu
def test_outputs_in_gaps():
    """Turned into the gaps between the inputs' tokens: as into memory of their own."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx, rot = Context(0), hi.Rotary(64)
    T, H, G, D = 37, 4, 2, 64
    wide = torch.randn((T, 2 * (H + G), D), device="cuda:0")
    pos = torch.arange(T, dtype=torch.int32, device="cuda:0") * 31
    q, qo, k, ko = wide[:, :H], wide[:, H:2 * H], wide[:, 2 * H:2 * H + G], wide[:, 2 * H + G:]
    want = [torch.empty((T, h, D), device="cuda:0") for h in (H, G)]
    torch.cuda.synchronize()
    hi.rotary_into(ctx, rot, pos, q, want[0], k, want[1])
    hi.rotary_into(ctx, rot, pos, q, qo, k, ko)
    ctx.synchronize()
    assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
