"""Calls around histories whose outputs overlap each other or an input, wherever they begin, are refused; nothing reaches a device."""
import ctypes as C
import random

import pytest

from hydra_amd import _lib as L

EHIP = -4
# Every byte −1: a context of no device, so that a call that passes the checks goes no further than choosing it.
NO_DEVICE = C.create_string_buffer(b"\xff" * 65536, 65536)
CTX, BASE = C.addressof(NO_DEVICE), 1 << 30


def history(**kw):
    d = dict(k=1 << 20, v=2 << 20, k_scales=3 << 20, v_scales=4 << 20, lengths=5 << 20, sequences=2, kv_heads=2, head_dim=64,
             format=3, rows=100, ring=0, pinned=0)
    d.update(kw)
    return L.HistoryC(**d)


def attend(tokens, q, q_stride, out, lse, type_=0, sequences=2):
    d = L.HistoryDescC(tokens, 2, type_, 0, 0, 0, 0.125, q_stride)
    return L.lib().hh_history_attention(CTX, C.byref(d), C.byref(history(sequences=sequences)), None, BASE + q, 256, None, BASE + out,
                                        None if lse is None else BASE + lse)


def held(at, step, size, n):
    return {(at + i * step) // 4 + j for i in range(n) for j in range(size // 4)}


@pytest.mark.parametrize("seed", range(4))
def test_attention(seed):
    rng = random.Random(seed)
    seen = {True: 0, False: 0}
    for _ in range(400):
        type_, tokens, S = rng.randrange(3), rng.choice([1, 2, 3]), rng.choice([1, 2])
        size, n = (4, 2, 2)[type_], tokens * S
        row = 2 * 64 * size
        stride = rng.choice([128, 128, 128 + 64, 256, 384, 520])
        q, out = 16 * rng.randint(0, 150), 16 * rng.randint(0, 300)
        if rng.random() < 0.3:
            out = q
        lse = None if rng.random() < 0.4 else 4 * rng.randint(0, 1500)
        a, b = held(q, stride * size, row, n), held(out, row, row, n)
        c = set() if lse is None else held(lse, 8, 8, n)
        bad = bool(a & b and not (q == out and (stride == 128 or n == 1)) or c & a or c & b)
        seen[bad] += 1
        assert attend(tokens, q, stride, out, lse, type_, S) == (-1 if bad else EHIP), (tokens, S, q, stride, out, lse, type_)
    assert min(seen.values()) > 20


def read(k, v, type_=0):
    return L.lib().hh_history_read(CTX, C.byref(history()), type_, 64, 3, 256, BASE + k, BASE + v)


def test_reads():
    bytes_ = 2 * 3 * 2 * 64 * 4
    assert read(0, bytes_) == EHIP and read(bytes_, 0) == EHIP
    assert read(0, bytes_ - 16) == -1 and read(bytes_ - 16, 0) == -1 and read(0, 16) == -1
    assert read(0, bytes_ // 2, 1) == EHIP and read(0, bytes_ // 2 - 16, 2) == -1


def write(**kw):
    return L.lib().hh_history_write(CTX, C.byref(history(**kw)), 0, 64, 1 << 16, 0, 3, 256)


def test_histories_of_overlapping_tensors():
    codes, scales = 2 * 2 * 100 * 64, 2 * 2 * 100 * 2
    assert write() == EHIP
    for k in (1 << 20, 2 << 20):     # at both ends of each other tensor
        for name, size in (("v", codes), ("k_scales", scales), ("v_scales", scales), ("lengths", 8)):
            if name == "v" and k == 2 << 20:
                continue
            kw = dict(k=k, v=7 << 20)
            align = {"v": 16, "lengths": 8}.get(name, 8)
            assert write(**{**kw, name: k + codes}) == EHIP and write(**{**kw, name: k - size}) == EHIP
            assert write(**{**kw, name: k + codes - align}) == -1 and write(**{**kw, name: k - size + align}) == -1 or size == align
    assert write(k_scales=(4 << 20) - scales + 8) == -1 and write(v_scales=(2 << 20) + 16) == -1
    assert write(lengths=(3 << 20) + 4) == -1
    f16 = dict(format=1, k_scales=None, v_scales=None)
    assert write(**f16) == EHIP and write(**f16, v=(1 << 20) + 2 * codes) == EHIP and write(**f16, v=(1 << 20) + 2 * codes - 16) == -1


def test_advances():
    advance = lambda counts: L.lib().hh_history_advance(CTX, C.byref(history()), 3, (5 << 20) + counts)
    assert advance(8) == EHIP and advance(-8) == EHIP and advance(4) == -1 and advance(-4) == -1 and advance(0) == -1
