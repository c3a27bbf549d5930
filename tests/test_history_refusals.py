"""Calls around histories that the C entries and the Python functions refuse: nothing reaches a device."""
import ctypes as C

import pytest

from hydra_amd import _lib as L


def history(**kw):
    d = dict(k=1 << 20, v=2 << 20, k_scales=3 << 20, v_scales=4 << 20, lengths=5 << 20, sequences=2, kv_heads=2, head_dim=64,
             format=3, rows=100, ring=0, pinned=0)
    d.update(kw)
    return L.HistoryC(**d)


HISTORY = [
    (dict(sequences=0), -1), (dict(sequences=4097), -1), (dict(kv_heads=0), -6), (dict(kv_heads=257), -6), (dict(head_dim=96), -6),
    (dict(format=0), -1), (dict(format=5), -1), (dict(rows=0), -1), (dict(rows=(1 << 28) + 1), -1), (dict(pinned=-1), -1),
    (dict(pinned=3), -1), (dict(ring=1, pinned=100), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(lengths=None), -1),
    (dict(v=1 << 20), -1), (dict(k=(1 << 20) + 8), -2), (dict(v=(1 << 20) + 8), -2), (dict(k_scales=None), -1),
    (dict(v_scales=None), -1), (dict(v_scales=3 << 20), -1), (dict(k_scales=(3 << 20) + 4), -2), (dict(v_scales=(4 << 20) + 2), -2),
]


def write(h, ctx=64, type_=0, k=64, v=128, stride=0, tokens=3, counts=256):
    return L.lib().hh_history_write(ctx, None if h is None else C.byref(h), type_, k, v, stride, tokens, counts)


def read(h, ctx=64, type_=0, starts=64, tokens=3, counts=256, k=64, v=128):
    return L.lib().hh_history_read(ctx, None if h is None else C.byref(h), type_, starts, tokens, counts, k, v)


def attend(h, prefix=None, ctx=64, q=64, counts=256, out=128, entry="hh_history_attention", **kw):
    d = dict(tokens=3, q_heads=4, type=0, window=0, first=0, max_length=0, sm_scale=0.125, q_stride=0)
    d.update(kw)
    dc = L.HistoryDescC(**d)
    args = [ctx, C.byref(dc), None if h is None else C.byref(h), None if prefix is None else C.byref(prefix)]
    if entry == "hh_history_reserve":
        return L.lib().hh_history_reserve(*args)
    return L.lib().hh_history_attention(*args, q, counts, None, out, None)


@pytest.mark.parametrize("kw,code", HISTORY)
def test_histories(kw, code):
    h = history(**kw)
    assert write(h) == code and read(h) == code and attend(h) == code
    assert L.lib().hh_history_advance(64, C.byref(h), 3, 256) == code
    assert attend(h, entry="hh_history_reserve") == code
    assert L.lib().hh_last_error()


def test_missing_objects():
    assert write(None) == -1 and read(None) == -1 and attend(None) == -1
    h = history()
    assert write(h, ctx=None) == -1 and read(h, ctx=None) == -1 and attend(h, ctx=None) == -1
    assert L.lib().hh_history_advance(None, C.byref(h), 3, 256) == -1
    assert attend(h, ctx=None, entry="hh_history_reserve") == -1


@pytest.mark.parametrize("kw,code", [
    (dict(type_=3), -1), (dict(type_=-1), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(counts=None), -1), (dict(k=72), -2),
    (dict(v=72), -2), (dict(stride=127), -6), (dict(stride=130), -2), (dict(stride=132, type_=1), -2), (dict(stride=1 << 31), -6),
    (dict(tokens=0), -1), (dict(tokens=65537), -1),
])
def test_writes(kw, code):
    assert write(history(), **kw) == code


def test_too_many_heads():
    h = history(sequences=4096, kv_heads=65)
    assert write(h) == -1 and attend(h, q_heads=65) == -1
    assert attend(history(sequences=4096, kv_heads=64), tokens=129, q_heads=64) == -1
    assert attend(history(sequences=4096, kv_heads=64), tokens=128, q_heads=64, q=72) == -2


def test_too_many_tokens():
    assert write(history(sequences=4096), tokens=1025) == -1
    assert attend(history(sequences=4096), tokens=1025) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(type_=3), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(starts=None), -1), (dict(counts=None), -1), (dict(k=72), -2),
    (dict(v=72), -2), (dict(k=128), -1), (dict(tokens=0), -1), (dict(tokens=65537), -1),
])
def test_reads(kw, code):
    assert read(history(), **kw) == code


def test_advances():
    h = history()
    assert L.lib().hh_history_advance(64, C.byref(h), 0, 256) == -1
    assert L.lib().hh_history_advance(64, C.byref(h), 3, None) == -1
    assert L.lib().hh_history_advance(64, C.byref(h), 3, h.lengths) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(q_heads=0), -6), (dict(q_heads=5), -6), (dict(q_heads=34), -6), (dict(type=3), -1), (dict(window=-1), -1), (dict(first=-1, window=3), -1),
    (dict(first=2), -1), (dict(max_length=-1), -1), (dict(sm_scale=0.0), -1), (dict(sm_scale=float("nan")), -1),
    (dict(sm_scale=float("inf")), -1), (dict(sm_scale=3e38), -1), (dict(q_stride=255), -6), (dict(q_stride=257), -2), (dict(q_stride=260, type=2), -2),
    (dict(q_stride=1 << 31), -6), (dict(tokens=0), -1), (dict(tokens=65537), -1),
])
def test_attention_descriptions(kw, code):
    assert attend(history(), **kw) == code
    assert attend(history(), entry="hh_history_reserve", **kw) == code


def test_attention_pointers():
    h = history()
    for kw, code in ((dict(q=None), -1), (dict(counts=None), -1), (dict(out=None), -1), (dict(q=72), -2), (dict(out=72), -2)):
        assert attend(h, **kw) == code


def test_types_over_formats():
    for fmt, types in ((1, (0, 1)), (2, (2,)), (3, (0, 1, 2)), (4, (0, 1, 2))):
        for t in range(3):
            # An accepted pair goes on to the next check, the alignment of q.
            assert attend(history(format=fmt), type=t, q=72) == (-2 if t in types else -1), (fmt, t)


def test_rings_need_a_window_that_they_hold():
    ring = dict(ring=1, pinned=4)      # 96 rows besides the pinned
    assert attend(history(**ring)) == -1
    assert attend(history(**ring), window=95) == -1
    assert attend(history(**ring), window=94, q=72) == -2
    assert attend(history(**ring), window=97, tokens=1) == -1
    assert attend(history(**ring), window=96, tokens=1, q=72) == -2
    assert attend(history(**ring), window=2 ** 31 - 1, tokens=65536) == -1
    assert attend(history(**ring), window=10, first=5) == -1
    assert attend(history(**ring), window=10, first=4, q=72) == -2


def test_prefixes():
    h, p = history(), dict(sequences=1)
    assert attend(h, history(**p), q=72) == -2
    for kw, code in ((dict(sequences=2), -1), (dict(ring=1), -1), (dict(kv_heads=4), -6), (dict(head_dim=128), -6), (dict(format=4), -6),
                     (dict(rows=0), -1), (dict(k=None), -1)):
        assert attend(h, history(**{**p, **kw})) == code
    assert attend(h, history(**p), window=5) == -1


def test_python():
    import torch
    from hydra_amd import history as hi
    n = torch.zeros(2, dtype=torch.int32)
    code = lambda *shape: torch.zeros(shape, dtype=torch.uint8)
    k8, s8 = code(2, 3, 10, 64), code(2, 3, 10, 2)
    h = hi.History(k8, k8.clone(), n, s8, s8.clone())
    assert (h.sequences, h.kv_heads, h.rows, h.head_dim, h.format) == (2, 3, 10, 64, hi.MXFP8)
    assert hi.History(code(2, 3, 10, 32), code(2, 3, 10, 32), n, s8, s8.clone()).format == hi.MXFP4
    x = torch.zeros((2, 3, 10, 128), dtype=torch.bfloat16)
    assert hi.History(x, x.clone(), n).format == hi.BF16
    bad = [lambda: hi.History(k8, k8.clone(), n),                                   # codes without scales
           lambda: hi.History(x, x.clone(), n, s8, s8.clone()),                     # numbers with scales
           lambda: hi.History(x.float(), x.float(), n),
           lambda: hi.History(k8[..., :48].contiguous(), k8[..., :48].contiguous(), n, s8, s8.clone()),
           lambda: hi.History(k8[:, :, ::2], k8[:, :, ::2], n, s8, s8.clone()),     # rows apart
           lambda: hi.History(k8, k8.clone(), n.long(), s8, s8.clone()),
           lambda: hi.History(k8, k8.clone(), n, s8, s8[:, :, :5].contiguous()),
           lambda: hi.History(x[0], x[0], n),
           lambda: hi.History.empty(1, 1, 4, 64, format="int8", device="cpu"),
           lambda: hi.Rotary(64, scaling="other", device="cpu")]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(L.HydraHIPError):
        hi.Rotary(64, rotated=63, device="cpu")
    assert hi._tokens(x, "x", x.shape, torch.bfloat16, x.device) == 10 * 128
    wide = torch.zeros((2, 5, 9 * 64))
    q = wide[..., 64:5 * 64].unflatten(-1, (4, 64))
    assert hi._tokens(q, "q", q.shape, torch.float32, q.device) == 9 * 64
    for t in (q[:, ::2].expand(2, 3, 4, 64)[:, :, :, ::2], q.transpose(2, 3), q[:, :3], q[:1, :1].expand(2, 5, 4, 64)):
        with pytest.raises(ValueError):
            hi._tokens(t, "q", t.shape, torch.float32, q.device)


def test_python_describes_calls_as_the_header_does():
    """What is packed for the C entries is the structures', and what does not fit them is refused."""
    import torch
    from hydra_amd import history as hi
    for n in (1, 2):
        v = (64, 128, 3, 1 << 33, 5, 4096, 8192, 7, 9, 1 << 34)[:5 * n]
        a = (L.RotaryRowsC * n).from_buffer_copy(hi._ROWS[n - 1].pack(*v))
        assert tuple(getattr(a[i], f) for i in range(n) for f, _ in L.RotaryRowsC._fields_) == v
        assert hi._ROWS[n - 1].size == C.sizeof(a)
    h = hi.History.empty(2, 3, 10, 64, device="cpu")
    d = L.HistoryDescC.from_buffer_copy(hi._desc(h, 1, 2, torch.float16, 3, 4, 5, 0.25, 1 << 33))
    assert hi._DESC.size == C.sizeof(d)
    assert [getattr(d, f) for f, _ in L.HistoryDescC._fields_] == [1, 2, 1, 3, 4, 5, 0.25, 1 << 33]
    for kw in (dict(window=1 << 31), dict(first=-(1 << 31) - 1), dict(max_length=1 << 40), dict(sm_scale="1"), dict(tokens=1.5)):
        a = dict(tokens=1, window=0, first=0, max_length=0, sm_scale=1.0)
        a.update(kw)
        with pytest.raises(ValueError):
            hi._desc(h, a["tokens"], 6, torch.float32, a["window"], a["first"], a["max_length"], a["sm_scale"], 0)
    d = L.HistoryDescC.from_buffer_copy(hi._desc(h, 1, 2, torch.float16, 0, 0, 0, 1e39, 0))
    assert d.sm_scale == float("inf")        # which the entry refuses
