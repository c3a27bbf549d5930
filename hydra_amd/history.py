"""Rotary positions, histories in 16, 8 and 4 bits, and attention over them, on the HydraHIP C ABI (`hh_rotary`,
`hh_history_write`, `hh_history_read`, `hh_history_attention`).

A step of S sequences, each with up to N new tokens (one, or a part of a prompt), around a model's layers:

    per layer   rotary_into(ctx, rotary, positions, q, q, k, k)
                history_write(ctx, history, k, v, counts)
                history_attention_into(ctx, history, q, counts, out)
    then        history_advance(ctx, history, counts, N)

Every function enqueues on the context's stream and returns at once; tensors that another stream wrote must be complete, and
must live until the call has run. Nothing of a call is kept: positions, lengths and counts are read on the device, so a call
recorded with `Context.capture` follows them. The conventions of formats, positions and windows are include/hydra_hip.h's.
"""
from __future__ import annotations

import ctypes as C
import operator
import struct

import torch

from ._lib import HistoryC, RotaryDescC, check, lib
from .layer import Context
from .speculative import ELEM, _cuda, _ptr, _same, _spaced

F16, BF16, MXFP8, MXFP4 = 1, 2, 3, 4
FORMATS = {"f16": F16, "bf16": BF16, "mxfp8": MXFP8, "mxfp4": MXFP4}
SCALINGS = {"none": 0, "linear": 1, "yarn": 2}
_I32, _F32 = torch.int32, torch.float32


def _i32(**values):
    """Raises unless the values are 32-bit whole numbers: ctypes would cut off what does not fit."""
    for name, v in values.items():
        if not hasattr(v, "__index__") or not -(1 << 31) <= operator.index(v) < 1 << 31:
            raise ValueError(f"{name} must be a 32-bit whole number, not {v!r}")


class Rotary:
    """A model's rotary frequencies (hh_rotary_desc, hh_rotary_table), kept on the device. `rotated` columns of each head turn (0: all),
    as pairs over the first `span` columns (0: rotated)."""

    def __init__(self, head_dim: int, rotated: int = 0, span: int = 0, interleaved: bool = False, base: float = 10000.0,
                 scaling: str = "none", factor: float = 1.0, original_length: int = 0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, truncate: bool = True, device="cuda:0"):
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {sorted(SCALINGS)}, not {scaling!r}")
        _i32(head_dim=head_dim, rotated=rotated, span=span, original_length=original_length)
        self.c = RotaryDescC(head_dim, rotated or head_dim, span, int(bool(interleaved)), SCALINGS[scaling], original_length,
                             int(bool(truncate)), factor, beta_fast, beta_slow, base)
        table, magnitude = (C.c_double * max(1, self.c.rotated // 2))(), C.c_float()
        check(lib().hh_rotary_table(C.byref(self.c), table, C.byref(magnitude)))
        self.head_dim, self.magnitude = head_dim, magnitude.value
        self.turns = torch.tensor(list(table), dtype=torch.float64, device=device)


_ROWS = (struct.Struct("PPiqq"), struct.Struct("PPiqqPPiqq"))      # one and two RotaryRowsC: an array of structures takes five times as long to make


def _tokens(t, name, shape, dtype, device):
    """The elements between tokens of a [..][heads][d] tensor with packed heads and equally spaced tokens."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} tensor {tuple(shape)} on {device}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    row = shape[-1] * shape[-2]
    if t.is_contiguous():
        return row
    s, lead = t.stride(), shape[:-2]
    if s[-1] != 1 or (s[-2] != shape[-1] and shape[-2] > 1):
        raise ValueError(f"{name} must have packed heads, not strides {s}")
    step, over = None, 1
    for n, st in zip(reversed(lead), reversed(s[:-2])):
        if n == 1:
            continue
        if step is None:
            step = st
        elif st != step * over:
            raise ValueError(f"{name}: the tokens must be equally spaced, not with strides {s}")
        over *= n
    if step is None:
        return row
    if step < row:
        raise ValueError(f"{name}: tokens {step} elements apart overlap")
    return step


def rotary_into(ctx: Context, rotary: Rotary, positions, q, q_out, k=None, k_out=None):
    """Turns q, and k, by their tokens' positions (hh_rotary). q, q_out [..][q_heads][d], k, k_out [..][kv_heads][d], of one type, with
    equally spaced tokens; positions int32 [..]. An output is its input or apart from every tensor of the call. Returns the outputs."""
    dev, dtype = q.device, q.dtype
    _cuda(ctx, dev)
    if dtype not in ELEM or q.dim() < 2 or q.shape[-1] != rotary.head_dim:
        raise ValueError(f"q must be fp32, fp16 or bf16 [..][heads][{rotary.head_dim}], not {dtype} {tuple(q.shape)}")
    if rotary.turns.device != dev:
        raise ValueError(f"the frequencies are on {rotary.turns.device}, q on {dev}")
    shape = q.shape
    _same(positions, "positions", shape[:-2], _I32, dev)
    x = _tokens(q, "q", shape, dtype, dev)
    rows = (q.data_ptr(), q_out.data_ptr(), shape[-2], x, x if q_out is q else _tokens(q_out, "q_out", shape, dtype, dev))
    if k is not None:
        if k_out is None:
            raise ValueError("k needs k_out")
        other = k.shape
        if other[:-2] != shape[:-2] or other[-1] != shape[-1]:
            raise ValueError(f"k {tuple(other)} must have the tokens and head_dim of q {tuple(shape)}")
        x = _tokens(k, "k", other, dtype, dev)
        rows += (k.data_ptr(), k_out.data_ptr(), other[-2], x, x if k_out is k else _tokens(k_out, "k_out", other, dtype, dev))
    n = positions.numel()
    if n:   # tensors of nothing have no address
        count = len(rows) // 5
        check(lib().hh_rotary(ctx.handle, C.byref(rotary.c), rotary.turns.data_ptr(), rotary.magnitude, ELEM[dtype], n,
                              positions.data_ptr(), _ROWS[count - 1].pack(*rows), count))
    return (q_out, k_out) if k is not None else q_out


class History:
    """One layer's history (hh_history). k, v [S][kv_heads][rows][..]: fp16 or bf16 numbers, or uint8 codes: with scales of 32
    columns a byte, [S][kv_heads][rows][head_dim / 32], of head_dim (MXFP8) or head_dim / 2 (MXFP4) bytes a row. lengths int32 [S]. The tensors are
    the caller's and are updated in place."""

    def __init__(self, k, v, lengths, k_scales=None, v_scales=None, ring: bool = False, pinned: int = 0):
        dev = k.device
        if k.dim() != 4:
            raise ValueError(f"k must be [S][kv_heads][rows][columns], not {tuple(k.shape)}")
        _same(k, "k", k.shape, k.dtype, dev)
        _same(v, "v", k.shape, k.dtype, dev)
        S, G, rows, width = k.shape
        if k.dtype is torch.uint8:
            if k_scales is None or v_scales is None or k_scales.dim() != 4:
                raise ValueError("a history of codes needs k_scales and v_scales [S][kv_heads][rows][head_dim / 32]")
            D = 32 * k_scales.shape[3]
            for t, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
                _same(t, name, (S, G, rows, D // 32), torch.uint8, dev)
            if width not in (D, D // 2):
                raise ValueError(f"rows of {width} bytes are neither 8 nor 4 bits of {D} columns")
            format_ = MXFP8 if width == D else MXFP4
        elif k.dtype in (torch.float16, torch.bfloat16):
            if k_scales is not None or v_scales is not None:
                raise ValueError("scales belong to a history of codes")
            D, format_ = width, F16 if k.dtype is torch.float16 else BF16
        else:
            raise ValueError(f"k must be fp16, bf16 or uint8 codes, not {k.dtype}")
        _same(lengths, "lengths", (S,), _I32, dev)
        _i32(rows=rows, pinned=pinned)
        self.k, self.v, self.k_scales, self.v_scales, self.lengths = k, v, k_scales, v_scales, lengths
        self.sequences, self.kv_heads, self.rows, self.head_dim, self.format = S, G, rows, D, format_
        self.ring, self.pinned, self.device = bool(ring), pinned, dev
        self.c = HistoryC(k.data_ptr(), v.data_ptr(), _ptr(k_scales), _ptr(v_scales), lengths.data_ptr(), S, G, D, format_, rows,
                          int(self.ring), pinned)

    @classmethod
    def empty(cls, sequences: int, kv_heads: int, rows: int, head_dim: int, format: str = "mxfp8", ring: bool = False,
              pinned: int = 0, lengths=None, device="cuda:0"):
        """A history of its own tensors, zeros, which are complete when this returns; its lengths are 0, or `lengths`, which layers may share."""
        if format not in FORMATS:
            raise ValueError(f"format must be one of {sorted(FORMATS)}, not {format!r}")
        if lengths is None:
            lengths = torch.zeros(sequences, dtype=_I32, device=device)
        shape = (sequences, kv_heads, rows)
        if format in ("f16", "bf16"):
            new = lambda: torch.zeros(shape + (head_dim,), dtype=torch.float16 if format == "f16" else torch.bfloat16, device=device)
            h = cls(new(), new(), lengths, ring=ring, pinned=pinned)
        else:
            code = lambda: torch.zeros(shape + (head_dim if format == "mxfp8" else head_dim // 2,), dtype=torch.uint8, device=device)
            scale = lambda: torch.zeros(shape + (head_dim // 32,), dtype=torch.uint8, device=device)
            h = cls(code(), code(), lengths, scale(), scale(), ring=ring, pinned=pinned)
        if h.device.type == "cuda":   # a context's stream does not wait for torch's, which fills them
            torch.cuda.current_stream(h.device).synchronize()
        return h


def history_write(ctx: Context, history: History, k, v, counts):
    """A step's keys and values into the history (hh_history_write): k, v fp32, fp16 or bf16 [S][N][kv_heads][d], spaced alike,
    which may be slices with equally spaced tokens; counts int32 [S]."""
    dev = history.device
    _cuda(ctx, dev)
    if k.dtype not in ELEM or k.dim() != 4:
        raise ValueError(f"k must be fp32, fp16 or bf16 [S][N][kv_heads][d], not {k.dtype} {tuple(k.shape)}")
    N = k.shape[1]
    shape = (history.sequences, N, history.kv_heads, history.head_dim)
    stride = _spaced(k, "k", k.shape, k.stride(), shape, k.dtype, dev)
    if _spaced(v, "v", v.shape, v.stride(), shape, k.dtype, dev) != stride:
        raise ValueError("k and v must be spaced alike")
    _same(counts, "counts", (history.sequences,), _I32, dev)
    check(lib().hh_history_write(ctx.handle, C.byref(history.c), ELEM[k.dtype], k.data_ptr(), v.data_ptr(), stride, N,
                                 counts.data_ptr()))


def history_read_into(ctx: Context, history: History, starts, counts, k, v):
    """Positions starts[s] + i, i < counts[s], as numbers into k and v, packed fp32, fp16 or bf16 [S][N][kv_heads][d]
    (hh_history_read); starts, counts int32 [S]. Returns k and v."""
    dev = history.device
    _cuda(ctx, dev)
    if k.dtype not in ELEM or k.dim() != 4:
        raise ValueError(f"k must be fp32, fp16 or bf16 [S][N][kv_heads][d], not {k.dtype} {tuple(k.shape)}")
    N = k.shape[1]
    for t, name in ((k, "k"), (v, "v")):
        _same(t, name, (history.sequences, N, history.kv_heads, history.head_dim), k.dtype, dev)
    _same(starts, "starts", (history.sequences,), _I32, dev)
    _same(counts, "counts", (history.sequences,), _I32, dev)
    check(lib().hh_history_read(ctx.handle, C.byref(history.c), ELEM[k.dtype], starts.data_ptr(), N, counts.data_ptr(),
                                k.data_ptr(), v.data_ptr()))
    return k, v


def history_advance(ctx: Context, history: History, counts, tokens: int):
    """history.lengths += counts (each 0..tokens), the end of a step (hh_history_advance)."""
    _cuda(ctx, history.device)
    _same(counts, "counts", (history.sequences,), _I32, history.device)
    _i32(tokens=tokens)
    check(lib().hh_history_advance(ctx.handle, C.byref(history.c), tokens, counts.data_ptr()))


_DESC = struct.Struct("iiiiiifq")            # a HistoryDescC


def _desc(history, tokens, q_heads, dtype, window, first, max_length, sm_scale, q_stride):
    try:
        return _DESC.pack(tokens, q_heads, ELEM[dtype], window, first, max_length,
                          history.head_dim ** -0.5 if sm_scale is None else sm_scale, q_stride)
    except struct.error as e:
        raise ValueError(f"tokens, window, first and max_length must be 32-bit whole numbers, sm_scale a number: {e}") from None


def history_attention_into(ctx: Context, history: History, q, counts, out, lse=None, sinks=None, window: int = 0, first: int = 0,
                           sm_scale: float | None = None, max_length: int = 0, prefix: History | None = None):
    """Attention of a step's tokens over the history that they have been written to, and a shared `prefix` before it
    (hh_history_attention). q, out fp32, fp16 or bf16 [S][N][q_heads][d] (q may be a slice with equally spaced tokens); counts int32 [S];
    sinks bf16 (or int16 bits) [q_heads]; lse fp32 [S][N][q_heads]. `out` may be a packed q. Returns `out`."""
    dev = history.device
    _cuda(ctx, dev)
    if q.dtype not in ELEM or q.dim() != 4:
        raise ValueError(f"q must be fp32, fp16 or bf16 [S][N][q_heads][d], not {q.dtype} {tuple(q.shape)}")
    S, N, H, D = q.shape
    if S != history.sequences or D != history.head_dim:
        raise ValueError(f"q {tuple(q.shape)} does not fit a history of {history.sequences} sequences and heads of {history.head_dim}")
    stride = _spaced(q, "q", q.shape, q.stride(), q.shape, q.dtype, dev)
    _same(out, "out", q.shape, q.dtype, dev)
    _same(counts, "counts", (S,), _I32, dev)
    if lse is not None:
        _same(lse, "lse", (S, N, H), _F32, dev)
    if sinks is not None:
        _same(sinks, "sinks", (H,), sinks.dtype if sinks.dtype is torch.int16 else torch.bfloat16, dev)
    if prefix is not None and prefix.device != dev:
        raise ValueError(f"the prefix is on {prefix.device}, the history on {dev}")
    d = _desc(history, N, H, q.dtype, window, first, max_length, sm_scale, stride)
    check(lib().hh_history_attention(ctx.handle, d, C.byref(history.c), None if prefix is None else C.byref(prefix.c),
                                     q.data_ptr(), counts.data_ptr(), _ptr(sinks), out.data_ptr(), _ptr(lse)))
    return out


def history_reserve(ctx: Context, history: History, tokens: int, q_heads: int, dtype, window: int = 0, first: int = 0,
                    max_length: int = 0, prefix: History | None = None):
    """Pre-sizes the context's workspace for calls that a graph will record (hh_history_reserve): attention of up to `tokens` tokens
    a sequence over histories up to max_length (0: the rows) and prefixes up to the rows of `prefix`."""
    if dtype not in ELEM:
        raise ValueError(f"dtype must be fp32, fp16 or bf16, not {dtype}")
    d = _desc(history, tokens, q_heads, dtype, window, first, max_length, None, 0)
    check(lib().hh_history_reserve(ctx.handle, d, C.byref(history.c), None if prefix is None else C.byref(prefix.c)))
