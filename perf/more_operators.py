"""Histories that are quantised as they are written, and what a serving step does around them, as cases that can
be timed and compared.

A case is one pass of one operator through `hydra_amd.history`:

  rotary     rotary positions of a step's queries and keys;
  store      a step's keys and values into a history, and the same rows read back as numbers;
  attend     a step's tokens (one a stream, or a prompt) over a history, with a window and first tokens that stay
             visible, or over all of it;
  prefix     the same for streams that share a long prefix.

With `own` false, `run` computes the same in elementary torch operations. All states share one context, as a
program has one. Histories are [sequence][kv head][row][column]: F16, BF16, or e4m3 / e2m1 codes (MXFP8, MXFP4) with an
e8m0 scale byte per 32 columns.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# A format's largest number, 448 and 6, as mantissa and exponent.
LARGEST = {"mxfp8": (0.875, 9), "mxfp4": (0.75, 3)}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _rotary(**kw):
    return {"kind": "rotary", "tokens": 1, "q_heads": 64, "kv_heads": 8, "head_dim": 64, "rotated": 64, "interleaved": False,
            "type": "f32", "base": 150000.0, "factor": 1.0, "yarn": False, "original_length": 4096, "far": 131072, **kw}


def _store(**kw):
    return {"kind": "store", "sequences": 1, "tokens": 1, "kv_heads": 8, "head_dim": 64, "type": "f32", "format": "mxfp8",
            "rows": 4096, "ring": False, "pinned": 0, **kw}


def _attend(**kw):
    return {"kind": "attend", "sequences": 1, "tokens": 1, "q_heads": 64, "kv_heads": 8, "head_dim": 64, "type": "f32",
            "format": "mxfp8", "length": 4096, "window": 0, "first": 0, "ring": False, "sinks": False, "shared": 0, **kw}


def listed():
    return [
        # One stream's next token: the smallest call. Frequencies blended for a context 32 times as long.
        _rotary(name="rotary_token", factor=32.0, yarn=True),
        # A decoding batch of many streams, interleaved pairs, 16-bit activations.
        _rotary(name="rotary_batch_interleaved", tokens=200, q_heads=24, kv_heads=4, head_dim=128, rotated=128, interleaved=True,
                type="f16", base=10000.0),
        # A long prompt, a quarter of each head rotated.
        _rotary(name="rotary_prompt_16384", tokens=16384, q_heads=16, kv_heads=2, head_dim=256, rotated=64, type="bf16",
                base=10000000.0),
        # A step of 32 streams into the rings of a sliding-window layer, fp32 from the projection.
        _store(name="store_step_32", sequences=32, rows=192, ring=True, pinned=4),
        # Two ragged prompts at 4 bits.
        _store(name="store_prompt_8000", sequences=2, tokens=8000, head_dim=128, type="bf16", format="mxfp4", rows=8100),
        # A step of 16 streams in a sliding-window layer: the 128 newest keys and the first 4.
        _attend(name="window_step_16", sequences=16, length=5000, window=128, first=4, ring=True, sinks=True),
        # A step of eight ragged streams at long histories, 8 bits.
        _attend(name="long_step_8", sequences=8, length=32768, sinks=True),
        # One stream at a very long history, 4 bits, heads of 256.
        _attend(name="long_step_131071", q_heads=16, kv_heads=2, head_dim=256, type="bf16", format="mxfp4", length=131071),
        # A prompt over the history that it has just been written to.
        _attend(name="prompt_4096", tokens=4096, type="bf16", length=0, sinks=True),
        # A part of each of two prompts, behind what came before, window and first tokens over a 16-bit history.
        _attend(name="prompt_window_1024", sequences=2, tokens=6001, q_heads=32, head_dim=128, type="f16", format="f16", length=2500,
                window=1024, first=4),
        # Four streams with a short instruction in common.
        _attend(name="prefix_4", kind="prefix", sequences=4, q_heads=24, kv_heads=4, format="f16", length=50, shared=1000),
        # Sixty-four streams behind one long document.
        _attend(name="prefix_64", kind="prefix", sequences=64, type="bf16", length=500, shared=24576, sinks=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, its logarithm uniform."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


HEADS = [(64, 8), (32, 8), (16, 2), (24, 4), (8, 8), (5, 1), (16, 1)]


def draw(rng):
    kind = rng.choice(["rotary", "store", "store", "attend", "attend", "attend", "attend", "prefix", "prefix"])
    q_heads, kv_heads = rng.choice(HEADS)
    head_dim = rng.choice([64, 64, 128, 256])
    type_ = rng.choice(["f32", "f16", "bf16"])
    format_ = rng.choice(["mxfp8", "mxfp8", "mxfp4", "bf16" if type_ == "bf16" else "f16"])
    if kind == "rotary":
        rotated = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 2 * rng.randint(1, head_dim // 2)])
        most = min(16384, 75_000_000 // ((q_heads + kv_heads) * head_dim * (2 if type_ == "f32" else 1)))
        scaled = rng.random() < 0.5
        return _rotary(tokens=_spread(rng, 1, most), q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rotated=rotated,
                       interleaved=rng.random() < 0.4, type=type_, base=rng.choice([10000.0, 150000.0, 1000000.0, 10000000.0]),
                       factor=round(rng.uniform(2, 40), 1) if scaled else 1.0, yarn=scaled and rng.random() < 0.6,
                       original_length=rng.choice([2048, 4096, 8192]), far=_spread(rng, 1000, 1000000))
    if kind == "store":
        tokens = _spread(rng, 1, 8192)
        sequences = _spread(rng, 1, max(1, min(64, 14_000_000 // (tokens * kv_heads * head_dim))))
        tokens = max(1, min(tokens, 14_000_000 // (sequences * kv_heads * head_dim)))
        ring = rng.random() < 0.4
        return _store(sequences=sequences, tokens=tokens, kv_heads=kv_heads, head_dim=head_dim, type=type_, format=format_,
                      rows=tokens + _spread(rng, 16, 1024), ring=ring, pinned=rng.choice([0, 1, 4, 16]) if ring else 0)
    shared = min(_spread(rng, 64, 32768), 32_000_000 // (kv_heads * head_dim)) if kind == "prefix" else 0
    shape = rng.choice(["step", "step", "few", "prompt"] if kind == "attend" else ["step", "step", "few"])
    tokens = {"step": 1, "few": rng.randint(2, 16), "prompt": _spread(rng, 17, 4096)}[shape]
    window = _spread(rng, 16, 2048) if kind == "attend" and rng.random() < 0.4 else 0
    # Histories of up to 80 million numbers a batch, and 130 GFLOP a pass.
    length = min(_spread(rng, 1, 4096 if kind == "prefix" or shape == "prompt" else 131072), 40_000_000 // (kv_heads * head_dim))
    sequences = _spread(rng, 1, max(1, min(64, 40_000_000 // ((length + tokens) * kv_heads * head_dim))))
    tokens = max(1, min(tokens, 130_000_000_000 // (4 * sequences * q_heads * head_dim * (length + shared + 2048))))
    return _attend(kind=kind, sequences=sequences, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                   type=type_, format=format_, length=length, window=window, first=rng.choice([0, 1, 4, 16]) if window else 0,
                   ring=window > 0 and rng.random() < 0.6, sinks=rng.random() < 0.5, shared=shared)


# ---- inputs ------------------------------------------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + part) & 0x7FFFFFFFFFFF)


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return torch.empty(shape, dtype=dtype, device=DEV).normal_(0.0, std, generator=g)


def _whole(g, low, high, shape):
    """Whole numbers low..high."""
    return torch.randint(low, high + 1, shape, dtype=torch.int32, device=DEV, generator=g)


def _ragged(g, sequences, most):
    """Numbers of up to `most`, from half of it: of a single sequence `most`."""
    if sequences == 1:
        return torch.full((1,), most, dtype=torch.int32, device=DEV)
    return _whole(g, (most + 1) // 2, most, (sequences,))


def _rows_like(g, shape, dtype):
    """Keys or values [..][heads][columns]: some columns of a head are larger than others."""
    size = torch.exp(0.4 * _normal(g, shape[-2:]))
    return (_normal(g, shape) * size).to(dtype)


def _filled(g, sequences, rows, kv_heads, head_dim, format_):
    """The codes and scales of a history that holds numbers in every row."""
    x = _rows_like(g, (sequences, rows, kv_heads, head_dim), torch.float32).transpose(1, 2)
    return _encode(x, format_)


def _rotary_inputs(case, seed):
    g = _generator(seed, 1)
    T, D, dtype = case["tokens"], case["head_dim"], TYPES[case["type"]]
    return {"q": _normal(g, (T, case["q_heads"], D), dtype), "k": _normal(g, (T, case["kv_heads"], D), dtype),
            "positions": _whole(g, 0, case["far"] - 1, (T,))}


def _store_inputs(case, seed):
    g = _generator(seed, 2)
    S, N, G, D = (case[k] for k in ("sequences", "tokens", "kv_heads", "head_dim"))
    dtype = TYPES[case["type"]]
    # A ring goes on for ever; a history of fixed rows has room for the step.
    start = _whole(g, 0, 100000 if case["ring"] else max(0, case["rows"] - N), (S,))
    return {"k_new": _rows_like(g, (S, N, G, D), dtype), "v_new": _rows_like(g, (S, N, G, D), dtype), "lengths": start,
            "counts": _ragged(g, S, N)}


def _attend_rows(case):
    """Rows of a stream's history: a ring holds the window of each of the step's tokens and a few more."""
    if case["ring"]:
        return case["first"] + case["window"] + case["tokens"] + 15
    return case["length"] + case["tokens"]


def _attend_inputs(case, seed):
    g = _generator(seed, 3)
    S, N, H, G, D = (case[k] for k in ("sequences", "tokens", "q_heads", "kv_heads", "head_dim"))
    s = {"q": _normal(g, (S, N, H, D), TYPES[case["type"]]), "counts": _ragged(g, S, N), "lengths": _ragged(g, S, case["length"]),
         "sinks": _normal(g, (H,), torch.bfloat16) if case["sinks"] else None}
    s["k"], s["k_scales"] = _filled(g, S, _attend_rows(case), G, D, case["format"])
    s["v"], s["v_scales"] = _filled(g, S, _attend_rows(case), G, D, case["format"])
    if case["shared"]:
        s["prefix_k"], s["prefix_k_scales"] = _filled(g, 1, case["shared"], G, D, case["format"])
        s["prefix_v"], s["prefix_v_scales"] = _filled(g, 1, case["shared"], G, D, case["format"])
        s["prefix_lengths"] = torch.full((1,), case["shared"], dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    if case["kind"] == "rotary":
        s = _rotary_inputs(case, seed)
        s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
        s["frequencies"], s["magnitude"] = _frequencies(case)
    elif case["kind"] == "store":
        s = _store_inputs(case, seed)
        S, _, G, D = s["k_new"].shape
        empty = torch.zeros((S, G, case["rows"], D), device=DEV)
        for name in ("k", "v"):
            s[name], s[name + "_scales"] = _encode(empty, case["format"])
            s[name + "_out"] = torch.zeros_like(s[name + "_new"])
    else:
        s = _attend_inputs(case, seed)
        s["out"], s["lse"] = torch.zeros_like(s["q"]), torch.zeros(s["q"].shape[:3], device=DEV)
    s["case"] = case
    torch.cuda.synchronize()
    return s


# ---- the framework's operators -------------------------------------------------------------------

_context = None


def _run_own(s):
    global _context
    from hydra_amd import history as hi
    if _context is None:
        from hydra_amd.layer import Context
        _context = Context(0)
    ctx, case, kind = _context, s["case"], s["case"]["kind"]
    if kind == "rotary":
        if "rotary" not in s:       # the frequencies that a program keeps for a model
            s["rotary"] = hi.Rotary(case["head_dim"], rotated=case["rotated"], interleaved=case["interleaved"], base=case["base"],
                                    scaling="yarn" if case["yarn"] else "linear" if case["factor"] != 1 else "none",
                                    factor=case["factor"], original_length=case["original_length"], device=DEV)
        hi.rotary_into(ctx, s["rotary"], s["positions"], s["q"], s["q_out"], s["k"], s["k_out"])
        return s["q_out"], s["k_out"]
    if "history" not in s:          # the handle that a program keeps for a layer's history
        s["history"] = hi.History(s["k"], s["v"], s["lengths"], k_scales=s["k_scales"], v_scales=s["v_scales"],
                                  ring=case["ring"], pinned=case["pinned"] if kind == "store" else case["first"] if case["ring"] else 0)
        if case.get("shared"):
            s["prefix"] = hi.History(s["prefix_k"], s["prefix_v"], s["prefix_lengths"], k_scales=s["prefix_k_scales"],
                                     v_scales=s["prefix_v_scales"])
    if kind == "store":
        hi.history_write(ctx, s["history"], s["k_new"], s["v_new"], s["counts"])
        hi.history_read_into(ctx, s["history"], s["lengths"], s["counts"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    hi.history_attention_into(ctx, s["history"], s["q"], s["counts"], s["out"], lse=s["lse"], sinks=s["sinks"],
                              window=case["window"], first=case["first"], max_length=case["length"] + case["tokens"],
                              prefix=s.get("prefix"))
    return s["out"], s["lse"]


def run(s):
    if own:
        return _run_own(s)
    return {"rotary": _rotary_plain, "store": _store_plain, "attend": _attend_plain, "prefix": _attend_plain}[s["case"]["kind"]](s)


# ---- plain forms -----------------------------------------------------------------------------------

def _frequencies(case):
    """Radians a position of each pair, in 64 bits, and the factor of what is rotated."""
    n, base, factor = case["rotated"], case["base"], case["factor"]
    f = base ** (-torch.arange(0, n, 2, dtype=torch.float64, device=DEV) / n)
    if not case["yarn"]:
        return f / factor, 1.0

    def pair_of(turns):     # the pair that turns this often within the original context
        return n * math.log(case["original_length"] / (2 * math.pi * turns)) / (2 * math.log(base))

    low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), n - 1)
    ramp = ((torch.arange(n // 2, dtype=torch.float64, device=DEV) - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _rotary_plain(s):
    case = s["case"]
    n = case["rotated"]
    angle = s["positions"].double().view(-1, 1, 1) * s["frequencies"]
    cos, sin = (s["magnitude"] * torch.cos(angle)).float(), (s["magnitude"] * torch.sin(angle)).float()
    for name in ("q", "k"):
        x = s[name][..., :n].float()
        a, b = (x[..., ::2], x[..., 1::2]) if case["interleaved"] else (x[..., :n // 2], x[..., n // 2:])
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1 if case["interleaved"] else -2).flatten(-2)
        s[name + "_out"][..., :n] = y.to(s[name].dtype)
        s[name + "_out"][..., n:] = s[name][..., n:]
    return s["q_out"], s["k_out"]


def _powers():
    """What the scale bytes stand for, up to 2^127."""
    return torch.tensor([2.0 ** (b - 127) for b in range(255)], device=DEV)


def _encode(x, format_):
    """fp32 [..][columns] -> codes and scale bytes: the least power of two under which nothing passes the format's largest
    number; numbers to the nearest, ties to even."""
    if format_ in ("f16", "bf16"):
        return x.to(TYPES[format_]).contiguous(), None
    groups = x.contiguous().view(*x.shape[:-1], -1, 32)
    top = groups.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)
    exponent = (exponent - LARGEST[format_][1] + (mantissa > LARGEST[format_][0])).clamp(min=-126)
    y = groups * _powers()[(127 - exponent).long()]
    scales = (exponent + 127).squeeze(-1).to(torch.uint8)
    if format_ == "mxfp8":
        return y.to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2), scales
    code = torch.zeros(y.shape, dtype=torch.uint8, device=x.device)
    for i in range(7):      # past the middle of two numbers; at it, to the one of even code
        middle = (E2M1[i] + E2M1[i + 1]) / 2
        code += (y.abs() >= middle) if i % 2 else (y.abs() > middle)
    code += 8 * torch.signbit(y)
    code = code.flatten(-2)
    return code[..., ::2] + 16 * code[..., 1::2], scales


def _decode(codes, scales):
    """The numbers in fp32."""
    if scales is None:
        return codes.float()
    if codes.shape[-1] == 32 * scales.shape[-1]:
        x = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1 + [-v for v in E2M1], device=codes.device)
        x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    return (x.view(*scales.shape, 32) * _powers()[scales.long()].unsqueeze(-1)).flatten(-2)


def _store_plain(s):
    case = s["case"]
    S, N, G, D = s["k_new"].shape
    rows, pinned = case["rows"], case["pinned"]
    position = s["lengths"].long().view(S, 1) + torch.arange(N, device=DEV)
    row = torch.where(position < pinned, position, pinned + (position - pinned) % (rows - pinned)) if case["ring"] else position
    i, t = (torch.arange(N, device=DEV) < s["counts"].view(S, 1)).nonzero(as_tuple=True)
    r = row[i, t]
    for name in ("k", "v"):
        codes, scales = _encode(s[name + "_new"].float(), case["format"])
        s[name][i, :, r] = codes[i, t]
        if scales is not None:
            s[name + "_scales"][i, :, r] = scales[i, t]
        held = _decode(s[name][i, :, r], None if scales is None else s[name + "_scales"][i, :, r])
        s[name + "_out"][i, t] = held.to(s[name + "_out"].dtype)
    return s["k_out"], s["v_out"]


def _attend_plain(s):
    case = s["case"]
    S, N, H, D = s["q"].shape
    G, window, first = case["kv_heads"], case["window"], case["first"]
    rows = s["k"].shape[2]
    row = torch.arange(rows, device=DEV)
    part = lambda name, i: _decode(s[name][i], None if s[name + "_scales"] is None else s[name + "_scales"][i])
    prefix = (part("prefix_k", 0), part("prefix_v", 0)) if case["shared"] else None
    for i in range(S):
        length, count = s["lengths"][i].long(), s["counts"][i]
        q_at = length + torch.arange(N, device=DEV).view(N, 1)
        at = row
        if case["ring"]:    # the newest position that a row holds
            span = rows - first
            newest = row + span * torch.div(length + count - 1 - row, span, rounding_mode="floor")
            at = torch.where(row < first, row, torch.where(newest < first, 2 ** 30, newest))
        sees = at <= q_at
        if window:
            sees = sees & ((at > q_at - window) | (at < first))
        k, v = part("k", i), part("v", i)
        if prefix is not None:
            k, v = torch.cat([prefix[0], k], 1), torch.cat([prefix[1], v], 1)
            sees = torch.cat([torch.ones((N, case["shared"]), dtype=torch.bool, device=DEV), sees], 1)
        q = s["q"][i].float().view(N, G, H // G, D).transpose(0, 1).reshape(G, -1, D)
        x = (torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(D))).view(G, N, H // G, -1)
        x = x.masked_fill(~sees.unsqueeze(1), -math.inf)
        sink = torch.full((H,), -math.inf, device=DEV) if s["sinks"] is None else s["sinks"].float()
        sink = sink.view(G, 1, H // G, 1)
        top = torch.maximum(x.amax(-1, keepdim=True), sink)
        p = torch.exp(x - top)
        den = p.sum(-1, keepdim=True) + torch.exp(sink - top)
        out = (torch.matmul(p.view(G, N * (H // G), -1), v).view(G, N, H // G, D) / den).transpose(0, 1).reshape(N, H, D)
        lse = (top + torch.log(den)).squeeze(-1).transpose(0, 1).reshape(N, H)
        real = torch.arange(N, device=DEV).view(N, 1) < count
        s["out"][i] = torch.where(real.unsqueeze(-1), out, s["out"][i].float()).to(s["out"].dtype)
        s["lse"][i] = torch.where(real, lse, s["lse"][i])
    return s["out"], s["lse"]


# ---- what a pass cannot do without ---------------------------------------------------------------

def _mean(sequences, most):
    return most if sequences == 1 else (most + (most + 1) // 2) / 2


def _held(format_, numbers):
    return numbers * {"f16": 2, "bf16": 2, "mxfp8": 1 + 1 / 32, "mxfp4": 0.5 + 1 / 32}[format_]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "rotary":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": n * case["head_dim"] * 2.0 * size + 4 * case["tokens"], "flops": n * case["rotated"] * 3.0}
    S, N, G, D = (case[k] for k in ("sequences", "tokens", "kv_heads", "head_dim"))
    tokens = _mean(S, N)
    if case["kind"] == "store":
        numbers = 2 * S * tokens * G * D
        return {"bytes": numbers * 2.0 * size + 2 * _held(case["format"], numbers), "flops": 0}
    H, length, window = case["q_heads"], _mean(S, case["length"]), case["window"]
    keys = length + tokens
    each = length + tokens / 2                      # keys that a token sees
    if window:
        each = min(each, window + case["first"])
        keys = min(keys, window + case["first"] + tokens)
    return {"bytes": _held(case["format"], 2.0 * (S * keys + case["shared"]) * G * D) + S * tokens * H * (2 * D * size + 4),
            "flops": 4.0 * S * tokens * H * D * (each + case["shared"])}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------

def _numbers(codes, scales):
    """What a history holds, from the bits."""
    if scales is None:
        return codes.double()
    c = codes.long()
    if c.shape[-1] == 32 * scales.shape[-1]:
        e, m, negative = (c >> 3) & 15, (c & 7).double(), c >> 7
        x = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.pow(2.0, (e - 10).double()))
    else:
        c = torch.stack([c % 16, c // 16], -1).view(*c.shape[:-1], -1)
        e, m, negative = (c >> 1) & 3, (c & 1).double(), c >> 3
        x = torch.where(e == 0, m / 2, (2 + m) * torch.pow(2.0, (e - 2).double()))
    x = torch.where(negative == 1, -x, x)
    return x * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, dim=-1)


def _exact_rotary(case, seed):
    s = _rotary_inputs(case, seed)
    n, factor = case["rotated"], case["factor"]
    outputs = []
    turns, m = [], 1.0
    for i in range(n // 2):
        f = math.exp(-2 * i / n * math.log(case["base"]))
        if case["yarn"]:
            m = 1 + math.log(factor) / 10
            index = [n / 2 * math.log(case["original_length"] / (b * 2 * math.pi)) / math.log(case["base"]) for b in (32, 1)]
            low, high = max(0, math.floor(index[0])), min(n - 1, math.ceil(index[1]))
            keep = 1 - min(1.0, max(0.0, (i - low) / (high - low if high > low else 0.001)))
            f = f * keep + f / factor * (1 - keep)
        else:
            f = f / factor
        turns.append(f)
    angle = s["positions"].double()[:, None, None] * torch.tensor(turns, dtype=torch.float64, device=DEV)
    for x in (s["q"].double(), s["k"].double()):
        first = torch.arange(n // 2, device=DEV) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else n // 2)
        turned = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.full_like(angle, m), angle)
        y = x.clone()
        y[..., first], y[..., second] = turned.real, turned.imag
        outputs.append(y)
    return tuple(outputs)


def _exact_store(case, seed):
    s = _store_inputs(case, seed)
    outputs = []
    for x in (s["k_new"].double(), s["v_new"].double()):
        if case["format"] in ("f16", "bf16"):
            y = x.to(TYPES[case["format"]]).double()
        else:
            if case["format"] == "mxfp8":
                held = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]
            else:
                held = E2M1
            held = torch.tensor(held, dtype=torch.float64, device=DEV)
            groups = x.reshape(-1, 32)
            top = groups.abs().amax(1, keepdim=True)
            scale = torch.pow(2.0, torch.round(torch.log2((top / held[-1]).clamp(min=2.0 ** -126))))
            scale = torch.where(top > held[-1] * scale, 2 * scale, scale)
            y = groups / scale
            above = torch.searchsorted(held, y.abs().contiguous()).clamp(max=len(held) - 1)
            below = (above - 1).clamp(min=0)
            up, down = held[above] - y.abs(), y.abs() - held[below]
            pick = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
            y = (torch.sign(y) * held[pick] * scale).view(x.shape)
        there = torch.arange(x.shape[1], device=DEV)[None, :] < s["counts"][:, None]
        outputs.append(y * there[:, :, None, None])
    return tuple(outputs)


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    S, N, H, D = s["q"].shape
    G, rows = case["kv_heads"], s["k"].shape[2]
    out = torch.zeros((S, N, H, D), dtype=torch.float64, device=DEV)
    lse = torch.zeros((S, N, H), dtype=torch.float64, device=DEV)
    for i in range(S):
        length, count = int(s["lengths"][i]), int(s["counts"][i])
        end = length + count
        position = torch.arange(end, device=DEV)
        if case["ring"]:
            span = rows - case["first"]
            position = position[(position < case["first"]) | (position >= end - span)]
            where = torch.where(position < case["first"], position, case["first"] + (position - case["first"]) % span)
        else:
            where = position
        mine = torch.arange(length, end, device=DEV)[:, None]
        mask = position[None, :] <= mine
        if case["window"]:
            mask &= (mine - position[None, :] < case["window"]) | (position[None, :] < case["first"])
        held = {}
        for name in ("k", "v"):
            sc = s[name + "_scales"]
            held[name] = _numbers(s[name][i][:, where], None if sc is None else sc[i][:, where])
            if case["shared"]:
                sc = s["prefix_" + name + "_scales"]
                held[name] = torch.cat([_numbers(s["prefix_" + name][0], None if sc is None else sc[0]), held[name]], 1)
        if case["shared"]:
            mask = torch.cat([torch.ones((count, case["shared"]), dtype=torch.bool, device=DEV), mask], 1)
        for h in range(H):
            g = h // (H // G)
            x = s["q"][i, :count, h].double() @ held["k"][g].T / math.sqrt(D)
            x = torch.where(mask, x, -math.inf)
            if s["sinks"] is not None:
                x = torch.cat([x, s["sinks"][h].double().expand(count, 1)], 1)
            lse[i, :count, h] = torch.logsumexp(x, 1)
            out[i, :count, h] = torch.softmax(x, 1)[:, :mask.shape[1]] @ held["v"][g]
    return out, lse


def exact(case, seed):
    return {"rotary": _exact_rotary, "store": _exact_store, "attend": _exact_attend, "prefix": _exact_attend}[case["kind"]](case, seed)
