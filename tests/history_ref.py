"""Plain implementations in 64 bits of the history operators: formats, rows of positions, attention, rotary positions."""
import math

import numpy as np

E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
HELD = {"mxfp8": np.array(E4M3), "mxfp4": np.array(E2M1)}


def encode(x, fmt):
    """Numbers [..][columns] -> (codes, scale bytes, the numbers that they stand for)."""
    x = np.asarray(x, np.float64)
    held = HELD[fmt]
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(g).max(-1, keepdims=True)
    odd = ~np.isfinite(top)
    e = np.full(top.shape, -126, np.int64)
    for i in np.argwhere(~odd & (top > 0)):
        i = tuple(i)
        p = int(math.floor(math.log2(top[i]))) - 10
        while top[i] > held[-1] * 2.0 ** p:
            p += 1
        e[i] = max(p, -126)
    y = np.abs(np.where(odd, 0.0, g)) / 2.0 ** e.astype(np.float64)
    above = np.searchsorted(held, y).clip(max=len(held) - 1)
    below = (above - 1).clip(min=0)
    up, down = held[above] - y, y - held[below]
    pick = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    values = np.where(odd, np.nan, np.copysign(held[pick] * 2.0 ** e.astype(np.float64), g)).reshape(x.shape)
    codes = (pick + len(held if fmt == "mxfp4" else np.zeros(128)) * np.signbit(np.where(odd, 0.0, g))).reshape(x.shape).astype(np.uint8)
    if fmt == "mxfp4":
        codes = codes[..., ::2] + 16 * codes[..., 1::2]
    return codes, np.where(odd, 255, e + 127)[..., 0].astype(np.uint8), values


def row_of(p, rows, ring, pinned):
    if not ring:
        return p if p < rows else -1
    return p if p < pinned else pinned + (p - pinned) % (rows - pinned)


def attention(q, k, v, lengths, counts, sinks, scale, window=0, first=0, ring=False, pinned=0, prefix=None, prefix_length=0):
    """{(s, i, head): output}, {..: lse} of the tokens that there are. k, v numbers [S][G][rows][D]; prefix (k, v) [G][rows][D]."""
    S, N, H, D = q.shape
    G, rows = k.shape[1], k.shape[2]
    out, lse = {}, {}
    for s in range(S):
        length = min(max(0, int(lengths[s])), 1 << 30)
        for i in range(min(N, max(0, int(counts[s])))):
            own = length + i
            low = max(0, own - window + 1) if window else 0
            last = own if ring else min(own, rows - 1)
            at = [row_of(p, rows, ring, pinned) for p in list(range(0, min(first, low, last + 1))) + list(range(low, last + 1))]
            for h in range(H):
                g = h // (H // G)
                kk, vv = k[s, g, at], v[s, g, at]
                if prefix is not None:
                    n = min(max(0, prefix_length), prefix[0].shape[1])
                    kk, vv = np.concatenate([prefix[0][g, :n], kk]), np.concatenate([prefix[1][g, :n], vv])
                x = scale * (kk @ q[s, i, h])
                if sinks is not None:
                    x = np.append(x, sinks[h])
                if x.size == 0:
                    out[s, i, h], lse[s, i, h] = np.zeros(D), -math.inf
                    continue
                top = x.max()
                e = np.exp(x - top)
                den = e.sum()
                out[s, i, h] = (e[:len(kk)] / den) @ vv
                lse[s, i, h] = top + math.log(den)
    return out, lse


def frequencies(rotated, span, base, scaling, factor, length, fast, slow, truncate):
    """(radians a position of each pair, the outputs' factor)."""
    f = [base ** (-2.0 * i / span) for i in range(rotated // 2)]
    if scaling == "none":
        return f, 1.0
    if scaling == "linear":
        return [x / factor for x in f], 1.0
    ends = [span / 2 * math.log(length / (2 * math.pi * b)) / math.log(base) for b in (fast, slow)]
    if truncate:
        ends = [math.floor(ends[0]), math.ceil(ends[1])]
    low, high = max(ends[0], 0), min(ends[1], span - 1)
    high = max(high, low + 0.001)
    ramp = [min(max((i - low) / (high - low), 0), 1) for i in range(len(f))]
    return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1


def rotary(x, positions, f, magnitude, span, interleaved):
    """x [T][heads][d] in 64 bits -> (turned, the sum of magnitudes that each output is made of)."""
    y, size = x.copy(), np.abs(x)
    for i, w in enumerate(f):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + span // 2)
        angle = positions.astype(np.float64) * w
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        y[..., a] = magnitude * (x[..., a] * c - x[..., b] * s)
        y[..., b] = magnitude * (x[..., b] * c + x[..., a] * s)
        size[..., a] = size[..., b] = magnitude * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size
