"""Verification of drafted tokens (hh_draft_verify) against the rule as it is stated, one sequence after
the other in 64 bits: paths, counts and tokens are equal. The random numbers are inputs; the kernel's
probabilities and sums are fp64 (errors near 1e-13), so that a border falls between the two once in 1e8 draws."""
import ctypes as C

import numpy as np
import pytest

MODES = ["given", "iid", "distinct"]


def softmax(x, t):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        e = np.where(x == top, 1.0, np.exp((x - top) / t))
    return e / e.sum()


def reference(target, draft, mode, tokens, parents, counts, u, uf, t, most):
    """(path, accepted, next) of one sequence."""
    N, V = target.shape
    count = min(max(int(counts), 0), N)
    path = [-1] * N
    if count == 0:
        return path, 0, -1
    cur, line = 0, [0]
    while True:
        kids = [n for n in range(cur + 1, count) if parents[n] == cur][:most]
        found = None
        if t == 0:
            x = np.where(np.isnan(target[cur]), -np.inf, target[cur].astype(np.float64))
            best = int(np.argmax(x)) if x.max() > -np.inf else -1
            found = next((n for n in kids if tokens[n] == best and best >= 0), None)
            after = best
        else:
            p = full = softmax(target[cur], t)
            q = None if mode == "given" else softmax(draft[cur], t)
            for n in kids:
                x = int(tokens[n])
                qx = 1.0 if q is None else (q[x] if 0 <= x < V else 0.0)
                if 0 <= x < V and float(u[n]) * qx < p[x]:
                    found = n
                    break
                p = p.copy() if q is None else np.maximum(p - q, 0)
                if 0 <= x < V:
                    p[x] = 0
                if p.sum() > 0:
                    p /= p.sum()
                if mode == "distinct" and 0 <= x < V:
                    q = q.copy()
                    q[x] = 0
                    if q.sum() > 0:
                        q /= q.sum()
            if found is None:
                if not p.sum() > 0:
                    p = full
                c = np.cumsum(p)
                after = -1 if not c[-1] > 0 else min(int((c <= float(uf) * c[-1]).sum()), int(np.nonzero(p)[0][-1]))
        if found is None:
            path[:len(line)] = line
            return path, len(line), after
        cur = found
        line.append(cur)


def inputs(torch, S, N, V, kind, mode, branch, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[kind]
    target = torch.empty((S, N, V)).exponential_(1.0, generator=g) * spread
    draft = (target + 0.6 * torch.randn((S, N, V), generator=g)).to(dt)
    target = target.to(dt)
    parents = torch.tensor([[(i - 1) // branch for i in range(N)]] * S, dtype=torch.int32)
    tokens = torch.zeros((S, N), dtype=torch.int32)
    for s in range(S):
        for n in range(1, N):
            p = softmax(draft[s, (n - 1) // branch].float().numpy(), 1.0)
            if mode == "iid":
                tokens[s, n] = int(np.searchsorted(np.cumsum(p), float(torch.rand((), generator=g))).clip(0, V - 1))
            else:
                tokens[s, n] = int(np.argsort(-p, kind="stable")[min((n - 1) % branch, V - 1)])
    return dict(target=target, draft=None if mode == "given" else draft, tokens=tokens, parents=parents,
                counts=torch.full((S,), N, dtype=torch.int32), u=torch.rand((S, N), generator=g), uf=torch.rand((S,), generator=g))


def call(torch, ctx, t, mode, temperature=1.0, most=0, target=None, draft=None):
    from hydra_amd import speculative as sp
    d = {k: None if x is None else x.to("cuda:0") for k, x in t.items()}
    S, N, _ = t["target"].shape
    path = torch.full((S, N), 99, dtype=torch.int32, device="cuda:0")
    acc, nxt = (torch.full((S,), 99, dtype=torch.int32, device="cuda:0") for _ in range(2))
    torch.cuda.synchronize()
    sp.draft_verify_into(ctx, d["target"] if target is None else target, d["tokens"], d["parents"], d["counts"], d["u"], d["uf"],
                         path, acc, nxt, draft=d["draft"] if draft is None else draft, distinct=mode == "distinct",
                         temperature=temperature, max_children=most)
    ctx.synchronize()
    return path.cpu(), acc.cpu(), nxt.cpu()


def check(t, mode, got, temperature=1.0, most=0):
    num = lambda x: None if x is None else x.float().numpy()
    for s in range(t["target"].shape[0]):
        want = reference(num(t["target"][s]), None if t["draft"] is None else num(t["draft"][s]), mode, t["tokens"][s].tolist(),
                         t["parents"][s].tolist(), int(t["counts"][s]), t["u"][s], t["uf"][s], temperature, most or 10**6)
        assert (got[0][s].tolist(), int(got[1][s]), int(got[2][s])) == (want[0], want[1], want[2]), f"sequence {s}"


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("S,N,V,kind,branch,temperature", [
    (1, 1, 1, "f32", 1, 1.0),
    (3, 2, 2, "f16", 1, 1.0),
    (4, 6, 7, "f32", 2, 0.7),
    (5, 9, 64, "bf16", 3, 1.0),
    (2, 64, 257, "f32", 1, 1.3),         # a line of 64
    (2, 64, 300, "f16", 63, 1.0),        # 63 children of one node
    (4, 21, 2048, "f32", 4, 0.5),
    (3, 13, 2049, "bf16", 3, 1.0),
    (2, 9, 12345, "f32", 2, 0.9),
    (1, 5, 100003, "f16", 4, 1.0),
    (2, 9, 131073, "f32", 2, 0.9),       # chunks of 4096, a tail of one
    (3, 6, 140001, "bf16", 5, 1.1),
])
def test_verify(mode, S, N, V, kind, branch, temperature):
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] verify {mode} S={S} N={N} V={V} {kind} branch={branch}", flush=True)
    ctx = Context(0)
    try:
        for seed in range(3 if V < 50000 else 1):
            t = inputs(torch, S, N, V, kind, mode, branch, seed * 7 + V)
            check(t, mode, call(torch, ctx, t, mode, temperature), temperature)
            for most in (1, 2):
                check(t, mode, call(torch, ctx, t, mode, temperature, most), temperature, most)
    finally:
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
def test_many_leaves(mode):
    """Logits enough (71 MB) that the leaves' statistics wait for the rounds: paths that end at leaves and at nodes with
    children, counts from none on, leaves of nothing, NaN and +inf, nodes without a parent, more children than are tried."""
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        S, N, V = 72, 63, 4003
        print(f"[gpu] verify many leaves {mode}", flush=True)
        t = inputs(torch, S, N, V, "f32", mode, 3, 5)
        t["counts"][:8] = torch.tensor([0, 1, 2, 5, 40, 64, -3, 62], dtype=torch.int32)
        for s in range(8, 24):                                   # every leaf of these, one way each
            T, way = t["target"][s, 21:], s % 4
            if way == 0:
                T[:] = float("-inf")
            elif way == 1:
                T[:, ::3] = float("nan")
            elif way == 2:
                T[:, [5, 4002]] = float("inf")
            else:
                T[:, 1:] = float("-inf")
        t["parents"][24, 3::5] = torch.tensor([-7, 80, 62, -1, 63, -1, -1, 99, 60, 61, -1, 0][:len(range(3, 63, 5))], dtype=torch.int32)
        t["u"][8:24] *= 0.2                                      # mostly accepted: paths down to the leaves
        for most in (0, 2):
            check(t, mode, call(torch, ctx, t, mode, 0.9, most), 0.9, most)
    finally:
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_greedy(kind):
    """Ties go to the lowest token; the random numbers are not needed."""
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        for V in (1, 5, 1000, 4097, 50001):
            t = inputs(torch, 6, 10, V, kind, "given", 3, V)
            t["target"][0, :, : V // 2] = t["target"][0].amax()      # ties
            t["target"][1, 0] = float("-inf")
            t["target"][2, 0, 0] = float("nan")
            t["target"][3, 0, V - 1] = float("inf")
            t["tokens"][4, 1:] = -1
            best = torch.where(t["target"].isnan(), float("-inf"), t["target"].float()).argmax(-1)
            t["tokens"][5, 1:] = best[5][t["parents"][5, 1:].long()].int()
            for most in (0, 1, 2):
                check(t, "given", call(torch, ctx, t, "given", 0.0, most), 0.0, most)
            chain = dict(t, parents=torch.arange(-1, 9, dtype=torch.int32).expand(6, 10).contiguous())
            chain["tokens"] = torch.cat([t["tokens"][:, :1], best[:, :-1].int()], 1).contiguous()
            chain["tokens"][1, 5] += 1
            check(chain, "given", call(torch, ctx, chain, "given", 0.0, 1), 0.0, 1)
            without = dict(t, u=None, uf=None)
            assert all(torch.equal(a, b) for a, b in zip(call(torch, ctx, without, "given", 0.0), call(torch, ctx, t, "given", 0.0)))
    finally:
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
def test_odd_rows_and_tokens(mode):
    """Masked vocabularies, NaN, +inf, rows of nothing, tokens outside the vocabulary or tried twice, a draft equal to
    the target, no overlap at all, counts from none to too many, parents that are no earlier nodes."""
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    inf, nan = float("inf"), float("nan")
    try:
        S, N, V = 12, 7, 1500
        for seed in range(4):
            t = inputs(torch, S, N, V, "f32", mode, 3, seed)
            T, D = t["target"], t["draft"]
            T[0, :, 10:] = -inf                              # a top-k filter
            T[1, :, ::2] = nan
            T[2, 0, [3, 1400]] = inf
            T[3, 0] = -inf                                   # nothing to draw
            T[4, :, 700:] = -inf
            t["tokens"][5, 1:] = torch.tensor([-1, V, 2**31 - 1, -5, 0, 1], dtype=torch.int32)
            t["tokens"][6, 2:4] = t["tokens"][6, 1]
            t["counts"][7], t["counts"][8], t["counts"][9] = 0, 3, 100
            t["parents"][9] = torch.tensor([3, 0, 2, -4, 1, 9, 1], dtype=torch.int32)
            if D is not None:
                D[4, :, :700] = -inf                         # no token in common
                D[10] = T[10]
                D[11, 0] = nan
            T[8, 0] = torch.finfo(torch.float32).min    # rows masked by the lowest value: all of it, and but for two
            T[8, 1:] = torch.finfo(torch.float32).min
            T[8, 1:, [77, 901]] = torch.tensor([1.0, 2.0])
            T[5, 3:] *= 1e30                                # far apart
            t["u"][10] = 1 - 2.0 ** -24
            t["uf"][0], t["uf"][1] = 0.0, 1 - 2.0 ** -24
            check(t, mode, call(torch, ctx, t, mode))
    finally:
        ctx.close()


@pytest.mark.gpu
@pytest.mark.parametrize("mode,branch", [("iid", 1), ("iid", 2), ("distinct", 2), ("given", 2)])
def test_tokens_are_distributed_as_the_target(mode, branch):
    """The first token that comes out of 4096 sequences of one distribution: chi-square against it. 7 degrees of
    freedom: above 29.9 once in 10^4 by chance (the seed is fixed)."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    S, V, N = 4096, 8, 1 + branch
    g = torch.Generator().manual_seed(11)
    row, drow = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = softmax(row.numpy(), 1.0), softmax(drow.numpy(), 1.0)
    if mode == "iid":
        tokens = torch.multinomial(torch.tensor(q).expand(S, V), branch, replacement=True, generator=g)
    elif mode == "distinct":
        tokens = torch.multinomial(torch.tensor(q).expand(S, V), branch, replacement=False, generator=g)
    else:
        tokens = torch.tensor([2, 5]).expand(S, 2)
    t = dict(target=row.expand(S, N, V).contiguous(), draft=None if mode == "given" else drow.expand(S, N, V).contiguous(),
             tokens=torch.cat([torch.zeros((S, 1)), tokens], 1).int(), parents=torch.tensor([[-1] + [0] * branch] * S, dtype=torch.int32),
             counts=torch.full((S,), N, dtype=torch.int32), u=torch.rand((S, N), generator=g), uf=torch.rand((S,), generator=g))
    ctx = Context(0)
    try:
        path, acc, nxt = call(torch, ctx, t, mode)
    finally:
        ctx.close()
    first = torch.where(acc > 1, t["tokens"].gather(1, path[:, 1:2].clamp(min=0).long()).squeeze(1), nxt)
    seen = np.bincount(first.numpy(), minlength=V)
    assert 0 < int((acc > 1).sum()) < S
    assert ((seen - S * p) ** 2 / (S * p)).sum() < 29.9


@pytest.mark.gpu
@pytest.mark.parametrize("mode,temperature", [("given", 0.0), ("given", 1.0), ("iid", 1.0), ("distinct", 1.0)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_that_begin_anywhere(kind, mode, temperature):
    """Rows at every offset within a vector, the draft's at others than the target's, about whole chunks; what lies between
    the rows is NaN and +inf."""
    import torch
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        for V in (1, 3, 1021, 1024, 2048):
            print(f"[gpu] verify offsets {mode} {kind} V={V}", flush=True)
            t = inputs(torch, 3, 7, V, kind, mode, 2, V)
            for off, gap in ((0, 1), (1, 4), (2, 3), (3, 2), (1, 0)):
                def view(x, off, gap):
                    if x is None:
                        return None
                    wide = torch.full((off + 21 * (V + gap),), float("inf"), dtype=x.dtype, device="cuda:0")
                    wide[::2] = float("nan")
                    v = wide[off:].view(3, 7, V + gap)[:, :, :V]
                    v.copy_(x)
                    return v
                check(t, mode, call(torch, ctx, t, mode, temperature, target=view(t["target"], off, gap),
                                    draft=view(t["draft"], 3 - off, gap + 1)), temperature)
    finally:
        ctx.close()


@pytest.mark.gpu
def test_strided_rows_and_replays():
    """Logits that are slices of padded rows, recorded and replayed on new inputs beside eager calls of another shape."""
    import torch
    from hydra_amd import speculative as sp
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        S, N, V = 3, 10, 1001
        t = inputs(torch, S, N, V, "bf16", "iid", 3, 5)
        wide_t, wide_d = (torch.full((S, N, V + 6), float("nan"), dtype=torch.bfloat16, device="cuda:0") for _ in range(2))
        tv, dv = wide_t[..., 3:3 + V], wide_d[..., :V]
        tv.copy_(t["target"])
        dv.copy_(t["draft"])
        check(t, "iid", call(torch, ctx, t, "iid", target=tv, draft=dv))
        sp.reserve(ctx, verify=(S, N, V), verify_dtype=torch.bfloat16)
        other = inputs(torch, 1, 4, 300, "f32", "distinct", 2, 6)
        d = {k: x.to("cuda:0") for k, x in t.items()}
        path = torch.zeros((S, N), dtype=torch.int32, device="cuda:0")
        acc, nxt = (torch.zeros(S, dtype=torch.int32, device="cuda:0") for _ in range(2))
        torch.cuda.synchronize()
        graph = ctx.capture(lambda: sp.draft_verify_into(ctx, tv, d["tokens"], d["parents"], d["counts"], d["u"], d["uf"], path, acc,
                                                         nxt, draft=dv))
        for rep in range(4):
            t = inputs(torch, S, N, V, "bf16", "iid", 3, 50 + rep)
            tv.copy_(t["target"])
            dv.copy_(t["draft"])
            for k in ("tokens", "u", "uf"):
                d[k].copy_(t[k])
            check(other, "distinct", call(torch, ctx, other, "distinct"))
            torch.cuda.synchronize()
            graph.launch()
            ctx.synchronize()
            check(t, "iid", (path.cpu(), acc.cpu(), nxt.cpu()))
        with pytest.raises(Exception):       # a larger workspace while the graph lives
            big = inputs(torch, 64, 64, 50, "f32", "iid", 3, 6)
            call(torch, ctx, big, "iid")
        graph.close()
        check(big, "iid", call(torch, ctx, big, "iid"))
    finally:
        ctx.close()


# ---- refusals (no GPU) ------------------------------------------------------------------------------

def _call(desc=None, **kw):
    from hydra_amd import _lib
    d = dict(sequences=1, nodes=4, vocab=100, type=0, draft=1, max_children=0, temperature=1.0, target_stride=0, draft_stride=0)
    d.update(desc or {})
    a = dict(target=16, draft=16, tokens=16, parents=16, counts=16, u=16, uf=16, path=16, accepted=16, nxt=16)
    a.update(kw)
    return _lib.lib().hh_draft_verify(C.create_string_buffer(4096), C.byref(_lib.VerifyDescC(**d)), *a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(desc=dict(sequences=0)), -1), (dict(desc=dict(nodes=65)), -1), (dict(desc=dict(vocab=0)), -1), (dict(desc=dict(vocab=1 << 25)), -1),
    (dict(desc=dict(type=3)), -1), (dict(desc=dict(draft=3)), -1), (dict(desc=dict(max_children=64)), -1),
    (dict(desc=dict(max_children=-1)), -1), (dict(desc=dict(temperature=-1.0)), -1), (dict(desc=dict(temperature=float("inf"))), -1),
    (dict(desc=dict(temperature=float("nan"))), -1), (dict(desc=dict(temperature=1e-9)), -1), (dict(desc=dict(target_stride=99)), -6),
    (dict(desc=dict(sequences=4096, nodes=64, vocab=1 << 24)), -1),
    (dict(desc=dict(draft_stride=99)), -6), (dict(target=None), -1), (dict(draft=None), -1), (dict(tokens=None), -1), (dict(parents=None), -1),
    (dict(counts=None), -1), (dict(u=None), -1), (dict(uf=None), -1), (dict(path=None), -1), (dict(accepted=None), -1), (dict(nxt=None), -1),
])
def test_verify_refusals(kw, code):
    assert _call(**kw) == code


def test_null_context():
    from hydra_amd._lib import lib
    assert lib().hh_draft_verify(None, None, *[None] * 10) == -1
    assert lib().hh_draft_reserve(None, None, None, 0, None) == -1
