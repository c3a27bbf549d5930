"""Verification (hh_draft_verify) where the draft's distributions are sharp: most of the mass on one token, and again on one of
the rest, as low temperatures and confident models make them. The draft off the tokens tried is normalised by its own largest
entry, so that no gap between the logits is too wide. Oracle: the rule as it is stated, in 64 bits, the draft as logarithms."""
import numpy as np
import pytest

from test_draft_verify import call, softmax


def normal(x):
    """exp(x) over its sum; entries of +inf share it; all zero where nothing is left."""
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    with np.errstate(invalid="ignore"):
        e = np.where(x == top, 1.0, np.exp(x - top))
    return e / e.sum()


def oracle(target, draft, distinct, tokens, parents, count, u, uf, t):
    """(path, accepted, next) of one sequence."""
    N, V = target.shape
    cur, line = 0, [0]
    while True:
        p = full = softmax(target[cur], t)
        lq = draft[cur].astype(np.float64) / t
        for n in (n for n in range(cur + 1, count) if parents[n] == cur):
            x, q = int(tokens[n]), normal(lq)
            if float(u[n]) * q[x] < p[x]:
                cur = n
                line.append(n)
                break
            p = np.maximum(p - q, 0)
            p[x] = 0
            if p.sum() > 0:
                p /= p.sum()
            if distinct:
                lq[x] = -np.inf
        else:
            p = p if p.sum() > 0 else full
            c = np.cumsum(p)
            after = min(int((c <= float(uf) * c[-1]).sum()), int(np.nonzero(p)[0][-1]))
            return line + [-1] * (N - len(line)), len(line), after


def drawn(torch, g, draft, parents, t, distinct):
    """Children's tokens drawn from the draft's rows, in the order of their index."""
    S, N, V = draft.shape
    tokens = torch.zeros((S, N), dtype=torch.int32)
    for s in range(S):
        for n in range(N):
            kids = [m for m in range(n + 1, N) if int(parents[s, m]) == n]
            noise = -torch.empty((len(kids), V), dtype=torch.float64).exponential_(1.0, generator=g).log()
            x = draft[s, n].double() / t
            if distinct and kids:
                tokens[s, kids] = (x + noise[0]).topk(len(kids)).indices.int()
            elif kids:
                tokens[s, kids] = (x + noise).argmax(-1).int()
    return tokens


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["distinct", "iid"])
@pytest.mark.parametrize("V,N,branch,gap,levels,temperature", [
    (4, 3, 2, 40.0, 1, 1.0),
    (8, 5, 4, 200.0, 1, 1.0),
    (300, 13, 3, 80.0, 1, 1.0),
    (300, 21, 4, 60.0, 3, 0.5),           # each of the first four far behind the one before it
    (1500, 13, 3, 45.0, 2, 0.05),         # 900 nats: beyond the range of an exponential in 64 bits
    (5000, 13, 4, 200.0, 3, 0.1),         # 2000 nats, three times
    (9001, 9, 2, 1.0, 2, 1e-3),
    (140001, 6, 5, 40.0, 1, 1.0),         # chunks of 4096
])
def test_sharp_drafts(mode, V, N, branch, gap, levels, temperature):
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] verify sharp {mode} V={V} N={N} branch={branch} gap={gap} T={temperature}", flush=True)
    S = 24 if V < 10000 else 3
    g = torch.Generator().manual_seed(V + N)
    target = torch.randn((S, N, V), generator=g) * 2 * temperature
    draft = torch.randn((S, N, V), generator=g) * temperature
    for i in range(levels):               # a token each, `gap` above all below it
        at = torch.randint(0, V, (S, N, 1), generator=g)
        draft.scatter_(2, at, gap * (levels - i))
        # The target puts a part of its mass there too, else a rejection is certain.
        target.scatter_add_(2, at, torch.full(at.shape, 4.0 * temperature))
    draft[1, 0, V // 2] = float("inf")    # before all others, then gone
    parents = torch.tensor([[(i - 1) // branch for i in range(N)]] * S, dtype=torch.int32)
    distinct = mode == "distinct"
    t = dict(target=target, draft=draft, parents=parents, tokens=drawn(torch, g, draft, parents, temperature, distinct),
             counts=torch.full((S,), N, dtype=torch.int32), u=torch.rand((S, N), generator=g), uf=torch.rand((S,), generator=g))
    ctx = Context(0)
    try:
        path, acc, nxt = call(torch, ctx, t, mode, temperature)
    finally:
        ctx.close()
    for s in range(S):
        want = oracle(target[s].numpy(), draft[s].numpy(), distinct, t["tokens"][s].tolist(), parents[s].tolist(), N, t["u"][s],
                      t["uf"][s], float(np.float32(temperature)))
        assert (path[s].tolist(), int(acc[s]), int(nxt[s])) == want, f"sequence {s}"


@pytest.mark.gpu
@pytest.mark.parametrize("logits,temperature", [([0, -40, -41, -42], 1.0), ([0, -9, -9.5, -10], 0.01), ([0, -80, -150, -151], 1.0)])
def test_tokens_of_a_sharp_draft_are_distributed_as_the_target(logits, temperature):
    """The first token that comes out of 4096 sequences, two children drawn without putting back. Chi-square of 3 degrees
    of freedom: above 21.1 once in 10^4 by chance (the seed is fixed)."""
    import torch
    from hydra_amd.layer import Context
    S, V, N = 4096, 4, 3
    g = torch.Generator().manual_seed(17)
    p = np.array([0.1, 0.1, 0.2, 0.6])
    parents = torch.tensor([[-1, 0, 0]] * S, dtype=torch.int32)
    draft = torch.tensor(logits, dtype=torch.float32).expand(S, N, V).contiguous()
    target = torch.tensor(np.log(p) * temperature, dtype=torch.float32).expand(S, N, V).contiguous()
    noise = -torch.empty((S, V), dtype=torch.float64).exponential_(1.0, generator=g).log()
    two = (draft[:, 0].double() / temperature + noise).topk(2).indices.int()
    t = dict(target=target, draft=draft, parents=parents, tokens=torch.cat([torch.zeros((S, 1), dtype=torch.int32), two], 1),
             counts=torch.full((S,), N, dtype=torch.int32), u=torch.rand((S, N), generator=g), uf=torch.rand((S,), generator=g))
    ctx = Context(0)
    try:
        path, acc, nxt = call(torch, ctx, t, "distinct", temperature)
    finally:
        ctx.close()
    first = torch.where(acc > 1, t["tokens"].gather(1, path[:, 1:2].clamp(min=0).long()).squeeze(1), nxt)
    seen = np.bincount(first.numpy(), minlength=V)
    assert ((seen - S * p) ** 2 / (S * p)).sum() < 21.1, seen / S


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["distinct", "iid"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_draft_equal_to_the_target_leaves_nothing(kind, mode):
    """A child without a token is rejected whatever the distributions; where they are equal nothing is left of the target then,
    and the next token is drawn from the target itself, also where the rows lie at other offsets in memory."""
    import torch
    from hydra_amd.layer import Context
    S, N, V, T = 16, 4, 3001, 0.7
    dtype = {"f32": torch.float32, "bf16": torch.bfloat16}[kind]
    g = torch.Generator().manual_seed(23)
    rows = (torch.randn((S, N, V), generator=g) * 3).to(dtype)
    parents = torch.tensor([[-1, 0, 0, 0]] * S, dtype=torch.int32)
    tokens = drawn(torch, g, rows.float(), parents, T, mode == "distinct")
    t = dict(target=rows, draft=rows.clone(), parents=parents, tokens=tokens, counts=torch.full((S,), N, dtype=torch.int32),
             u=torch.rand((S, N), generator=g), uf=torch.rand((S,), generator=g))
    tokens[:, 1] = torch.where(torch.arange(S) % 2 == 0, -1, V)
    p = np.stack([softmax(rows[s, 0].float().numpy(), float(np.float32(T))) for s in range(S)])
    c = p.cumsum(1)
    want = (c <= (t["uf"].numpy().astype(np.float64) * c[:, -1])[:, None]).sum(1).tolist()
    ctx = Context(0)
    try:
        for off in (0, 1, 2, 3):
            print(f"[gpu] verify equal rows {mode} {kind} offset {off}", flush=True)
            wide = torch.zeros(S * N * (V + 7) + 4, dtype=dtype, device="cuda:0")
            draft = wide[off:off + S * N * (V + 7)].view(S, N, V + 7)[..., :V]
            draft.copy_(rows)
            path, acc, nxt = call(torch, ctx, t, mode, T, draft=draft)
            assert acc.tolist() == [1] * S and nxt.tolist() == want
    finally:
        ctx.close()
