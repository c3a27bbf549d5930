"""Decoding with drafted tokens as a program does it: a small model's layers (Runner: tree attention in the
hook, the FFN block behind it), verification, commit, accumulated weights and eviction, eager and as one
graph. Greedy decoding with any drafts gives the tokens that decoding one at a time gives."""
import ctypes as C

import numpy as np
import pytest

from hydra_amd import formats as F
from hydra_amd import synth

pytestmark = pytest.mark.gpu

H, QH, KVH, D, VOCAB, ROWS = 256, 8, 2, 64, 512, 192
DESCS = [
    F.MoEDesc(hidden=H, intermediate=128, experts=6, top_k=2, quant=F.QUANT_MXFP4, activation=F.ACT_SWIGLU_OAI,
              router=F.ROUTER_TOPK_SOFTMAX, expert_bias=1),
    F.MoEDesc(hidden=H, intermediate=128, experts=5, top_k=2, quant=F.QUANT_BF16, activation=F.ACT_SILU,
              router=F.ROUTER_SOFTMAX_TOPK_RENORM),
]


class Model:
    """S sequences of up to N drafted tokens at a time; everything that a step touches is allocated here."""

    def __init__(self, torch, ctx, S, N, ring=None, bounded=False):
        from hydra_amd import speculative as sp
        from hydra_amd._lib import MatrixC
        from hydra_amd.layer import MoELayer, Runner, to_device
        self.torch, self.sp, self.ctx, self.S, self.N = torch, sp, ctx, S, N
        dev = "cuda:0"
        rng = np.random.default_rng(5)
        mat = lambda rows, cols, i, std: (lambda w: (MatrixC(F.QUANT_BF16, rows, cols, 64, C.c_void_p(w.data_ptr()), None, None, None), w))(
            to_device(synth.bf16_normal(90 + i, "w", rows * cols, 0.0, std), dev))
        self.qkv = [mat((QH + 2 * KVH) * D, H, i, 0.06) for i in range(2)]
        self.o = [mat(H, QH * D, 10 + i, 0.06) for i in range(2)]
        self.head = mat(VOCAB, H, 20, 0.06)
        g = torch.Generator().manual_seed(1)
        self.emb = torch.randn((VOCAB, H), generator=g).to(dev) * 2
        self.sinks = torch.randn((2, QH), generator=g).bfloat16().to(dev)
        norm = to_device(synth.f32_to_bf16(rng.uniform(0.5, 1.5, H).astype(np.float32)), dev)
        layers = [(MoELayer(synth.make_layer(d, seed=70 + i), ctx), {"pre_norm": norm, "eps": 1e-5}, None) for i, d in enumerate(DESCS)]
        self.runner = Runner(ctx, layers)
        self.runner.reserve(S * N)
        f32 = lambda *shape: torch.zeros(shape, device=dev)
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
        half = lambda *shape: torch.zeros(shape, dtype=torch.float16, device=dev)
        self.hidden, self.logits = f32(S * N, H), f32(S, N, VOCAB)
        self.fused, self.mixed, self.back = f32(2, S, N, QH + 2 * KVH, D), f32(2, S, N, QH, D), f32(S * N, H)
        self.dk, self.dv, self.lse = half(2, S, N, KVH, D), half(2, S, N, KVH, D), f32(2, S, N, QH)
        self.tokens, self.parents, self.path = i32(S, N), i32(S, N), i32(S, N)
        self.counts, self.accepted, self.next = i32(S), i32(S), i32(S)
        self.lengths, self.position = i32(S), i32(S)
        rows = [ring or ROWS, ROWS]
        self.window = [31 if ring else 0, 0]     # the same for every N: the two runs are of one model
        self.caches = [sp.KVCache(half(S, r, KVH, D), half(S, r, KVH, D), self.lengths, ring=bool(ring) and i == 0,
                                  weights=f32(S, KVH, r) if bounded else None, positions=i32(S, KVH, r) if bounded else None,
                                  next_position=self.position if bounded else None) for i, r in enumerate(rows)]
        self.set = sp.CacheSet(self.caches)
        for c in self.caches:
            sp.reserve(ctx, c, nodes=N, q_heads=QH, q_dtype=torch.float32, layers=2 if bounded else 0, verify=(S, N, VOCAB))
        torch.cuda.synchronize()

    def gemm(self, m, x, y, tokens):
        from hydra_amd._lib import check, lib
        check(lib().hh_expert_gemm(self.ctx.handle, C.byref(m[0]), C.c_void_p(x.data_ptr()), tokens, C.c_void_p(y.data_ptr())))

    def hook(self, l):
        T = self.S * self.N
        self.gemm(self.qkv[l], self.hidden, self.fused[l], T)
        x = self.fused[l]
        self.dk[l].copy_(x[:, :, QH:QH + KVH])
        self.dv[l].copy_(x[:, :, QH + KVH:])
        self.sp.attention_tree_into(self.ctx, self.caches[l], x[:, :, :QH], self.dk[l], self.dv[l], self.parents, self.counts,
                                    self.mixed[l], lse=self.lse[l], sinks=self.sinks[l], window=self.window[l])
        self.gemm(self.o[l], self.mixed[l], self.back, T)
        self.hidden.add_(self.back)

    def enqueue(self, keep=0, recent=0):
        torch, sp = self.torch, self.sp
        with torch.cuda.stream(self.ctx.stream):
            torch.index_select(self.emb, 0, self.tokens.view(-1), out=self.hidden)
        self.runner.forward(self.hidden, self.hook)
        self.gemm(self.head, self.hidden, self.logits, self.S * self.N)
        sp.draft_verify_into(self.ctx, self.logits, self.tokens, self.parents, self.counts, None, None, self.path, self.accepted,
                             self.next, temperature=0.0)
        sp.cache_commit(self.ctx, self.set, self.dk, self.dv, self.path, self.accepted)
        if keep:
            for l, c in enumerate(self.caches):
                sp.attention_weights_into(self.ctx, c, self.fused[l][:, :, :QH], self.lse[l], self.path, self.accepted)
            sp.cache_evict(self.ctx, self.set, keep, recent)

    def step(self, tokens, parents, counts, run=None, **kw):
        """One step on host inputs: (accepted tokens behind the pending one, next token) of each sequence."""
        torch = self.torch
        self.ctx.synchronize()
        for t, x in ((self.tokens, tokens), (self.parents, parents), (self.counts, counts)):
            t.copy_(torch.as_tensor(np.asarray(x), dtype=torch.int32))
        torch.cuda.synchronize()
        (run or (lambda: self.enqueue(**kw)))()
        self.ctx.synchronize()
        path, acc, nxt = self.path.cpu().numpy(), self.accepted.cpu().numpy(), self.next.cpu().numpy()
        return [[int(tokens[s][path[s, i]]) for i in range(1, acc[s])] for s in range(self.S)], [int(x) for x in nxt]


FIRST = [7, 300, 41]


def one_by_one(torch, count, **kw):
    """Each sequence's first `count` tokens, one at a time."""
    from hydra_amd.layer import Context
    ctx = Context(0)
    try:
        m = Model(torch, ctx, 3, 1, **kw)
        out, cur = [[], [], []], list(FIRST)
        for _ in range(count):
            _, cur = m.step([[t] for t in cur], [[-1]] * 3, [1, 1, 1])
            for s in range(3):
                out[s].append(cur[s])
        return out
    finally:
        ctx.close()


def drafts(rng, true, N):
    """A tree behind the pending token: some of the true continuation, some of it wrong, and other branches."""
    tokens, parents, at = [0], [-1], {0: 0}      # node -> how many of `true` lead to it (−1: off the line)
    for i in range(1, N):
        p = int(rng.integers(max(0, i - 4), i))
        depth = at[p]
        right = depth >= 0 and depth < len(true) and rng.random() < 0.7
        tokens.append(true[depth] if right else int(rng.integers(VOCAB)))
        at[i] = depth + 1 if depth >= 0 and depth < len(true) and tokens[-1] == true[depth] else -1
        parents.append(p)
    return tokens, parents


@pytest.mark.parametrize("ring", [None, 40])
@pytest.mark.parametrize("captured", [False, True])
def test_greedy_decoding_is_the_same_with_drafts(ring, captured):
    """Layers' outputs do not depend on the batch; attention sums in another order, so logits differ by 1e-5 of
    their size and the argmax of 512 does not."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] speculative step ring={ring} captured={captured}", flush=True)
    want = one_by_one(torch, 60, ring=ring)
    assert len(set(want[0])) > 5      # not a loop of one token
    rng = np.random.default_rng(2)
    ctx = Context(0)
    try:
        m = Model(torch, ctx, 3, 9, ring=ring)
        graph = None
        got, cur, accepted, steps = [[], [], []], list(FIRST), 0, 0
        while min(len(g) for g in got) < 40:
            toks, pars, cnts = [], [], []
            for s in range(3):
                t, p = drafts(rng, want[s][len(got[s]):], 9)
                t[0] = cur[s]
                toks.append(t)
                pars.append(p)
                cnts.append(int(rng.integers(1, 10)))
            if captured and graph is None and steps == 2:
                ctx.synchronize()
                graph = ctx.capture(m.enqueue)
            acc, nxt = m.step(toks, pars, cnts, run=graph.launch if graph else None)
            steps += 1
            for s in range(3):
                got[s] += acc[s] + [nxt[s]]
                accepted += len(acc[s])
                cur[s] = nxt[s]
            if max(len(g) for g in got) > 55:
                break
        if graph:
            graph.close()
    finally:
        ctx.close()
    for s in range(3):
        assert got[s] == want[s][:len(got[s])]
    assert accepted > 20 and steps < 40
    assert m.lengths.tolist() == [len(g) for g in got]


@pytest.mark.parametrize("captured", [False, True])
def test_bounded_histories(captured):
    """Every step ends with the eviction: histories stay within the budget, hold each position once, and the newest."""
    import torch
    from hydra_amd.layer import Context
    print(f"[gpu] bounded histories captured={captured}", flush=True)
    keep, recent, N, S = 48, 16, 9, 3
    rng = np.random.default_rng(4)
    ctx = Context(0)
    try:
        m = Model(torch, ctx, S, N, bounded=True)
        cur, graph, made = list(FIRST), None, [0, 0, 0]
        for step in range(30):
            toks, pars = zip(*[drafts(rng, [], N) for _ in range(S)])
            toks = [[cur[s]] + list(t[1:]) for s, t in enumerate(toks)]
            if captured and step == 3:
                ctx.synchronize()
                graph = ctx.capture(lambda: m.enqueue(keep, recent))
            acc, cur = m.step(toks, pars, [N] * S, run=graph.launch if graph else None, keep=keep, recent=recent)
            for s in range(S):
                made[s] += 1 + len(acc[s])
        for s in range(S):
            assert int(m.position[s]) == made[s] and int(m.lengths[s]) == min(made[s], keep)
            for c in m.caches:
                n = int(m.lengths[s])
                pos = c.positions[s, :, :n].cpu().numpy()
                for row in pos:
                    assert len(set(row.tolist())) == n and row.min() >= 0 and row.max() == made[s] - 1
                    assert set(range(made[s] - min(recent, made[s]), made[s])) <= set(row.tolist())
                w = c.weights[s, :, :n]
                assert torch.isfinite(w).all() and (w >= 0).all()
        if graph:
            graph.close()
    finally:
        ctx.close()
