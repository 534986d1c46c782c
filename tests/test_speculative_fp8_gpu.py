"""Caches in 8 bits in use: stored, attended and verified together, as examples/speculative_decode.py does."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import speculative_decode as S  # noqa: E402
from dropkv_b200 import (attention_fp8, block_tables, load_rows_fp8, qk_norm_rope, store_rows_fp8,  # noqa: E402
                         verify_draft)

pytestmark = pytest.mark.gpu


def _prompts(model, lens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, model.vocab, (n,), generator=g, device="cuda") for n in lens]


def _dense_step(model, caches, tokens, lens, seen, parents):
    """Logits of the nodes in fp32 torch; all rows, the nodes' own too, as they stand in the pages."""
    m, T = model, tokens.shape[1]
    if parents is None:
        mask = torch.ones(T, T, dtype=torch.bool, device=tokens.device).tril().expand(len(tokens), T, T)
        depth = torch.arange(T, device=tokens.device).expand(len(tokens), T)
    else:
        mask, depth = S.tree_mask_from_parents(parents)
    norm = lambda y: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    out = []
    for b in range(tokens.shape[0]):
        n = int(lens[b])
        slots = torch.tensor([[int(caches.table[b, j // caches.block]) * caches.block + j % caches.block for j in range(n + T)]],
                             device=tokens.device)
        x = m.embed[tokens[b]].float()
        pos = int(seen[b]) + depth[b]
        see = torch.cat([torch.ones(T, n, dtype=torch.bool, device=x.device), mask[b]], 1)
        for layer, w in enumerate(m.w):
            K, V = load_rows_fp8(caches.K[layer], caches.V[layer], caches.K_scales[layer], caches.V_scales[layer], slots,
                                 torch.float32)
            q = (norm(x) @ w["qkv"].float()).view(T, -1, m.D)[:, :m.Hq].transpose(0, 1)
            q, c, s = norm(q) * w["qn"].float(), m.cos[pos], m.sin[pos]
            lo, hi = q[..., :m.D // 2], q[..., m.D // 2:]
            q = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
            g = m.Hq // m.Hkv
            sc = torch.einsum("hqd,hkd->hqk", q, K[0].repeat_interleave(g, 0)) * m.D ** -0.5
            o = torch.einsum("hqk,hkd->hqd", sc.masked_fill(~see, float("-inf")).softmax(-1), V[0].repeat_interleave(g, 0))
            x = x + o.transpose(0, 1).reshape(T, -1) @ w["out"].float()
            x = x + torch.nn.functional.silu(norm(x) @ w["up"].float()) @ w["down"].float()
        out.append(norm(x) @ m.head.float())
    return torch.stack(out)


@pytest.mark.parametrize("lens,tree", [((300, 47, 130), 13), ((20,), 1), ((64, 9), 33), ((150, 31), None)])
def test_a_step_matches_dense_attention_over_the_stored_rows(lens, tree):
    model = S.Decoder(layers=3, dtype=torch.float16)
    caches = S.PagedCaches8(model, len(lens), pages=256)
    last = caches.load(_prompts(model, lens, 2))
    for _ in range(2):
        root = last.argmax(-1)
        tokens, parents = S.draft_tree(root, model.followers, tree) if tree else (S.draft_chain(root, model.draft, 5, 1.0), None)
        before = caches.lens.clone(), caches.seen.clone()
        logits, keep = caches.verify(tokens, parents)
        want = _dense_step(model, caches, tokens, *before, parents)
        # as over 16-bit caches: some 30 roundings of 2^-11 of values of order 1 on the way to a logit of
        # standard deviation 3 (what the pages hold is the same on both sides)
        assert float((logits.float() - want).abs().max()) < 30 * 2.0 ** -11 * 3 * 4
        if parents is None:
            at = torch.arange(tokens.shape[1], device="cuda")
            place = torch.where(at <= torch.arange(len(lens), device="cuda")[:, None], at, -1)
        else:
            place, _, _ = S.accept(tokens, parents, logits.argmax(-1))
        keep(place)
        assert torch.equal(caches.lens, before[0] + (place >= 0).sum(1).int())
        last = logits[:, 0]


def test_kept_rows_of_a_tree_are_the_nodes_rows():
    """What ``keep`` moves to the front of the slots is what the pages then hold, to a rounding."""
    model = S.Decoder(layers=1, dtype=torch.float16)
    caches = S.PagedCaches8(model, 2, pages=64)
    last = caches.load(_prompts(model, (90, 33), 5))
    tokens, parents = S.draft_tree(last.argmax(-1), model.followers, 9)
    lens = caches.lens.clone()
    logits, keep = caches.verify(tokens, parents)
    pools = caches.K[0], caches.V[0], caches.K_scales[0], caches.V_scales[0]
    at = lambda b, j: int(caches.table[b, j // caches.block]) * caches.block + j % caches.block  # noqa: E731
    nodes = load_rows_fp8(*pools, torch.tensor([[at(b, int(lens[b]) + i) for i in range(9)] for b in range(2)], device="cuda"), torch.float32)
    place = torch.tensor([[0, -1, 1, -1, -1, -1, -1, 2, -1]] * 2, device="cuda")
    keep(place)
    kept = load_rows_fp8(*pools, torch.tensor([[at(b, int(lens[b]) + i) for i in range(3)] for b in range(2)], device="cuda"), torch.float32)
    for a, b, scales in zip(nodes, kept, pools[2:]):
        a = a[:, :, [0, 2, 7]]
        # both are roundings of the same row: each by 2^-4 of the value at most, or by half of a scale's smallest step
        assert bool(((a - b).abs() <= 2 * (2.0 ** -4 / (1 - 2.0 ** -4) * torch.maximum(a.abs(), b.abs()) + 2.0 ** -10 * scales.max())).all())


@pytest.mark.parametrize("drafted,temperature", [(4, 1.0), (0, 0.7), (7, 0.3)])
def test_sampling_runs(drafted, temperature):
    model = S.Decoder(layers=2)
    torch.manual_seed(0)
    out, rate = S.sample(model, _prompts(model, (200, 33, 5), 3), 5, drafted, temperature)
    assert 1.0 <= rate <= drafted + 1
    assert all(5 <= len(o) <= 5 * (drafted + 1) and all(0 <= t < model.vocab for t in o) for o in out)


def test_a_captured_step_follows_its_inputs():
    """A decode step of the operators in one CUDA graph: replayed on other inputs, in place, it gives what the
    calls give."""
    B, Hq, Hkv, T, D, block, V = 3, 8, 2, 5, 64, 16, 5003
    g = torch.Generator(device="cuda").manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    lens = torch.tensor([40, 7, 100], dtype=torch.int32, device="cuda")
    held = (lens + block - 1) // block
    free = torch.randperm(64, generator=g, device="cuda").int()
    table = torch.full((B, 12), -1, dtype=torch.int32, device="cuda")
    table[:, :7] = torch.arange(64, 64 + 7 * B, device="cuda").view(B, 7)
    Q, K, W = (rnd(B, T, h, D).bfloat16().transpose(1, 2) for h in (Hq, Hkv, Hkv))
    pools = [rnd(96, Hkv, block, D).to(torch.float8_e4m3fn) for _ in range(2)] + [torch.full((96, Hkv), 2.0 ** -7, device="cuda") for _ in range(2)]
    ang = torch.rand(200, D // 2, generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    target, draft = rnd(B, T, V), rnd(B, T - 1, V)
    tokens, uniforms = torch.randint(0, V, (B, T - 1), generator=g, device="cuda"), torch.rand(B, T, generator=g, device="cuda")

    def step(pools):
        t = block_tables(lens + T, block, free, 12, T, new_lens=torch.full_like(lens, T), table=table, held=held)
        at = lens.long()[:, None] + torch.arange(T, device="cuda")
        q, k = qk_norm_rope(Q, K, cos, sin, at)
        store_rows_fp8(k, W, t.slots, *pools)
        few = attention_fp8(q[:, :, :1], *pools, lens, t.table, window=50, sinks=4)
        return [*t, few, attention_fp8(q, *pools, lens, t.table), *load_rows_fp8(*pools, t.slots),
                *verify_draft(target, tokens, uniforms, draft_logits=draft)]

    copies = lambda: [p.clone() for p in pools]  # noqa: E731
    step(copies())
    mine = copies()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(mine)
    for change in range(2):
        if change:
            lens.copy_(torch.tensor([64, 0, 31], device="cuda"))
            held.copy_((lens + block - 1) // block)
            Q.copy_(Q.flip(0)), target.mul_(0.5), uniforms.mul_(0.3)
        for m, p in zip(mine, pools):
            m.copy_(p)
        graph.replay()
        torch.cuda.synchronize()
        want_pools = copies()
        for a, b in zip(got, step(want_pools)):
            assert torch.equal(a, b)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(mine, want_pools))
