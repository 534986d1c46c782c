"""The paged operators together, as examples/speculative_decode.py runs them."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import speculative_decode as S  # noqa: E402
from dropkv_b200 import block_tables, qk_norm_rope, token_logprobs, tree_attention  # noqa: E402

pytestmark = pytest.mark.gpu


def _dense_step(model, caches, tokens, parents):
    """Logits of the nodes in fp32 torch, the stored rows gathered from the pages."""
    m = model
    mask, depth = S.tree_mask_from_parents(parents)
    out = []
    for b in range(tokens.shape[0]):
        n = int(caches.lens[b])
        slots = [int(caches.table[b, j // caches.block]) * caches.block + j % caches.block for j in range(n)]
        page = torch.tensor([s // caches.block for s in slots], device=tokens.device, dtype=torch.long)
        at = torch.tensor([s % caches.block for s in slots], device=tokens.device, dtype=torch.long)
        x = m.embed[tokens[b]].float()
        pos = int(caches.seen[b]) + depth[b]
        norm = lambda y: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
        for layer, w in enumerate(m.w):
            qkv = (norm(x) @ w["qkv"].float()).view(len(x), -1, m.D)
            q, k, v = (t.transpose(0, 1) for t in qkv.split([m.Hq, m.Hkv, m.Hkv], dim=1))
            c, s = m.cos[pos], m.sin[pos]
            turn = lambda y, wt: (lambda z: torch.cat([z[..., :m.D // 2] * c - z[..., m.D // 2:] * s,  # noqa: E731
                                                       z[..., m.D // 2:] * c + z[..., :m.D // 2] * s], -1))(norm(y) * wt.float())
            q, k = turn(q, w["qn"]), turn(k, w["kn"])
            K = torch.cat([caches.K[layer][page, :, at].float().transpose(0, 1), k], 1)
            V = torch.cat([caches.V[layer][page, :, at].float().transpose(0, 1), v], 1)
            see = torch.cat([torch.ones(len(x), n, dtype=torch.bool, device=x.device), mask[b]], 1)
            g = m.Hq // m.Hkv
            sc = torch.einsum("hqd,hkd->hqk", q, K.repeat_interleave(g, 0)) * m.D ** -0.5
            o = torch.einsum("hqk,hkd->hqd", sc.masked_fill(~see, float("-inf")).softmax(-1), V.repeat_interleave(g, 0))
            x = x + o.transpose(0, 1).reshape(len(x), -1) @ w["out"].float()
            x = x + torch.nn.functional.silu(norm(x) @ w["up"].float()) @ w["down"].float()
        out.append(norm(x) @ m.head.float())
    return torch.stack(out)


def _prompts(model, lens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, model.vocab, (n,), generator=g, device="cuda") for n in lens]


@pytest.mark.parametrize("lens,tree", [((300, 47, 130), 13), ((20,), 1), ((64, 9), 33)])
def test_a_step_matches_dense_attention_over_the_stored_rows(lens, tree):
    model = S.Decoder(layers=3, dtype=torch.float16)
    caches = S.PagedCaches(model, len(lens), pages=256)
    last = caches.load(_prompts(model, lens, 2))
    for _ in range(2):                               # a second step stands on the first's kept rows
        root = S.token_logprobs(last, last.argmax(-1), top_k=1).top_tokens[:, 0]
        tokens, parents = S.draft_tree(root, model.followers, tree)
        want = _dense_step(model, caches, tokens, parents)
        logits, keep = caches.verify(tokens, parents)
        # fp16 activations and weights through 3 layers of products: each rounding is 2^-11 of
        # values of order 1, some 30 of them on the way to a logit of standard deviation 3
        assert float((logits.float() - want).abs().max()) < 30 * 2.0 ** -11 * 3 * 4
        place, _, _ = S.accept(tokens, parents, logits.argmax(-1))
        keep(place)
        last = logits[:, 0]


def test_a_pool_that_runs_out_of_pages_ends_the_loop():
    model = S.Decoder(layers=1, dtype=torch.float16)
    prompts = _prompts(model, (300, 100), 4)             # 90 and 30 rows kept: eight pages of 16
    few = S.PagedCaches(model, 2, pages=7)
    with pytest.raises(RuntimeError, match="8 pages wanted of 7"):
        few.load(prompts)
    narrow = S.PagedCaches(model, 2, pages=64, max_blocks=5)
    with pytest.raises(RuntimeError, match="90 rows of at most 80"):
        narrow.load(prompts)


def test_accept_takes_the_longest_agreeing_path():
    tokens = torch.tensor([[5, 6, 7, 8, 9, 6], [1, 2, 3, 4, 4, 4]], device="cuda")
    parents = torch.tensor([[-1, 0, 0, 2, 3, 0], [-1, 0, 1, 2, 3, 4]], device="cuda")
    choice = torch.tensor([[7, 0, 8, 1, 0, 0], [9, 3, 4, 4, 4, 4]], device="cuda")
    place, taken, nxt = S.accept(tokens, parents, choice)
    assert place.tolist() == [[0, -1, 1, 2, -1, -1], [0, -1, -1, -1, -1, -1]]
    assert taken.tolist() == [3, 1] and nxt.tolist() == [1, 9]


def test_trees_decode_what_single_tokens_do():
    """Greedy decoding with trees keeps the tokens that one token a step gives: both run the
    same operators, whose results for a row do not depend on the drafts beside it by more than
    rounding; the prompts' choices are no near ties."""
    model = S.Decoder(layers=2, dtype=torch.float16)
    prompts = _prompts(model, (200, 33), 3)
    single, rate1 = S.decode(model, prompts, steps=6, tree=1)
    many, rate = S.decode(model, prompts, steps=6, tree=13)
    assert rate1 == 1.0 and rate > 1.0
    for a, b in zip(single, many):
        n = min(len(a), len(b))
        assert n >= 6 and a[:n] == b[:n]


def test_a_captured_step_follows_its_inputs():
    """A decode step of four operators in one CUDA graph: replayed on other inputs, in place,
    it gives what the calls give."""
    B, Hq, Hkv, T, D, block, V = 3, 8, 2, 4, 64, 16, 5003
    g = torch.Generator(device="cuda").manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    lens = torch.tensor([40, 7, 100], dtype=torch.int32, device="cuda")
    held = (lens + block - 1) // block
    free = torch.randperm(64, generator=g, device="cuda").int()
    table = torch.full((B, 12), -1, dtype=torch.int32, device="cuda")
    table[:, :7] = torch.arange(64, 64 + 7 * B, device="cuda").view(B, 7)
    Q, K, W = (rnd(B, T, h, D).bfloat16().transpose(1, 2) for h in (Hq, Hkv, Hkv))
    pages = [rnd(96, Hkv, block, D).bfloat16() for _ in range(2)]
    ang = torch.rand(200, D // 2, generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    logits = rnd(1300, V)                         # more rows than a wave of CTAs: two launches
    tokens = torch.randint(0, V, (1300,), generator=g, device="cuda")

    def step(pages):
        t = block_tables(lens + T, block, free, 12, T, new_lens=torch.full_like(lens, T), table=table, held=held)
        at = lens.long()[:, None] + torch.arange(T, device="cuda")
        q, k = qk_norm_rope(Q, K, cos, sin, at, V=W, slots=t.slots, K_pages=pages[0], V_pages=pages[1])
        return [*t, q, k, tree_attention(q, *pages, lens, block_table=t.table), *token_logprobs(logits, tokens, top_k=3)]

    step([p.clone() for p in pages])              # (nothing is loaded for the first time while capturing)
    mine = [p.clone() for p in pages]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(mine)
    for change in range(2):
        if change:
            lens.copy_(torch.tensor([64, 0, 31], device="cuda"))
            held.copy_((lens + block - 1) // block)
            Q.copy_(Q.flip(0)), logits.mul_(0.5)
        for m, p in zip(mine, pages):
            m.copy_(p)
        graph.replay()
        torch.cuda.synchronize()
        want_pages = [p.clone() for p in pages]
        for a, b in zip(got, step(want_pages)):
            assert torch.equal(a, b)
        assert all(torch.equal(a, b) for a, b in zip(mine, want_pages))
