"""The paged operators together, as examples/speculative_decode.py runs them."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import speculative_decode as S  # noqa: E402

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
