"""Speculative decoding over paged, evicted caches: the paged operators in one loop.

    python examples/speculative_decode.py [--steps 8] [--tree 16] [--layers 4]
    python examples/speculative_decode.py --sample 0.8 [--drafted 4]

A small decoder with random weights (rotary positions, normed heads, grouped queries)
prefills a ragged batch of prompts. Every layer's K/V is evicted with ``compress_varlen``,
whose kept lengths exist on the GPU only; ``block_tables`` hands out pages for them there
and ``store_rows`` moves the kept rows in. Then, step by step, a tree of drafted tokens
is verified in one pass of the decoder: ``block_tables`` gives the nodes slots,
``qk_norm_rope`` writes their rows to the pages at the positions of their depths,
``tree_attention`` attends, ``token_logprobs`` gives each node's likeliest next token, and
the longest drafted path that agrees with the decoder's own choices
is kept. The result is what greedy decoding gives, one or more tokens a step.

With ``--sample`` tokens are drawn at a temperature, over caches in 8 bits: ``store_rows_fp8``
quantises kept and drafted rows as it writes them, ``attention_fp8`` attends over the
pages as they are, and ``verify_draft`` accepts a chain of drawn tokens so that the result is
distributed as the decoder's own samples.

The draft here is a table of likely followers of each token, which is what the decoder says
with no layers in between. A real one would come from a smaller model; nothing else would
change.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from dropkv_b200 import (attention_fp8, block_tables, compress_varlen, qk_norm_rope, store_rows, store_rows_fp8,  # noqa: E402
                         token_logprobs, tree_attention, tree_mask_from_parents, verify_draft)


class Decoder:
    """Weights of a decoder drawn from a seed, and its dense prefill."""

    def __init__(self, layers=4, hidden=512, Hq=8, Hkv=2, D=64, vocab=1000, positions=8192, seed=0, device="cuda",
                 dtype=torch.bfloat16):
        g = torch.Generator(device=device).manual_seed(seed)
        self.layers, self.hidden, self.Hq, self.Hkv, self.D, self.vocab = layers, hidden, Hq, Hkv, D, vocab
        self.device, self.dtype = torch.device(device), dtype
        draw = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g, device=device)).to(dtype)  # noqa: E731
        self.embed = draw(vocab, hidden)
        self.head = draw(hidden, vocab, scale=3 * hidden ** -0.5)
        self.w = [dict(qkv=draw(hidden, (Hq + 2 * Hkv) * D, scale=hidden ** -0.5),
                       out=draw(Hq * D, hidden, scale=0.3 * (Hq * D) ** -0.5),
                       up=draw(hidden, 2 * hidden, scale=hidden ** -0.5),
                       down=draw(2 * hidden, hidden, scale=0.5 * (2 * hidden) ** -0.5),
                       qn=1 + draw(D, scale=0.1), kn=1 + draw(D, scale=0.1)) for _ in range(layers)]
        self.draft = self.norm(self.embed) @ self.head                       # [vocab, vocab]: the draft's logits
        self.followers = token_logprobs(self.draft, torch.arange(vocab, device=device),
                                        top_k=3).top_tokens                  # [vocab, 3]: its likeliest
        freq = 10000.0 ** (-torch.arange(0, D, 2, device=device) / D)
        angle = torch.arange(positions, device=device)[:, None] * freq
        self.cos, self.sin = angle.cos(), angle.sin()

    def norm(self, x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).to(self.dtype)

    def project(self, x, w):
        """Q, K, V of tokens x [B, T, hidden] as [B, heads, T, D] views."""
        B, T, _ = x.shape
        q, k, v = (self.norm(x) @ w["qkv"]).view(B, T, -1, self.D).split([self.Hq, self.Hkv, self.Hkv], dim=2)
        return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)

    def after(self, x, attended, w):
        """The layer after its attention [B, Hq, T, D]."""
        B, T, _ = x.shape
        x = x + attended.transpose(1, 2).reshape(B, T, -1) @ w["out"]
        return x + torch.nn.functional.silu(self.norm(x) @ w["up"]) @ w["down"]

    def prefill(self, tokens):
        """A prompt [L] through the decoder: (per layer (Q, K, V) with heads normed and
        rotated, logits of its last token)."""
        L = tokens.shape[0]
        x, kept = self.embed[tokens][None], []
        at = torch.arange(L, device=self.device)
        causal = at[:, None] >= at[None, :]
        for w in self.w:
            q, k, v = self.project(x, w)
            q, k = qk_norm_rope(q, k, self.cos, self.sin, at, q_weight=w["qn"], k_weight=w["kn"])
            g = self.Hq // self.Hkv
            s = torch.einsum("bhqd,bhkd->bhqk", q.float(), k.float().repeat_interleave(g, 1)) * self.D ** -0.5
            p = s.masked_fill(~causal, float("-inf")).softmax(-1)
            o = torch.einsum("bhqk,bhkd->bhqd", p, v.float().repeat_interleave(g, 1)).to(self.dtype)
            x = self.after(x, o, w)
            kept.append((q, k, v))
        return kept, (self.norm(x[:, -1]) @ self.head)[0]


class PagedCaches:
    """The batch's evicted caches in pages: one pool of K and V for each layer, one block
    table for all of them."""

    def __init__(self, model: Decoder, batch: int, pages: int, block: int = 16, max_blocks: int = 64):
        self.model, self.block, self.max_blocks = model, block, max_blocks
        shape = (pages, model.Hkv, block, model.D)
        self.K = [torch.zeros(shape, dtype=model.dtype, device=model.device) for _ in range(model.layers)]
        self.V = [torch.zeros(shape, dtype=model.dtype, device=model.device) for _ in range(model.layers)]
        self.free = torch.randperm(pages, device=model.device).int()
        self.table = self.held = None
        self.lens = torch.zeros(batch, dtype=torch.int32, device=model.device)   # rows stored
        self.seen = torch.zeros(batch, dtype=torch.int64, device=model.device)   # tokens seen: positions go on from here

    def store(self, layer, k, v, slots):
        store_rows(k, v, slots, self.K[layer], self.V[layer])

    def attend(self, layer, q, k, v, positions, slots, mask):
        """A layer's attention of new tokens, their rows written to their slots: (attended, keys)."""
        m, w = self.model, self.model.w[layer]
        q, k = qk_norm_rope(q, k, m.cos, m.sin, positions, q_weight=w["qn"], k_weight=w["kn"], V=v, slots=slots,
                            K_pages=self.K[layer], V_pages=self.V[layer])
        return tree_attention(q, self.K[layer], self.V[layer], self.lens, tree_mask=mask, block_table=self.table), k

    def grow(self, lens, new_lens, max_new):
        """Pages for requests of these lengths, and the slots of their new tokens. Rows without a
        page would be left out and not seen, so a pool or a table that is too small ends the loop."""
        t = block_tables(lens, self.block, self.free, self.max_blocks, max_new, new_lens=new_lens, table=self.table,
                         held=self.held)
        used, longest = torch.stack([t.used[0], lens.max().long()]).tolist()  # (a read back)
        if used > len(self.free) or longest > self.max_blocks * self.block:
            raise RuntimeError(f"{used} pages wanted of {len(self.free)} free, {longest} rows of at most "
                               f"{self.max_blocks * self.block}")
        self.table, self.held = t.table, t.held
        self.free = self.free[used:]
        return t.slots

    def load(self, prompts, keep_ratio=0.3, window=8, kernel_size=11):
        """Prefill, evict and store; returns each prompt's last logits."""
        m = self.model
        prefilled = [m.prefill(p) for p in prompts]
        self.seen = torch.tensor([len(p) for p in prompts], device=m.device)
        slots, most = None, max(len(p) for p in prompts)
        for layer in range(m.layers):
            Q, K, V = zip(*(kept[layer] for kept, _ in prefilled))
            keep_len, outs = compress_varlen(list(Q), list(K), list(V), window, kernel_size, keep_ratio)
            if slots is None:  # the kept lengths do not depend on the layer
                self.lens = keep_len.clone()
                slots = self.grow(self.lens, None, most)
            for b, (_, k, v) in enumerate(outs):  # rows past keep_len have slot -1
                self.store(layer, k, v, slots[b:b + 1, :k.shape[2]])
        return torch.stack([logits for _, logits in prefilled])

    def verify(self, tokens, parents):
        """One pass of the decoder over drafted trees (tokens, parents [B, T]; None: chains):
        logits of every node [B, T, vocab], and a function that keeps accepted nodes."""
        m, T = self.model, tokens.shape[1]
        if parents is None:
            mask, depth = None, torch.arange(T, device=m.device)
        else:
            mask, depth = tree_mask_from_parents(parents)
        slots = self.grow(self.lens + T, torch.full_like(self.lens, T), T)
        positions = self.seen[:, None] + depth
        x, rows = m.embed[tokens], []
        for layer, w in enumerate(m.w):
            q, k, v = m.project(x, w)
            o, k = self.attend(layer, q, k, v, positions, slots, mask)
            x = m.after(x, o, w)
            rows.append((k, v))

        def keep(place):
            """place [B, T]: a node's place among the accepted ones, or -1. Their rows move to
            the front of the nodes' slots (a chain's are there); the others are forgotten."""
            if parents is not None:
                to = torch.where(place >= 0, torch.gather(slots, 1, place.clamp(min=0)), -1)
                for layer, (k, v) in enumerate(rows):
                    self.store(layer, k, v, to)
            taken = (place >= 0).sum(1)
            self.lens = self.lens + taken.int()
            self.seen = self.seen + taken

        return m.norm(x) @ m.head, keep


class PagedCaches8(PagedCaches):
    """The same with pages in 8 bits and a scale for each page and head."""

    def __init__(self, model: Decoder, batch: int, pages: int, block: int = 16, max_blocks: int = 64):
        super().__init__(model, batch, pages, block, max_blocks)
        self.K = [k.to(torch.float8_e4m3fn) for k in self.K]
        self.V = [v.to(torch.float8_e4m3fn) for v in self.V]
        scales = lambda: [torch.ones(pages, model.Hkv, device=model.device) for _ in range(model.layers)]  # noqa: E731
        self.K_scales, self.V_scales = scales(), scales()

    def store(self, layer, k, v, slots):
        store_rows_fp8(k, v, slots, self.K[layer], self.V[layer], self.K_scales[layer], self.V_scales[layer])

    def attend(self, layer, q, k, v, positions, slots, mask):
        m, w = self.model, self.model.w[layer]
        q, k = qk_norm_rope(q, k, m.cos, m.sin, positions, q_weight=w["qn"], k_weight=w["kn"])
        self.store(layer, k, v, slots)
        return attention_fp8(q, self.K[layer], self.V[layer], self.K_scales[layer], self.V_scales[layer], self.lens,
                             self.table, tree_mask=mask), k


def draft_tree(root, followers, T):
    """(tokens, parents [B, T]): the next token [B] as the root, likely followers of each node
    below it (``followers`` [vocab, K])."""
    K = followers.shape[1]
    above, which = [-1] + [i // K for i in range(T - 1)], [0] + [i % K for i in range(T - 1)]
    tokens = root[:, None].repeat(1, T)
    for i in range(1, T):
        tokens[:, i] = followers[tokens[:, above[i]], which[i]]
    return tokens, torch.tensor(above, device=root.device).expand(len(root), T)


def accept(tokens, parents, choice):
    """The longest path from the root whose tokens are the decoder's own choices: (place of
    each node on it, or -1; the choice after its last node). ``choice`` [B, T]: likeliest
    token after each node. Parents come before children, so one pass over the nodes does."""
    B, T = tokens.shape
    place = torch.full((B, T), -1, dtype=torch.int64, device=tokens.device)
    place[:, 0] = 0  # the root is the decoder's choice already
    for i in range(1, T):
        p = parents[:, i:i + 1]
        agrees = (torch.gather(place, 1, p) >= 0) & (torch.gather(choice, 1, p) == tokens[:, i:i + 1])
        place[:, i:i + 1] = torch.where(agrees, torch.gather(place, 1, p) + 1, -1)
    # of equal children one path only: the deepest node's ancestors
    depth, last = place.max(1)
    on = torch.zeros_like(place, dtype=torch.bool)
    node = last.clone()
    for _ in range(T):
        on.scatter_(1, node.clamp(min=0)[:, None], True)
        node = torch.where(node > 0, torch.gather(parents, 1, node.clamp(min=0)[:, None])[:, 0], node)
    place = torch.where(on & (place >= 0), place, -1)
    return place, depth + 1, torch.gather(choice, 1, last[:, None])[:, 0]


def draft_chain(root, logits, T, temperature):
    """Tokens [B, T + 1]: the next token [B] and T after it, each drawn from the draft's
    logits ([vocab, vocab]) of the one before."""
    tokens = [root]
    for _ in range(T):
        tokens.append(torch.multinomial((logits[tokens[-1]].float() / temperature).softmax(-1), 1)[:, 0])
    return torch.stack(tokens, 1)


def sample(model, prompts, steps, drafted, temperature=1.0, keep_ratio=0.3, pages=512, block=16):
    """Continuations drawn at a temperature, over caches in 8 bits: (list of token lists,
    tokens a step)."""
    caches = PagedCaches8(model, len(prompts), pages, block)
    last = caches.load(prompts, keep_ratio)
    B, out = len(prompts), [[] for _ in prompts]
    none = torch.empty(B, 0, dtype=torch.int64, device=model.device)
    root = verify_draft(last[:, None], none, torch.rand(B, 1, device=model.device), temperature=temperature).next_token
    for _ in range(steps):
        tokens = draft_chain(root, model.draft, drafted, temperature)
        logits, keep = caches.verify(tokens, None)
        v = verify_draft(logits, tokens[:, 1:], torch.rand(B, drafted + 1, device=model.device),
                         draft_logits=model.draft[tokens[:, :-1]], temperature=temperature)
        at = torch.arange(drafted + 1, device=model.device)
        keep(torch.where(at <= v.accepted[:, None], at, -1))
        root = v.next_token
        for b, (n, row) in enumerate(zip(v.accepted.tolist(), tokens.tolist())):
            out[b] += row[:n + 1]
    return out, sum(map(len, out)) / (steps * B)


def decode(model, prompts, steps, tree, keep_ratio=0.3, pages=512, block=16):
    """Greedy continuation of the prompts: (list of token lists, tokens a step)."""
    caches = PagedCaches(model, len(prompts), pages, block)
    last = caches.load(prompts, keep_ratio)
    root, out = token_logprobs(last, last.argmax(-1), top_k=1).top_tokens[:, 0], [[] for _ in prompts]
    for _ in range(steps):
        tokens, parents = draft_tree(root, model.followers, tree)
        logits, keep = caches.verify(tokens, parents)
        best = token_logprobs(logits, tokens, top_k=1)
        place, _, root = accept(tokens, parents, best.top_tokens[..., 0])
        keep(place)
        for b, (p, row) in enumerate(zip(place.tolist(), tokens.tolist())):
            out[b] += [t for _, t in sorted((at, t) for at, t in zip(p, row) if at >= 0)]
    return out, sum(map(len, out)) / (steps * len(prompts))


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--tree", type=int, default=16)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--sample", type=float, metavar="T", help="draw tokens at this temperature, over caches in 8 bits")
    ap.add_argument("--drafted", type=int, default=4, help="tokens drafted a step with --sample")
    a = ap.parse_args()
    model = Decoder(layers=a.layers)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, model.vocab, (n,), generator=g, device="cuda") for n in (300, 47, 512)]
    if a.sample is not None:
        torch.manual_seed(2)
        out, rate = sample(model, prompts, a.steps, a.drafted, a.sample)
    else:
        out, rate = decode(model, prompts, a.steps, a.tree)
    for p, o in zip(prompts, out):
        print(f"prompt of {len(p)}: {o}")
    print(f"{rate:.2f} tokens a step and sequence")


if __name__ == "__main__":
    main()
