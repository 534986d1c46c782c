"""The snippets of the integration guide on paged caches, run as they stand on small inputs."""

import os
import re

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def snippet(name):
    """The first block of Python that imports ``name``."""
    with open(os.path.join(ROOT, "INTEGRATION.md")) as f:
        blocks = re.findall(r"```python\n(.*?)```", f.read(), re.S)
    return next(b for b in blocks if re.search(rf"import .*\b{name}\b", b))


def inputs(T, fp8):
    """What a program has in hand before the snippet: two sequences that keep 70 and 130 rows."""
    g = torch.Generator(device="cuda").manual_seed(0)
    B, Hq, Hkv, D, pages, vocab = 2, 8, 2, 128, 12, 100
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    angle = torch.arange(400, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device="cuda") / D)
    pool = [torch.zeros(pages, Hkv, 64, D, device="cuda").to(torch.float8_e4m3fn if fp8 else torch.bfloat16) for _ in "KV"]
    d = dict(torch=torch, B=B, T=T, max_blocks=4, max_keep=130, keep_lens=ints(70, 130), new_lens=ints(T, T),
             free_pages=torch.randperm(pages, generator=g, device="cuda").int(), seen=torch.tensor([[300], [200]], device="cuda"),
             K_c=draw(B, Hkv, 130, D), V_c=draw(B, Hkv, 130, D), K_pages=pool[0], V_pages=pool[1], cos=angle.cos(), sin=angle.sin(),
             q_weight=draw(D), k_weight=draw(D), tokens=torch.randint(0, vocab, (B, T), generator=g, device="cuda"),
             parents=torch.tensor([[-1, 0, 0, 1]], device="cuda").expand(B, T), children=torch.randint(0, vocab, (B, T), generator=g, device="cuda"))
    if fp8:
        d.update(K_scales=torch.zeros(pages, Hkv, device="cuda"), V_scales=torch.zeros(pages, Hkv, device="cuda"),
                 positions=d["seen"] + torch.arange(T, device="cuda"), Q_new=draw(B, Hq, T, D), K_new=draw(B, Hkv, T, D),
                 V_new=draw(B, Hkv, T, D), logits=draw(B, T, vocab), draft_logits=draw(B, T - 1, vocab))
    else:
        d.update(Q=draw(B, Hq, T, D), K=draw(B, Hkv, T, D), V=draw(B, Hkv, T, D), logits=draw(B, T, vocab))
    return d


def attended(q, rows_k, rows_v, lens, see):
    """Attention over the first ``lens`` rows and T new ones, in 32 bits."""
    out = torch.empty_like(q, dtype=torch.float32)
    g, T = q.shape[1] // rows_k.shape[1], q.shape[2]
    for b, n in enumerate(lens):
        k, v = (x[b, :, :n + T].float().repeat_interleave(g, 0) for x in (rows_k, rows_v))
        z = q[b].float() @ k.transpose(1, 2) * q.shape[-1] ** -0.5
        z[:, :, n:] = z[:, :, n:].masked_fill(~see[b], float("-inf"))
        out[b] = torch.softmax(z, -1) @ v
    return out


def test_trees_over_pages():
    T, d = 4, inputs(4, False)
    code, ns = snippet("tree_attention"), dict(d)
    exec("from dropkv_b200 import *\n" + code, ns)
    rows = [torch.zeros(2, 2, 134, 128, device="cuda").bfloat16() for _ in "KV"]
    for b, n in enumerate((70, 130)):
        for r, kept, new in zip(rows, (d["K_c"], d["V_c"]), (ns["k"], d["V"])):
            r[b, :, :n], r[b, :, n:n + T] = kept[b, :, :n], new[b]
    want = attended(ns["q"], *rows, (70, 130), ns["mask"])
    # 16-bit weights and output: 2^-8 of rows of size 4 at most
    assert float((ns["out"].float() - want).abs().max()) < 4 * 2.0 ** -7
    assert ns["lp"].top_tokens.shape == (2, T, 8)


def test_chains_over_pages_in_8_bits():
    T, d = 4, inputs(4, True)
    code, ns = snippet("attention_fp8"), dict(d)
    exec("from dropkv_b200 import *\n" + code, ns)
    kept = torch.arange(130, device="cuda") < torch.tensor([[70], [130]], device="cuda")
    rows = []
    for back, given, new in ((ns["K"], d["K_c"], ns["k"]), (ns["V"], d["V_c"], d["V_new"])):
        # what was stored is read back: off by half a step of 8 bits at most, zeros past the rows
        off = (back.float() - given.float()).abs()
        assert bool((off <= 2.0 ** -4 * given.float().abs() + 2.0 ** -9)[kept[:, None, :, None].expand_as(off)].all())
        assert not back.transpose(1, 2)[~kept].any()
        r = torch.zeros(2, 2, 134, 128, device="cuda")
        for b, n in enumerate((70, 130)):
            r[b, :, :n], r[b, :, n:n + T] = given[b, :, :n].float(), new[b].float()
        rows.append(r)
    chain = torch.ones(2, T, T, dtype=torch.bool, device="cuda").tril()
    want = attended(ns["q"], *rows, (70, 130), chain)
    # rows rounded to 8 bits (2^-4 each): logits of size 12 off by some 2^-4 of sqrt(128) terms; far from what other rows would give
    got = ns["out"].float()
    assert float((got - want).norm() / want.norm()) < 0.2
    other = attended(ns["q"], rows[0].flip(2), rows[1].flip(2), (70, 130), chain)
    assert float((got - other).norm() / other.norm()) > 0.5
    v = ns["v"]
    assert v.accepted.shape == v.next_token.shape == (2,) and v.accept_prob.shape == (2, T - 1)
    assert bool(((v.next_token >= 0) & (v.next_token < 100)).all())
