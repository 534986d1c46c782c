"""The operators of a speculative step over paged, evicted KV caches, as measured cases.

A ragged batch of compressed caches (DropKV keeps another number of rows of every
sequence, and those counts exist on the GPU only) lives in pages of a shared pool:

* ``block_tables``   hands out pages and gives every new token its slot;
* ``store_rows``     writes K/V rows (the eviction's outputs, accepted drafts) to slots;
* ``qk_norm_rope``   norms the heads of queries and keys, rotates them by their
                     positions and writes K/V rows to slots in the same pass;
* ``tree_attention`` attends with a tree of drafted tokens over a cache, paged or in
                     row buffers;
* ``token_logprobs`` log probabilities of given tokens, entropy and top alternatives.

``run`` computes each in its plain form in 32 bits, or, where ``own`` is true, by the
calls of ``dropkv_b200``.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
# query heads, KV heads, head size of the attention layers this repository's tests and benchmark use
_HEADS = [(32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 2, 64), (8, 8, 128)]


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small serving batch: a page more for a few requests, a slot for each
        dict(name="tables_step", op="tables", B=32, block=16, longest=2048, new=1, extend=True),
        # 128 caches compressed to at most a tenth of 128K tokens enter the pool at once
        dict(name="tables_prefill", op="tables", B=128, block=64, longest=13107, new=13107, extend=False),
        # one Llama layer's kept rows (a tenth of 128K) go to their pages
        dict(name="store_layer", op="store", B=1, Hkv=8, D=128, N=13107, block=64, ragged=False, nhd=False,
             dtype="bf16"),
        # the accepted rows of four short drafts, the rest of each skipped; pages ordered by token, then head
        dict(name="store_ragged", op="store", B=4, Hkv=2, D=64, N=103, block=16, ragged=True, nhd=True, dtype="fp16"),
        # one decode token of one sequence: latency
        dict(name="rope_token", op="rope", B=1, L=1, heads=0, R=128, norm=False, interleaved=False, store=True,
             block=64, dtype="bf16"),
        # a prefill chunk of 4096 tokens whose model norms its heads
        dict(name="rope_chunk", op="rope", B=1, L=4096, heads=0, R=128, norm=True, interleaved=False, store=False,
             block=64, dtype="bf16"),
        # an odd batch with half of each head rotated, in neighbouring pairs, written to pages too
        dict(name="rope_partial", op="rope", B=3, L=1037, heads=2, R=32, norm=True, interleaved=True, store=True,
             block=16, dtype="fp16"),
        # eight drafted tokens over a short cache in row buffers: latency
        dict(name="tree_short", op="tree", B=1, T=8, heads=2, longest=819, paged=False, block=0, dtype="bf16"),
        # a wide tree over one Llama layer's compressed cache (a tenth of 128K)
        dict(name="tree_layer", op="tree", B=1, T=64, heads=0, longest=13107, paged=True, block=64, dtype="bf16"),
        # a ragged batch of long caches in small pages, seven query heads to a KV head
        dict(name="tree_batch", op="tree", B=8, T=32, heads=1, longest=65536, paged=True, block=16, dtype="fp16"),
        # verifying 16 drafted nodes with their children's tokens, an odd vocabulary: latency
        dict(name="logprobs_step", op="logprobs", N=16, C=4, V=50257, top=5, temperature=0.7, dtype="fp16"),
        # scoring a prompt of 2048 tokens over a large vocabulary
        dict(name="logprobs_prompt", op="logprobs", N=2048, C=1, V=151936, top=20, temperature=1.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["tables", "store", "rope", "tree", "logprobs"])
    if op == "tables":
        extend = rng.random() < 0.5
        longest = _log(rng, 1, 13107)
        return dict(op=op, B=_log(rng, 1, 128), block=rng.choice([8, 16, 32, 64, 128, 256]), longest=longest,
                    new=min(longest, _log(rng, 1, 300)) if extend else longest, extend=extend)
    if op == "store":
        _, Hkv, D = rng.choice(_HEADS)
        n = _log(rng, 1, 13107 * 8 * 128 // (Hkv * D))
        B = min(n, _log(rng, 1, 16))
        return dict(op=op, B=B, Hkv=Hkv, D=D, N=n // B, block=rng.choice([8, 16, 32, 64, 128]),
                    ragged=rng.random() < 0.5, nhd=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]))
    if op == "rope":
        h = rng.randrange(len(_HEADS))
        Hq, Hkv, D = _HEADS[h]
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        n = _log(rng, 1, 4096 * 40 * 128 * 2 // ((Hq + 3 * Hkv) * D * _BYTES[dtype]))
        B = min(n, _log(rng, 1, 16))
        return dict(op=op, B=B, L=n // B, heads=h, R=rng.choice([D, D, D // 2, D // 4]), norm=rng.random() < 0.6,
                    interleaved=rng.random() < 0.3, store=rng.random() < 0.5, block=rng.choice([8, 16, 32, 64, 128]),
                    dtype=dtype)
    if op == "tree":
        h = rng.randrange(len(_HEADS))
        Hq, Hkv, D = _HEADS[h]
        T = _log(rng, 1, 64)
        B = _log(rng, 1, 8)
        most = 8 * 65536 * 4 * 128 * 32 * 7 // (B * Hkv * D * max(T * Hq // Hkv, 32 * 7))
        paged = rng.random() < 0.6
        return dict(op=op, B=B, T=T, heads=h, longest=_log(rng, 1, min(131072, most)), paged=paged,
                    block=rng.choice([8, 16, 32, 64, 128, 256]) if paged else 0, dtype=rng.choice(["bf16", "fp16"]))
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    V = rng.choice([32000, 50257, 151936, _log(rng, 1000, 151936)])
    return dict(op=op, N=_log(rng, 1, 2048 * 151936 * 2 // (V * _BYTES[dtype])), C=rng.choice([1, 1, 2, 5, 16]), V=V,
                top=rng.choice([0, 1, 5, 20, 32]), temperature=rng.choice([1.0, 0.6, 1.3]), dtype=dtype)


def _lengths(B, longest):
    """Cached lengths of a ragged batch: spread evenly from an eighth of the longest up to it."""
    return [max(1, longest - (longest - longest // 8) * i // max(1, B - 1)) for i in range(B)] if B > 1 else [longest]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _tree(rs, T):
    """A draft tree of T nodes, parents before children: (mask of a node's ancestors and itself, depths)."""
    mask, depth = np.zeros((T, T), bool), np.zeros(T, np.int64)
    for i in range(T):
        p = -1 if i == 0 else int(rs.randint(max(-1, i - 9), i))  # children stay near their parents
        if p >= 0:
            mask[i] = mask[p]
            depth[i] = depth[p] + 1
        mask[i, i] = True
    return mask, depth


def _pages(rs, lens, block, spare):
    """Pages for sequences of these lengths, in shuffled order: (table [B, most], pages in the pool)."""
    need = [-(-n // block) for n in lens]
    pool = sum(need) + spare
    order = rs.permutation(pool)
    table = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _slots_of(table, block, first, count):
    """Slot of tokens first .. first + count - 1 of one request."""
    t = np.arange(first, first + count)
    return table[t // block].astype(np.int64) * block + t % block


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    rs = np.random.RandomState((int(seed) * 7919 + 13) % (1 << 31))
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    s = dict(op=case["op"], case=case)
    if case["op"] == "tables":
        B, block = case["B"], case["block"]
        lens = np.array(_lengths(B, case["longest"]), np.int32)[rs.permutation(B)]
        new = np.minimum(lens, case["new"]).astype(np.int32)
        s["max_blocks"] = -(-case["longest"] // block) + 1
        if case["extend"]:  # the pages that the tokens before these hold already
            before, pool = _pages(rs, list(lens - new), block, int(new.sum()) // block + 2 * B + 1)
            table = np.full((B, s["max_blocks"]), -1, np.int32)
            table[:, :before.shape[1]] = before[:, :s["max_blocks"]]
            held = (-(-(lens - new) // block)).astype(np.int32)
            free = np.setdiff1d(np.arange(pool, dtype=np.int32), table[table >= 0])
            s.update(table=cuda(table), held=cuda(held))
        else:
            free = np.arange(int((-(-lens // block)).sum()) + 7, dtype=np.int32)
            s.update(table=None, held=None)
        s.update(lens=cuda(lens), new_lens=cuda(new), free=cuda(rs.permutation(free).astype(np.int32)))
    elif case["op"] == "store":
        B, Hkv, D, N, dt = case["B"], case["Hkv"], case["D"], case["N"], _DTYPES[case["dtype"]]
        kept = np.array(_lengths(B, N))[rs.permutation(B)] if case["ragged"] else np.full(B, N)
        table, pool = _pages(rs, list(kept), case["block"], 2)
        slots = np.full((B, N), -1, np.int64)
        for b in range(B):
            slots[b, :kept[b]] = _slots_of(table[b], case["block"], 0, int(kept[b]))
        s.update(K=_randn(g, B, Hkv, N, D, dtype=dt), V=_randn(g, B, Hkv, N, D, dtype=dt), slots=cuda(slots))
        s["K_pages"], s["V_pages"] = _pool(pool, Hkv, case["block"], D, dt, case["nhd"])
    elif case["op"] == "rope":
        Hq, Hkv, D = _HEADS[case["heads"]]
        B, L, R, dt = case["B"], case["L"], case["R"], _DTYPES[case["dtype"]]
        # a model's projections: one row of all heads for each token, seen as [B, heads, L, D]
        s["Q"], s["K"], s["V"] = (_randn(g, B, L, h, D, dtype=dt).transpose(1, 2) for h in (Hq, Hkv, Hkv))
        P = 131072
        freq = 500000.0 ** (-np.arange(0, R, 2) / R)
        angle = np.arange(P)[:, None] * freq[None, :]
        s["cos"], s["sin"] = cuda(np.cos(angle).astype(np.float32)), cuda(np.sin(angle).astype(np.float32))
        start = rs.randint(0, P - L + 1, B)
        s["positions"] = cuda(start[:, None] + np.arange(L)[None, :])
        s["q_weight"] = s["k_weight"] = None
        if case["norm"]:
            s["q_weight"] = (1 + 0.1 * _randn(g, D)).to(dt)
            s["k_weight"] = (1 + 0.1 * _randn(g, D)).to(dt)
        if case["store"]:
            before = 5  # rows that the sequences hold already
            table, pool = _pages(rs, [before + L] * B, case["block"], 2)
            s["slots"] = cuda(np.stack([_slots_of(table[b], case["block"], before, L) for b in range(B)]))
            s["K_pages"], s["V_pages"] = _pool(pool, Hkv, case["block"], D, dt, False)
    elif case["op"] == "tree":
        Hq, Hkv, D = _HEADS[case["heads"]]
        B, T, dt = case["B"], case["T"], _DTYPES[case["dtype"]]
        lens = np.array(_lengths(B, case["longest"]), np.int64)[rs.permutation(B)]
        trees = [_tree(rs, T)[0] for _ in range(B)]
        s.update(Q=_randn(g, B, T, Hq, D, dtype=dt).transpose(1, 2), cache_lens=cuda(lens.astype(np.int32)),
                 mask=cuda(np.stack(trees)), table=None)
        if case["paged"]:
            table, pool = _pages(rs, list(lens + T), case["block"], 1)
            shape = (pool, Hkv, case["block"], D)
            s["table"] = cuda(table)
        else:
            shape = (B, Hkv, int(lens.max()) + T + 37, D)
        K = _randn(g, *shape, dtype=dt)
        K[..., int(rs.randint(D))] *= 4  # an outlier channel, as keys have
        s.update(K=K, V=_randn(g, *shape, dtype=dt))
    else:
        N, C, V, dt = case["N"], case["C"], case["V"], _DTYPES[case["dtype"]]
        logits = 2.5 * torch.randn(N, V, generator=g, device="cuda")
        best = torch.randint(0, V // 8, (N, 8), generator=g, device="cuda")  # a few likely tokens in each row
        best += V // 8 * torch.arange(8, device="cuda")
        logits.scatter_(1, best, 12 + 3 * _randn(g, N, 8))
        s["logits"] = logits.to(dt)
        s["tokens"] = torch.cat([best[:, :1], torch.randint(0, V, (N, C - 1), generator=g, device="cuda")], 1) \
            if C > 1 else best[:, 0].contiguous()
    return s


def _pool(pages, Hkv, block, D, dt, nhd):
    """An empty K and V pool [pages, Hkv, block, D]; nhd: a page's rows by token, then head."""
    shape = (pages, block, Hkv, D) if nhd else (pages, Hkv, block, D)
    k, v = torch.zeros(shape, dtype=dt, device="cuda"), torch.zeros(shape, dtype=dt, device="cuda")
    return (k.transpose(1, 2), v.transpose(1, 2)) if nhd else (k, v)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_RUN_OWN if own else _RUN)[state["op"]](state)


def _own_tables(s):
    from dropkv_b200 import block_tables
    r = block_tables(s["lens"], s["case"]["block"], s["free"], s["max_blocks"], s["case"]["new"],
                     new_lens=s["new_lens"], table=s["table"], held=s["held"])
    return [r.table, r.held, r.slots, r.used]


def _own_store(s):
    from dropkv_b200 import store_rows
    store_rows(s["K"], s["V"], s["slots"], s["K_pages"], s["V_pages"])
    return [s["K_pages"], s["V_pages"]]


def _own_rope(s):
    from dropkv_b200 import qk_norm_rope
    pages = dict(V=s["V"], slots=s["slots"], K_pages=s["K_pages"], V_pages=s["V_pages"]) if s["case"]["store"] else {}
    out = qk_norm_rope(s["Q"], s["K"], s["cos"], s["sin"], s["positions"], q_weight=s["q_weight"],
                       k_weight=s["k_weight"], eps=1e-6, interleaved=s["case"]["interleaved"], **pages)
    return list(out) + ([s["K_pages"], s["V_pages"]] if pages else [])


def _own_tree(s):
    from dropkv_b200 import tree_attention
    return tree_attention(s["Q"], s["K"], s["V"], s["cache_lens"], tree_mask=s["mask"], block_table=s["table"])


def _own_logprobs(s):
    from dropkv_b200 import token_logprobs
    c = s["case"]
    r = token_logprobs(s["logits"], s["tokens"], top_k=c["top"], temperature=c["temperature"])
    return [r.logprob, r.entropy] + ([r.top_logprobs, r.top_tokens] if c["top"] else [])


def _plain_tables(s):
    block, lens, new, free = s["case"]["block"], s["lens"].long(), s["new_lens"].long(), s["free"]
    B, most, F = lens.numel(), s["max_blocks"], free.numel()
    held = s["held"].long() if s["held"] is not None else torch.zeros_like(lens)
    take = ((lens + block - 1) // block - held).clamp(min=0)
    ends = take.cumsum(0)
    first = ends - take
    got = torch.minimum((F - first).clamp(min=0), take)
    col = torch.arange(most, device=lens.device)[None, :]
    at = (first[:, None] + col - held[:, None]).clamp(0, max(F - 1, 0))
    old = s["table"] if s["table"] is not None else torch.full((B, most), -1, dtype=torch.int32, device=lens.device)
    drawn = (col >= held[:, None]) & (col < (held + got)[:, None])
    table = torch.where(drawn, free[at], torch.where(col < held[:, None], old, -1)).int()
    i = torch.arange(s["case"]["new"], device=lens.device)[None, :]
    t = (lens - new)[:, None] + i
    page = torch.gather(table.long(), 1, (t // block).clamp(max=most - 1))
    slots = torch.where((i < new[:, None]) & (page >= 0) & (t // block < most), page * block + t % block, -1)
    return [table, (held + got).clamp(max=most).int(), slots, ends[-1:]]


def _scatter(pages, rows, slots, block):
    """rows [B, H, N, D] into pages [pages, H, block, D] at slots [B, N]; negative slots are left out."""
    take = slots >= 0
    at = slots[take]
    pages[at // block, :, at % block] = rows.transpose(1, 2)[take]


def _plain_store(s):
    _scatter(s["K_pages"], s["K"], s["slots"], s["case"]["block"])
    _scatter(s["V_pages"], s["V"], s["slots"], s["case"]["block"])
    return [s["K_pages"], s["V_pages"]]


def _normed_rotated(x, weight, cos, sin, R, interleaved):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    c, d = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([c, d], -1).flatten(-2) if interleaved else torch.cat([c, d], -1)
    return torch.cat([r, y[..., R:]], -1).to(x.dtype)


def _plain_rope(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    q = _normed_rotated(s["Q"], s["q_weight"], cos, sin, c["R"], c["interleaved"])
    k = _normed_rotated(s["K"], s["k_weight"], cos, sin, c["R"], c["interleaved"])
    if not c["store"]:
        return [q, k]
    _scatter(s["K_pages"], k, s["slots"], c["block"])
    _scatter(s["V_pages"], s["V"], s["slots"], c["block"])
    return [q, k, s["K_pages"], s["V_pages"]]


def _plain_tree(s):
    Q, K, V, lens = s["Q"], s["K"], s["V"], s["cache_lens"].long()
    B, Hq, T, D = Q.shape
    Hkv = K.shape[1]
    if s["table"] is not None:
        at = s["table"].long().clamp(min=0)
        K, V = (x[at].transpose(1, 2).reshape(B, Hkv, -1, D) for x in (K, V))
    j = torch.arange(K.shape[2], device=Q.device)
    node = j[None, None, :] - lens[:, None, None]                       # [B, 1, L]: the key's node, negative in the cache
    seen = torch.gather(s["mask"], 2, node.clamp(0, T - 1).expand(B, T, -1))
    seen = torch.where(node < 0, True, seen & (node < T))               # [B, T, L]
    q = Q.float().reshape(B, Hkv, Hq // Hkv, T, D)
    scores = torch.einsum("bhgtd,bhld->bhgtl", q, K.float()) * D ** -0.5
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    V = V.float().masked_fill((j[None, :] >= lens[:, None] + T)[:, None, :, None], 0.0)
    out = torch.einsum("bhgtl,bhld->bhgtd", p, V) / p.sum(-1, keepdim=True)
    return out.reshape(B, Hq, T, D).to(Q.dtype)


def _plain_logprobs(s):
    c = s["case"]
    logits, tokens = s["logits"].float(), s["tokens"]
    x = logits / c["temperature"]
    shifted = x - x.amax(-1, keepdim=True)
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    at = tokens if tokens.dim() == 2 else tokens[:, None]
    logprob = torch.gather(shifted, 1, at) - log_total
    entropy = log_total[:, 0] - torch.where(e > 0, e * shifted, 0.0).sum(-1) / total[:, 0]
    out = [logprob.reshape(tokens.shape), entropy]
    if c["top"]:
        ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :c["top"]].contiguous()
        out += [torch.gather(shifted, 1, ids) - log_total, ids]
    return out


_RUN = dict(tables=_plain_tables, store=_plain_store, rope=_plain_rope, tree=_plain_tree, logprobs=_plain_logprobs)
_RUN_OWN = dict(tables=_own_tables, store=_own_store, rope=_own_rope, tree=_own_tree, logprobs=_own_logprobs)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "tables":
        B, most = case["B"], -(-case["longest"] // case["block"]) + 1
        # lengths in and out, the table in (where there is one) and out, the pages handed out, the slots
        pages = sum(-(-min(n, case["new"]) // case["block"]) for n in _lengths(B, case["longest"]))
        table = B * most * 4 * (2 if case["extend"] else 1)
        return dict(bytes=B * (16 if case["extend"] else 12) + table + pages * 4 + B * case["new"] * 8 + 8, flops=0)
    if case["op"] == "store":
        rows = sum(_lengths(case["B"], case["N"])) if case["ragged"] else case["B"] * case["N"]
        return dict(bytes=rows * case["Hkv"] * case["D"] * _BYTES[case["dtype"]] * 4 + case["B"] * case["N"] * 8, flops=0)
    if case["op"] == "rope":
        Hq, Hkv, D = _HEADS[case["heads"]]
        n, e = case["B"] * case["L"], _BYTES[case["dtype"]]
        rows = 2 * (Hq + Hkv) + (3 * Hkv if case["store"] else 0)  # K is written twice, V read and written
        return dict(bytes=n * (rows * D * e + 8 + case["R"] * 4 + (8 if case["store"] else 0)),
                    flops=n * (Hq + Hkv) * (3 * case["R"] + (4 * D if case["norm"] else 0)))
    if case["op"] == "tree":
        Hq, Hkv, D = _HEADS[case["heads"]]
        keys = sum(_lengths(case["B"], case["longest"])) + case["B"] * case["T"]
        rows = case["B"] * case["T"] * Hq
        pages = keys // case["block"] * 4 if case["paged"] else 0
        return dict(bytes=keys * Hkv * D * 4 + rows * D * 4 + pages + case["B"] * (4 + case["T"] ** 2),
                    flops=4 * keys * case["T"] * Hq * D)
    N, V = case["N"], case["V"]
    return dict(bytes=N * V * _BYTES[case["dtype"]] + N * (case["C"] * 12 + 4 + case["top"] * 12), flops=5 * N * V)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"tables": _exact_tables, "store": _exact_store, "rope": _exact_rope, "tree": _exact_tree,
            "logprobs": _exact_logprobs}[case["op"]](s, case)


def _exact_tables(s, case):
    lens, new, free = (s[k].tolist() for k in ("lens", "new_lens", "free"))
    most, block = s["max_blocks"], case["block"]
    old = s["table"].tolist() if s["table"] is not None else [[]] * len(lens)
    held = s["held"].tolist() if s["held"] is not None else [0] * len(lens)
    table = np.full((len(lens), most), -1, np.int32)
    slots = np.full((len(lens), case["new"]), -1, np.int64)
    asked, have = 0, []
    for b, n in enumerate(lens):
        row = old[b][:held[b]]
        want = max(0, -(-n // block) - held[b])
        row = (row + free[asked:asked + want])[:most]
        asked += want
        table[b, :len(row)] = row
        have.append(len(row))
        for i in range(new[b]):
            t = n - new[b] + i
            if t // block < len(row) and row[t // block] >= 0:
                slots[b, i] = row[t // block] * block + t % block
    return [table, np.array(have, np.int32), slots, np.array([asked], np.int64)]


def _placed(pages, rows, slots, block):
    """The pool in 64 bits with rows [B, H, N, D] put at slots, one sequence after another."""
    out = pages.double().transpose(1, 2).contiguous()                   # [pages, block, H, D]
    flat = out.view(-1, *out.shape[2:])
    for b in range(slots.shape[0]):
        keep = torch.nonzero(slots[b] >= 0)[:, 0]
        flat[slots[b, keep]] = rows[b].double().permute(1, 0, 2)[keep]
    return out.transpose(1, 2)


def _exact_store(s, case):
    return [_placed(s["K_pages"], s["K"], s["slots"], case["block"]),
            _placed(s["V_pages"], s["V"], s["slots"], case["block"])]


def _exact_rope(s, case):
    R, pos = case["R"], s["positions"]
    cos, sin = s["cos"].double()[pos], s["sin"].double()[pos]           # [B, L, R / 2]
    pairs = torch.arange(R // 2, device=pos.device)
    lo, hi = (2 * pairs, 2 * pairs + 1) if case["interleaved"] else (pairs, pairs + R // 2)

    def turned(x, w):
        y = x.double().clone()
        if w is not None:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6) * w.double()
        z = torch.complex(y[..., lo], y[..., hi]) * torch.complex(cos, sin)[:, None]
        y[..., lo], y[..., hi] = z.real, z.imag
        return y

    q, k = turned(s["Q"], s["q_weight"]), turned(s["K"], s["k_weight"])
    if not case["store"]:
        return [q, k]
    return [q, k, _placed(s["K_pages"], k, s["slots"], case["block"]),
            _placed(s["V_pages"], s["V"], s["slots"], case["block"])]


def _exact_tree(s, case):
    Q, mask = s["Q"].double(), s["mask"]
    B, Hq, T, D = Q.shape
    Hkv = s["K"].shape[1]
    out = torch.empty(B, Hq, T, D, dtype=torch.float64, device=Q.device)
    for b, n in enumerate(s["cache_lens"].tolist()):
        if s["table"] is not None:
            ids = s["table"][b, :-(-(n + T) // case["block"])].long()
        for h in range(Hkv):
            if s["table"] is not None:
                k, v = (s[x][ids, h].reshape(-1, D)[:n + T].double() for x in "KV")
            else:
                k, v = (s[x][b, h, :n + T].double() for x in "KV")
            for hq in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = Q[b, hq] @ k.T / math.sqrt(D)
                z[:, n:] = torch.where(mask[b], z[:, n:], -math.inf)
                out[b, hq] = torch.softmax(z, -1) @ v
    return out


def _exact_logprobs(s, case):
    logits, tokens = s["logits"], s["tokens"]
    at = tokens.reshape(len(tokens), -1)
    logprob, entropy, tops, ids = [], [], [], []
    for a in range(0, len(tokens), 128):  # by 128 rows: a row takes 8 bytes for every word
        z = torch.log_softmax(logits[a:a + 128].double() / case["temperature"], -1)
        logprob.append(torch.gather(z, 1, at[a:a + 128]))
        entropy.append(-(z.exp() * z).sum(-1))
        if case["top"]:
            order = torch.argsort(-logits[a:a + 128].double(), dim=-1, stable=True)[:, :case["top"]]
            ids.append(order)
            tops.append(torch.gather(z, 1, order))
    out = [torch.cat(logprob).reshape(tokens.shape), torch.cat(entropy)]
    return out + ([torch.cat(tops), torch.cat(ids)] if case["top"] else [])
