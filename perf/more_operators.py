"""The operators of a decode step over caches held in 8 bits, as measured cases.

The pages of a pool hold rows in e4m3 with one power-of-two scale for each page and head
(a row's value is its 8 bits times the scale of its page):

* ``store_rows_fp8``  quantises K/V rows as they are written to slots: a page's scale grows
                      with its largest value, and rows that stand there already follow it;
* ``load_rows_fp8``   reads rows back;
* ``attention_fp8``   attends over such a cache: single tokens, drafted trees, prompt chunks,
                      all of it or the last rows and a few first ones;
* ``verify_draft``    accepts drafted tokens against the target's probabilities by given
                      random numbers and draws the token after them.

``run`` computes each in its plain form in 32 bits (the probabilities in 64, as a token is
found by a long sum), or, where ``own`` is true, by the calls of ``dropkv_b200``.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_E4M3 = torch.float8_e4m3fn
# query heads, KV heads, head size of the attention layers this repository's tests and benchmark use
_HEADS = [(32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 2, 64), (8, 8, 128)]


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one Llama layer's kept rows (a tenth of 128K tokens) enter their pages, and are read back for a check
        dict(name="store_layer", op="store", B=1, Hkv=8, D=128, N=13107, before=0, block=64, nhd=False, dtype="bf16"),
        # a decode step of 64 requests: one row each into pages that hold rows already, read back with them
        dict(name="store_step", op="store", B=64, Hkv=2, D=64, N=1, before=819, block=16, nhd=True, dtype="fp16"),
        # a ragged batch of long caches is read back to be evicted again
        dict(name="load_long", op="load", B=8, Hkv=4, D=128, N=65536, block=16, nhd=False, dtype="fp16"),
        # a short cache read back in 32 bits: latency
        dict(name="load_short", op="load", B=1, Hkv=2, D=64, N=819, block=64, nhd=True, dtype="fp32"),
        # a decode step over 32 compressed caches of up to a tenth of 128K tokens
        dict(name="attend_step", op="attend", B=32, T=1, heads=0, longest=13107, block=64, window=0, sinks=0, tree=False,
             dtype="bf16"),
        # a decode step over few, long caches in small pages, seven query heads to a KV head
        dict(name="attend_long", op="attend", B=8, T=1, heads=1, longest=65536, block=16, window=0, sinks=0, tree=False,
             dtype="fp16"),
        # a decode step that sees the last rows and four first ones of long caches: latency
        dict(name="attend_window", op="attend", B=4, T=1, heads=2, longest=65536, block=16, window=1000, sinks=4, tree=False,
             dtype="bf16"),
        # a drafted tree over one Llama layer's compressed cache
        dict(name="attend_tree", op="attend", B=1, T=64, heads=0, longest=13107, block=64, window=0, sinks=0, tree=True,
             dtype="bf16"),
        # a prompt chunk of 4096 tokens over the compressed cache of those before it
        dict(name="attend_chunk", op="attend", B=1, T=4096, heads=0, longest=13107, block=64, window=0, sinks=0, tree=False,
             dtype="bf16"),
        # verifying five drafted tokens of four sequences, an odd vocabulary: latency
        dict(name="verify_step", op="verify", B=4, T=5, V=50257, draft=True, ragged=False, temperature=0.7, dtype="fp16"),
        # verifying a large batch over a large vocabulary, drafts of up to seven tokens
        dict(name="verify_batch", op="verify", B=64, T=7, V=151936, draft=True, ragged=True, temperature=1.0, dtype="bf16"),
        # a draft without probabilities (a table of followers)
        dict(name="verify_table", op="verify", B=16, T=4, V=32000, draft=False, ragged=False, temperature=1.0, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["store", "load", "attend", "attend", "verify"])
    block = rng.choice([8, 16, 32, 64, 128, 256])
    if op == "store":
        _, Hkv, D = rng.choice(_HEADS)
        append = rng.random() < 0.5
        n = _log(rng, 1, (1024 if append else 13107) * 8 * 128 // (Hkv * D))
        B = min(n, _log(rng, 1, 64))
        return dict(op=op, B=B, Hkv=Hkv, D=D, N=n // B, before=_log(rng, 1, 2048) if append else 0, block=block,
                    nhd=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "load":
        _, Hkv, D = rng.choice(_HEADS)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        n = _log(rng, 1, 8 * 65536 * 4 * 128 * 2 // (Hkv * D * _BYTES[dtype]))
        B = min(n, _log(rng, 1, 16))
        return dict(op=op, B=B, Hkv=Hkv, D=D, N=n // B, block=block, nhd=rng.random() < 0.5, dtype=dtype)
    if op == "attend":
        h = rng.randrange(len(_HEADS))
        Hq, Hkv, D = _HEADS[h]
        T = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 4096)])
        B = _log(rng, 1, 4 if T > 64 else 64)
        most = min(8 * 65536 * 4 * 128 // (B * Hkv * D), 4096 * 32 * 15155 * 128 // (B * T * Hq * D) - T)
        tree = T <= 64 and rng.random() < 0.5
        window = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(op=op, B=B, T=T, heads=h, longest=_log(rng, 1, max(1, min(131072, most))), block=block,
                    window=max(window, T) if tree and window else window, sinks=rng.choice([0, 1, 4, 100]) if window else 0,
                    tree=tree, dtype=rng.choice(["bf16", "fp16"]))
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    V = rng.choice([32000, 50257, 151936, _log(rng, 1000, 151936)])
    T = rng.choice([1, 3, 5, 7, _log(rng, 1, 16)])
    most = 64 * 15 * 151936 * 2 // ((2 * T + 1) * V * _BYTES[dtype])
    return dict(op=op, B=_log(rng, 1, max(1, min(256, most))), T=T, V=V, draft=rng.random() < 0.7, ragged=rng.random() < 0.4,
                temperature=rng.choice([1.0, 0.6, 1.3]), dtype=dtype)


def _lengths(B, longest):
    """Lengths of a ragged batch: spread evenly from an eighth of the longest up to it."""
    return [max(1, longest - (longest - longest // 8) * i // max(1, B - 1)) for i in range(B)] if B > 1 else [longest]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _tree(rs, T):
    """A draft tree of T nodes, parents before children: the mask of a node's ancestors and itself."""
    mask = np.zeros((T, T), bool)
    for i in range(T):
        p = -1 if i == 0 else int(rs.randint(max(-1, i - 9), i))  # children stay near their parents
        if p >= 0:
            mask[i] = mask[p]
        mask[i, i] = True
    return mask


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


def _slots(table, block, first, ends, most):
    """Slots [B, most] of tokens first_b .. ends_b - 1 of each request, -1 past them."""
    out = np.full((len(ends), most), -1, np.int64)
    for b, (lo, hi) in enumerate(zip(first, ends)):
        t = np.arange(lo, hi)
        out[b, :hi - lo] = table[b][t // block].astype(np.int64) * block + t % block
    return out


def _pool(g, pages, H, block, D, nhd=False, outlier=None):
    """Pages of drawn rows in 8 bits and their scales: (pages [pages, H, block, D], scales [pages, H])."""
    x = torch.randn(pages, H, block, D, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-1, 2, (pages, H, 1, 1), generator=g, device="cuda"))  # pages differ in size
    if outlier is not None:
        x[..., outlier] *= 4  # a channel larger than the others, as keys have
    scale = _scale_for(x.abs().amax((2, 3)))
    x8 = (x / scale[:, :, None, None]).to(_E4M3)
    if nhd:  # a page's rows by token, then head
        x8 = x8.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(_E4M3)
    return x8, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    rs = np.random.RandomState((int(seed) * 7919 + 13) % (1 << 31))
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    s = dict(op=case["op"], case=case)
    if case["op"] in ("store", "load"):
        B, H, D, N, block, dt = (case[k] for k in ("B", "Hkv", "D", "N", "block", "dtype"))
        if case["op"] == "load":
            lens = np.array(_lengths(B, N))[rs.permutation(B)]
            table, pool = _pages(rs, list(lens), block, 1)
            s["slots"] = cuda(_slots(table, block, [0] * B, lens, N))
        else:
            before = np.array(_lengths(B, case["before"]))[rs.permutation(B)] if case["before"] else np.zeros(B, int)
            table, pool = _pages(rs, list(before + N), block, 1)
            s["slots"] = cuda(_slots(table, block, before, before + N, N))
            start = before // block * block  # the rows of the touched pages are read back
            s["back"] = cuda(_slots(table, block, start, before + N, N + min(block, case["before"])))
            rows = torch.exp2(torch.randint(-1, 3, (B, 1, N, 1), generator=g, device="cuda"))  # rows differ in size
            s["K"], s["V"] = ((rows * torch.randn(B, H, N, D, generator=g, device="cuda")).to(_DTYPES[dt]) for _ in "KV")
        s["K_pages"], s["K_scales"] = _pool(g, pool, H, block, D, case["nhd"])
        s["V_pages"], s["V_scales"] = _pool(g, pool, H, block, D, case["nhd"])
    elif case["op"] == "attend":
        Hq, Hkv, D = _HEADS[case["heads"]]
        B, T, dt = case["B"], case["T"], _DTYPES[case["dtype"]]
        lens = np.array(_lengths(B, case["longest"]), np.int64)[rs.permutation(B)]
        table, pool = _pages(rs, list(lens + T), case["block"], 1)
        s.update(Q=_randn(g, B, T, Hq, D, dtype=dt).transpose(1, 2), cache_lens=cuda(lens.astype(np.int32)),
                 table=cuda(table), mask=cuda(np.stack([_tree(rs, T) for _ in range(B)])) if case["tree"] else None)
        s["K_pages"], s["K_scales"] = _pool(g, pool, Hkv, case["block"], D, outlier=int(rs.randint(D)))
        s["V_pages"], s["V_scales"] = _pool(g, pool, Hkv, case["block"], D)
    else:
        B, T, V, dt = case["B"], case["T"], case["V"], _DTYPES[case["dtype"]]
        logits = 2.5 * torch.randn(B, T + 1, V, generator=g, device="cuda")
        best = torch.randint(0, V // 8, (B, T + 1, 8), generator=g, device="cuda")  # a few likely tokens in each row
        best += V // 8 * torch.arange(8, device="cuda")
        logits.scatter_(2, best, 10 + 2 * _randn(g, B, T + 1, 8))
        s["target"] = logits.to(dt)
        draft = (logits[:, :T] + 0.4 * _randn(g, B, T, V)).to(dt)  # a smaller model's, near the target's
        if case["draft"]:
            q = torch.softmax(draft.float() / case["temperature"], -1)
            tokens = torch.multinomial(q.view(B * T, V), 1, generator=g).view(B, T)
        else:
            tokens = draft.argmax(-1)
        if case["ragged"]:
            drafted = cuda(rs.randint(0, T + 1, (B, 1)))
            tokens = torch.where(torch.arange(T, device="cuda") < drafted, tokens, -1)
        s.update(draft=draft if case["draft"] else None, tokens=tokens,
                 uniforms=torch.rand(B, T + 1, generator=g, device="cuda"))
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_RUN_OWN if own else _RUN)[state["op"]](state)


def _own_store(s):
    from dropkv_b200 import load_rows_fp8, store_rows_fp8
    pool = (s["K_pages"], s["V_pages"], s["K_scales"], s["V_scales"])
    store_rows_fp8(s["K"], s["V"], s["slots"], *pool)
    return [*load_rows_fp8(*pool, s["back"], dtype=s["K"].dtype), s["K_scales"], s["V_scales"]]


def _own_load(s):
    from dropkv_b200 import load_rows_fp8
    return list(load_rows_fp8(s["K_pages"], s["V_pages"], s["K_scales"], s["V_scales"], s["slots"],
                              dtype=_DTYPES[s["case"]["dtype"]]))


def _own_attend(s):
    from dropkv_b200 import attention_fp8
    c = s["case"]
    return attention_fp8(s["Q"], s["K_pages"], s["V_pages"], s["K_scales"], s["V_scales"], s["cache_lens"], s["table"],
                         tree_mask=s["mask"], window=c["window"] or None, sinks=c["sinks"])


def _own_verify(s):
    from dropkv_b200 import verify_draft
    r = verify_draft(s["target"], s["tokens"], s["uniforms"], draft_logits=s["draft"], temperature=s["case"]["temperature"])
    return [r.accepted, r.next_token, r.accept_prob]


def _scale_for(largest):
    """The smallest power of two (2^-126 at least) that brings a largest value to at most 448."""
    m, e = torch.frexp(largest.double() / 448)
    return torch.exp2((e - (m == 0.5).int()).clamp(min=-126).double()).float().masked_fill(largest == 0, 2.0 ** -126)


def _stored(x, slots, pages, scales):
    """Rows x [B, H, N, D] to slots of pages in 8 bits; pages and scales change in place."""
    P, H, block, D = pages.shape
    take = slots >= 0
    page, off = slots[take] // block, slots[take] % block
    rows = x.transpose(1, 2)[take].float()                                                       # [n, H, D]
    largest = torch.zeros(P, H, device=x.device).index_reduce_(0, page, rows.abs().amax(-1), "amax")
    touched = torch.zeros(P, dtype=torch.bool, device=x.device).index_fill_(0, page, True)
    started = torch.zeros(P, dtype=torch.bool, device=x.device).index_fill_(0, page[off == 0], True)
    before = scales.masked_fill(started[:, None], 0.0)
    after = torch.where(touched[:, None], torch.maximum(_scale_for(largest), before), scales)
    grown = (touched & ~started)[:, None] & (after > before)
    old = (pages.float() * (before / after)[:, :, None, None]).to(_E4M3).view(torch.uint8)
    raw = pages.view(torch.uint8)
    raw.copy_(torch.where(grown[:, :, None, None], old, raw))
    raw[page, :, off] = (rows / after[page][..., None]).to(_E4M3).view(torch.uint8)
    scales.copy_(after)


def _read(pages, scales, slots, dtype):
    """Rows at slots [B, N] in `dtype`: [B, H, N, D], zeros where a slot is negative."""
    block = pages.shape[2]
    at = slots.clamp(min=0)
    x = pages.view(torch.uint8)[at // block, :, at % block].view(_E4M3).float() * scales[at // block][..., None]
    return x.masked_fill((slots < 0)[:, :, None, None], 0.0).to(dtype).transpose(1, 2).contiguous()


def _plain_store(s):
    _stored(s["K"], s["slots"], s["K_pages"], s["K_scales"])
    _stored(s["V"], s["slots"], s["V_pages"], s["V_scales"])
    return [_read(s["K_pages"], s["K_scales"], s["back"], s["K"].dtype),
            _read(s["V_pages"], s["V_scales"], s["back"], s["K"].dtype), s["K_scales"], s["V_scales"]]


def _plain_load(s):
    dt = _DTYPES[s["case"]["dtype"]]
    return [_read(s["K_pages"], s["K_scales"], s["slots"], dt), _read(s["V_pages"], s["V_scales"], s["slots"], dt)]


def _plain_attend(s):
    c, Q, lens = s["case"], s["Q"], s["cache_lens"].long()
    B, Hq, T, D = Q.shape
    Hkv, g = s["K_pages"].shape[1], Hq // s["K_pages"].shape[1]
    at = s["table"].long().clamp(min=0)
    K, V = ((s[x + "_pages"].view(torch.uint8)[at].view(_E4M3).float() * s[x + "_scales"][at][..., None, None])
            .transpose(1, 2).reshape(B, Hkv, -1, D) for x in "KV")
    j = torch.arange(K.shape[2], device=Q.device)
    node = j[None, None, :] - lens[:, None, None]                       # [B, 1, L]: the key's node, negative in the cache
    i = torch.arange(T, device=Q.device)
    if s["mask"] is None:
        depth = i[None, :].expand(B, T)
        seen = node <= i[:, None]
        near = node > (i - c["window"])[:, None]
    else:
        depth = (s["mask"].sum(-1) - 1).clamp(min=0)
        seen = torch.gather(s["mask"], 2, node.clamp(0, T - 1).expand(B, T, -1))
        seen = torch.where(node < 0, True, seen & (node < T))           # [B, T, L]
        near = (node >= 0) | (node > (depth - c["window"])[..., None])
    if c["window"]:
        seen = seen & (near | (j < c["sinks"]))
    V = V.masked_fill((j[None, :] >= lens[:, None] + T)[:, None, :, None], 0.0)
    q = Q.float().reshape(B, Hkv, g, T, D)
    out = torch.empty(B, Hkv, g, T, D, device=Q.device)
    heads = max(1, min(Hkv, 2 ** 31 // (B * g * T * K.shape[2])))       # as many at a time as fit a few GB
    for h in range(0, Hkv, heads):
        z = torch.einsum("bhgtd,bhld->bhgtl", q[:, h:h + heads], K[:, h:h + heads]) * D ** -0.5
        z = z.masked_fill(~seen[:, None, None], float("-inf"))
        p = torch.exp(z - z.amax(-1, keepdim=True))
        out[:, h:h + heads] = torch.einsum("bhgtl,bhld->bhgtd", p, V[:, h:h + heads]) / p.sum(-1, keepdim=True)
    return out.reshape(B, Hq, T, D).to(Q.dtype)


def _probabilities(logits, temperature):
    x = logits.double() / temperature
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    tokens, u = s["tokens"], s["uniforms"].double()
    B, T = tokens.shape
    p = _probabilities(s["target"], s["case"]["temperature"])           # [B, T + 1, V]
    drafted = tokens >= 0
    at = tokens.clamp(min=0)[..., None]
    px = torch.gather(p[:, :T], 2, at)[..., 0]
    if s["draft"] is not None:
        q = _probabilities(s["draft"], s["case"]["temperature"])
        qx = torch.gather(q, 2, at)[..., 0]
    else:
        q = torch.zeros_like(p[:, :T]).scatter_(2, at, 1.0)
        qx = torch.ones_like(px)
    ok = drafted & (u[:, :T] * qx < px)
    prob = torch.where(drafted, (px / qx).clamp(max=1), 0.0)
    accepted = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device=tokens.device)
    n = accepted.clamp(max=T - 1)
    rejected = (accepted < T) & drafted[b, n]
    r = p[b, accepted]
    r = torch.where(rejected[:, None], (r - q[b, n]).clamp(min=0), r)
    c = r.cumsum(-1)
    nxt = (c <= u[:, T:] * c[:, -1:]).sum(-1)
    return [accepted, nxt.clamp(max=p.shape[-1] - 1), prob.float()]


_RUN = dict(store=_plain_store, load=_plain_load, attend=_plain_attend, verify=_plain_verify)
_RUN_OWN = dict(store=_own_store, load=_own_load, attend=_own_attend, verify=_own_verify)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] in ("store", "load"):
        B, H, D, N, block, e = (case[k] for k in ("B", "Hkv", "D", "N", "block", "dtype"))
        e = _BYTES[e]
        if case["op"] == "load":  # rows that are there in, all rows out, slots and scales
            rows = sum(_lengths(B, N))
            return dict(bytes=2 * H * D * (rows + B * N * e) + B * N * 8 + rows // block * H * 8, flops=0)
        # rows in, in 8 bits out and in again with their pages' earlier ones, all of these out; slots and scales
        ends = _lengths(B, case["before"]) if case["before"] else [0] * B
        back = sum(N + n % block for n in ends)
        pages = sum(-(-(n % block + N) // block) for n in ends)
        return dict(bytes=2 * H * D * (B * N * (e + 1) + back * (1 + e)) + 16 * B * N + pages * H * 16, flops=0)
    if case["op"] == "attend":
        Hq, Hkv, D = _HEADS[case["heads"]]
        T, w = case["T"], case["window"]
        keys = seen = 0
        for n in _lengths(case["B"], case["longest"]):
            i = np.arange(T)
            if w:
                first = np.maximum(n + i - w + 1, 0)
                mine = np.minimum(case["sinks"], first) + n + i + 1 - first
                keys += min(case["sinks"], int(first[0])) + n + T - int(first[0])
            else:
                mine = n + i + 1
                keys += n + T
            seen += int(mine.sum())
        rows = case["B"] * T * Hq
        return dict(bytes=keys * Hkv * D * 2 + keys // case["block"] * (Hkv * 8 + 4) + rows * D * 4 + case["B"] * 4
                    + (case["B"] * T * T if case["tree"] else 0), flops=4 * seen * Hq * D)
    B, T, V, e = case["B"], case["T"], case["V"], _BYTES[case["dtype"]]
    rows = B * (T + 1) + (B * T if case["draft"] else 0)
    return dict(bytes=rows * V * e + B * T * 12 + B * (T + 1) * 4 + B * 16, flops=4 * rows * V)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "load": _exact_load, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](s, case)


def _e4m3(y):
    """The nearest value with three bits behind the first, ties to even; steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_read(values, slots, block):
    """Rows of values [pages, H, block, D] (64 bits) at slots."""
    flat = values.transpose(1, 2).reshape(-1, values.shape[1], values.shape[3])
    out = flat[slots.clamp(min=0)]
    out[slots < 0] = 0
    return out.transpose(1, 2)


def _exact_store(s, case):
    block, out, scales = case["block"], [], []
    for name in "KV":
        x, x8, sc = s[name].double(), s[name + "_pages"].double(), s[name + "_scales"].double()
        slots = s["slots"]
        pages = torch.unique(slots[slots >= 0] // block).tolist()
        where = {}
        for b, row in enumerate((slots // block).tolist()):
            for n, p in enumerate(row):
                if slots[b, 0] >= 0:
                    where.setdefault(p, []).append((b, n))
        for p in pages:
            b, n0, n1 = where[p][0][0], where[p][0][1], where[p][-1][1] + 1
            rows = x[b, :, n0:n1]                                        # [H, rows, D]
            first = int(slots[b, n0]) % block
            largest = rows.abs().amax((1, 2)) / 448
            want = torch.exp2(torch.ceil(torch.log2(largest.clamp(min=2.0 ** -126))))
            if first:
                want = torch.maximum(want, sc[p])
                x8[p] = torch.where((want > sc[p])[:, None, None], _e4m3(x8[p] * (sc[p] / want)[:, None, None]), x8[p])
            sc[p] = want
            x8[p, :, first:first + n1 - n0] = _e4m3(rows / want[:, None, None])
        out.append(_exact_read(x8 * sc[:, :, None, None], s["back"], block))
        scales.append(sc)
    return out + scales


def _exact_load(s, case):
    return [_exact_read(s[x + "_pages"].double() * s[x + "_scales"].double()[:, :, None, None], s["slots"], case["block"])
            for x in "KV"]


def _exact_attend(s, case):
    Q, w = s["Q"].double(), case["window"]
    B, Hq, T, D = Q.shape
    Hkv = s["K_pages"].shape[1]
    g = Hq // Hkv
    out = torch.empty(B, Hq, T, D, dtype=torch.float64, device=Q.device)
    for b, n in enumerate(s["cache_lens"].tolist()):
        ids = s["table"][b, :-(-(n + T) // case["block"])].long()
        hide = torch.zeros(T, n + T, dtype=torch.bool, device=Q.device)
        at = torch.arange(n + T, device=Q.device)
        for i0 in range(0, T, 512):
            i = torch.arange(i0, min(T, i0 + 512), device=Q.device)
            place = n + i
            if s["mask"] is not None:
                place = n + s["mask"][b, i].sum(-1) - 1
                hide[i, n:] = ~s["mask"][b, i]
            else:
                hide[i] = at[None, :] > place[:, None]
            if w:
                far = (at[None, :] <= place[:, None] - w) & (at >= case["sinks"])[None, :]
                if s["mask"] is not None:
                    far[:, n:] = False
                hide[i] |= far
        for h in range(Hkv):
            k, v = ((s[x + "_pages"].view(torch.uint8)[ids, h].view(_E4M3).double()
                     * s[x + "_scales"][ids, h].double()[:, None, None]).reshape(-1, D)[:n + T] for x in "KV")
            for hq in range(h * g, (h + 1) * g):
                z = (Q[b, hq] @ k.T / math.sqrt(D)).masked_fill_(hide, -math.inf)
                out[b, hq] = torch.softmax(z, -1) @ v
    return out


def _exact_verify(s, case):
    tokens, u, tau = s["tokens"].tolist(), s["uniforms"].tolist(), case["temperature"]
    T, V = case["T"], case["V"]
    accepted, following, prob = [], [], np.zeros((len(tokens), T))
    for b, row in enumerate(tokens):
        n, rest, counting = 0, None, True
        for i in range(T):
            if row[i] < 0:
                counting = False
                continue
            p = torch.softmax(s["target"][b, i].double() / tau, 0)
            if s["draft"] is not None:
                q = torch.softmax(s["draft"][b, i].double() / tau, 0)
            else:
                q = torch.zeros_like(p)
                q[row[i]] = 1
            px, qx = float(p[row[i]]), float(q[row[i]])
            prob[b, i] = min(1.0, px / qx)
            if not counting:
                continue
            if u[b][i] * qx >= px:
                rest, counting = torch.relu(p - q), False
            else:
                n += 1
        if rest is None:
            rest = torch.softmax(s["target"][b, n].double() / tau, 0)
        sums = torch.cumsum(rest, 0)
        following.append(min(V - 1, int(torch.searchsorted(sums, u[b][T] * float(sums[-1]), right=True))))
        accepted.append(n)
    return [torch.tensor(accepted), torch.tensor(following), torch.from_numpy(prob)]
