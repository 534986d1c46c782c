"""``tree_attention`` against the formula in 64 bits.

Tolerance, for one output: the softmax weights are rounded to the input type before the
product with V (unit roundoff u: 2^-8 bf16, 2^-11 fp16) while their sum is not, which
moves the output by at most 2 u A with A = sum_j p_j |v_j|; scores are sums of D products
in fp32, off by less than 2^-13 here (|s| of at most 40, D of at most 128), hence another
2^-13 A; and the output is rounded once, u |o|. fp16 weights under its smallest normal
lose up to 2^-25 each, of a largest weight of at least 1: n 2^-25 max|v|.
"""

import pytest
import torch

from dropkv_b200 import block_tables, store_rows, tree_attention, tree_mask_from_parents

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _want(Q, K, V, lens, mask, scale):
    """(o, sum p |v|) in 64 bits; K, V [B, Hkv, rows, D], rows past a length never used."""
    B, Hq, T, D = Q.shape
    Hkv, rows = K.shape[1], K.shape[2]
    o = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=Q.device)
    a = torch.zeros_like(o)
    for b in range(B):
        n = min(max(int(lens[b]), 0), rows)
        m = min(n + T, rows)
        see = torch.ones(T, m, dtype=torch.bool, device=Q.device)
        see[:, n:] = (mask[b] if mask.dim() == 3 else mask)[:, :m - n]
        for i in range(T):
            j = see[i].nonzero()[:, 0]
            if not len(j):
                continue
            k = K[b][:, j].double().repeat_interleave(Hq // Hkv, 0)
            v = V[b][:, j].double().repeat_interleave(Hq // Hkv, 0)
            p = torch.softmax(torch.einsum("hd,hjd->hj", Q[b, :, i].double(), k) * scale, -1)
            o[b, :, i] = torch.einsum("hj,hjd->hd", p, v)
            a[b, :, i] = torch.einsum("hj,hjd->hd", p, v.abs())
    return o, a


def _close(got, Q, K, V, lens, mask, scale=None):
    scale = Q.shape[-1] ** -0.5 if scale is None else scale
    o, a = _want(Q, K, V, lens, mask, scale)
    u = ROUNDOFF[Q.dtype]
    tol = u * o.abs() + (2 * u + 2.0 ** -13) * a
    if Q.dtype == torch.float16:
        tol = tol + K.shape[2] * 2.0 ** -25 * 6 + 2.0 ** -25
    bad = ~((got.double() - o).abs() <= tol) & ~(o.isnan() & got.isnan()) & ~(got.double() == o)
    assert not bool(bad.any()), \
        f"{int(bad.sum())} of {o.numel()} off, worst {float(((got.double() - o).abs() / tol).nan_to_num().max()):.2f} x"


def _random_tree(T, g, B=None):
    par = torch.tensor([[-1 if i == 0 else int(torch.randint(max(-1, i - 6), i, (1,), generator=g)) for i in range(T)]
                        for _ in range(B or 1)])
    mask, _ = tree_mask_from_parents(par)
    return mask if B else mask[0]


def _inputs(B, Hq, Hkv, T, D, lens, dtype, seed, cap=None, kscale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cap = max(lens) + T if cap is None else cap
    Q = torch.randn(B, T, Hq, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
    K = (kscale * torch.randn(B, Hkv, cap, D, generator=g, device="cuda")).to(dtype)
    V = torch.randn(B, Hkv, cap, D, generator=g, device="cuda").to(dtype)
    return Q, K, V, torch.tensor(lens, dtype=torch.int32, device="cuda")


SHAPES = [
    # B, Hq, Hkv, T, D, lens
    (1, 8, 2, 1, 64, [0]),                    # one node, an empty cache
    (1, 32, 8, 1, 128, [1]),
    (1, 14, 2, 8, 64, [819]),
    (2, 32, 8, 5, 128, [127, 128]),           # tree tiles around a tile's end
    (2, 28, 4, 13, 128, [250, 3]),            # 91 rows to a KV head
    (1, 32, 8, 33, 128, [1000]),              # 132 rows: just past one row tile
    (1, 32, 8, 64, 128, [700]),               # 256 rows
    (1, 28, 4, 40, 128, [300]),               # 280 rows: past two row tiles
    (3, 8, 8, 16, 128, [0, 511, 40]),         # MHA, one empty cache
    (1, 16, 2, 100, 64, [2000]),              # 800 rows
    (1, 4, 1, 256, 64, [70]),                 # the most nodes, MQA
    (5, 4, 1, 3, 128, [4000, 1, 0, 129, 2500]),  # a ragged batch
    (1, 32, 1, 2, 64, [9000]),                # one KV head: its keys are split over every SM
]


@pytest.mark.parametrize("B,Hq,Hkv,T,D,lens", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_in_buffers(B, Hq, Hkv, T, D, lens, dtype):
    Q, K, V, n = _inputs(B, Hq, Hkv, T, D, lens, dtype, seed=T + D)
    mask = _random_tree(T, torch.Generator().manual_seed(T), B).cuda()
    got = tree_attention(Q, K, V, n, tree_mask=mask)
    _close(got, Q, K, V, lens, mask)
    assert torch.equal(got, tree_attention(Q, K, V, n, tree_mask=mask))   # the same bits every time


def _paged(K, V, lens, T, block, seed, nhd, fill=0.0, extra=2):
    """The rows [0, lens + T) of row buffers in shuffled pages: (K pages, V pages, table)."""
    B, H, cap, D = K.shape
    need = [n + T for n in lens]
    pages = sum(-(-n // block) for n in need) + extra
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int().cuda()
    t = block_tables(torch.tensor(need, dtype=torch.int32, device="cuda"), block, free,
                     max(-(-n // block) for n in need) + 1, cap)
    shape = (pages, block, H, D) if nhd else (pages, H, block, D)
    Kp, Vp = (torch.full(shape, fill, dtype=K.dtype, device="cuda") for _ in range(2))
    if nhd:
        Kp, Vp = Kp.transpose(1, 2), Vp.transpose(1, 2)
    store_rows(K, V, t.slots, Kp, Vp)
    return Kp, Vp, t.table


@pytest.mark.parametrize("B,Hq,Hkv,T,D,lens", [s for s in SHAPES if s[3] != 256])
@pytest.mark.parametrize("block,nhd", [(8, False), (16, True), (64, False), (256, True)])
def test_rows_in_pages(B, Hq, Hkv, T, D, lens, block, nhd):
    dtype = torch.bfloat16 if block != 64 else torch.float16
    Q, K, V, n = _inputs(B, Hq, Hkv, T, D, lens, dtype, seed=T + block)
    mask = _random_tree(T, torch.Generator().manual_seed(block)).cuda()
    # rows that no request holds are NaN: they must not matter
    Kp, Vp, table = _paged(K, V, lens, T, block, seed=T, nhd=nhd, fill=float("nan"))
    got = tree_attention(Q, Kp, Vp, n, tree_mask=mask, block_table=table)
    _close(got, Q, K, V, lens, mask)
    # where the rows lie does not change a bit
    assert torch.equal(got, tree_attention(Q, K, V, n, tree_mask=mask))


@pytest.mark.parametrize("B,Hq,Hkv,T,D,most,paged", [
    (90, 8, 4, 3, 128, 300, True),      # few rows, several short pieces of caches to a CTA
    (61, 8, 4, 3, 64, 40, False),       # caches of one tile: every piece is whole
    (40, 32, 4, 20, 128, 700, True),    # 160 rows: two groups of rows, several pieces to a CTA
    (30, 28, 4, 50, 64, 500, True),     # 350 rows: more than a segment's
])
def test_many_short_caches(B, Hq, Hkv, T, D, most, paged):
    rs = torch.Generator().manual_seed(B)
    lens = torch.randint(0, most, (B,), generator=rs).tolist()
    Q, K, V, n = _inputs(B, Hq, Hkv, T, D, lens, torch.bfloat16, seed=B)
    mask = _random_tree(T, rs, B).cuda()
    if paged:
        Kp, Vp, table = _paged(K, V, lens, T, 16, seed=B, nhd=False)
        got = tree_attention(Q, Kp, Vp, n, tree_mask=mask, block_table=table)
    else:
        got = tree_attention(Q, K, V, n, tree_mask=mask)
    some = [0, 1, B // 3, B // 2, B - 1]
    _close(got[some], Q[some], K[some], V[some], [lens[b] for b in some], mask[some])
    alone = torch.stack([tree_attention(Q[b:b + 1], K[b:b + 1], V[b:b + 1], n[b:b + 1], tree_mask=mask[b])[0] for b in range(B)])
    # each is as near to the definition as the tolerance says: twice that between the two
    u = ROUNDOFF[torch.bfloat16]
    assert float((got.double() - alone.double()).abs().max()) <= 2 * (u * 6 + (2 * u + 2.0 ** -13) * 6)


@pytest.mark.parametrize("B,Hq,Hkv,T,D,most,q_tma", [
    (90, 8, 4, 3, 128, 300, True),      # several short pieces to a CTA
    (60, 16, 2, 16, 128, 1500, True),   # 128 rows, taken in turn, in pieces of many lengths
    (60, 16, 2, 16, 128, 1500, False),
    (30, 28, 4, 50, 64, 500, False),    # 350 rows: pieces of two groups of rows and of one, in one CTA
    (24, 24, 4, 60, 128, 900, False),   # 360 rows of 128
])
def test_every_cache_of_a_ragged_batch(B, Hq, Hkv, T, D, most, q_tma):
    rs = torch.Generator().manual_seed(B + T)
    lens = torch.randint(0, most, (B,), generator=rs).tolist()
    Q, K, V, n = _inputs(B, Hq, Hkv, T, D, lens, torch.bfloat16, seed=B + T)
    if not q_tma:
        Q = torch.stack([Q, Q], -1)[..., 0]
    mask = _random_tree(T, rs, B).cuda()
    _close(tree_attention(Q, K, V, n, tree_mask=mask), Q, K, V, lens, mask)


@pytest.mark.parametrize("long,short", [(450, 90), (230, 60), (1000, 20)])
def test_short_pieces_after_long_ones(long, short):
    # CTAs that end a segment of several tiles, which two groups take in turn, and go on with
    # segments of one: a group has no work in some pieces and is at others for long
    B, T = 90, 4
    lens = [long - (b % 7) if b % 3 == 0 else short for b in range(B)]
    Q, K, V, n = _inputs(B, 8, 4, T, 128, lens, torch.bfloat16, seed=long)
    want = tree_attention(Q, K, V, n)
    some = [0, 1, 2, 45, B - 1]
    chain = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    _close(want[some], Q[some], K[some], V[some], [lens[b] for b in some], chain)
    for _ in range(40):
        assert torch.equal(tree_attention(Q, K, V, n), want)


@pytest.mark.parametrize("lens", [[350], [330, 350, 450, 470, 620], [360, 900]])
@pytest.mark.parametrize("strided_q", [False, True])
def test_nodes_in_the_third_tile_and_past_it(lens, strided_q):
    # segments of four tiles and more to a CTA, taken in turn, with nodes from the third tile on: the
    # softmax of that tile looks into V while the loads before it in the slot are the other group's
    B, Hkv, T, D = 37, 4, 64, 128
    lens = [lens[b % len(lens)] for b in range(B)]
    Q, K, V, n = _inputs(B, 8, Hkv, T, D, lens, torch.bfloat16, seed=21)
    if strided_q:
        Q = torch.stack([Q, Q], -1)[..., 0]
    par = torch.tensor([-1] + [0] * 20 + [3] * 10 + [25] * 33)
    mask = tree_mask_from_parents(par)[0].cuda()
    clean = tree_attention(Q, K, V, n, tree_mask=mask)
    some = [0, 1, 2, B - 1]
    _close(clean[some], Q[some], K[some], V[some], [lens[b] for b in some], mask)
    nodes = (3, 25, 40)
    hit = torch.zeros(B, 8, T, D, dtype=torch.bool, device="cuda")
    for b, m in enumerate(lens):
        for i, node in enumerate(nodes):
            V[b, :, m + node, 7 + i] = float("nan") if b % 2 else float("inf")
            hit[b, :, mask[:, node], 7 + i] = True
    for _ in range(20):
        got = tree_attention(Q, K, V, n, tree_mask=mask)
        assert torch.equal(got[~hit], clean[~hit])
        assert not bool(got[hit].isfinite().any())


def test_a_long_cache_in_small_pages_with_few_rows():
    lens, T = [30000, 7], 4
    Q, K, V, n = _inputs(2, 28, 4, T, 128, lens, torch.float16, seed=12)
    mask = _random_tree(T, torch.Generator().manual_seed(12)).cuda()
    Kp, Vp, table = _paged(K, V, lens, T, 8, seed=3, nhd=False)
    got = tree_attention(Q, Kp, Vp, n, tree_mask=mask, block_table=table)
    _close(got, Q, K, V, lens, mask)


def test_chain_is_causal_and_scale():
    Q, K, V, n = _inputs(2, 8, 2, 9, 128, [333, 60], torch.bfloat16, seed=1)
    got = tree_attention(Q, K, V, n, scale=0.2)
    _close(got, Q, K, V, [333, 60], torch.ones(9, 9, dtype=torch.bool, device="cuda").tril(), scale=0.2)


def test_row_buffers_with_spare_capacity_and_garbage_past_the_rows():
    B, Hq, Hkv, T, D, lens = 2, 32, 8, 6, 128, [500, 130]
    Q, K, V, n = _inputs(B, Hq, Hkv, T, D, lens, torch.float16, seed=2, cap=900)
    mask = _random_tree(T, torch.Generator().manual_seed(2)).cuda()
    for b, m in enumerate(lens):
        K[b, :, m + T:], V[b, :, m + T:] = float("inf"), float("nan")
    got = tree_attention(Q, K, V, n, tree_mask=mask)
    _close(got, Q, K, V, lens, mask)
    wide = torch.full((B, 900, Hkv, 2 * D), float("nan"), dtype=K.dtype, device="cuda")
    wide[..., :D] = K.transpose(1, 2)                     # rows of another stride
    assert torch.equal(got, tree_attention(Q, wide[..., :D].transpose(1, 2), V, n, tree_mask=mask))
    strided = Q.new_zeros(B, Hq, T, 2 * D)
    strided[..., ::2] = Q                                 # Q of any strides
    assert torch.equal(got, tree_attention(strided[..., ::2], K, V, n, tree_mask=mask))


def test_dimensions_of_one_may_have_any_stride():
    Q, K, V, n = _inputs(1, 4, 1, 1, 64, [60], torch.bfloat16, seed=13)
    odd = lambda t: t.as_strided(t.shape, [5 if m == 1 else s for m, s in zip(t.shape, t.stride())])  # noqa: E731
    assert torch.equal(tree_attention(Q, K, V, n), tree_attention(odd(Q), odd(K), odd(V), n))


def test_mask_of_any_strides():
    Q, K, V, n = _inputs(2, 8, 4, 10, 64, [50, 200], torch.bfloat16, seed=3)
    mask = _random_tree(10, torch.Generator().manual_seed(3), 2).cuda()
    got = tree_attention(Q, K, V, n, tree_mask=mask)
    flipped = mask.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(got, tree_attention(Q, K, V, n, tree_mask=flipped))
    same = mask[:1].expand(2, 10, 10)
    assert torch.equal(tree_attention(Q, K, V, n, tree_mask=same), tree_attention(Q, K, V, n, tree_mask=mask[0]))


def test_rows_that_see_nothing_are_zero():
    Q, K, V, n = _inputs(2, 8, 2, 4, 128, [0, 5], torch.bfloat16, seed=4)
    mask = torch.eye(4, dtype=torch.bool, device="cuda")
    mask[2] = False
    K[0, :, 2], V[0, :, 2] = float("nan"), float("inf")   # node 2 of sequence 0: seen by none
    K[1, :, 7], V[1, :, 7] = float("nan"), float("nan")   # and of sequence 1
    got = tree_attention(Q, K, V, n, tree_mask=mask)
    assert bool((got[0, :, 2] == 0).all())
    _close(got, Q, K, V, [0, 5], mask)                    # node 2 of sequence 1 sees the cache alone


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_infinities_and_nan_stay_with_the_nodes_that_see_them(bad):
    lens, T = [200], 12
    Q, K, V, n = _inputs(1, 8, 2, T, 64, lens, torch.bfloat16, seed=5)
    par = torch.tensor([-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 6])
    mask = tree_mask_from_parents(par)[0].cuda()
    clean = tree_attention(Q, K, V, n, tree_mask=mask)
    V[0, 1, 200 + 2, 7] = bad                             # node 2, one column of one KV head
    got = tree_attention(Q, K, V, n, tree_mask=mask)
    sees = mask[:, 2]
    hit = torch.zeros(1, 8, T, 64, dtype=torch.bool, device="cuda")
    hit[0, 4:, sees, 7] = True
    assert torch.equal(got[~hit], clean[~hit])
    assert bool((got[hit].isnan() if bad != bad else got[hit] == bad).all())
    V[0, 1, 200 + 2, 7] = 0
    clean = tree_attention(Q, K, V, n, tree_mask=mask)
    K[0, 1, 200 + 2, 3] = float("nan")                    # a key that is not a number: its viewers' rows alone
    got = tree_attention(Q, K, V, n, tree_mask=mask)
    hit[0, 4:, sees] = True
    assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores_and_rising_maxima(dtype):
    # keys that grow along the cache: the running maximum rises in every tile, by more than any lazy margin
    lens, T = [1500], 7
    Q, K, V, n = _inputs(1, 8, 2, T, 128, lens, dtype, seed=6)
    K *= torch.linspace(0, 3.5, K.shape[2], device="cuda")[:, None].to(dtype)
    mask = _random_tree(T, torch.Generator().manual_seed(6)).cuda()
    _close(tree_attention(Q, K, V, n, tree_mask=mask), Q, K, V, lens, mask)
    K = K.flip(2).contiguous()
    _close(tree_attention(Q, K, V, n, tree_mask=mask), Q, K, V, lens, mask)


def test_lengths_past_the_capacity_and_missing_pages():
    T, block = 4, 16
    Q, K, V, n = _inputs(3, 4, 2, T, 64, [100, 126, 60], torch.float16, seed=7, cap=128)
    chain = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    _close(tree_attention(Q, K, V, n), Q, K, V, [100, 126, 60], chain)   # the second's last two nodes do not fit
    n2 = torch.tensor([-5, 500, 128], dtype=torch.int32, device="cuda")
    _close(tree_attention(Q, K, V, n2), Q, K, V, [-5, 500, 128], chain)
    # the first request's second page is missing: its keys are not seen
    Kp, Vp, table = _paged(K, V, [100, 100, 60], T, block, seed=1, nhd=False)
    table[0, 1], table[2, 0] = -1, Kp.shape[0]
    n3 = torch.tensor([100, 100, 60], dtype=torch.int32, device="cuda")
    got = tree_attention(Q, Kp, Vp, n3, block_table=table)
    cut = lambda x, lo, hi: torch.cat([x[:, :, :lo], x[:, :, hi:]], 2)  # noqa: E731
    _close(got[:1], Q[:1], cut(K[:1], 16, 32), cut(V[:1], 16, 32), [84], chain)
    _close(got[1:2], Q[1:2], K[1:2], V[1:2], [100], chain)
    _close(got[2:], Q[2:], cut(K[2:], 0, 16), cut(V[2:], 0, 16), [44], chain)
    none = tree_attention(Q, Kp, Vp, n3, block_table=torch.full_like(table, -1))
    assert bool((none == 0).all())


def test_pools_beyond_32_bits():
    T, block, D, Hkv = 3, 64, 128, 2
    pages = 2 ** 31 // (Hkv * block * D) + 9            # elements of the pool pass 2^31
    Q, K, V, n = _inputs(1, 4, Hkv, T, D, [200], torch.bfloat16, seed=8)
    Kp = torch.empty(pages, Hkv, block, D, dtype=torch.bfloat16, device="cuda")
    Vp = torch.empty_like(Kp)
    free = torch.tensor([pages - 1, 3, pages - 7, pages // 2], dtype=torch.int32, device="cuda")
    t = block_tables(torch.tensor([200 + T], dtype=torch.int32, device="cuda"), block, free, 4, 200 + T)
    store_rows(K, V, t.slots, Kp, Vp)
    mask = _random_tree(T, torch.Generator().manual_seed(8)).cuda()
    _close(tree_attention(Q, Kp, Vp, n, tree_mask=mask, block_table=t.table), Q, K, V, [200], mask)


def test_matches_decode_attention_on_a_chain():
    from dropkv_b200 import decode_attention
    Q, K, V, n = _inputs(1, 32, 8, 4, 128, [2996], torch.bfloat16, seed=9)
    a, b = tree_attention(Q, K, V, n).double(), decode_attention(Q, K, V).double()
    o, w = _want(Q, K, V, [2996], torch.ones(4, 4, dtype=torch.bool, device="cuda").tril(), 128 ** -0.5)
    u = 2.0 ** -8
    assert bool(((a - b).abs() <= 2 * (u * o.abs() + (2 * u + 2.0 ** -13) * w)).all())   # each is that near to o


def test_on_another_stream_and_in_a_graph():
    Q, K, V, n = _inputs(2, 32, 8, 8, 128, [700, 90], torch.bfloat16, seed=10)
    want = tree_attention(Q, K, V, n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = tree_attention(Q, K, V, n)
        b = tree_attention(Q, K, V, n)
    side.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = tree_attention(Q, K, V, n)
    graph.replay()
    assert torch.equal(c, want)
    n.copy_(torch.tensor([33, 694], dtype=torch.int32))     # lengths are read when the graph runs
    graph.replay()
    assert torch.equal(c, tree_attention(Q, K, V, n))


def test_outputs_are_there_for_the_next_kernel():
    # caches of one tile in long buffers: there is nothing to join, and the kernel that would join
    # must not end, and let the next one on the stream begin, before the outputs are written
    lens = [100, 3, 77, 90, 1, 60, 99, 50]
    Q, K, V, n = _inputs(8, 32, 8, 20, 128, lens, torch.bfloat16, seed=14, cap=4096)
    want = tree_attention(Q, K, V, n)
    torch.cuda.synchronize()
    copies = []
    for _ in range(60):
        out = tree_attention(Q, K, V, n)
        copies.append(out.clone())
        out.zero_()
    torch.cuda.synchronize()
    assert all(torch.equal(c, want) for c in copies)


def test_empty_batch():
    z = torch.zeros(0, 8, 3, 64, device="cuda").half()
    k = torch.zeros(0, 2, 16, 64, device="cuda").half()
    assert tree_attention(z, k, k, torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 8, 3, 64)


def test_refusals():
    Q, K, V, n = _inputs(1, 8, 2, 4, 64, [10], torch.bfloat16, seed=11)
    with pytest.raises(TypeError):
        tree_attention(Q.float(), K.float(), V.float(), n)
    with pytest.raises(TypeError):
        tree_attention(Q, K, V, n.long())
    with pytest.raises(TypeError):
        tree_attention(Q, K, V, n, tree_mask=torch.ones(4, 4, device="cuda"))
    with pytest.raises(ValueError):
        tree_attention(Q, K, V, n, tree_mask=torch.ones(3, 3, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError):
        tree_attention(Q[:, :7], K, V, n)
    with pytest.raises(ValueError):
        tree_attention(Q, K, V, n, block_table=n)
    with pytest.raises(ValueError):
        tree_attention(Q, K.repeat_interleave(2, -1)[..., ::2], V, n)
