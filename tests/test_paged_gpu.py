"""Pages, slots, rows and rotations: ``block_tables``, ``store_rows``, ``qk_norm_rope``.

Whole numbers and copied rows have to be equal; ``qk_norm_rope`` is compared with the
formula in 64 bits. Its tolerance: one rounding to the output type (unit roundoff u:
2^-8 bf16, 2^-11 fp16, 2^-24 fp32) of a value whose fp32 computation -- a sum of D
squares, rsqrt, three products and a sum -- is off by at most 2^-18 of the larger member
of the rotated pair; fp16 results under the smallest normal add 2^-25.
"""

import pytest
import torch

from dropkv_b200 import block_tables, qk_norm_rope, store_rows

pytestmark = pytest.mark.gpu

ROUNDOFF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _tables_want(lens, new, table, held, free, block, max_blocks, max_new):
    want_t, want_s, want_h, at = [], [], [], 0
    for b, n in enumerate(lens):
        n = max(n, 0)
        nn = min(max(new[b], 0), n)
        h = min(max(held[b], 0), max_blocks)
        need = max(0, min(-(-n // block), max_blocks) - h)
        row = (list(table[b][:h]) if h else []) + free[at:at + need]
        at += need
        want_h.append(len(row))
        want_t.append(row + [-1] * (max_blocks - len(row)))
        row = want_t[-1]
        s = []
        for i in range(max_new):
            t = n - nn + i
            ok = i < nn and t // block < max_blocks and row[t // block] >= 0
            s.append(row[t // block] * block + t % block if ok else -1)
        want_s.append(s)
    return want_t, want_h, want_s, at


@pytest.mark.parametrize("lens,block,max_blocks,max_new", [
    ([1], 16, 1, 1),
    ([0, 17, 16, 1, 0, 33], 16, 4, 40),      # empty requests, page ends, one token over
    ([5, 9, 13], 1, 20, 13),                 # pages of one row
    ([100, 7, 300], 7, 60, 300),             # a block size that is no power of two
    ([64] * 300, 64, 3, 64),                 # more requests than a CTA has threads
    ([5000, 1, 4097], 128, 50, 5000),        # more slots than a CTA writes
    ([40, -3, 8], 8, 4, 50),                 # a negative length counts as 0; the table is too short for one
])
def test_block_tables_fresh(lens, block, max_blocks, max_new):
    total = sum(-(-max(n, 0) // block) for n in lens)
    free = torch.randperm(total + 3, generator=torch.Generator().manual_seed(1)).tolist()
    got = block_tables(_i32(lens), block, _i32(free), max_blocks, max_new)
    t, h, s, used = _tables_want(lens, lens, None, [0] * len(lens), free, block, max_blocks, max_new)
    assert got.table.tolist() == t and got.held.tolist() == h and got.slots.tolist() == s and got.used.tolist() == [used]


@pytest.mark.parametrize("block", [1, 2, 3, 7, 48, 100, 1 << 20, (1 << 31) - 1])
def test_block_tables_quotients_up_to_the_largest_length(block):
    """Slots of the last tokens of caches whose length is next to a page's end, and to 2^31."""
    top = 2 ** 31 - 1
    lens = [min(top, max(1, k * block + d)) for k in (1, 2, 5) for d in (-1, 0, 1)] + [top]
    wide = min(-(-top // block), 4096)                       # longer caches run out of columns
    t = block_tables(_i32(lens), block, torch.arange(0, dtype=torch.int32, device="cuda"), wide, 6,
                     new_lens=_i32([6] * len(lens)),
                     table=torch.arange(wide, dtype=torch.int32, device="cuda").expand(len(lens), wide).contiguous(),
                     held=_i32([wide] * len(lens)))
    for b, n in enumerate(lens):
        new = min(6, n)
        want = [(tok if tok // block < wide else -1) for tok in range(n - new, n)] + [-1] * (6 - new)
        assert t.slots[b].tolist() == want, (n, block)


def test_block_tables_extends_held_pages_and_a_step_can_follow_a_step():
    block, max_blocks = 16, 5
    lens = [15, 16, 0, 60, 80]
    free = list(range(100, 140))
    a = block_tables(_i32(lens), block, _i32(free), max_blocks, 80)
    used = int(a.used)
    free = free[used:]
    new = [1, 2, 5, 0, 30]                    # the last outgrows its table row: no slots there
    lens = [n + m for n, m in zip(lens, new)]
    b = block_tables(_i32(lens), block, _i32(free), max_blocks, 7, new_lens=_i32(new), table=a.table, held=a.held)
    t, h, s, used = _tables_want(lens, new, a.table.tolist(), a.held.tolist(), free, block, max_blocks, 7)
    assert b.table.tolist() == t and b.held.tolist() == h and b.slots.tolist() == s and b.used.tolist() == [used]
    assert torch.equal(b.table[:, 0][b.held > 1], a.table[:, 0][b.held > 1])


def test_a_captured_step_moves_along_its_free_list_on_the_device():
    """The next call wants the list without the pages already taken. Where nobody reads ``used``
    back, the list is shifted by it on the device, and a graph of a step hands out new pages
    every time it runs."""
    B, T, block, wide, F = 3, 9, 4, 24, 60
    free = torch.randperm(F, generator=torch.Generator().manual_seed(5)).int().cuda()
    lens, held, taken = _i32([7, 0, 16]), _i32([0, 0, 0]), torch.zeros(1, dtype=torch.int64, device="cuda")
    table = torch.full((B, wide), -1, dtype=torch.int32, device="cuda")
    new, at = _i32([T] * B), torch.arange(F, device="cuda")

    def step():
        left = torch.where(at + taken < F, free[(at + taken).clamp(max=F - 1)], -1)
        t = block_tables(lens + T, block, left, wide, T, new_lens=new, table=table, held=held)
        return t, lens + T, taken + t.used

    def keep(r):
        for to, x in zip((table, held, lens, taken), (r[0].table, r[0].held, r[1], r[2])):
            to.copy_(x)

    start = [x.clone() for x in (lens, held, taken, table)]
    keep(step())                                  # (nothing is loaded for the first time while capturing)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
        keep(got)
    for x, y in zip((lens, held, taken, table), start):
        x.copy_(y)
    l, h, f, tab = [7, 0, 16], [0] * B, free.tolist(), None
    for _ in range(5):
        graph.replay()
        l = [n + T for n in l]
        tab, h, s, used = _tables_want(l, [T] * B, tab, h, f, block, wide, T)
        f = f[used:]
        assert got[0].table.tolist() == tab and got[0].held.tolist() == h and got[0].slots.tolist() == s
        assert int(taken) == F - len(f)


def test_block_tables_short_free_list():
    # 2 + 3 + 1 pages asked for, 4 there: the second request gets two of three, the third none
    got = block_tables(_i32([32, 48, 10]), 16, _i32([9, 8, 7, 6]), 4, 48)
    assert got.table.tolist() == [[9, 8, -1, -1], [7, 6, -1, -1], [-1] * 4]
    assert got.held.tolist() == [2, 2, 0] and got.used.tolist() == [6]
    s = got.slots.tolist()
    assert s[1][31] == 6 * 16 + 15 and s[1][32:] == [-1] * 16 and s[2] == [-1] * 48
    none = block_tables(_i32([4]), 4, _i32([]), 1, 4)
    assert none.table.tolist() == [[-1]] and none.held.tolist() == [0] and none.used.tolist() == [1]
    empty = block_tables(_i32([]), 4, _i32([1]), 1, 4)
    assert empty.table.shape == (0, 1) and empty.used.tolist() == [0]


def test_block_tables_slots_beyond_32_bits():
    page = 2 ** 31 - 2
    got = block_tables(_i32([130]), 128, _i32([page, page - 1]), 2, 130)
    assert got.slots[0, 127].item() == page * 128 + 127 and got.slots[0, 129].item() == (page - 1) * 128 + 1


def _put(pages, rows, slots):
    """Plain store: rows [B, H, N, D] to slots [B, N] of pages [P, H, block, D] (in place)."""
    P, _, block, _ = pages.shape
    for b, n in torch.nonzero((slots >= 0) & (slots < P * block)).tolist():
        s = int(slots[b, n])
        pages[s // block, :, s % block] = rows[b, :, n]


def _slots(B, N, total, seed, skip=0.2):
    g = torch.Generator().manual_seed(seed)
    s = torch.randperm(max(total, B * N), generator=g)[:B * N].reshape(B, N)  # some may lie beyond the pool
    s[torch.rand(B, N, generator=g) < skip] = -1
    return s


@pytest.mark.parametrize("B,H,N,D,pages,block,dtype,layout", [
    (1, 1, 1, 64, 1, 1, torch.bfloat16, "plain"),
    (2, 8, 133, 128, 20, 16, torch.bfloat16, "plain"),
    (3, 2, 50, 64, 200, 1, torch.float16, "nhd"),
    (2, 3, 37, 33, 30, 7, torch.float16, "plain"),       # odd rows: 2-byte copies
    (2, 3, 37, 33, 30, 7, torch.float32, "nhd"),         # odd rows of 4-byte elements
    (1, 4, 300, 96, 40, 8, torch.float32, "view"),
    (4, 2, 20, 128, 3, 16, torch.bfloat16, "view"),      # fewer rows than slots: those beyond are left out
])
def test_store_rows(B, H, N, D, pages, block, dtype, layout):
    g = torch.Generator(device="cuda").manual_seed(N)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    if layout == "view":   # a [B, N, H, D] projection with room around each row; K and V of different strides
        K, V = rnd(B, N, H, D + 8)[..., 4:4 + D].transpose(1, 2), rnd(B, H, N + 2, D)[:, :, 1:-1]
    else:
        K, V = rnd(B, H, N, D), rnd(B, H, N, D)
    Kp, Vp = ((rnd(pages, block, H, D).transpose(1, 2), rnd(pages, H, block, D)) if layout == "nhd"
              else (rnd(pages, H, block, D), rnd(pages, H, block, D)))
    slots = _slots(B, N, pages * block, seed=N)
    slots[0, 0] = pages * block  # just outside
    want = Kp.clone(), Vp.clone()
    _put(want[0], K, slots), _put(want[1], V, slots)
    store_rows(K, V, slots.cuda(), Kp, Vp)
    assert torch.equal(Kp, want[0]) and torch.equal(Vp, want[1])


def test_store_rows_nothing_to_store_and_offsets_beyond_32_bits():
    z = torch.zeros(2, 3, 0, 8, device="cuda")
    pool = torch.ones(2, 3, 4, 8, device="cuda")
    store_rows(z, z, torch.zeros(2, 0, dtype=torch.int64, device="cuda"), pool, pool.clone())
    assert bool((pool == 1).all())
    pages = 2 ** 31 // (16 * 128) + 5        # elements of the pool pass 2^31
    Kp = torch.empty(pages, 1, 16, 128, dtype=torch.bfloat16, device="cuda")
    Vp = torch.empty_like(Kp)
    K, V = torch.randn(2, 1, 1, 3, 128, device="cuda").bfloat16()
    slots = torch.tensor([[0, pages * 16 - 1, (pages - 1) * 16]], device="cuda")
    store_rows(K, V, slots, Kp, Vp)
    for i, s in enumerate(slots[0].tolist()):
        assert torch.equal(Kp[s // 16, 0, s % 16], K[0, 0, i]) and torch.equal(Vp[s // 16, 0, s % 16], V[0, 0, i])


def _rope_want(x, w, eps, cos, sin, pos, interleaved):
    """(rotated and normed rows, the larger member of each element's pair), in 64 bits."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    R = 2 * cos.shape[1]
    out, big = y.clone(), y.abs()
    P = cos.shape[0]
    ok = ((pos >= 0) & (pos < P))[:, None, :, None]
    at = pos.clamp(0, max(P - 1, 0))
    c, s = (torch.where(ok, t.double()[at][:, None], float("nan")) for t in (cos, sin))
    i = torch.arange(R // 2, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    a, b = y[..., lo], y[..., hi]
    out[..., lo], out[..., hi] = a * c - b * s, b * c + a * s
    m = torch.maximum(a.abs(), b.abs())
    big[..., lo], big[..., hi] = m, m
    return out, big


def _rope_close(got, want, big, dtype):
    tol = ROUNDOFF[dtype] * want.abs() + 2.0 ** -18 * big + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    bad = ~((got.double() - want).abs() <= tol) & ~(want.isnan() & got.isnan())
    assert not bool(bad.any()), f"{int(bad.sum())} elements off, worst {float((got.double() - want).abs().nan_to_num().max())}"


@pytest.mark.parametrize("B,Hq,Hkv,L,D,R", [
    (1, 32, 8, 1, 128, 128),      # one token
    (2, 14, 2, 37, 64, 64),
    (1, 28, 4, 130, 128, 64),     # half of each head turns
    (3, 3, 3, 5, 96, 96),         # MHA, odd head counts
    (2, 4, 1, 9, 80, 20),         # sizes off 16-byte vectors
    (1, 2, 1, 7, 33, 30),         # an odd head size
    (1, 4, 2, 6, 256, 256),
    (1, 4, 2, 6, 512, 128),
    (2, 4, 2, 3, 64, 0),          # nothing turns: norm alone
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("norm,interleaved,paged", [(False, False, False), (True, False, True), (True, True, False),
                                                    (False, True, True)])
def test_qk_norm_rope(B, Hq, Hkv, L, D, R, dtype, norm, interleaved, paged):
    g = torch.Generator(device="cuda").manual_seed(D + L + R)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    # projections viewed [B, H, L, D]; V of another layout
    Q, K = (3 * rnd(B, L, h, D).to(dtype).transpose(1, 2) for h in (Hq, Hkv))
    V = rnd(B, Hkv, L, D).to(dtype)
    P = 4000
    ang = torch.arange(P, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, R, 2, device="cuda") / max(R, 1))
    cos, sin = ang.cos().float(), ang.sin().float()
    pos = torch.randint(0, P, (B, L), generator=g, device="cuda")
    w = [(1 + 0.3 * rnd(D)).to(dtype) if norm else None for _ in range(2)]
    pages = {}
    if paged:
        block, n = 8, -(-B * L // 8) + 1
        pages = dict(V=V, slots=_slots(B, L, n * block, seed=L).cuda(),
                     K_pages=rnd(n, block, Hkv, D).to(dtype).transpose(1, 2), V_pages=rnd(n, Hkv, block, D).to(dtype))
        Kp, Vp = pages["K_pages"].clone(), pages["V_pages"].clone()
    q, k = qk_norm_rope(Q, K, cos, sin, pos, q_weight=w[0], k_weight=w[1], eps=1e-5, interleaved=interleaved, **pages)
    for got, x, wt in ((q, Q, w[0]), (k, K, w[1])):
        assert got.dtype == dtype and got.is_contiguous()
        _rope_close(got, *_rope_want(x, wt, 1e-5, cos, sin, pos, interleaved), dtype)
    if paged:
        _put(Kp, k, pages["slots"].cpu()), _put(Vp, V, pages["slots"].cpu())
        assert torch.equal(pages["K_pages"], Kp) and torch.equal(pages["V_pages"], Vp)


@pytest.mark.parametrize("B,Hq,Hkv,L,D,R", [
    (1, 32, 8, 4096, 128, 128),   # 40 heads, 48 with V's: ten and twelve groups of two rounds of two rows
    (3, 14, 2, 1037, 64, 32),     # seven groups a token: the second round has two rows, or four, of fourteen
    (1, 9, 3, 4099, 128, 64),     # 12 heads, or 15: the last group's last row is missing
    (2, 5, 1, 3001, 64, 64),      # 6 heads, or 7
    (1, 1, 1, 9001, 128, 128),    # fewer heads than a group could take
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm,interleaved,paged", [(False, False, False), (True, False, False), (True, False, True),
                                                    (True, True, False), (False, True, True)])
def test_qk_norm_rope_over_many_tokens(B, Hq, Hkv, L, D, R, dtype, norm, interleaved, paged):
    """Enough tokens that a group of lanes takes several of its token's rows, in several rounds."""
    test_qk_norm_rope(B, Hq, Hkv, L, D, R, dtype, norm, interleaved, False)
    if not paged:
        return
    g = torch.Generator(device="cuda").manual_seed(L)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    Q, K, V = (rnd(B, L, h, D).transpose(1, 2) for h in (Hq, Hkv, Hkv))
    ang = torch.rand(300, R // 2, generator=g, device="cuda") * 6
    pos = torch.randint(0, 300, (B, L), generator=g, device="cuda")
    w = [rnd(D) if norm else None for _ in range(2)]
    block, pages = 16, -(-B * L // 16) + 3
    slots = _slots(B, L, pages * block, seed=L).cuda()
    Kp, Vp = rnd(pages, Hkv, block, D), rnd(pages, Hkv, block, D)
    want = Kp.clone().transpose(1, 2).reshape(-1, Hkv, D), Vp.clone().transpose(1, 2).reshape(-1, Hkv, D)
    q, k = qk_norm_rope(Q, K, ang.cos(), ang.sin(), pos, q_weight=w[0], k_weight=w[1], interleaved=interleaved, V=V,
                        slots=slots, K_pages=Kp, V_pages=Vp)
    q2, k2 = qk_norm_rope(Q, K, ang.cos(), ang.sin(), pos, q_weight=w[0], k_weight=w[1], interleaved=interleaved)
    assert torch.equal(q, q2) and torch.equal(k, k2)       # (checked above against the formula)
    keep = (slots >= 0) & (slots < pages * block)
    for to, rows, got in ((want[0], k, Kp), (want[1], V, Vp)):
        to[slots[keep]] = rows.transpose(1, 2)[keep]
        assert torch.equal(got.transpose(1, 2).reshape(-1, Hkv, D), to)


def test_qk_norm_rope_shared_positions_views_and_unknown_positions():
    B, Hq, Hkv, L, D = 2, 8, 2, 11, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    # rows off 16-byte boundaries, spare columns around them
    Q = torch.randn(B, Hq, L, D + 3, generator=g, device="cuda").bfloat16()[..., 1:1 + D]
    K = torch.randn(B, Hkv, L, D + 3, generator=g, device="cuda").bfloat16()[..., 2:2 + D]
    ang = torch.rand(50, D // 2, generator=g, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, 50, (L,), generator=g, device="cuda")
    pos[3], pos[5] = -1, 50
    q, k = qk_norm_rope(Q, K, cos, sin, pos)
    for got, x in ((q, Q), (k, K)):
        want, big = _rope_want(x, None, 0, cos, sin, pos.expand(B, L), False)
        assert bool(got[:, :, [3, 5]].isnan().all())
        _rope_close(got, want, big, torch.bfloat16)
    e, _ = qk_norm_rope(Q[:, :, :0], K[:, :, :0], cos, sin, pos[:0])
    assert e.shape == (B, Hq, 0, D)


def test_qk_norm_rope_norms_zeros_and_one_side_only():
    x = torch.zeros(1, 2, 3, 64, device="cuda", dtype=torch.float16)
    one = torch.ones(64, device="cuda", dtype=torch.float16)
    ang = torch.zeros(4, 32, device="cuda")
    y = torch.full_like(x, 2.0)
    q, k = qk_norm_rope(x, y, ang.cos(), ang.sin(), torch.arange(3, device="cuda"), q_weight=one)
    assert bool((q == 0).all()) and torch.equal(k, y)     # zeros stay zeros; K has no norm


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,interleaved", [(128, False), (128, True), (80, False)])
def test_qk_norm_rope_what_does_not_turn_stays(D, interleaved, dtype):
    """Elements behind the rotation come through bit by bit, infinities, NaN and -0 among them,
    and reach no other element."""
    g = torch.Generator(device="cuda").manual_seed(D)
    R, L = 32, 9
    Q = torch.randn(1, 6, L, D, generator=g, device="cuda").to(dtype)
    Q[0, 0, :, R:] = float("inf")
    Q[0, 1, :, R + 1::2] = float("nan")
    Q[0, 2, :, R::3] = -0.0
    K = Q[:, :2].clone()
    ang = torch.rand(L, R // 2, generator=g, device="cuda") * 6
    q, k = qk_norm_rope(Q, K, ang.cos(), ang.sin(), torch.arange(L, device="cuda"), interleaved=interleaved)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(q[..., R:].isnan(), Q[..., R:].isnan()) and bool(q[..., :R].isfinite().all())
    keep = ~Q[..., R:].isnan()
    assert torch.equal(q[..., R:].view(bits)[keep], Q[..., R:].contiguous().view(bits)[keep])
    assert torch.equal(k.view(bits), q[:, :2].contiguous().view(bits))


def test_calls_on_another_stream():
    side = torch.cuda.Stream()
    K = torch.randn(1, 2, 64, 64, device="cuda").half()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        t = block_tables(_i32([64]), 16, _i32([3, 1, 0, 2]), 4, 64)
        Kp, Vp = (torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.float16) for _ in range(2))
        store_rows(K, K, t.slots, Kp, Vp)
    side.synchronize()
    assert torch.equal(Kp[t.table[0].long()].transpose(0, 1).reshape(2, 64, 64), K[0])


def test_dimensions_of_one_may_have_any_stride():
    g = torch.Generator(device="cuda").manual_seed(8)
    odd = lambda t: t.as_strided(t.shape, [7 if n == 1 else s for n, s in zip(t.shape, t.stride())])  # noqa: E731
    K, V = torch.randn(2, 1, 1, 5, 64, generator=g, device="cuda").half()
    slots = torch.tensor([[3, 1, -1, 0, 2]], device="cuda")
    a = [torch.zeros(1, 1, 16, 64, device="cuda").half() for _ in range(4)]
    store_rows(odd(K), odd(V), slots, odd(a[0]), odd(a[1]))
    store_rows(K, V, slots, a[2], a[3])
    assert torch.equal(a[0], a[2]) and torch.equal(a[1], a[3]) and bool((a[0] != 0).any())
    ang = torch.rand(9, 32, generator=g, device="cuda")
    pos = torch.arange(5, device="cuda")
    q, k = qk_norm_rope(odd(K), odd(V), ang.cos(), ang.sin(), pos)
    q2, k2 = qk_norm_rope(K, V, ang.cos(), ang.sin(), pos)
    assert torch.equal(q, q2) and torch.equal(k, k2)


def test_refusals():
    x = torch.zeros(1, 2, 3, 64, device="cuda").half()
    pool = torch.zeros(2, 2, 16, 64, device="cuda").half()
    s = torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    c = torch.zeros(10, 32, device="cuda")
    with pytest.raises(TypeError):
        block_tables(_i32([3]).long(), 16, _i32([0]), 1, 3)
    with pytest.raises(ValueError):
        block_tables(_i32([3]), 16, _i32([0]), 1, 3, table=_i32([[0]]))
    with pytest.raises(ValueError):
        block_tables(_i32([3]), 16, _i32([0]), 2, 3, table=_i32([[0]]), held=_i32([1]))
    with pytest.raises(ValueError):
        store_rows(x, x, s, pool[:, :1], pool[:, :1])
    with pytest.raises(TypeError):
        store_rows(x, x, s, pool.float(), pool.float())
    with pytest.raises(TypeError):
        store_rows(x, x, s.int(), pool, pool)
    with pytest.raises(ValueError):
        store_rows(x[..., ::2], x[..., ::2], s, pool[..., :32], pool[..., :32])
    with pytest.raises(ValueError):
        qk_norm_rope(x, x, c, c, s[0], V=x, slots=s)
    with pytest.raises(ValueError):
        qk_norm_rope(x, x, c, c, s[0, :2])
    with pytest.raises(TypeError):
        qk_norm_rope(x, x, c.half(), c.half(), s[0])
    with pytest.raises(ValueError):
        qk_norm_rope(x, x, c, c, s[0], q_weight=c[0])
