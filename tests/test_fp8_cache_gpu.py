"""Rows of caches in 8 bits: ``store_rows_fp8`` and ``load_rows_fp8`` against their definition.

Nothing here has a tolerance: a page's scale is a power of two, the 8 bits are the nearest ones
(ties to even) of a value over it, and what is read back is their product, rounded once to the
output type. All of that is computed exactly in 64 bits.
"""

import pytest
import torch

from dropkv_b200 import block_tables, load_rows_fp8, store_rows_fp8

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def nearest8(y):
    """The e4m3 value nearest to y (64 bits), ties to even; NaN for what is no number."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.where(y.isfinite(), torch.round(y / step) * step, torch.nan)


def scale_for(x):
    m = torch.where(x.isfinite(), x, 0.0).abs().max().item() if x.numel() else 0.0
    e = -126
    while m > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Pool:
    """A pool and its definition: values (8 bits, as numbers) and scales in 64 bits on the host."""

    def __init__(self, pages, H, block, D, nhd=False, seed=0, junk=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape = (pages, block, H, D) if nhd else (pages, H, block, D)
        make = lambda: torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)  # noqa: E731
        raw = [make(), make()]
        if not junk:  # any bits but NaN's
            raw = [torch.where((r & 0x7f) == 0x7f, 0x38, r).to(torch.uint8) for r in raw]
        self.K, self.V = (r.view(E4M3) if not nhd else r.view(E4M3).transpose(1, 2) for r in raw)
        self.Ks, self.Vs = (torch.exp2(torch.randint(-9, 3, (pages, H), generator=g, device="cuda").float()) for _ in "KV")
        self.block = block
        self.want = [x.float().double().cpu() for x in (self.K, self.V)]
        self.scales = [s.double().cpu() for s in (self.Ks, self.Vs)]
        self.known = torch.ones(pages, block, dtype=torch.bool)

    @property
    def tensors(self):
        return self.K, self.V, self.Ks, self.Vs

    def store(self, K, V, slots):
        store_rows_fp8(K, V, slots, *self.tensors)
        n_slots, H = self.K.shape[0] * self.block, self.K.shape[1]
        rows = {}
        for b, row in enumerate(slots.tolist()):
            for n, s in enumerate(row):
                if 0 <= s < n_slots:
                    rows.setdefault(s // self.block, []).append((s % self.block, b, n))
        for p, items in rows.items():
            offs = [o for o, _, _ in items]
            if 0 in offs:
                self.known[p] = False
            self.known[p, offs] = True
            for x, want, scales in zip((K, V), self.want, self.scales):
                x = x.double().cpu()
                for h in range(H):
                    new = torch.stack([x[b, h, n] for _, b, n in items])
                    s, old = scale_for(new), scales[p, h].item()
                    if 0 not in offs:
                        s = max(s, old)
                        if s > old:
                            want[p, h] = nearest8(want[p, h] * (old / s))
                    want[p, h, offs] = nearest8(new / s)
                    scales[p, h] = s

    def check(self):
        for t, want, s, ws in zip((self.K, self.V), self.want, (self.Ks, self.Vs), self.scales):
            assert torch.equal(s.double().cpu(), ws)
            known = self.known[:, None, :, None].expand(t.shape)
            got = t.float().double().cpu()
            assert torch.equal(got[known].nan_to_num(777.0), want[known].nan_to_num(777.0))


def rows(B, H, N, D, dtype, seed, layout="bhnd"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "bhnd":
        x = torch.randn(B, H, N, D, generator=g, device="cuda")
    else:  # a model's projections [B, N, H, D], seen as [B, H, N, D]
        x = torch.randn(B, N, H, D, generator=g, device="cuda").transpose(1, 2)
    x = x * torch.exp2(torch.randint(-3, 4, (B, 1, N, 1), generator=g, device="cuda").float())
    return x.to(dtype)


def chain_slots(table, block, first, ends, most):
    out = torch.full((len(ends), most), -1, dtype=torch.int64)
    for b, (lo, hi) in enumerate(zip(first, ends)):
        for i, t in enumerate(range(lo, hi)):
            out[b, i] = table[b][t // block] * block + t % block
    return out.cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,D,block,lens,nhd,layout", [
    (1, 8, 128, 64, [200], False, "bhnd"),          # whole pages and a part of one
    (3, 2, 64, 16, [33, 1, 16], True, "bnhd"),      # one row; a page's end; pages by token, then head
    (2, 1, 128, 8, [70, 9], False, "bnhd"),         # small pages: several begin in a window of 32 rows
    (1, 2, 128, 256, [300], False, "bhnd"),         # a page larger than what stays in registers
    (2, 3, 24, 7, [20, 15], False, "bhnd"),         # sizes that fit no vector
    (1, 1, 1, 1, [5], False, "bhnd"),               # pages of one row of one element
    (1, 1, 96, 1024, [1500], False, "bhnd"),        # the largest pages
    (1, 2, 512, 32, [40], False, "bhnd"),           # long rows
])
def test_a_cache_is_written_and_read_back(B, H, D, block, lens, nhd, layout, dtype):
    need = [-(-n // block) for n in lens]
    pool = Pool(sum(need) + 2, H, block, D, nhd, seed=1, junk=True)
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(2)).tolist()
    table = [[order.pop() for _ in range(n)] for n in need]
    N = max(lens)
    K, V = rows(B, H, N, D, dtype, 3, layout), rows(B, H, N, D, dtype, 4, layout)
    slots = chain_slots(table, block, [0] * B, lens, N)
    pool.known[:] = False  # nothing is said of pages that are never written
    pool.store(K, V, slots)
    pool.check()
    for out_dtype in (dtype, torch.float32):
        for x, want, s in zip(load_rows_fp8(*pool.tensors, slots, dtype=out_dtype), pool.want, pool.scales):
            value = (want * s[:, :, None, None]).to(out_dtype)
            for b in range(B):
                for n in range(N):
                    p, o = divmod(int(slots[b, n]), block)
                    there = value[p, :, o] if slots[b, n] >= 0 else torch.zeros(H, D, dtype=out_dtype)
                    assert torch.equal(x[b, :, n].cpu(), there)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,D,block", [(2, 64, 16), (8, 128, 64), (1, 128, 256), (2, 20, 24)])
def test_rows_are_appended_step_by_step(H, D, block, dtype):
    """Pages fill up over calls of one and several rows; a scale that grows takes the rows before along."""
    B, total = 3, 2 * block + 5
    pool = Pool(3 * B + 1, H, block, D, seed=5)
    pool.known[:] = False
    table = [[3 * b + 2, 3 * b, 3 * b + 1] for b in range(B)]
    at, step, i = [0, 3, block - 1], [1, 2, 1], 0
    K0, V0 = rows(B, H, 3, D, dtype, 8), rows(B, H, 3, D, dtype, 9)
    pool.store(K0, V0, chain_slots([table[0], table[1], table[2]], block, [0, 0, 0], [0, 3, 0], 3))
    lead = rows(1, H, block - 1, D, dtype, 10)
    pool.store(lead, lead, chain_slots([table[2]], block, [0], [block - 1], block - 1))
    while min(at) < total and i < 40:
        i += 1
        n = [min(s * (1 + i % 4), total - a) for a, s in zip(at, step)]
        most = max(max(n), 1)
        K, V = rows(B, H, most, D, dtype, 20 + i), rows(B, H, most, D, dtype, 70 + i)
        K *= 2.0 ** (i % 9 - 4)
        pool.store(K, V, chain_slots(table, block, at, [a + m for a, m in zip(at, n)], most))
        at = [a + m for a, m in zip(at, n)]
        pool.check()


def test_rows_without_a_slot_stand_between_a_pages_rows():
    """Accepted nodes of drafted trees: few of many rows, in one or two pages, gaps of up to 255 rows."""
    H, D, block, N = 2, 128, 16, 700
    pool = Pool(6, H, block, D, seed=6)
    slots = torch.full((3, N), -1, dtype=torch.int64)
    slots[0, [3, 9, 40, 41, 200, 455]] = torch.arange(6) + 2 * block + 5      # gaps of 158 and 254 rows
    slots[1, [0, 31, 32, 63, 64, 319]] = torch.tensor([10, 11, 12, 13, 14, 15])
    slots[1, [320, 690]] = torch.tensor([0, 1]) + 3 * block                   # a gap of 369: of a page of its own
    slots[1, 690] = 4 * block + 7
    slots[2, 699] = 5 * block + 15                                            # the last row alone
    K, V = rows(3, H, N, D, torch.bfloat16, 11), rows(3, H, N, D, torch.bfloat16, 12)
    pool.store(K, V, slots.cuda())
    pool.check()


def test_slots_outside_the_pool_are_left_out():
    pool = Pool(3, 2, 16, 64, seed=7)
    K, V = rows(1, 2, 6, 64, torch.float16, 13), rows(1, 2, 6, 64, torch.float16, 14)
    slots = torch.tensor([[47, 48, -1, 1 << 40, -(1 << 40), 46]], device="cuda")
    slots[0, 5] = -7
    pool.store(K, V, slots)
    pool.check()
    k, v = load_rows_fp8(*pool.tensors, slots, dtype=torch.float32)
    assert k[:, :, 1:].abs().max() == 0 and v[:, :, 1:].abs().max() == 0 and k[:, :, 0].abs().max() > 0
    empty = torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    assert load_rows_fp8(*pool.tensors, empty)[0].shape == (1, 2, 0, 64)
    store_rows_fp8(K[:, :, :0], V[:, :, :0], empty, *pool.tensors)
    pool.check()


@pytest.mark.parametrize("value", [0.0, 1e-45, 1e-38, 448.0, 448.0625, 449.0, 480.0, 65504.0, 3.3e38, 2.0 ** -126, 7.0 * 2 ** -130])
def test_scales_at_the_ends_of_the_range(value):
    pool = Pool(2, 1, 16, 64, seed=8)
    K = torch.full((1, 1, 16, 64), value, device="cuda")
    K[0, 0, 3, 5] = -value / 3
    K[0, 0, 4] = 0
    slots = torch.arange(16, 32, device="cuda")[None]
    pool.store(K, 2.0 ** -20 * K, slots)
    pool.check()
    # 3.3e38 is 248.3 * 2^120, whose nearest 8 bits say 256 * 2^120 = 2^128: infinity in fp32, as read back
    k, _ = load_rows_fp8(*pool.tensors, slots, dtype=torch.float32)
    assert torch.equal(k[0, 0].cpu(), (pool.want[0][1, 0] * pool.scales[0][1, 0]).float())
    assert k.isfinite().all() or value > 3e38


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block", [16, 512])
def test_values_that_are_no_numbers_stay_apart(dtype, block):
    """NaN and infinities become NaN; a page's scale is that of the finite values."""
    pool = Pool(2, 2, block, 128, seed=9)
    K, V = rows(1, 2, block, 128, dtype, 15), rows(1, 2, block, 128, dtype, 16)
    K[0, 0, 3, 7], K[0, 1, block - 1, 0], V[0, 1, 0, 127] = float("nan"), float("inf"), float("-inf")
    V[0, 0] = float("nan")                                  # nothing finite: the smallest scale
    slots = torch.arange(block, device="cuda")[None]
    pool.store(K, V, slots)
    pool.check()
    assert pool.Vs[0, 0].item() == 2.0 ** -126
    more = rows(1, 2, 1, 128, dtype, 17) * 64               # the page grows: NaN stays NaN
    pool.known[0, 5] = True
    pool.store(more, more, slots[:, 5:6])
    pool.check()


def test_a_page_that_is_handed_out_again_starts_anew():
    pool = Pool(1, 1, 16, 64, seed=10)
    big, small = torch.full((1, 1, 16, 64), 1e6, device="cuda"), torch.full((1, 1, 3, 64), 1e-3, device="cuda")
    pool.store(big, big, torch.arange(16, device="cuda")[None])
    pool.store(small, small, torch.arange(3, device="cuda")[None])
    pool.check()
    assert pool.Ks[0, 0].item() < 1e-4
    pool.Ks.fill_(float("nan"))                             # a scale that is none: the rows before mean nothing
    pool.store(small[:, :, :1], small[:, :, :1], torch.tensor([[0]], device="cuda"))
    pool.check()


def test_slots_past_32_bits():
    """A pool of over 2^32 slots: stores and loads find its last pages."""
    block, D = 1024, 1
    pages = (1 << 32) // block + 3
    K = torch.zeros(pages, 1, block, D, dtype=torch.uint8, device="cuda").view(E4M3)
    V = torch.zeros(pages, 1, block, D, dtype=torch.uint8, device="cuda").view(E4M3)
    Ks, Vs = torch.ones(pages, 1, device="cuda"), torch.ones(pages, 1, device="cuda")
    x = torch.arange(1, 5, device="cuda").float().view(1, 1, 4, 1)
    slots = torch.tensor([[0, (1 << 32) + block, (1 << 32) + block + 1, pages * block - 1]], device="cuda")
    store_rows_fp8(x, 3 * x, slots, K, V, Ks, Vs)
    k, v = load_rows_fp8(K, V, Ks, Vs, slots, dtype=torch.float32)
    assert torch.equal(k, x) and torch.equal(v, 3 * x)
    assert Ks[1:-2].min() == 1 and K.view(torch.uint8).count_nonzero().item() == 4


def test_block_tables_slots_and_another_stream():
    """The slots that block_tables hands out on the device, all on a stream of the caller's, captured and replayed."""
    B, H, D, block = 4, 2, 64, 16
    lens = torch.tensor([40, 1, 16, 25], dtype=torch.int32, device="cuda")
    pool = Pool(12, H, block, D, seed=11, junk=True)
    K, V = rows(B, H, 40, D, torch.bfloat16, 18), rows(B, H, 40, D, torch.bfloat16, 19)
    free = torch.randperm(12, device="cuda").int()
    bt = block_tables(lens, block, free, 4, 40)
    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=st):
        store_rows_fp8(K, V, bt.slots, *pool.tensors)
        out = load_rows_fp8(*pool.tensors, bt.slots)
    K.mul_(2), V.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    other = Pool(12, H, block, D, seed=11, junk=True)
    other.known[:] = False
    other.store(K, V, bt.slots)
    other.check()
    for got, want in zip(out, load_rows_fp8(*other.tensors, bt.slots)):
        assert torch.equal(got, want)
