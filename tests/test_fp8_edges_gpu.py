"""Caches in 8 bits at the ends of what a call may ask for: nothing at all, the largest groups of heads, pools past
32 bits, prompts that begin inside a page, inputs of every stride."""

import pytest
import torch

from dropkv_b200 import attention_fp8, load_rows_fp8, store_rows_fp8, verify_draft
from test_fp8_attention_gpu import E4M3, Case
from test_fp8_cache_gpu import Pool, chain_slots, rows

pytestmark = pytest.mark.gpu


def _pool(pages=3, H=2, block=16, D=64):
    return (torch.zeros(pages, H, block, D, device="cuda").to(E4M3), torch.zeros(pages, H, block, D, device="cuda").to(E4M3),
            torch.ones(pages, H, device="cuda"), torch.ones(pages, H, device="cuda"))


@pytest.mark.parametrize("T", [1, 40])
def test_attention_over_nothing(T):
    ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(2, 4, T, 64, device="cuda").bfloat16()
    for pool, table in ((_pool(), ints(2, 0)), (_pool(pages=0), ints(2, 5))):     # no pages a sequence; no pages
        out = attention_fp8(q, *pool, ints(2), table)
        assert out.shape == q.shape and not out.any()
    assert attention_fp8(q[:0], *_pool(), ints(0), ints(0, 5)).shape == (0, 4, T, 64)
    assert attention_fp8(q[:, :, :0], *_pool(), ints(2), ints(2, 5)).shape == (2, 4, 0, 64)
    assert attention_fp8(q[:, :0], *_pool(), ints(2), ints(2, 5)).shape == (2, 0, T, 64)


def test_rows_of_nothing():
    slots = torch.full((2, 3), 5, dtype=torch.int64, device="cuda")
    x = torch.randn(2, 2, 3, 64, device="cuda").bfloat16()
    store_rows_fp8(x, x, slots, *_pool(pages=0))
    for k in load_rows_fp8(*_pool(pages=0), slots):
        assert k.shape == (2, 2, 3, 64) and not k.any()
    pool = _pool()
    store_rows_fp8(x[:, :, :0], x[:, :, :0], slots[:, :0], *pool)
    store_rows_fp8(x[:0], x[:0], slots[:0], *pool)
    assert not any(p.float().any() for p in pool[:2]) and all((s == 1).all() for s in pool[2:])
    assert load_rows_fp8(*pool, slots[:, :0])[0].shape == (2, 2, 0, 64)
    v = verify_draft(torch.zeros(0, 4, 10, device="cuda"), torch.zeros(0, 3, dtype=torch.int64, device="cuda"),
                     torch.zeros(0, 4, device="cuda"))
    assert v.accepted.shape == v.next_token.shape == (0,) and v.accept_prob.shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T", [((128, 1, 64), 1), ((128, 1, 128), 3), ((130, 2, 64), 2), ((127, 1, 128), 5), ((34, 2, 64), 9)])
def test_large_groups_of_heads(heads, T, dtype):
    Case(*heads, [200, 3], T, 16, dtype, seed=30).check()


@pytest.mark.parametrize("block", [512, 1024])
@pytest.mark.parametrize("T", [1, 20])
def test_large_pages(T, block):
    Case(8, 2, 128, [1500, 10], T, block, torch.bfloat16, seed=31).check()


@pytest.mark.parametrize("T", [1, 24])
def test_pools_past_32_bits(T):
    """Pages at the far end of a pool of more than 2^32 bytes give what they give in a small one."""
    c = Case(8, 2, 128, [300, 90], T, 16, torch.bfloat16, seed=32)
    want = c.check()
    pages, n = (1 << 32) // (2 * 16 * 128) + 5000, c.K.shape[0]
    for name in ("K", "V"):
        far = torch.empty(pages, 2, 16, 128, dtype=torch.uint8, device="cuda")
        far[-n:] = getattr(c, name).view(torch.uint8)
        setattr(c, name, far.view(E4M3))
    for name in ("ks", "vs"):
        far = torch.empty(pages, 2, device="cuda")
        far[-n:] = getattr(c, name)
        setattr(c, name, far)
    c.table = torch.where(c.table >= 0, c.table + (pages - n), -1)
    assert torch.equal(attention_fp8(c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,D,block", [(2, 128, 64), (3, 64, 16), (1, 128, 256), (1, 64, 1)])
@pytest.mark.parametrize("first", [0, 1, -1])
def test_prompts_that_begin_anywhere_in_a_page(first, H, D, block, dtype):
    """Rows from a page's start, one past it and one before the next, to within a row of a page's end."""
    first %= block
    for total in (block, 3 * block - 1, 3 * block, 3 * block + 1):
        pool = Pool(6, H, block, D, seed=40)
        table = [[4, 0, 5, 2, 1]]
        x = rows(1, H, total, D, dtype, 41)
        pool.store(x, -2 * x, chain_slots(table, block, [first], [first + total], total))
        pool.check()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_whole_page_with_what_is_no_number(bad):
    pool = Pool(3, 2, 64, 128, seed=42)
    x = rows(1, 2, 128, 128, torch.bfloat16, 43)
    y = x.clone()
    x[0, 1, 70, 5] = bad
    pool.store(x, y, chain_slots([[2, 0]], 64, [0], [128], 128))
    pool.check()


def test_rows_of_every_stride():
    """Heads that share their rows, rows that lie apart, rows off 16 bytes."""
    wide = rows(1, 1, 80, 130, torch.bfloat16, 44)
    for x in (wide[..., :128].expand(1, 2, 80, 128), wide[..., 1:129].expand(1, 2, 80, 128),
              rows(1, 2, 160, 128, torch.bfloat16, 45)[:, :, ::2]):
        pool = Pool(4, 2, 32, 128, seed=46)
        pool.store(x, x, chain_slots([[3, 1, 0]], 32, [0], [80], 80))
        pool.check()


def test_masks_of_every_stride():
    c = Case(8, 2, 128, [200, 70], 24, 16, torch.bfloat16, seed=47)
    mask = torch.rand(2, 24, 24, generator=torch.Generator().manual_seed(1)) < 0.4
    mask = (mask & torch.ones(24, 24, dtype=torch.bool).tril() | torch.eye(24, dtype=torch.bool)).cuda()
    want = c.check(mask=mask)
    wide = torch.zeros(2, 24, 27, dtype=torch.bool, device="cuda")
    for other in (mask.transpose(1, 2).contiguous().transpose(1, 2), wide[..., 1:25].copy_(mask)):
        assert torch.equal(c.check(mask=other), want)
    one = mask[:1].expand(2, 24, 24)
    assert torch.equal(c.check(mask=one), c.check(mask=mask[0]))
