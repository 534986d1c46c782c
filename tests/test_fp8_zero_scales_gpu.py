"""Pages whose scale is 0: they hold zeros, as a quantiser by the largest magnitude leaves a page of zeros. Their rows are
seen like others (a logit of 0, nothing of V), and become zeros of the new scale where rows are added to them."""

import pytest
import torch

from dropkv_b200 import load_rows_fp8, store_rows_fp8
from test_fp8_attention_gpu import E4M3, Case
from test_fp8_cache_gpu import Pool, chain_slots, rows
from test_fp8_precision_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T", [((8, 2, 128), 1), ((14, 2, 64), 2), ((8, 2, 128), 4), ((8, 4, 64), 30), ((28, 4, 128), 90)])
@pytest.mark.parametrize("of", ["K", "V", "KV"])
def test_attention_sees_pages_of_zeros(heads, T, of, dtype):
    """Every third page, its bits what they were; then all of them."""
    for step in (3, 1):
        c = Case(*heads, [500, 0, 70], T, 16, dtype, seed=60)
        for name, scales in (("K", c.ks), ("V", c.vs)):
            if name in of:
                for b, n in enumerate(c.lens):
                    scales[c.table[b, :-(-(n + T) // 16):step].long()] = 0.0
        got = check(c)
        check(c, window=100 + T, sinks=20)
        if step == 1 and "V" in of:
            assert got.abs().max() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 80])
def test_rows_added_to_a_page_of_zeros(D, dtype):
    pool = Pool(4, 2, 16, D, seed=61)
    for s, want, w8 in ((pool.Ks, pool.scales[0], pool.want[0]), (pool.Vs, pool.scales[1], pool.want[1])):
        s[2, 0] = 0.0
        want[2, 0] = 0.0
        w8[2, 0] = 0.0
    x = rows(1, 2, 5, D, dtype, 62)
    pool.store(x, -x, chain_slots([[2, 0]], 16, [7], [12], 5))
    pool.check()
    k, v = load_rows_fp8(*pool.tensors, chain_slots([[2, 0]], 16, [0], [7], 7), dtype=dtype)
    assert not k[0, 0].any() and not v[0, 0].any() and k[0, 1].any()


def test_zeros_in_a_page_of_zeros_stay():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    pages, scales = [z(2, 2, 16, 64).to(E4M3) for _ in "KV"], [z(2, 2) for _ in "KV"]
    x = z(1, 2, 3, 64).bfloat16()
    store_rows_fp8(x, x, torch.tensor([[5, 6, 7]], device="cuda"), *pages, *scales)
    assert all(not p.float().any() for p in pages) and all((s[0] == 2.0 ** -126).all() and not s[1].any() for s in scales)
