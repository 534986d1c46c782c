"""Pages whose scale is 0: they hold zeros, as a quantiser by the largest magnitude leaves a page of zeros. Their rows are
seen like others (a logit of 0, nothing of V)."""

import pytest
import torch

from test_fp8_attention_gpu import Case
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
