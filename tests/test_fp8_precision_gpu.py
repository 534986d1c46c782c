"""``attention_fp8`` where a careless split of the queries, or one reference for all rows' weights, loses what the
output is made of: small elements beside a large channel, pages whose scales of V lie far apart.

The tolerance of an output element, from arithmetic, with u the output type's unit roundoff (2^-8 bf16, 2^-11 fp16), p the
weights of its row, and sv a page's scale of V:

* the output is rounded once: u |o|;
* weights are rounded to fp16: 2^-11 sum p |v|; one under fp16's smallest normal number by half of 2^-24 at most, where 2^7 stands
  for (at least) the row's largest product of a weight and a scale: 2^-32 max(p sv) 448 for each key. Exponentials by the hardware's
  2^x and sums in fp32 add less than 2^-16 sum p |v|;
* a logit is off by d = scale (e w sum |k| + D 2^-23 sum |q k|) + 2^-22 |logit|: with w the power of two that brings the row's largest
  query to at most 448, the parts of a query leave e w. A part has the nearest 8 bits of what those before it left. bf16, two
  parts: the first leaves at most 2^-10 of what is under 2^-6 (half a step there), and of the rest no more than 3 bits, which the second holds;
  of 2^-10 the second leaves at most 2^-14, by three bits of its own or as a multiple of 2^-9 / 16. So e = 2^-14; a third part (fp16)
  leaves an eighth of that or less: e = 2^-17. Weights then change by a factor within exp(+-2 d) of one another.
"""

import math

import pytest
import torch

from dropkv_b200 import attention_fp8
from test_fp8_attention_gpu import E4M3, U, Case

pytestmark = pytest.mark.gpu
LEFT = {torch.bfloat16: 2.0 ** -14, torch.float16: 2.0 ** -17}


def values(x, s, page, h, row):
    """Rows of a head in 64 bits; a page with a scale of 0 holds zeros."""
    y = x.view(torch.uint8)[page, h, row].view(E4M3).double() * s[page, h].double()[:, None]
    return y.masked_fill((s[page, h] == 0)[:, None], 0.0)


def check(c, window=None, sinks=0, scale=None):
    got = attention_fp8(c.Q, c.K, c.V, c.ks, c.vs, c.cache_lens, c.table, window=window, sinks=sinks, scale=scale)
    f, u, g = scale or c.D ** -0.5, U[c.Q.dtype], c.Hq // c.Hkv
    for b in range(c.B):
        see = c.seen(None, window, sinks, b).cuda()
        at = torch.arange(see.shape[1], device="cuda")
        page, row = c.table[b].long()[at // c.block].clamp(0, c.K.shape[0] - 1), at % c.block
        for h in range(c.Hkv):
            k, v = (values(x, s, page, h, row).masked_fill(~see.any(0)[:, None], 0.0) for x, s in ((c.K, c.ks), (c.V, c.vs)))
            sv = c.vs[page, h].double().masked_fill(~see.any(0), 0.0)
            q = c.Q[b, h * g:(h + 1) * g].double()
            w = torch.exp2(torch.ceil(torch.log2(q.abs().amax(-1, keepdim=True) / 448)))
            z = f * q @ k.T
            d = f * (LEFT[c.Q.dtype] * w * k.abs().sum(-1) + c.D * 2.0 ** -23 * q.abs() @ k.abs().T) + 2.0 ** -22 * z.abs()
            d = (d * see).amax(-1, keepdim=True)
            p = torch.softmax(z.masked_fill(~see, -math.inf), -1).masked_fill(~see, 0.0)
            want, size, peak = p @ v, p @ v.abs(), 448 * (p * sv).amax(-1, keepdim=True)
            tol = (u * want.abs() + (2.0 ** -11 + 2.0 ** -16 + torch.expm1(2 * d)) * size + see.sum(-1, keepdim=True) * 2.0 ** -32 * peak
                   + 2.0 ** -25)
            # (what is within its tolerance of the type's range, or past it, may be an infinity)
            err = (got[b, h * g:(h + 1) * g].double() - want).abs().masked_fill(want.abs() + tol > torch.finfo(got.dtype).max, 0.0)
            assert bool((err <= tol).all()), (b, h, float((err / tol).nan_to_num(1e9).max()), float(err.max()), float(want.abs().max()))
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T", [((8, 2, 128), 1), ((8, 2, 64), 4), ((8, 4, 128), 5), ((8, 2, 128), 5), ((8, 2, 64), 40),
                                     ((28, 4, 128), 33)])
@pytest.mark.parametrize("down", [10, 11, 12])
def test_small_elements_beside_a_large_channel(heads, T, down, dtype):
    """One channel of 448, the others under 2^-down, whose signs are those of the keys, so that what is lost of them adds
    up; keys are 0 in the large channel, so that the logits are made of the small ones alone. V goes with the logits, so that
    the output is some 0.8 of its largest value, and 0 where the logits are lost."""
    c = Case(*heads, [300, 70], T, 16, dtype, seed=50)
    Hq, _, D = heads
    g = torch.Generator(device="cuda").manual_seed(51)
    pm = lambda *s: torch.randint(0, 2, s, generator=g, device="cuda") * 2.0 - 1  # noqa: E731
    sign = pm(D)
    x = 2.0 ** -down * (0.55 + 0.43 * torch.rand(c.B, T, Hq, D, generator=g, device="cuda")) * sign
    x[..., 0] = 448 * pm(c.B, T, Hq)
    c.Q = (32 * x).to(dtype).transpose(1, 2)
    shape = (*c.K.shape[:3], 1)
    size = 8 * pm(*shape) * (0.5 + 0.5 * torch.rand(shape, generator=g, device="cuda"))
    for name, scales, of in (("K", c.ks, sign.clone()), ("V", c.vs, pm(D))):
        raw = getattr(c, name).view(torch.uint8)
        if name == "K":
            of[0] = 0
        raw.copy_(torch.where((raw & 0x7f) == 0x7f, raw, (size * of).to(E4M3).view(torch.uint8)))  # (rows that none sees keep NaN)
        scales.copy_(torch.where(scales.isnan(), scales, 2.0 ** -5))
    check(c, scale=2.0 ** (down - 9) * 128 / D)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T", [((8, 2, 128), 4), ((4, 2, 64), 6), ((8, 2, 128), 16), ((14, 2, 64), 40), ((8, 2, 128), 200)])
@pytest.mark.parametrize("far", [12, 24, 40])
def test_pages_that_a_token_does_not_see(heads, T, far, dtype):
    """The later tokens' pages hold values 2^far times the others': the earlier tokens, which do not see them, lose nothing.
    (What the later ones give is past fp16's range, and looked at in bf16 alone.)"""
    half = T // 2
    c = Case(*heads, [208 - half, (16 if half <= 16 else 1000) - half], T, 8, dtype, seed=52)
    for b, n in enumerate(c.lens):
        c.vs[c.table[b, (n + half) // 8:(n + T - 1) // 8 + 1].long()] *= 2.0 ** far
    check(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,T", [((8, 2, 128), 1), ((4, 2, 64), 6), ((8, 2, 128), 16), ((14, 2, 64), 40), ((8, 2, 128), 200)])
@pytest.mark.parametrize("far,first", [(12, False), (30, False), (30, True), (60, False), (60, True)])
def test_pages_that_weigh_nothing(heads, T, far, first, dtype):
    """Pages with large values and logits of -100: they add nothing, and take no bits of the others. Some pages' values are
    far smaller still, and some are zeros, whose scale is the least there is."""
    c = Case(*heads, [700, 90], T, 16, dtype, seed=53, q_scale=0.2)
    h = torch.Generator().manual_seed(54)
    c.Q[..., 0] = 4.0
    c.K.view(torch.uint8)[..., 0].masked_fill_((c.K.view(torch.uint8)[..., 0] & 0x7f) != 0x7f, 0)
    vs, V = c.vs.clone(), c.V.view(torch.uint8)
    for b, n in enumerate(c.lens):
        ids = c.table[b, :-(-(n + T) // 16)].long()
        kind = torch.randint(0, 4, (len(ids),), generator=h)
        kind[-1] = 0
        if first:   # the large ones in front
            kind = torch.cat([kind[:-1].sort(descending=True).values, kind[-1:]])
        large, small, zero = (ids[(kind == i).cuda()] for i in (3, 2, 1))
        c.vs[large] = vs[large] * 2.0 ** far
        c.ks[large] = 1.0
        c.K.view(torch.uint8)[large, ..., 0] = torch.tensor([-25.0]).to(E4M3).view(torch.uint8).item()   # times 4: -100 times `scale`
        c.K.view(torch.uint8)[large, ..., 1:] = 0
        c.vs[small] = vs[small] * 2.0 ** -20
        c.vs[zero] = 2.0 ** -126
        V[zero] = 0
    check(c, scale=1.0)
    check(c, scale=1.0, window=300, sinks=40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [8, 9, 16, 17])
def test_both_sides_of_the_kernels_border(T, D, dtype):
    """Query rows of a KV head up to which one kernel answers, and one more."""
    c = Case(8, 8, D, [700, 5, 129], T, 16, dtype, seed=55)
    check(c)
    check(c, window=50, sinks=3)
