"""``token_logprobs`` against the formulas in 64 bits.

Tolerance: with x in units of the temperature, an exponent and a logarithm in fp32 are off
by at most 2^-21 (1 + |x - max x|) and a sum of V terms, in runs of at most V / 256 and a
tree over them, by (V / 256 + 32) 2^-24 of itself; the same for the entropy, whose terms
weigh exponents of up to the entropy's own size. Ids have to be equal.
"""

import math

import pytest
import torch

from dropkv_b200 import token_logprobs

pytestmark = pytest.mark.gpu


def _check(logits, tokens, top_k, temperature=1.0):
    got = token_logprobs(logits, tokens, top_k=top_k, temperature=temperature)
    V = logits.shape[-1]
    x = logits.double() / temperature
    z = torch.log_softmax(x, -1)
    at = tokens if tokens.dim() == logits.dim() else tokens.unsqueeze(-1)
    lp = torch.gather(z, -1, at.clamp(0, V - 1)).masked_fill((at < 0) | (at >= V), -math.inf).reshape(tokens.shape)
    h = torch.special.entr(z.exp()).sum(-1)
    run = (V / 256 + 32) * 2.0 ** -24
    far = (x.amax(-1) - x.masked_fill(x == -math.inf, math.inf).amin(-1)).nan_to_num(0.0, 0.0, 0.0)
    ok = lambda g, w, tol: bool((((g.double() - w).abs() <= tol) | (g.double() == w)  # noqa: E731
                                 | (g.isnan() & w.isnan())).all())
    near = lambda w: run + 2.0 ** -21 * (1 + w.abs().nan_to_num(0.0, 0.0, 0.0) + math.log(V))  # noqa: E731
    assert ok(got.logprob, lp, near(lp))
    assert ok(got.entropy, h, 4 * (run + 2.0 ** -21) * (1 + h.nan_to_num(0.0) + math.log(V)) + 0 * far)
    assert got.logprob.shape == tokens.shape and got.entropy.shape == logits.shape[:-1]
    if not top_k:
        assert got.top_logprobs is None and got.top_tokens is None
        return got
    # larger first, NaN above all, ties to the lower index
    key = torch.where(logits.isnan(), math.inf, logits.double())
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    nan_first = torch.argsort(torch.gather(logits.isnan().int(), -1, order), dim=-1, descending=True, stable=True)
    ids = torch.gather(order, -1, nan_first)[..., :top_k]
    assert torch.equal(got.top_tokens, ids)
    w = torch.gather(z, -1, ids)
    assert ok(got.top_logprobs, w, near(w))
    return got


@pytest.mark.parametrize("N,V", [(1, 1), (1, 7), (3, 255), (2, 1024), (5, 4097), (16, 50257), (1, 151936), (300, 8193),
                                 (2, 32000), (700, 1000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rows(N, V, dtype):
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = (4 * torch.randn(N, V, generator=g, device="cuda")).to(dtype)
    _check(logits, torch.randint(0, V, (N,), generator=g, device="cuda"), min(V, 20))
    _check(logits, torch.randint(0, V, (N, 3), generator=g, device="cuda"), 0, temperature=0.6)


@pytest.mark.parametrize("top_k", [1, 2, 31, 32, 33, 64])
@pytest.mark.parametrize("order", ["random", "rising", "falling", "equal", "two values", "first big"])
def test_top_alternatives_in_any_order(top_k, order):
    V = 20011
    g = torch.Generator(device="cuda").manual_seed(top_k)
    x = torch.linspace(-30, 30, V, device="cuda")
    x = {"random": x[torch.randperm(V, generator=g, device="cuda")], "rising": x, "falling": x.flip(0),
         "equal": torch.zeros_like(x), "two values": (torch.rand(V, generator=g, device="cuda") < 0.01).float(),
         "first big": torch.where(torch.arange(V, device="cuda") < 70, 5.0, x)}[order]
    for dtype in (torch.float32, torch.bfloat16):
        _check(x.to(dtype).expand(2, V).contiguous(), torch.zeros(2, dtype=torch.int64, device="cuda"), top_k)


@pytest.mark.parametrize("top_k", [1, 20, 64])
@pytest.mark.parametrize("order", ["rising", "rising in steps", "random"])
@pytest.mark.parametrize("dtype,first", [(torch.bfloat16, 0), (torch.bfloat16, 3), (torch.float16, 1), (torch.float32, 0),
                                         (torch.float32, 1)])
def test_more_candidates_than_the_list_holds(top_k, order, dtype, first):
    """Logits that rise along rows of many chunks overflow the list of candidates, whose chunks are then
    gone through again: rows that clusters share, and more rows than CTAs, 74 chunks each in
    fp32. In the second kind all rows are one row of memory."""
    V, N = 151936, 1200
    g = torch.Generator(device="cuda").manual_seed(top_k)
    x = torch.linspace(-30, 30, V, device="cuda")
    x = {"rising": x, "rising in steps": (x * 8).floor() / 8, "random": x[torch.randperm(V, generator=g, device="cuda")]}[order]
    room = torch.zeros(V + 8, dtype=dtype, device="cuda")
    row = room[first:first + V]
    row.copy_(x)
    token = torch.tensor([V - 77], device="cuda")
    one = _check(row[None], token, top_k)
    many = token_logprobs(row.expand(N, V), token.expand(N), top_k=top_k)
    assert bool((many.top_tokens == one.top_tokens).all())
    # two results that are each as near to the definition as _check allows
    run = 2 * ((V / 256 + 32) * 2.0 ** -24 + 2.0 ** -21 * (1 + 60 + math.log(V)))
    assert float((many.logprob - one.logprob).abs().max()) <= run
    assert float((many.top_logprobs - one.top_logprobs).abs().max()) <= run
    assert float((many.entropy - one.entropy).abs().max()) <= 4 * run


def test_masked_vocabularies_and_tokens_outside():
    V = 3001
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(5, V, generator=g, device="cuda")
    x[0, 5:] = -math.inf                         # five words left: fewer than the alternatives asked for
    x[1, :] = torch.finfo(torch.float32).min     # the lowest value everywhere
    x[2, ::2] = torch.finfo(torch.float32).min
    x[3, :] = -math.inf                          # nothing left
    tokens = torch.tensor([[3, 2900, -1], [0, V, V - 1], [1, 2, -100], [0, 1, 2], [9, 2 ** 40, 10]], device="cuda")
    got = _check(x, tokens, 8)
    assert bool(got.entropy[3].isnan()) and got.logprob[0, 1] == -math.inf
    assert abs(float(got.entropy[1]) - math.log(V)) < 1e-4


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_that_are_no_distribution_are_nan_and_alone(bad):
    V = 5000
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(4, V, generator=g, device="cuda").half()
    x[1, 4321] = bad
    if bad != bad:
        x[1, 77] = -bad                          # the other sign
    got = _check(x, torch.arange(4, device="cuda"), 5)
    assert bool(got.entropy[1].isnan()) and bool(got.logprob[1].isnan()) and not bool(got.entropy[[0, 2, 3]].isnan().any())
    assert got.top_tokens[1, 0] == (4321 if bad == bad else 77)


def test_large_logits_do_not_overflow():
    x = torch.tensor([[60000.0, 59990.0, -60000.0, 0.0]], device="cuda")
    got = token_logprobs(x, torch.tensor([[0, 1, 2, 3]], device="cuda"))
    want = torch.log_softmax(x.double(), -1)
    # the logits' own scale: one rounding of x log2(e) at 86562, 2^-8, cancels; differences keep 24 bits
    assert bool(((got.logprob - want).abs() <= 2.0 ** -22 * want.abs() + 2.0 ** -7).all())


@pytest.mark.parametrize("temperature", [1e-38, 2e-39, 1e-40, 1e-45])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_temperatures_whose_inverse_overflows(temperature, dtype):
    """All of the probability is the largest logits'; the log probability of what lies 0.25 below
    them is under -2^120, or past fp32's range."""
    x = torch.tensor([[3.0, 2.75, -math.inf, 3.0, -5.0], [0.5, -0.25, 0.0, 0.25, -2.0]], device="cuda").to(dtype)
    got = token_logprobs(x, torch.arange(5, device="cuda").expand(2, 5), top_k=3, temperature=temperature)
    assert got.logprob[0, [0, 3]].tolist() == pytest.approx([-math.log(2)] * 2, abs=2.0 ** -20)
    assert got.logprob[1, 0].item() == 0 and bool((got.logprob[0, [1, 2, 4]] < -2.0 ** 120).all())
    assert bool((got.logprob[1, 1:] < -2.0 ** 120).all())
    assert got.entropy.tolist() == pytest.approx([math.log(2), 0.0], abs=2.0 ** -20)
    assert got.top_tokens.tolist() == [[0, 3, 1], [0, 3, 2]]
    wide = torch.zeros(2, 9001, device="cuda", dtype=dtype)    # many chunks, a maximum that moves
    wide[0, 8000], wide[1, ::2] = 1.0, -1.0
    got = token_logprobs(wide, torch.tensor([8000, 1], device="cuda"), temperature=temperature)
    assert got.logprob.tolist() == pytest.approx([0.0, -math.log(4500)], abs=2.0 ** -18)
    assert got.entropy.tolist() == pytest.approx([0.0, math.log(4500)], abs=2.0 ** -18)


def test_strides_and_leading_dimensions():
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(6, 2 * 777 + 5, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 777, (6,), generator=g, device="cuda")
    for view in (wide[:, 3:780], wide[:, 1:1555:2], wide[:1, :777].expand(6, 777), wide[::2, :777]):
        a = token_logprobs(view, t[:len(view)], top_k=3)
        b = token_logprobs(view.contiguous(), t[:len(view)], top_k=3)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    x = wide[:, :777].reshape(2, 3, 777)
    a = token_logprobs(x, t.reshape(2, 3), top_k=2)
    b = token_logprobs(x.reshape(6, 777), t, top_k=2)
    assert a.logprob.shape == (2, 3) and a.top_tokens.shape == (2, 3, 2)
    assert all(torch.equal(u.flatten(), v.flatten()) for u, v in zip(a, b))
    one = token_logprobs(x[0, 0], t[0], top_k=2)
    assert one.logprob.shape == () and torch.equal(one.top_tokens, b.top_tokens[0])
    none = token_logprobs(wide[:0], t[:0])
    assert none.logprob.shape == (0,)


def test_rows_beyond_32_bits():
    V = 40000
    base = torch.empty(2 ** 31 + 4 * V, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((2, V), (2 ** 31 + 2 * V, 1))
    x.copy_(torch.randn(2, V, device="cuda"))
    _check(x, torch.tensor([5, 39999], device="cuda"), 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-1e30, -1.2e38, -1.7e38, -2.5e38, -3.3e38])
def test_masks_of_any_low_value(low, dtype):
    """A mask's value may be finite and so low that a few of it overflow: its share is 0."""
    V = 9001
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (3 * torch.randn(4, V, generator=g, device="cuda")).to(dtype)
    x[0, :4500] = low          # whole threads and the first chunk hold nothing else
    x[1, 1::2] = low
    x[2, :] = low
    x[2, 8500] = 1.0
    x[3, 4096:] = low
    got = _check(x, torch.tensor([8000, 2, 8500, 1], device="cuda"), 5)
    assert bool(got.entropy.isfinite().all())


def test_more_rows_than_a_wave_of_ctas_and_the_next_kernel():
    # the rows past whole waves go in a second launch beside the first: both have ended for the next
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(1500, 20000, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 20000, (1500,), generator=g, device="cuda")
    want = _check(x, t, 5)
    for _ in range(10):
        got = token_logprobs(x, t, top_k=5)
        copies = [y.clone() for y in got]
        for y in got:
            y.zero_()
        assert all(torch.equal(a, b) for a, b in zip(copies, want))


def test_rows_split_over_clusters_beside_other_work():
    # a row's CTAs begin when the SMs that other work holds come free; none writes into the shared
    # memory of one that has not begun
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(40, 9000, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 9000, (40,), generator=g, device="cuda")
    want = _check(x, t, 20)
    work = torch.randn(1 << 22, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = []
    for _ in range(30):
        with torch.cuda.stream(side):
            work.mul_(1.0001)
        got.append(token_logprobs(x, t, top_k=20))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for y in got for a, b in zip(y, want))


def test_on_another_stream():
    x = torch.randn(7, 9000, device="cuda")
    t = torch.arange(7, device="cuda")
    want = token_logprobs(x, t, top_k=9)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [token_logprobs(x, t, top_k=9) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
