"""``verify_draft`` against its definition in 64 bits. Tokens and counts have to be equal.

``accept_prob`` is a ratio of softmax values in fp32: an exponential of the difference of the logits over the rows'
maxima (2^-22), a quotient and a product (2^-24 each) with the two rows' sums, and off by what these are: sums of positive fp32 terms over 256 threads (each at
most V / 256 / 8 additions one after another; errors of 2^-24 each of a part of the sum, and 2^-22 of a term's
exponential). 2^-17 relative bounds that for V up to 2^18.
"""

import math

import pytest
import torch

from dropkv_b200 import verify_draft

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def definition(target, tokens, uniforms, draft, tau):
    """(accepted, next, prob) of one sequence, in 64 bits."""
    T, V = tokens.numel(), target.shape[-1]
    n, rest, probs = 0, None, []
    ended = False
    for i in range(T):
        x = int(tokens[i])
        if not 0 <= x < V:
            probs.append(0.0)
            ended = ended or rest is None
            if rest is None and n == i:
                rest = "p"
            continue
        p = torch.softmax(target[i].double() / tau, 0)
        q = torch.softmax(draft[i].double() / tau, 0) if draft is not None else \
            torch.zeros(V, dtype=torch.float64, device=p.device).index_fill_(0, torch.tensor([x], device=p.device), 1.0)
        px, qx = float(p[x]), float(q[x])
        probs.append(math.nan if math.isnan(px) or math.isnan(qx) else (0.0 if px == 0 else min(1.0, px / qx) if qx else 1.0))
        if rest is None and n == i:
            if math.isnan(px) or math.isnan(qx):
                rest = "none"
            elif float(uniforms[i]) * qx < px:
                n += 1
            else:
                rest = (p - q).clamp(min=0)
                if not rest.sum() > 0:
                    rest = "p"
    if isinstance(rest, str) and rest == "none":
        return n, -1, probs
    if rest is None or isinstance(rest, str):
        rest = torch.softmax(target[n].double() / tau, 0)
    if bool(rest.isnan().any()):
        return n, -1, probs
    c = rest.cumsum(0)
    at = int((c <= float(uniforms[T]) * float(c[-1])).sum())
    return n, min(at, int(rest.nonzero().max())), probs


def check(target, tokens, uniforms, draft=None, tau=1.0):
    got = verify_draft(target, tokens, uniforms, draft_logits=draft, temperature=tau)
    want = [definition(target[b], tokens[b], uniforms[b], draft[b] if draft is not None else None, tau)
            for b in range(target.shape[0])]
    assert got.accepted.tolist() == [w[0] for w in want]
    assert got.next_token.tolist() == [w[1] for w in want]
    prob = torch.tensor([w[2] for w in want], dtype=torch.float64).reshape(got.accept_prob.shape)
    have = got.accept_prob.double().cpu()
    assert torch.equal(have.isnan(), prob.isnan())
    assert bool(((have - prob).abs().nan_to_num(0.0) <= 2.0 ** -17 * prob.nan_to_num(0.0)).all())
    return got


def logits(B, T, V, dtype, seed, noise=0.4, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = spread * torch.randn(B, T + 1, V, generator=g, device="cuda")
    t[:, :, : max(1, V // 50)] += 3
    d = t[:, :T] + noise * torch.randn(B, T, V, generator=g, device="cuda")
    u = torch.rand(B, T + 1, generator=g, device="cuda")
    d = d.to(dtype)
    tok = torch.multinomial(torch.softmax(d.float(), -1).reshape(B * T, V), 1, generator=g).view(B, T) if T and V > 1 else \
        torch.zeros(B, T, dtype=torch.int64, device="cuda")
    return t.to(dtype), tok, u, d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (2, 3, 2), (5, 4, 17), (3, 1, 127), (4, 5, 1000), (2, 7, 50257), (3, 2, 32000), (1, 3, 151936),
                                   (40, 6, 4099), (2, 0, 900), (1, 256, 64), (2, 17, 129)])
def test_drafts_with_probabilities(B, T, V, dtype):
    for seed in range(3):
        t, tok, u, d = logits(B, T, V, dtype, seed)
        check(t, tok, u, d, tau=(1.0, 0.6, 1.7)[seed])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", [(4, 4, 31), (3, 3, 50257), (30, 5, 2000)])
def test_drafts_without_probabilities(B, T, V, dtype):
    t, tok, u, d = logits(B, T, V, dtype, 5, noise=0.1, spread=1.0)
    tok = t[:, :T].argmax(-1)
    check(t, tok, u, None, tau=0.3)
    check(t, tok, u * 0.01, None, tau=0.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_flat_vocabulary_draws_every_token(dtype):
    """150 thousand words of one probability: cumulative sums a step of 7e-6 apart, which uniforms hit in fp32."""
    V = 151936
    u = torch.rand(64, 1, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    t = torch.zeros(64, 1, V, dtype=dtype, device="cuda")
    got = verify_draft(t, torch.zeros(64, 0, dtype=torch.int64, device="cuda"), u)
    want = (u[:, 0].double() * V).floor().long()     # the first whose sum, (t + 1) / V, passes u
    off = (u[:, 0].double() * V - (u[:, 0].double() * V).round()).abs()
    clear = off > 1e-6
    assert bool(clear.sum() >= 60) and torch.equal(got.next_token[clear], want[clear]) and got.accepted.abs().max() == 0


@pytest.mark.parametrize("draft", [True, False])
def test_padded_drafts(draft):
    t, tok, u, d = logits(6, 5, 333, torch.bfloat16, 7, noise=0.05)
    u[:, :5] *= 0.5
    for b, k in enumerate([0, 1, 3, 5, 2, 4]):
        tok[b, k:] = -1
    tok[4, 2], tok[5, 1] = 333, 1 << 40              # outside as well; what follows is not looked at
    check(t, tok, u, d if draft else None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_words_that_are_ruled_out(dtype):
    """-inf logits: of the draft's token in either distribution, and of most words."""
    t, tok, u, d = logits(8, 3, 777, dtype, 9, noise=0.1)
    t[0, 0, tok[0, 0]] = -math.inf                   # never accepted
    d[1, 0, tok[1, 0]] = -math.inf                   # q is 0 there: accepted
    t[2, :, 5:] = -math.inf                          # five words are left
    t[3] = -math.inf
    t[3, :, 776] = 1.0                               # one word is left
    d[4, :, 300:] = -math.inf
    tok[4] = d[4].argmax(-1)
    u[5] = 0.0                                       # all accepted, the first word with any weight drawn
    u[6] = 1 - 2.0 ** -24
    got = check(t, tok, u, d)
    assert got.accepted[0] == 0 and got.accept_prob[1, 0] == 1.0 and got.next_token[2] < 5 and got.next_token[3] == 776


def test_equal_distributions_and_borders():
    """p = q: everything is accepted, whatever the numbers. Borders next to the acceptance probability."""
    t, tok, u, _ = logits(4, 3, 1000, torch.float32, 11)
    u[:, :3] = 1 - 2.0 ** -24
    got = check(t, tok, u, t[:, :3].clone())
    assert got.accepted.tolist() == [3] * 4
    t, tok, u, d = logits(64, 1, 500, torch.float32, 12, noise=1.0)
    exact = [definition(t[b], tok[b], u[b], d[b], 1.0)[2][0] for b in range(64)]
    for ulps in (-1, 0, 1):                          # numbers an fp32 step around the probability: fp32 could not tell
        u[:, 0] = torch.tensor([min(x, 1 - 2.0 ** -24) for x in exact], device="cuda")
        if ulps:
            u[:, 0] = torch.nextafter(u[:, 0], torch.full((64,), float(ulps), device="cuda")).clamp(max=1 - 2.0 ** -24)
        check(t, tok, u, d)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_rows_that_are_no_distribution(value):
    t, tok, u, d = logits(7, 3, 600, torch.float16, 13, noise=0.02)
    u[:, :3] *= 0.3
    t[0, 0, 5], t[1, 2, 599], t[2, 3, 0], d[3, 1, 17] = value, value, value, value
    t[4, 1] = -math.inf
    d[5, 0] = -math.inf
    got = check(t, tok, u, d)
    assert got.next_token[:6].tolist() == [-1] * 6 and got.next_token[6] >= 0
    assert got.accepted[:6].tolist() == [0, 2, 3, 1, 1, 0]


@pytest.mark.parametrize("tau", [1e-6, 0.02, 50.0, 1e6])
@pytest.mark.parametrize("dtype", DTYPES)
def test_temperatures(tau, dtype):
    t, tok, u, d = logits(5, 2, 3000, dtype, 15)
    if tau < 1:
        tok = d.argmax(-1)
    check(t, tok, u, d, tau=tau)


def test_logits_far_from_zero():
    t, tok, u, d = logits(4, 2, 5000, torch.float32, 16)
    check(t + 3000.0, tok, u, d - 2000.0)
    check(t * 1e30, tok, u, d * 1e30, tau=1e6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(dtype):
    t, tok, u, d = logits(3, 4, 1001, dtype, 17)
    want = check(t, tok, u, d)
    wide = torch.randn(3, 6, 1003, device="cuda").to(dtype)
    wide[:, 1:, 1:1002] = t
    other = torch.randn(4, 3, 1001, device="cuda").to(dtype)
    other[:] = d.transpose(0, 1)
    strided = torch.zeros(3, 5, 1001, 2, dtype=dtype, device="cuda")
    strided[..., 0] = t
    for x in (wide[:, 1:, 1:1002], strided[..., 0]):
        got = check(x, tok.t().contiguous().t(), u, other.transpose(0, 1))
        # (rows that start elsewhere within 16 bytes are summed in another order: the probabilities, which check() has
        # compared, may differ by fp32's rounding)
        assert torch.equal(got.accepted, want.accepted) and torch.equal(got.next_token, want.next_token)


def test_captured_and_on_another_stream():
    t, tok, u, d = logits(9, 4, 9000, torch.bfloat16, 18)
    verify_draft(t, tok, u, d)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=st):
        out = verify_draft(t, tok, u, d)
    t2, tok2, u2, d2 = logits(9, 4, 9000, torch.bfloat16, 19)
    for a, b in zip((t, tok, u, d), (t2, tok2, u2, d2)):
        a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, check(t2, tok2, u2, d2)):
        assert torch.equal(a, b)


def test_what_is_kept_is_distributed_as_the_target():
    """One drafted token, 40000 times: frequencies of the first token kept against p. Of n draws a frequency's
    standard deviation is sqrt(p (1 - p) / n); six of them, for 12 words."""
    V, n = 12, 40000
    g = torch.Generator(device="cuda").manual_seed(20)
    t = torch.randn(1, 2, V, generator=g, device="cuda") * 1.5
    d = torch.randn(1, 1, V, generator=g, device="cuda") * 1.5
    tok = torch.multinomial(torch.softmax(d[0, 0], -1), n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 2, generator=g, device="cuda")
    r = verify_draft(t.expand(n, 2, V), tok, u, d.expand(n, 1, V))
    first = torch.where(r.accepted > 0, tok[:, 0], r.next_token)
    p = torch.softmax(t[0, 0].double(), -1)
    f = torch.bincount(first, minlength=V).double() / n
    assert bool(((f - p).abs() <= 6 * (p * (1 - p) / n).sqrt()).all())


def test_the_largest_sizes():
    t, tok, u, d = logits(1, 1, 1 << 21, torch.bfloat16, 40)
    check(t, tok, u, d)
    t, tok, u, d = logits(2, 256, 40, torch.float32, 41, noise=0.01)
    check(t, tok, u, d)


@pytest.mark.parametrize("draft", [True, False])
def test_uniforms_and_probabilities_near_zero(draft):
    """Acceptance where the ratio or the random number leaves fp32's range, and a number of 0, which accepts any token
    whose probability 64 bits hold."""
    gaps = [0.0, 30.0, 60.0, 69.0, 75.0, 88.0, 103.0, 500.0, 695.0, 705.0, 740.0, 760.0, math.inf]
    zs = [0.0, 2.0 ** -149, 1e-38, 1e-30, 1e-29, 1e-26, 2.0 ** -24, 0.5, 1 - 2.0 ** -24]
    B = len(gaps) * len(zs)
    t = torch.zeros(B, 2, 5, device="cuda")
    t[:, 0, 3] = -torch.tensor(gaps, device="cuda").repeat_interleave(len(zs))
    u = torch.full((B, 2), 0.5, device="cuda")
    u[:, 0] = torch.tensor(zs, device="cuda").repeat(len(gaps))
    tok = torch.full((B, 1), 3, dtype=torch.int64, device="cuda")
    d = None
    if draft:
        d = torch.zeros(B, 1, 5, device="cuda")
        d[::2, 0, 3] = -40.0
    got = verify_draft(t, tok, u, draft_logits=d)
    for b in range(B):
        n, nxt, _ = definition(t[b], tok[b], u[b], d[b] if draft else None, 1.0)
        assert (int(got.accepted[b]), int(got.next_token[b])) == (n, nxt), (b, gaps[b // len(zs)], zs[b % len(zs)])
