"""``verify_draft`` where a probability lies within a few parts in 10^13 of a random number.

Two words, the first with p = 1 / (1 + e^(-d / temperature)): of many d in fp32, those are taken whose p is off a multiple of
2^-24, u, by 3e-14 to 3e-13 of itself. Sums, exponentials and quotients in 64 bits are off by some 5e-15, here and in the
kernel, so which of the two is larger is certain. (A temperature rounded to fp32 is off by up to 6e-8.)
"""

import pytest
import torch

from dropkv_b200 import verify_draft

pytestmark = pytest.mark.gpu


def near_ties(tau, n=1 << 26):
    g = torch.Generator(device="cuda").manual_seed(1)
    d = (0.01 + 8 * torch.rand(n, generator=g, device="cuda", dtype=torch.float64)).float()
    p = 1 / (1 + torch.exp(-d.double() / tau))
    u = torch.round(p * 2.0 ** 24) / 2.0 ** 24
    off = (p - u).abs() / p
    take = (off > 3e-14) & (off < 3e-13) & (u < 1)
    return d[take], u[take].float(), (p > u)[take]


@pytest.mark.parametrize("tau", [1.0, 0.7, 1.3])
@pytest.mark.parametrize("up", [True, False])
def test_draws_and_decisions_near_a_tie(up, tau):
    d, u, first = near_ties(tau)
    n = d.numel()
    assert n > 100 and 0.3 < float(first.double().mean()) < 0.7
    # the larger word's logit is 0 and the other's -d, or d and 0
    rows = (torch.stack([d, torch.zeros_like(d)], 1) if up else torch.stack([torch.zeros_like(d), -d], 1)).view(n, 1, 2)
    none = torch.zeros(n, 0, dtype=torch.int64, device="cuda")
    drawn = verify_draft(rows, none, u[:, None], temperature=tau)
    assert torch.equal(drawn.next_token == 0, first)
    # the first word drafted by a draft without probabilities: accepted while u < p
    got = verify_draft(rows.expand(n, 2, 2), torch.zeros(n, 1, dtype=torch.int64, device="cuda"), torch.stack([u, u], 1),
                       temperature=tau)
    assert torch.equal(got.accepted == 1, first)
