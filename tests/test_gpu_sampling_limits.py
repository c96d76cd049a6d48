"""sample_tokens and verify_drafts where numbers are far apart or outside their
range: cuts among tokens that weigh next to nothing, random numbers below 0 and
above 1, logits whose differences pass float32.

Tokens are whole numbers and have to be equal to the reference's in float64.
Distributions are float32: off by half a step of rounding (2^-24 of the value),
by the weights' own error (2.2e-12, below 2^-38), and under top_k or top_p by the
rounding of the weights whose sum it is over (V 2^-46 of the largest: 2^-28 for
V = 2^18), together below 2^-23; and half a step of the smallest float32.

A random number of 1 has no token by the definition, since no running sum passes
the whole; what is drawn then has to be one of the tokens that stay."""
import math

import numpy as np
import pytest
import torch

from sampling_reference import sample, verify
from vramancer_amd import sampling

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
RTOL = 2.0 ** -23


def check(logits, u, **kw):
    probs = torch.full(logits.shape, 7.0, device=DEV)
    tokens = sampling.sample_tokens(logits, u, probs=probs, **kw)
    alone = sampling.sample_tokens(logits, u, **kw)
    want, rows = sample(logits, u, **kw)
    want_p = np.stack(rows)
    got = probs.double().cpu().numpy()
    assert ((got > 0) == (want_p.astype(np.float32) > 0)).all()
    assert (np.abs(got - want_p) <= RTOL * want_p + 2.0 ** -149).all()
    for drawn in (tokens.tolist(), alone.tolist()):
        for n, token in enumerate(drawn):
            assert token == int(want[n]) if u[n] < 1 or token < 0 else rows[n][token] > 0


def test_tokens_that_weigh_next_to_nothing_are_cut():
    x = torch.tensor([[0.0, -4.0, -4.5, -5.0], [-5.0, -4.5, -4.0, 0.0], [-4.0, -4.0, 0.0, -4.0]], device=DEV)
    u = torch.ones(3, device=DEV)
    for k in (1, 2, 3, 4):
        for t in (0.1, 0.05, 0.01, 0.005, 1e-4):
            check(x, u, temperature=t, top_k=k)
            check(x, u, temperature=t, top_k=k, top_p=0.9)
            check(x, u, temperature=t, top_k=k, top_p=1.0 - 2.0 ** -24)


def peaked(N, V, dtype, seed, spread):
    """A normal bulk and one token (a few in the second row) far above it."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((N, V), generator=g) * 2.5
    x[:, V // 3] = spread
    x[1, torch.randint(0, V, (5,), generator=g)] = spread - 1.0
    return x.to(dtype).to(DEV), torch.rand(N, generator=g).to(DEV)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 999, 8192, 8193, 40001])
@pytest.mark.parametrize("spread,t", [(45.0, 1.0), (22.0, 0.3), (8.0, 0.02), (60.0, 0.08), (30.0, 0.02)])
def test_cuts_far_below_the_largest(V, spread, t, dtype):
    x, u = peaked(4, V, dtype, V, spread)
    u[0], u[1] = 1.0, 0.0
    for k in (2, 20, 39, 700, 5000, V // 2, V - 1):
        if k < V:
            check(x, u, temperature=t, top_k=k)
    check(x, u, temperature=t, top_k=20, top_p=0.9)


@pytest.mark.parametrize("k", [3, 30, 4000, 20000])
def test_cuts_around_the_last_bins(k):
    # weights from 1 down to 2^-60 in steps of 2^-1/300: every bin, the last ones
    # among them, has tokens, here all in order, there spread over the row
    V = 18000
    l = -torch.arange(V).double() / 300 * math.log(2.0)
    g = torch.Generator().manual_seed(k)
    x = torch.stack([l, l.flip(0), l[torch.randperm(V, generator=g)], l * 0.9, l * 3.0, l - 5.0]).float().to(DEV)
    u = torch.tensor([1.0, 0.5, 0.999, 1.0, 1.0, 1.0], device=DEV)
    check(x, u, top_k=k)
    for n in (14400, 14700, 14850, 15000, 15300):
        check(x, u, top_k=n)
    check(x, u, top_k=k, top_p=0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [3000, 20001])
def test_cuts_wider_than_what_may_be_drawn(V, dtype):
    # masks that leave few tokens, some of which weigh nothing
    x, u = peaked(6, V, dtype, V, 20.0)
    x[0, 7:] = -math.inf
    x[1, ::3] = -math.inf
    x[2, 500:] = math.nan
    x[3] = -math.inf
    x[4, V // 2:] = torch.finfo(dtype).min
    x[5, :] = 2.0
    x[5, 3] = math.inf
    for k in (5, 100, 600, V // 2, V - 1):
        for t in (1.0, 0.02):
            check(x, u, temperature=t, top_k=k)
            check(x, u, temperature=t, top_k=k, top_p=0.95)


@pytest.mark.parametrize("shift,t", [(1e5, 1e-3), (-1e5, 1e-3), (3e4, 1e-4), (0.0, 1e-6), (1e30, 1e24), (-1e30, 1e23)])
@pytest.mark.parametrize("V", [2000, 10000])
def test_cuts_far_from_zero(V, shift, t):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn((4, V), generator=g).double() * t * 60 + shift).float().to(DEV)
    u = torch.tensor([1.0, 0.4, 0.9, 0.0], device=DEV)
    for k in (2, 300, 1500, V - 2):
        check(x, u, temperature=t, top_k=k)


def test_random_numbers_next_to_nothing():
    # few tokens that weigh anything to speak of, behind many that hardly do
    V = 30001
    g = torch.Generator().manual_seed(8)
    x = torch.randn((60, V), generator=g) - 30.0
    x[:, V // 2:] += 30.0
    x[::2, :V // 2] += 8.0
    u = torch.rand(60, generator=g) * 2.0 ** -torch.arange(0, 60).float()
    check(x.to(DEV), u.to(DEV), top_k=V - 10)
    check(x.to(DEV), u.to(DEV), top_k=V // 2 + 2000)
    check(x.to(DEV), u.to(DEV), top_p=1.0 - 2.0 ** -20)
    x[:, V // 2 + 30:] = -60.0
    check(x.to(DEV), u.to(DEV), top_k=3000)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("where", ["apart", "everywhere"])
def test_cuts_between_groups_far_from_each_other(where, dtype):
    # tokens in groups 60 to 90 bits below one another, in few parts of the row or
    # in each, so that the row's parts count from different maxima
    V = 50003
    g = torch.Generator().manual_seed(5)
    x = torch.randn((3, V), generator=g) * 2.5
    for n, (level, width) in enumerate(((160.0, 3), (110.0, 9), (50.0, 40))):
        at = (torch.arange(width) * (131 if where == "apart" else V // width) + 700 * n) % V
        x[:, at] = level + torch.rand((3, width), generator=g)
    x[2] = x[2].flip(0)
    x = x.to(dtype).to(DEV)
    u = torch.tensor([0.0, 0.37, 1.0], device=DEV)
    for t in (1.0, 0.6):
        for k in (2, 5, 12, 14, 52, 60, 900, 6000):
            check(x, u, temperature=t, top_k=k)


@pytest.mark.parametrize("V", [2_200_003, 4_500_001])  # (549 parts: more than one workgroup's threads)
def test_a_very_long_row_cut_far_below_its_largest(V):
    x, u = peaked(2, V, torch.float16, 3, 40.0)
    for kw in (dict(temperature=0.7, top_k=70), dict(temperature=0.7, top_k=5000), dict(top_p=0.3, temperature=20.0),
               dict(top_k=40, temperature=20.0)):
        check(x, u, **kw)


@pytest.mark.parametrize("V", [900, 20001])
def test_drafts_that_top_k_excludes_are_refused(V):
    # a random number of 0 accepts whatever has a probability
    B, K = 6, 3
    g = torch.Generator().manual_seed(V)
    x = torch.randn((B, K + 1, V), generator=g) * 2.5
    x[:, :, 5] = 40.0
    order = x.argsort(dim=-1, descending=True)
    d = torch.stack([order[b, :K, (20, 19, 18, 1, 700, 0)[b]] for b in range(B)])
    q = torch.full((B, K, V), 1.0 / V, device=DEV)
    x, d, ua, u = x.to(DEV), d.to(DEV), torch.zeros((B, K), device=DEV), torch.rand(B, generator=g).to(DEV)
    for probs in (q, None):
        for kw in (dict(top_k=20, temperature=0.7), dict(top_k=19, temperature=0.1), dict(top_k=20, top_p=0.99)):
            tokens, accepted = sampling.verify_drafts(x, d, ua, u, probs, **kw)
            want = verify(x, d, ua, u, probs, **kw)
            assert accepted.cpu().tolist() == want[1].tolist() and tokens.cpu().tolist() == want[0].tolist()
