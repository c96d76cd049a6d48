"""accept_uniforms outside [0, 1] are taken into it, a NaN as 0, as the draws'
random numbers are.  Tokens are whole numbers and have to be equal to the
reference's for the numbers inside."""
import math

import pytest
import torch

from sampling_reference import verify
from vramancer_amd import sampling

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("B,V", [(24, 400), (24, 9001), (4500, 1900)])  # (from 2^25 logits on: float32 sums first)
@pytest.mark.parametrize("cut", [False, True])
def test_random_numbers_outside_their_range(B, V, cut):
    K = 3
    kw = dict(top_k=V * 4 // 5) if cut else {}  # (what is cut weighs little: p stays near the softmax)
    g = torch.Generator().manual_seed(V)
    some = 24
    x = torch.randn((B, K + 1, V), generator=g)
    p = torch.softmax(x[:, :K], -1)
    d = p.argmax(-1)
    # q between 0.2 and 1.3 of p at the drafts: a number of 1 accepts some, one of 2 none of those above p / 2
    part = 0.2 + 1.1 * torch.rand((B, K, 1), generator=g)
    q = torch.full((B, K, V), 1e-6).scatter_(2, d[..., None], p.gather(2, d[..., None]) * part)
    inside = torch.tensor([0.0, 1.0, 0.0, 1.0, 0.0, 1.0, 0.5, 1.0])
    outside = torch.tensor([-1.0, 2.0, math.nan, math.inf, -math.inf, 1e30, 0.5, 1.0])
    which = torch.randint(0, 8, (B, K), generator=g)
    u = torch.rand(B, generator=g)
    x, d, q, u = x.to(DEV), d.to(DEV), q.to(DEV), u.to(DEV)
    tokens, accepted = sampling.verify_drafts(x, d, outside[which].to(DEV), u, q, **kw)
    want = verify(x[:some], d[:some], inside[which][:some], u[:some], q[:some], **kw)
    assert want[1].min() == 0 and want[1].max() == K
    assert accepted[:some].cpu().tolist() == want[1].tolist() and tokens[:some].cpu().tolist() == want[0].tolist()
    again = sampling.verify_drafts(x, d, inside[which].to(DEV), u, q, **kw)
    assert torch.equal(again[0], tokens) and torch.equal(again[1], accepted)
