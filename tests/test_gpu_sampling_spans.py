"""Large batches of drafts whose logits lie so far apart that float32 does not
hold their differences, or so near to 0 that it does not hold 1 / temperature.  Tokens are whole numbers and have to be equal to the
reference's in float64, whatever the batch's size."""
import pytest
import torch

from sampling_reference import verify
from vramancer_amd import sampling

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("B", [30, 700])  # (700: 2^25 logits, float32 sums first)
@pytest.mark.parametrize("most,t", [(3.3e38, 3e38), (3.3e38, 1e38), (2e38, 5e37), (3.3e38, float("inf")), (1e30, 2e29),
                                    (1e-37, 3e-38), (4e-39, 1e-39), (3e-41, 1e-41), (1e-43, 5e-44), (3e38, 1e-40)])
def test_logits_of_the_types_whole_range(B, most, t):
    K, V = 3, 12001
    g = torch.Generator(device=DEV).manual_seed(B)
    at = dict(generator=g, device=DEV)
    x = ((torch.rand((B, K + 1, V), **at) * 2 - 1).double() * most).float()
    p = torch.softmax((x.double() / t), -1)[:, :K]
    d = torch.randint(0, V, (B, K), **at)
    d[::2] = p.argmax(-1)[::2]
    up = 0.9 + 0.2 * torch.rand((B, K, 1), **at)
    q = (p * (0.5 + torch.rand((B, K, V), **at))).scatter(2, d[..., None], p.gather(2, d[..., None]) * up).float()
    ua, u = 1.0 - 0.2 * torch.rand((B, K), **at), torch.rand(B, **at)
    temp = torch.full((B,), t, device=DEV)
    tokens, accepted = sampling.verify_drafts(x, d, ua, u, q, temperature=temp)
    n = 30
    want = verify(x[:n], d[:n], ua[:n], u[:n], q[:n], temperature=temp[:n])
    assert want[1].min() == 0 and want[1].max() >= 1
    assert accepted[:n].cpu().tolist() == want[1].tolist()
    assert tokens[:n].cpu().tolist() == want[0].tolist()
