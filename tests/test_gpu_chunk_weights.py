"""The range of the softmax weights in chunk attention: a token that takes
nearly all of a row's weight (a sink) beside thousands of tokens with small,
equal ones.

Tolerance.  As in test_gpu_paged_chunk.py: u (reach + |out|), the float32
terms 32 x 2^-24 (D + 64) reach, and 2^-25 for small fp16 outputs.  fp16
weights have a least step: they are taken relative to a reference that keeps a
row's largest weight at 2^7 or more, so the step 2^-24, rounded to half of it,
is 2^-32 of the largest weight: 2^-32 sum_t |v_t| over the tokens that the row
sees, as the largest weight is at most the sum of all.
"""
import math

import pytest
import torch

from chunk_reference import FLOAT, HALF, attend, make_table
from vramancer_amd.paged_chunk import paged_attention_chunk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _say(msg):
    print(f"[case] {msg}", flush=True)


# low: ln of a small token's weight relative to the sink's
@pytest.mark.parametrize("low", [-10.0, -16.3])
@pytest.mark.parametrize("t,D", [("f16", 64), ("f16", 128), ("f16", 256), ("bf16", 64), ("f32", 64)])
@pytest.mark.parametrize("q_len,past", [(3, 4000), (20, 4000), (300, 4000), (1, 30000)])
@pytest.mark.parametrize("sink_at", ["first", "last"])
def test_sink_and_a_long_tail(t, D, low, q_len, past, sink_at):
    _say(f"sink {sink_at}, tail at {low}, {t} D={D}, {q_len} tokens after {past}")
    H, KH, PS, n = 4, 1, 16, q_len + past
    gen = torch.Generator().manual_seed(int(-low * 10) + D)
    P, table = make_table([n], PS, gen)
    q = torch.zeros((q_len, H, D))
    q[..., 0] = 8.0
    k, v = torch.zeros((n, D)), 0.5 + torch.rand((n, D), generator=gen)
    at = 0 if sink_at == "first" else past  # (every row sees it)
    k[at, 0] = -low * math.sqrt(D) / 8
    k[:, 1] = 3 * torch.randn(n, generator=gen)  # (no query looks there)
    v[at] = 0.0
    pool = torch.zeros((P, 1, 2, KH, PS, D))
    tokens = torch.arange(n)
    pages = table[0, tokens // PS].long()
    pool[pages, 0, 0, 0, tokens % PS], pool[pages, 0, 1, 0, tokens % PS] = k, v
    q, pool = q.to(FLOAT[t]), pool.to(FLOAT[t])
    lens, cu = torch.tensor([n], dtype=torch.int32), torch.tensor([0, q_len], dtype=torch.int32)
    lse = torch.empty((q_len, H), device=DEV)
    got = paged_attention_chunk(q.to(DEV), pool.to(DEV), table.to(DEV), lens.to(DEV), cu.to(DEV), 0, lse=lse)
    want, wlse, reach = attend(q, pool.double(), table, lens, cu, 0)
    u = HALF[q.dtype] if t != "f32" else 2.0 ** -17
    tol = HALF[q.dtype] * want.abs() + (u + 32 * 2.0 ** -24 * (D + 64)) * reach
    if t == "f16":
        tol += 2.0 ** -25 + 2.0 ** -32 * v.abs().sum(0).double()
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} tolerances, {float((err / want.abs()).max()):.2e} of it"
    assert (lse.cpu().double() - wlse).abs().le(1e-5 * (8 + wlse.abs())).all()


@pytest.mark.parametrize("q_len", [2, 200])
def test_rising_scores(q_len):
    """Scores that rise by a little in every block, so that the maximum lags
    behind them by as much as it may: fp16 weights stay below their largest."""
    _say(f"rising scores, {q_len} tokens")
    H, D, PS, n = 4, 64, 16, 2000
    gen = torch.Generator().manual_seed(3)
    P, table = make_table([n], PS, gen)
    q = torch.zeros((q_len, H, D))
    q[..., 0] = 8.0
    k, v = torch.zeros((n, D)), torch.randn((n, D), generator=gen)
    k[:, 0] = torch.arange(n) // 64 * 5.5 * math.log(2)  # 5.5 in base-2 logarithms a block
    pool = torch.zeros((P, 1, 2, 1, PS, D))
    tokens = torch.arange(n)
    pages = table[0, tokens // PS].long()
    pool[pages, 0, 0, 0, tokens % PS], pool[pages, 0, 1, 0, tokens % PS] = k, v
    q, pool = q.half(), pool.half()
    lens, cu = torch.tensor([n], dtype=torch.int32), torch.tensor([0, q_len], dtype=torch.int32)
    got = paged_attention_chunk(q.to(DEV), pool.to(DEV), table.to(DEV), lens.to(DEV), cu.to(DEV), 0).cpu().double()
    want, _, reach = attend(q, pool.double(), table, lens, cu, 0)
    # scores to 170: their float32 rounding, 2^-24 of 170 log2 e x 2, moves a weight by 2^-15 of itself
    tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -14) * reach + 2.0 ** -25 + 2.0 ** -32 * v.abs().sum(0).double()
    assert got.isfinite().all() and ((got - want).abs() <= tol).all()
