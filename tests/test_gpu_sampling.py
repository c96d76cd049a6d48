"""sample_tokens and verify_drafts against the definition in float64.

Tokens are whole numbers and have to be equal.  A distribution is float32: off
by half a step of rounding (2^-24 of the value), by the weights' own error
(below 2^-50), and under top_k or top_p by the rounding of the weights whose sum
it is over (V 2^-46 of the largest: 2^-28 for V = 2^18), together below 2^-23."""
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


def make(N, V, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((N, V), generator=g) * spread
    x[torch.arange(N), torch.randint(0, V, (N,), generator=g)] += 6.0
    return x.to(dtype).to(DEV), torch.rand(N, generator=g).to(DEV)


def check(logits, u, **kw):
    probs = torch.full(logits.shape, 7.0, device=DEV)
    tokens = sampling.sample_tokens(logits, u, probs=probs, **kw)
    assert torch.equal(tokens, sampling.sample_tokens(logits, u, **kw))  # the two paths of it
    want, rows = sample(logits, u, **kw)
    assert tokens.dtype == torch.int64 and tokens.cpu().tolist() == want.tolist()
    want = np.stack(rows)
    got = probs.double().cpu().numpy()
    assert ((got > 0) == (want.astype(np.float32) > 0)).all()
    assert (np.abs(got - want) <= RTOL * want + 2.0 ** -149).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 7, 63, 64, 257, 1000, 8191, 8192, 8193, 20001])
def test_plain(V, dtype):
    check(*make(5, V, dtype, V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_k", [1, 2, 50, 1000, 100000])
@pytest.mark.parametrize("V", [5, 999, 8200, 20001])
def test_top_k(V, top_k, dtype):
    check(*make(4, V, dtype, V + top_k), top_k=top_k, temperature=0.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top_p", [0.0, 1e-6, 0.3, 0.9, 0.999])
@pytest.mark.parametrize("V", [1, 5, 999, 8200, 20001])
def test_top_p(V, top_p, dtype):
    check(*make(4, V, dtype, V + int(100 * top_p)), top_p=top_p, temperature=1.3)


@pytest.mark.parametrize("dtype", TYPES)
def test_each_row_its_own(dtype):
    N = 33
    x, u = make(N, 5003, dtype, 3)
    g = torch.Generator().manual_seed(4)
    temp = torch.rand(N, generator=g) * 1.5 + 0.1
    temp[::5] = 0.0
    temp[1] = -1.0
    temp[2] = math.inf
    k = torch.randint(0, 60, (N,), generator=g, dtype=torch.int32)
    k[3], k[4] = -7, 5003
    p = torch.rand(N, generator=g)
    p[6], p[7] = 1.0, 2.0
    check(x, u, temperature=temp.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV))
    check(x, u, temperature=temp.to(DEV))


def test_nan_parameters():
    x, u = make(3, 1000, torch.float32, 11)
    t = torch.tensor([math.nan, 1.0, 1.0], device=DEV)
    p = torch.tensor([1.0, math.nan, 0.5], device=DEV)
    got = sampling.sample_tokens(x, u, temperature=t, top_p=p)
    want, _ = sample(x, u, temperature=torch.tensor([0.0, 1.0, 1.0]), top_p=torch.tensor([1.0, 1.0, 0.5]))
    assert got.cpu().tolist() == want.tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_k=700), dict(top_p=0.37), dict(top_k=900, top_p=0.61)])
def test_equal_logits(kw, dtype):
    # all equal, and a few values that many tokens share: the order is by index
    V = 9001
    flat = torch.full((2, V), 1.5)
    flat[1] = -torch.finfo(dtype).max  # the type's lowest value everywhere
    few = torch.randint(0, 4, (3, V), generator=torch.Generator().manual_seed(1)).float()
    zeros = torch.zeros((1, V))
    zeros[0, ::2] = -0.0  # equal to 0
    x = torch.cat([flat, few, zeros]).to(dtype).to(DEV)
    check(x, torch.tensor([0.123456, 0.999, 0.0, 0.5, 0.77, 0.3], device=DEV), **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20), dict(top_p=0.8), dict(temperature=0.0)])
def test_masked_and_not_finite(kw):
    V = 8500
    x, _ = make(9, V, torch.float32, 21)
    x[0] = -math.inf                         # no token
    x[1] = math.nan                          # no token
    x[2] = -math.inf
    x[2, 8300] = -50.0                       # one token
    x[3, ::2] = -math.inf                    # half of them
    x[4, 5::7] = math.nan
    x[5, 17] = x[5, 8400] = math.inf         # those two alone
    x[6, :] = torch.finfo(torch.float32).min
    x[6, 3] = 0.0
    x[7, :8192] = -math.inf                  # an empty first chunk
    x[8, 8192:] = -math.inf                  # an empty last one
    u = torch.tensor([0.5, 0.5, 0.9, 0.4, 0.3, 0.7, 0.6, 0.2, 0.8], device=DEV)
    check(x, u, **kw)
    got = sampling.sample_tokens(x, u, **kw).tolist()
    assert got[:3] == [-1, -1, 8300] and got[5] in (17, 8400)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=20, top_p=0.9)])
def test_random_numbers_at_the_ends(kw):
    x, _ = make(6, 8300, torch.bfloat16, 5)
    u = torch.tensor([0.0, 1.0, 1.0 - 2.0 ** -24, -3.0, 7.0, math.nan], device=DEV)
    check(x, u, **kw)


@pytest.mark.parametrize("kw", [dict(temperature=1e-4), dict(temperature=1e-38), dict(temperature=1e4),
                                dict(temperature=1e-4, top_k=5), dict(temperature=1e4, top_p=0.5),
                                dict(temperature=1e-38, top_p=0.5)])
def test_temperatures(kw):
    check(*make(4, 3001, torch.float32, 6), **kw)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    x, u = make(6, 5000, dtype, 8)
    check(x[:, 1:4000], u)                      # rows that start off their alignment
    check(x[::2, 3:4998], u[::2], top_k=40)
    check(x[:1].expand(6, 5000), u, top_p=0.7)  # a row for all
    check(x.t()[:6, :6], u)                     # (copied)
    check(x[:, ::2], u)


@pytest.mark.parametrize("V", [30000, 131072])
def test_crowded_bins(V):
    # float32 logits that lie within one step of the first pass's bins, and many
    # equal ones: the border's bin holds more tokens than fit a list
    g = torch.Generator().manual_seed(V)
    near = torch.rand((2, V), generator=g) * 1e-3
    near[1] = (near[1] * 4e3).round() / 4e3
    two = torch.zeros((1, V))
    two[0, torch.randperm(V, generator=g)[: V // 3]] = 2.0
    x = torch.cat([near, two]).to(DEV)
    u = torch.tensor([0.31, 0.62, 0.93], device=DEV)
    for kw in (dict(top_k=V // 2), dict(top_p=0.55), dict(top_k=V - 5, top_p=0.99)):
        check(x, u, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(top_k=9000), dict(top_p=0.45), dict(top_k=25000, top_p=0.8)])
def test_ties_of_both_signs(kw, dtype):
    # few values on both sides of 0, close together and far apart, in lists that
    # fit and that do not
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-3, 4, (4, 30001), generator=g).float()
    x = (x * torch.tensor([2.0 ** -12, 2.0 ** -5, 0.125, 1.0])[:, None]).to(dtype).to(DEV)
    check(x, torch.tensor([0.2, 0.45, 0.7, 0.95], device=DEV), **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [2047, 2048, 2049, 6145, 8191, 8192, 8193])
def test_rows_around_one_part(V, dtype):
    # lists that fit and that do not, each row with parameters of its own
    g = torch.Generator().manual_seed(V)
    x = torch.randn((12, V), generator=g) * 2.0
    x[0] = 0.75
    x[1] = -torch.finfo(dtype).max
    x[2] = torch.randint(0, 3, (V,), generator=g) * 0.01
    x[3] = -math.inf
    x[4] = math.nan
    x[4, V - 1] = -3.0
    x[5, : V // 2] = math.inf
    x[6, ::3] = -math.inf
    x = x.to(dtype).to(DEV)
    u = torch.rand(12, generator=g).to(DEV)
    k = torch.tensor([V // 2, V - 1, 1500, 5, 5, 700, 0, 1, 1000, V, 50, 40], dtype=torch.int32)
    p = torch.tensor([0.8, 1.0, 0.999, 0.5, 0.5, 0.3, 0.97, 0.5, 1.0, 0.9, 0.9, 1.0])
    t = torch.tensor([1.0, 0.7, 3.0, 1.0, 1.0, 1.0, 0.5, 1.0, 2.0, 0.6, 1.5, 0.0])
    check(x, u, temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV))
    check(x, u, top_k=V - 1)
    check(x, u, top_p=0.62, temperature=1.3)


def test_no_rows_and_out():
    x, u = make(4, 100, torch.float32, 9)
    assert sampling.sample_tokens(x[:0], u[:0]).shape == (0,)
    out = torch.full((4,), -5, dtype=torch.int64, device=DEV)
    ws = sampling.sample_workspace(4, 100, device=DEV)
    ws.fill_(255)
    got = sampling.sample_tokens(x, u, top_p=0.9, out=out, workspace=ws)
    assert got is out and out.cpu().tolist() == sample(x, u, top_p=0.9)[0].tolist()


def drafts_of(B, K, V, dtype, seed, near=0.7):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, K + 1, V), generator=g) * 2.5
    q = torch.softmax(x[:, :K] + torch.randn((B, K, V), generator=g) * near, -1)
    d = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, K) if K else torch.zeros((B, 0), dtype=torch.int64)
    return (x.to(dtype).to(DEV), d.to(DEV), torch.rand((B, K), generator=g).to(DEV), torch.rand(B, generator=g).to(DEV),
            q.to(DEV))


def many_drafts(B, K, V, dtype, seed):
    """The same, made on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((B, K + 1, V), generator=g, device=DEV) * 2.5
    q = torch.softmax(x[:, :K] + torch.randn((B, K, V), generator=g, device=DEV) * 0.7, -1)
    d = (q / -torch.rand((B, K, V), generator=g, device=DEV).clamp(min=1e-30).log()).argmax(-1)
    return (x.to(dtype), d, torch.rand((B, K), generator=g, device=DEV), torch.rand(B, generator=g, device=DEV), q)


def check_verify(x, d, ua, u, q=None, cu=None, **kw):
    tokens, accepted = sampling.verify_drafts(x, d, ua, u, draft_probs=q, cu_seqlens=cu, **kw)
    want_t, want_a = verify(x, d, ua, u, q, cu, **kw)
    assert tokens.dtype == torch.int64 and accepted.dtype == torch.int32
    assert accepted.cpu().tolist() == want_a.tolist()
    assert tokens.cpu().tolist() == want_t.tolist()
    return want_a


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_q", [True, False])
@pytest.mark.parametrize("V,K,B", [(1, 1, 2), (5, 3, 9), (1000, 4, 12), (8193, 2, 7), (20001, 5, 4), (300, 0, 3)])
def test_verify(V, K, B, with_q, dtype):
    x, d, ua, u, q = drafts_of(B, K, V, dtype, V + K)
    check_verify(x, d, ua, u, q if with_q else None)
    check_verify(x, d.int(), ua * 0.2, u, q if with_q else None, temperature=0.8, top_k=60, top_p=0.9)


def test_verify_every_length():
    # sequences that accept 0 .. K drafts
    B, K, V = 40, 6, 500
    x, d, ua, u, q = drafts_of(B, K, V, torch.float32, 1, near=0.3)
    got = check_verify(x, d, ua, u, q)
    assert set(got.tolist()) == set(range(K + 1))


def test_verify_ragged():
    B, K, V = 6, 4, 777
    g = torch.Generator().manual_seed(2)
    _, d, ua, u, q = drafts_of(B, K, V, torch.float16, 2)
    cu = torch.tensor([0, 1, 1, 6, 13, 15, 18], dtype=torch.int32)  # 1, 0, 5, 7 (more than K + 1), 2, 3 rows
    x = (torch.randn((21, V), generator=g) * 2).half().to(DEV)      # and three behind the last sequence
    for kw in (dict(), dict(temperature=torch.rand(B, generator=g).to(DEV), top_p=0.8)):
        check_verify(x, d, ua * 0.3, u, q, cu.to(DEV), **kw)
        check_verify(x, d, ua * 0.3, u, None, cu.long().to(DEV), **kw)


def test_verify_rows_behind_are_not_read():
    # rows behind the last sequence may hold anything, offsets past the rows are cut
    B, K, V = 3, 2, 300
    x, d, ua, u, q = drafts_of(B, K, V, torch.float32, 3)
    flat = torch.cat([x.reshape(-1, V), torch.full((4, V), math.nan, device=DEV)])
    cu = torch.tensor([0, 3, 6, 9], dtype=torch.int32, device=DEV)
    check_verify(flat, d, ua, u, q, cu)
    check_verify(flat[:7], d, ua, u, q, cu)  # the last sequence keeps one row


def test_verify_short_lists_and_bad_drafts():
    B, K, V = 5, 3, 600
    x, d, ua, u, q = drafts_of(B, K, V, torch.float32, 4, near=0.01)
    d[0, 0] = -1
    d[1, 1] = -1
    d[2, 0] = V
    d[3, 2] = 1 << 40
    ua = ua * 0.1
    check_verify(x, d, ua, u, q)
    check_verify(x, d, ua, u, None)


def test_verify_greedy_rows():
    B, K, V = 8, 3, 1200
    x, d, ua, u, q = drafts_of(B, K, V, torch.bfloat16, 5)
    d[:4] = x[:4, :K].float().argmax(-1)
    t = torch.zeros(B, device=DEV)
    t[::2] = 0.9
    got = check_verify(x, d, ua, u, q, temperature=t)
    assert got[1] == K and got[3] == K
    check_verify(x, d, ua, u, None, temperature=0.0, top_k=5)


def test_verify_masked():
    B, K, V = 6, 2, 900
    x, d, ua, u, q = drafts_of(B, K, V, torch.float32, 6)
    x[0, 0] = -math.inf            # nothing may follow: no draft is accepted, and no token drawn
    x[1, :, ::2] = -math.inf
    x[2, 1, d[2, 1]] = -math.inf   # a draft that the target forbids
    x[3, 0, :] = math.nan
    x[4, 0, 10] = math.inf
    q = q.clone()
    q[5, 0, 5] = math.nan
    q[5, 1, :] = -1.0
    check_verify(x, d, ua, u, q)
    check_verify(x, d, ua, u, q, top_p=0.9)


def test_verify_nothing_left():
    # q is at least p everywhere and the draft is refused all the same: the next token is p's own
    B, K, V = 4, 2, 9000
    x, d, ua, u, _ = drafts_of(B, K, V, torch.float32, 7)
    q = torch.full((B, K, V), 2.0, device=DEV)
    got = check_verify(x, d, ua * 0 + 0.9, u, q)
    assert got.sum() == 0
    check_verify(x, d, ua * 0 + 0.9, u, q, top_k=30)


def test_verify_strides():
    B, K, V = 4, 3, 1001
    x, d, ua, u, q = drafts_of(B, K, V, torch.float16, 8)
    wide = torch.zeros((B, K + 2, V + 5), dtype=torch.float16, device=DEV)
    wide[:, :K + 1, 2:V + 2] = x
    qs = torch.zeros((K, B, V + 3), device=DEV)
    qs[:, :, 1:V + 1] = q.transpose(0, 1)
    want = sampling.verify_drafts(x, d, ua, u, q)
    got = sampling.verify_drafts(wide[:, :K + 1, 2:V + 2], d.t().contiguous().t(), ua, u, qs[:, :, 1:V + 1].transpose(0, 1))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_verify(x, d, ua, u, q[:, :, :].contiguous())


def test_verified_tokens_are_the_targets():
    """The first token of a verified sequence has the target's distribution,
    whatever the draft's: over n sequences a token's share is binomial, within
    6 sigma of p for 8 tokens (chance below 2e-8)."""
    n, V = 60000, 8
    g = torch.Generator(device=DEV).manual_seed(9)
    target = torch.tensor([2.0, 1.0, 0.5, 0.0, -0.5, 1.5, -3.0, 0.2], device=DEV)
    draft = torch.tensor([-1.0, 2.0, 0.5, 1.0, 0.5, 0.0, 1.0, -2.0], device=DEV)
    q = torch.softmax(draft, -1)
    d = torch.multinomial(q.expand(n, V), 1, replacement=True, generator=g)
    ua, u = torch.rand((n, 1), generator=g, device=DEV), torch.rand(n, generator=g, device=DEV)
    tokens, accepted = sampling.verify_drafts(target.expand(n, 2, V), d, ua, u, q.expand(n, 1, V))
    p = torch.softmax(target.double(), -1).cpu()
    share = torch.bincount(tokens[:, 0], minlength=V).double().cpu() / n
    assert ((share - p).abs() <= 6 * (p * (1 - p) / n).sqrt()).all()
    agree = torch.minimum(p, q.double().cpu()).sum()
    assert abs(accepted.double().mean().item() - agree) <= 6 * math.sqrt(agree * (1 - agree) / n)


@pytest.mark.parametrize("B,K,V", [(3, 14, 700), (900, 2, 40), (300, 1, 20000), (90, 9, 40001), (9000, 3, 1000)])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=20, top_p=0.9)])
def test_verify_many(B, K, V, kw):
    # many drafts, many sequences: drafts tested in a launch of their own, and
    # from 2^25 logits on sums in float32 first
    x, d, ua, u, q = many_drafts(B, K, V, torch.bfloat16, B)
    ws = sampling.verify_workspace(B, K, V, device=DEV)
    ws.fill_(255)
    some = slice(0, B, max(1, B // 30))  # (the reference is slow)
    tokens, accepted = sampling.verify_drafts(x, d, ua, u, q, workspace=ws, **kw)
    want = verify(x[some], d[some], ua[some], u[some], q[some], **kw)
    assert tokens[some].cpu().tolist() == want[0].tolist() and accepted[some].cpu().tolist() == want[1].tolist()
    again = sampling.verify_drafts(x, d, ua, u, q, **kw)
    assert torch.equal(again[0], tokens) and torch.equal(again[1], accepted)


def borders(B, K, V, dtype, seed, near):
    """Drafts whose random number lies next to p / q, and draft distributions
    that are p but for 1e-6 of it (near) and a few tokens."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    at = dict(generator=g, device=DEV)
    x = (torch.randn((B, K + 1, V), **at) * 2.5).to(dtype)
    p = torch.softmax(x.double(), -1)[:, :K]
    q = p * (1 + near * torch.randn((B, K, V), **at))
    up = torch.randint(0, V, (B, K, 1), **at)
    down = torch.randint(0, V, (B, K, 9), **at)
    q = q.scatter(2, down, p.gather(2, down) * 0.3)
    d = p.argmax(-1) if near else up[..., 0]
    q = q.scatter(2, d[..., None], (p.gather(2, d[..., None]) * 1.7 + 1e-3).clamp(max=1.0)).float()
    ua = (p.gather(2, d[..., None]) / q.double().gather(2, d[..., None]))[..., 0].float()
    step = torch.randint(-3, 4, (B, K), **at)
    step[:, -1] = 4  # (the last is refused if the others pass)
    for i in range(1, 5):
        ua = torch.where(step >= i, torch.nextafter(ua, torch.full_like(ua, 2.0)), ua)
        ua = torch.where(step <= -i, torch.nextafter(ua, torch.zeros_like(ua)), ua)
    return x, d, ua, torch.rand(B, **at), q


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("near", [0.0, 1e-6, 1e-7])
@pytest.mark.parametrize("B,K,V,only", [(6, 3, 3000, None), (700, 3, 300, 60), (230, 2, 50001, 12), (12000, 3, 800, 100)])
def test_verify_at_the_borders(B, K, V, only, near, dtype):
    # small and large batches take different sums; both decide as 64 bits do
    x, d, ua, u, q = borders(B, K, V, dtype, V + B, near)
    tokens, accepted = sampling.verify_drafts(x, d, ua, u, q)
    n = only or B
    want = verify(x[:n], d[:n], ua[:n], u[:n], q[:n])
    assert accepted[:n].cpu().tolist() == want[1].tolist()
    assert tokens[:n].cpu().tolist() == want[0].tolist()
    if only:
        tokens, accepted = sampling.verify_drafts(x, d, ua, u)
        want = verify(x[:n], d[:n], ua[:n], u[:n])
        assert tokens[:n].cpu().tolist() == want[0].tolist() and accepted[:n].cpu().tolist() == want[1].tolist()


def test_verify_large_masked():
    # what test_verify_masked, _greedy_rows and _nothing_left hold, in a large batch
    B, K, V = 600, 3, 14001
    x, d, ua, u, q = many_drafts(B, K, V, torch.float32, 16)
    x[0, 0] = -math.inf
    x[1, :, ::2] = -math.inf
    x[2, 1, d[2, 1]] = -math.inf
    x[3, 0, :] = math.nan
    x[4, 0, 10] = math.inf
    x[5, 0, 700:] = math.nan
    q = q.clone()
    q[6, 0, 5] = math.nan
    q[7, 1, :] = -1.0
    q[8] = 2.0
    d[9, 0], d[10, 1] = -1, V
    t = torch.full((B,), 0.7, device=DEV)
    t[11:14] = 0.0
    t[14], t[15], t[16] = math.inf, 1e-38, 1e4
    d[12] = x[12, :K].argmax(-1)
    ua[8] = 0.9
    for kw in (dict(), dict(temperature=t)):
        for probs in (q, None):
            tokens, accepted = sampling.verify_drafts(x, d, ua, u, probs, **kw)
            part = {k: v[:40] for k, v in kw.items()}
            want = verify(x[:40], d[:40], ua[:40], u[:40], None if probs is None else q[:40], **part)
            assert tokens[:40].cpu().tolist() == want[0].tolist() and accepted[:40].cpu().tolist() == want[1].tolist()


@pytest.mark.parametrize("kw", [dict(), dict(top_k=70), dict(top_p=0.9)])
def test_a_very_long_row(kw):
    # more segments than the draw of a cut takes
    V = 2_200_003
    x, u = make(2, V, torch.float16, 3)
    check(x, u, **kw)


def test_rows_of_a_mixed_batch():
    # greedy, cut and whole rows, masked and empty ones, of one call
    N, V = 24, 9000
    x, u = make(N, V, torch.bfloat16, 31)
    x[5] = -math.inf
    x[6, 100:] = -math.inf
    x[7] = 2.0
    k = torch.zeros(N, dtype=torch.int32)
    k[::3] = torch.tensor([1, 5, 50, 4000, 5000, 8999, 9000, 20000], dtype=torch.int32)
    p = torch.ones(N)
    p[::2] = torch.linspace(0.0, 0.999, 12)
    t = torch.ones(N)
    t[::7] = 0.0
    check(x, u, temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV))
    ws = sampling.sample_workspace(N, V, device=DEV)
    ws.fill_(255)
    want = sampling.sample_tokens(x, u, temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV))
    got = sampling.sample_tokens(x, u, temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV), workspace=ws)
    assert torch.equal(got, want)


def test_repeats_and_streams():
    x, u = make(40, 30011, torch.bfloat16, 12)
    first = sampling.sample_tokens(x, u, top_p=0.9)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([sampling.sample_tokens(x, u, top_p=0.9) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(t, first) for g in got for t in g)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50, top_p=0.9)])
def test_captured(kw):
    """One graph of a draw and a verification, replayed with other numbers
    between eager calls."""
    B, K, V = 5, 3, 9001
    x, d, ua, u, q = drafts_of(B, K, V, torch.bfloat16, 13)
    temp = torch.full((B,), 0.8, device=DEV)
    sampling.verify_drafts(x, d, ua, u, q, temperature=temp, **kw)
    sampling.sample_tokens(x[:, 0], u, temperature=temp, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted = sampling.verify_drafts(x, d, ua, u, q, temperature=temp, **kw)
        drawn = sampling.sample_tokens(x[:, 0], u, temperature=temp, **kw)
    for seed in range(4):
        y, e, va, v, r = drafts_of(B, K, V, torch.bfloat16, 20 + seed)
        for to, fr in ((x, y), (d, e), (ua, va), (u, v), (q, r)):
            to.copy_(fr)
        temp.fill_(0.5 + 0.2 * seed)
        graph.replay()
        torch.cuda.synchronize()
        want = verify(y, e, va, v, r, temperature=temp, **kw)
        assert tokens.cpu().tolist() == want[0].tolist() and accepted.cpu().tolist() == want[1].tolist()
        assert drawn.cpu().tolist() == sample(y[:, 0], v, temperature=temp, **kw)[0].tolist()
        again = sampling.verify_drafts(x, d, ua, u, q, temperature=temp, **kw)
        assert torch.equal(again[0], tokens) and torch.equal(again[1], accepted)


def test_offsets_past_32_bits():
    # 70000 rows of 66000 16-bit logits: 9.2 GB, 4.6e9 elements
    N, V = 70000, 66000
    x = torch.zeros((N, V), dtype=torch.bfloat16, device=DEV)
    at = torch.arange(N, device=DEV) % V
    x[torch.arange(N, device=DEV), at] = 60.0  # (the others weigh V e^-60 together)
    u = torch.full((N,), 0.5, device=DEV)
    assert torch.equal(sampling.sample_tokens(x, u), at)
    del x
    torch.cuda.empty_cache()
