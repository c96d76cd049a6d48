"""paged_attention_chunk against float64 attention by the definition.

Tolerance per output element.  Let u be half a step of the query's type,
reach = sum_t p_t |v_t|.
* 16-bit products: queries, keys and codes enter exactly, scores are float32
  sums of D exact products; the weights are rounded once (at most 2^-9 relative
  for bf16, 2^-12 for fp16: at most 1 u each, u = 2^-8 / 2^-11 counting half a
  step relative to the value), the output once: u (reach + |out|).  Float32
  sums and exponentials of scores up to a few tens add below 2^-18 reach each:
  32 x 2^-24 x (D + 64) reach covers them.
* fp16 queries over int8 / fp8: the weights are a bf16 high and low part
  (2^-17), so only the output's rounding and the float32 terms count.
* float32 products: the float32 terms and the output's rounding.
* fp16 below 2^-14 are multiples of 2^-24: a rounding there is off by up to
  2^-25 whatever the value, which is more than 2^-11 of it (bf16 and float32
  have no such values in these tests).
lse: the float32 terms, absolute, times its size.
"""
import math

import pytest
import torch

from chunk_reference import FLOAT, HALF, attend, make_pool, make_table, to_gpu
from vramancer_amd import paged_chunk
from vramancer_amd.paged_chunk import chunk_workspace

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(params=["tight", "wide"], autouse=True)
def table_width(request):
    """The kernel is chosen by the batch's sizes, the table's width among
    them: every test runs with a table as wide as its longest sequence, and
    with one whose further entries are absent pages."""
    global _wide
    _wide = request.param == "wide"


def paged_attention_chunk(query, pool, table, lens, cu, layer, **kw):
    rows = query.shape[0] * query.shape[1]
    need = table.shape[1]
    if _wide and "workspace" not in kw and rows and table.dim() == 2:
        width = min(-(-(1 << 24) // (rows * pool.shape[4])), 1 << 15)
        if width > need:
            more = torch.full((table.shape[0], width - need), -1, dtype=table.dtype, device=table.device)
            table = torch.cat([table, more], 1)
    return paged_chunk.paged_attention_chunk(query, pool, table, lens, cu, layer, **kw)


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _batch(q_lens, past, PS, seed, drop=()):
    gen = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(q_lens, past)]
    P, table = make_table(lens, PS, gen)
    for b, i in drop:
        table[b, i] = P + 5 if (b + i) % 2 else -1
    cu = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    return gen, P, table, torch.tensor(lens, dtype=torch.int32), cu


def _tolerance(want, reach, q_type, wide, D, quant):
    u = HALF[q_type]
    soft = u if not wide and not (quant and q_type == torch.float16) else 2.0 ** -17
    tiny = 2.0 ** -25 if q_type == torch.float16 else 1e-30
    return u * want.abs() + (soft + 32 * 2.0 ** -24 * (D + 64)) * reach + tiny


def _check(qt, kv, q_lens, past, H, KH, D, PS, seed, layout=None, drop=(), tail=0, q_std=1.5, **kw):
    gen, P, table, lens, cu = _batch(q_lens, past, PS, seed, drop)
    L, layer = 2, 1
    pool, scales, vals = make_pool(kv, P, L, KH, PS, D, gen, layout)
    N = int(cu[-1]) + tail
    q = (torch.randn((N, H, D), generator=gen) * q_std).to(FLOAT[qt])
    g_pool, g_scales = to_gpu(pool, scales)
    out = torch.full((N, H, D), 7.0, dtype=q.dtype, device=DEV)
    lse = torch.full((N, H), 7.0, device=DEV)
    got = paged_attention_chunk(q.to(DEV), g_pool, table.to(DEV), lens.to(DEV), cu.to(DEV), layer, kv_scales=g_scales,
                                out=out, lse=lse, **kw)
    torch.cuda.synchronize()
    assert got is out
    want, wlse, reach = attend(q, vals, table, lens, cu, layer, **kw)
    n = int(cu[-1])
    assert (out[n:] == 7).all() and (lse[n:] == 7).all(), "rows behind the last sequence changed"
    wide = qt == "f32" or kv == "f32" or (kv in FLOAT and kv != qt)
    tol = _tolerance(want[:n], reach[:n], q.dtype, wide, D, kv not in FLOAT)
    err = (out[:n].cpu().double() - want[:n]).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).nan_to_num(9e9).max()):.2f} "
                           f"tolerances at {bad.nonzero()[0].tolist()}")
    got_l, want_l = lse[:n].cpu().double(), wlse[:n]
    none = want_l == -math.inf
    assert (got_l[none] == -math.inf).all() and (out[:n].cpu()[none] == 0).all()
    assert (got_l[~none] - want_l[~none]).abs().le(1e-5 * (8 + want_l[~none].abs())).all()
    return out


PAIRS = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "int8"), ("f16", "int8"), ("bf16", "fp8"), ("f16", "fp8"),
         ("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("f32", "int8"), ("f32", "fp8"), ("bf16", "f16"),
         ("f16", "bf16"), ("bf16", "f32")]


@pytest.mark.parametrize("qt,kv", PAIRS, ids=["-".join(p) for p in PAIRS])
@pytest.mark.parametrize("H,KH,D,PS", [(10, 2, 128, 16), (4, 4, 64, 16), (7, 1, 96, 16), (6, 2, 80, 32), (4, 2, 256, 16)])
def test_types_and_heads(qt, kv, H, KH, D, PS):
    _say(f"chunk {qt} over {kv} H={H} KH={KH} D={D} PS={PS}")
    _check(qt, kv, [33, 1, 70], [100, 47, 0], H, KH, D, PS, seed=D + H)


@pytest.mark.parametrize("q_lens,past", [
    ([1], [0]), ([1], [1]), ([1], [63]), ([2], [64]), ([17], [0]), ([64], [0]), ([65], [0]), ([127], [1]), ([129], [63]),
    ([0, 5, 0], [9, 20, 0]), ([1] * 70, list(range(70))), ([4] * 9, [300] * 9), ([300], [0]), ([3], [5000]),
    ([200, 1, 1, 1], [0, 700, 3, 0])], ids=lambda v: "x".join(map(str, v[:4])) + ("" if len(v) < 5 else f"n{len(v)}"))
@pytest.mark.parametrize("qt,kv", [("bf16", "bf16"), ("bf16", "int8"), ("f32", "f32")], ids=["bf16", "int8", "f32"])
def test_lengths(qt, kv, q_lens, past):
    _say(f"chunk {qt} over {kv} q {q_lens[:5]} past {past[:5]}")
    _check(qt, kv, q_lens, past, 6, 2, 64, 16, seed=sum(q_lens) + 7, tail=2)


@pytest.mark.parametrize("kv", ["f16", "int8", "fp8"])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 1000])
def test_window(kv, window):
    _say(f"chunk window {window} over {kv}")
    _check("f16", kv, [40, 150, 1], [300, 0, 90], 6, 2, 64, 16, seed=window, window=window)
    _check("f16", kv, [40, 9], [300, 0], 6, 2, 64, 16, seed=window, window=window, causal=False)


@pytest.mark.parametrize("qt,kv", [("bf16", "bf16"), ("f32", "f32")], ids=["bf16", "f32"])
def test_window_of_every_token(qt, kv):
    """The widest window is no window, for rows before a context's start too."""
    _say(f"chunk widest window {qt} over {kv}")
    gen, P, table, lens, cu = _batch([40, 9], [0, 70], 16, 77)
    lens = torch.tensor([11, 79], dtype=torch.int32)
    pool, _, vals = make_pool(kv, P, 1, 2, 16, 64, gen)
    q = torch.randn((49, 6, 64), generator=gen).to(FLOAT[qt])
    args = (q.to(DEV), pool.to(DEV), table.to(DEV), lens.to(DEV), cu.to(DEV), 0)
    out = paged_attention_chunk(*args, window=2 ** 31 - 1)
    assert torch.equal(out, paged_attention_chunk(*args))
    assert (out[:29] == 0).all() and (out[29:] != 0).any()


@pytest.mark.parametrize("qt,kv", [("bf16", "bf16"), ("f16", "fp8"), ("f32", "int8")], ids=["bf16", "fp8", "f32-int8"])
def test_not_causal(qt, kv):
    _say(f"chunk not causal {qt} over {kv}")
    _check(qt, kv, [40, 150, 1], [300, 0, 90], 6, 2, 128, 16, seed=3, causal=False)


@pytest.mark.parametrize("qt,kv", [("bf16", "bf16"), ("bf16", "int8"), ("f32", "f16")], ids=["bf16", "int8", "f32"])
def test_absent_pages_and_empty_rows(qt, kv):
    """Absent pages (-1, and past the pool) are skipped; a sequence whose
    pages are all absent, and rows before a context's start, give zeros."""
    _say(f"chunk absent pages {qt} over {kv}")
    drop = [(0, 0), (0, 3), (1, 0), (1, 1), (1, 2), (2, 1)]
    _check(qt, kv, [20, 30, 5], [60, 10, 30], 6, 2, 64, 16, seed=11, drop=drop)
    # context shorter than the chunk: the first rows are at negative positions
    gen, P, table, lens, cu = _batch([20, 6], [0, 3], 16, 12)
    pool, scales, vals = make_pool(kv, P, 1, 2, 16, 64, gen)
    lens = torch.tensor([7, 0], dtype=torch.int32)
    q = torch.randn((26, 6, 64), generator=gen).to(FLOAT[qt])
    gp, gs = to_gpu(pool, scales)
    out = paged_attention_chunk(q.to(DEV), gp, table.to(DEV), lens.to(DEV), cu.to(DEV), 0, kv_scales=gs).cpu()
    want, _, reach = attend(q, vals, table, lens, cu, 0)
    assert (out[:13] == 0).all() and (out[20:] == 0).all()
    tol = _tolerance(want, reach, q.dtype, qt == "f32", 64, kv == "int8")
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("qt,kv,D,PS", [("bf16", "bf16", 1, 16), ("f16", "f16", 30, 5), ("f32", "f32", 33, 3),
                                        ("bf16", "bf16", 72, 1), ("f16", "f16", 250, 7), ("bf16", "int8", 16, 4),
                                        ("f16", "fp8", 48, 12), ("bf16", "fp8", 144, 20), ("f32", "f16", 100, 40)])
def test_odd_head_dims_and_pages(qt, kv, D, PS):
    _say(f"chunk {qt} over {kv} D={D} PS={PS}")
    _check(qt, kv, [33, 1, 18], [50, 31, 0], 6, 2, D, PS, seed=D + PS)


@pytest.mark.parametrize("layout", ["plain", "inline"])
@pytest.mark.parametrize("kv", ["int8", "fp8"])
def test_pool_layouts(kv, layout):
    _say(f"chunk over {kv} {layout}")
    _check("bf16", kv, [33, 1, 70], [100, 47, 0], 10, 2, 128, 16, seed=5, layout=layout)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scale(scale):
    _say(f"chunk scale {scale}")
    _check("bf16", "bf16", [33, 5], [100, 47], 6, 2, 64, 16, seed=6, scale=scale, q_std=0.5)
    _check("f32", "f32", [33, 5], [100, 47], 6, 2, 64, 16, seed=6, scale=scale, q_std=0.5)


@pytest.mark.parametrize("window", [None, 30])
@pytest.mark.parametrize("qt,kv,D", [("bf16", "bf16", 64), ("f16", "f16", 128), ("f32", "f32", 64), ("bf16", "int8", 64),
                                     ("bf16", "fp8", 128), ("f16", "fp8", 64), ("f32", "fp8", 64), ("bf16", "f16", 64),
                                     ("f16", "f16", 256)])
@pytest.mark.parametrize("q_lens,past", [([40, 3], [70, 130]), ([200], [0]), ([4], [90])])
def test_values_that_are_not_finite(qt, kv, D, q_lens, past, window):
    """Infinities and NaN among keys and values that a row does not see (later
    tokens of its own chunk, tokens before its window) have no part in it; rows
    that see them get what the definition gives."""
    _say(f"not finite {qt} over {kv} D={D} q={q_lens} window={window}")
    gen, P, table, lens, cu = _batch(q_lens, past, 16, 31)
    pool, scales, vals = make_pool(kv, P, 1, 2, 16, D, gen)
    for b, (n, p) in enumerate(zip(q_lens, past)):
        # one token inside the chunk, one before it; the rest of the last page
        for t, x in ((p + n // 2, math.inf), (max(0, p - 20), math.nan)):
            pid, slot = int(table[b, t // 16]), t % 16
            vals[pid, 0, 1, 1, slot, 5] = x
            if kv in FLOAT:
                pool[pid, 0, 1, 1, slot, 5] = x
                pool[pid, 0, 0, 0, slot, 3] = x
                vals[pid, 0, 0, 0, slot, 3] = x
            elif kv == "int8":
                scales[pid, 0, 1, 1, slot] = x
                vals[pid, 0, 1, 1, slot] = pool_codes(pool, pid, slot).double() * x
            else:
                at = ((slot // 4 * 16 + 5) * (D // 16) + 0) * 4 + slot % 4
                pool.view(torch.uint8)[pid, 0, 1, 1].view(-1)[at] = 0x7f
                vals[pid, 0, 1, 1, slot, 5] = math.nan
        end = p + n
        if end % 16 and kv in FLOAT:
            pool[int(table[b, end // 16]), 0, :, :, end % 16:] = math.nan
    q = (torch.randn((int(cu[-1]), 6, D), generator=gen)).to(FLOAT[qt])
    gp, gs = to_gpu(pool, scales)
    got = paged_attention_chunk(q.to(DEV), gp, table.to(DEV), lens.to(DEV), cu.to(DEV), 0, kv_scales=gs,
                                window=window).cpu().double()
    want, _, reach = attend(q, vals, table, lens, cu, 0, window=window)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    wide = qt == "f32" or kv == "f32" or (kv in FLOAT and kv != qt)
    tol = _tolerance(want, reach, q.dtype, wide, D, kv not in FLOAT)
    assert ((got - want).abs() <= tol)[fine].all()
    assert fine.any() and not fine.all()


def pool_codes(pool, pid, slot):
    """int8 codes of V, kv-head 1, of a token of a stored pool."""
    D = pool.shape[-1]
    d = torch.arange(D)
    at = ((slot // 4 * 16 + d % 16) * (D // 16) + d // 16) * 4 + slot % 4
    return pool[pid, 0, 1, 1].reshape(-1)[at]


@pytest.mark.parametrize("t,D", [("bf16", 128), ("f16", 80), ("f32", 64)])
@pytest.mark.parametrize("q_lens", [[3, 1], [150, 20]], ids=["few", "many"])
def test_strides_and_alignment(t, D, q_lens):
    """Queries that are slices of a projection, rows and pools that start off
    16 bytes, outputs that do: the same bits as from dense, aligned ones."""
    _say(f"chunk strides {t} D={D} q={q_lens}")
    H, KH = 6, 2
    gen, P, table, lens, cu = _batch(q_lens, [70, 300], 16, 41)
    pool, _, _ = make_pool(t, P, 1, KH, 16, D, gen)
    pool, batch = pool.to(DEV), (table.to(DEV), lens.to(DEV), cu.to(DEV), 0)
    N = int(cu[-1])
    proj = torch.randn((N, (H + 2 * KH) * D + 1), generator=gen).to(FLOAT[t]).to(DEV)
    sliced = proj[:, 1:1 + H * D].view(N, H, D)
    want = paged_attention_chunk(sliced.contiguous(), pool, *batch)
    assert torch.equal(paged_attention_chunk(sliced, pool, *batch), want)
    turned = sliced.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged_attention_chunk(turned, pool, *batch), want)
    last = sliced.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(paged_attention_chunk(last, pool, *batch), want)
    odd_pool = torch.empty(pool.numel() + 1, dtype=pool.dtype, device=DEV)[1:].view(pool.shape).copy_(pool)
    assert torch.equal(paged_attention_chunk(sliced, odd_pool, *batch), want)
    out = torch.empty(want.numel() + 1, dtype=want.dtype, device=DEV)[1:].view(want.shape)
    assert torch.equal(paged_attention_chunk(sliced, pool, *batch, out=out), want)


@pytest.mark.parametrize("kv,page_bytes", [("bf16", 2 * 8 * 16 * 128 * 2), ("int8", 2 * 8 * 16 * 128)])
@pytest.mark.parametrize("q_lens", [[4, 1], [90, 40]], ids=["few", "many"])
def test_pool_past_32_bits(kv, page_bytes, q_lens):
    """Pages past 4 GiB of a pool give what the same pages give in a small one."""
    _say(f"chunk pool past 32 bits {kv} q={q_lens}")
    gen, P, table, lens, cu = _batch(q_lens, [100, 37], 16, 42)
    pool, scales, _ = make_pool(kv, P, 1, 8, 16, 128, gen, None if kv == "bf16" else "plain")
    pool = pool.to(DEV)
    scales = None if scales is None else scales.to(DEV)
    far = (1 << 32) // page_bytes + 3
    big = torch.empty((far + P, *pool.shape[1:]), dtype=pool.dtype, device=DEV)
    big[far:] = pool
    big_scales = None
    if scales is not None:
        big_scales = torch.zeros((far + P, *scales.shape[1:]), device=DEV)
        big_scales[far:] = scales
    q = torch.randn((int(cu[-1]), 16, 128), generator=gen).to(torch.bfloat16).to(DEV)
    far_table = torch.where(table >= 0, table + far, table).to(torch.int32)
    want = paged_attention_chunk(q, pool, table.to(DEV), lens.to(DEV), cu.to(DEV), 0, kv_scales=scales)
    got = paged_attention_chunk(q, big, far_table.to(DEV), lens.to(DEV), cu.to(DEV), 0, kv_scales=big_scales)
    assert torch.equal(got, want) and (want != 0).any()


def test_no_pages_and_no_tokens():
    _say("chunk without pages")
    pool = torch.zeros((2, 1, 2, 2, 16, 64), dtype=torch.bfloat16, device=DEV)
    q = torch.ones((5, 4, 64), dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    table = torch.empty((1, 0), dtype=torch.int32, device=DEV)
    for n in (0, 5):
        out = paged_attention_chunk(q, pool, table, torch.tensor([n], dtype=torch.int32, device=DEV), cu, 0)
        assert (out == 0).all()
    assert paged_attention_chunk(q[:0], pool, table, cu[:1], cu, 0).shape == (0, 4, 64)
