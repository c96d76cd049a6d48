"""qk_norm_rope and rope_append against float64.

Tolerances.  A row's norm and rotation are a few float32 operations and a sum
of at most 256 squares in a tree over lanes: at most 24 roundings in a chain,
24 x 2^-24 of the pair's size, written 2^-19 with room for the square root and
the division.  The result is rounded once: half a step u relative, or 2^-25
for an fp16 value below 2^-14.
int8: the scale is amax / 127 within those float32 errors; a value is off by
half a step of its code.  e4m3: half a step is 2^-4 of a normal code, 2^-10 of
the scale below 2^-6 of it; re-encoded codes are rounded once more.
"""
import pytest
import torch

from chunk_reference import FLOAT, HALF, make_pool, make_table, norm_rope, rope_angles, to_gpu
from vramancer_amd import kv_quant
from vramancer_amd.paged_chunk import rope_append
from vramancer_amd.rope import qk_norm_rope, rope_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = 2.0 ** -19


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _close(got, want, size, what):
    u = HALF[got.dtype]
    got = got.cpu().double()
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 1e-30
    assert torch.equal(got.isnan(), want.isnan()), what
    err = (got - want).abs().nan_to_num(0)
    tol = (u * want.abs() + F32 * size + tiny).nan_to_num(1)
    assert (err <= tol).all(), f"{what}: worst {float((err / tol).max()):.2f} tolerances"


def _gpu(t):
    return None if t is None else t.to(DEV)


def test_table():
    got = rope_table(2000, 64, base=500000.0, attention_scaling=0.5, device="cpu")
    want = rope_angles(2000, 64, 500000.0) * 0.5
    assert got.dtype == torch.float32 and (got - want).abs().max() <= 2.0 ** -24
    freq = torch.rand(16)
    assert torch.equal(rope_table(9, 32, inv_freq=freq, device=DEV).cpu()[:, :16],
                       torch.cos(torch.arange(9.0, dtype=torch.float64)[:, None] * freq.double()).float())


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,rot,inter,norm,N,H,KH", [
    (128, 128, False, True, 37, 10, 2), (128, 64, False, True, 5, 7, 1), (64, 64, True, False, 129, 4, 4),
    (64, 32, True, True, 1, 3, 1), (96, 96, False, True, 18, 6, 2), (80, 16, False, False, 9, 5, 5),
    (256, 256, False, True, 7, 3, 1), (256, 128, True, True, 7, 3, 1), (16, 16, False, True, 300, 2, 1),
    (30, 20, False, True, 11, 3, 1), (33, 32, True, True, 11, 3, 2), (1, 0, False, True, 4, 2, 1),
    (250, 100, False, True, 3, 2, 2), (128, 0, False, True, 20, 4, 2)])
def test_norm_and_rotation(t, D, rot, inter, norm, N, H, KH):
    _say(f"norm rope {t} D={D} rot={rot} interleaved={inter} norm={norm} N={N}")
    gen = torch.Generator().manual_seed(D + rot + N)
    qkv = (torch.randn((N, H + 2 * KH, D), generator=gen) * 2).to(FLOAT[t])
    q, k = qkv[:, :H], qkv[:, H:H + KH]
    qw, kw = ((torch.randn(D, generator=gen).to(FLOAT[t]) for _ in range(2)) if norm else (None, None))
    table = rope_angles(500, rot) if rot else None
    pos = torch.randint(0, 500, (N,), generator=gen)
    g = qkv.to(DEV)
    gq, gk = g[:, :H], g[:, H:H + KH]
    got = qk_norm_rope(gq, gk, _gpu(table), pos.to(DEV) if rot else None, _gpu(qw), _gpu(kw), 1e-5, inter)
    for x, w, y, name in ((q, qw, got[0], "query"), (k, kw, got[1], "key")):
        want, size = norm_rope(x, w, table, pos, 1e-5, inter)
        _close(y, want, size, name)
    # in place, one weight of another type, 32-bit positions
    a, b = gq.contiguous(), gk.contiguous()
    w32 = None if qw is None else qw.float().to(DEV)
    got2 = qk_norm_rope(a, b, _gpu(table), pos.to(DEV, torch.int32) if rot else None, w32, None, 1e-5, inter,
                        query_out=a, key_out=b)
    assert got2[0] is a and torch.equal(a, got[0])
    _close(b, *norm_rope(k, None, table, pos, 1e-5, inter), "key in place")


def test_positions_outside_the_table_and_alignment():
    """Rows at positions outside the table are NaN; rows that start off 16
    bytes, or whose strides do, give the same values."""
    _say("norm rope outside the table, unaligned")
    gen = torch.Generator().manual_seed(1)
    q, k = torch.randn((6, 3, 64), generator=gen).half(), torch.randn((6, 2, 64), generator=gen).half()
    w = torch.randn(64, generator=gen)
    table = rope_angles(10, 64)
    pos = torch.tensor([0, 9, 10, -1, 5, 1 << 40])
    got = qk_norm_rope(q.to(DEV), k.to(DEV), table.to(DEV), pos.to(DEV), w.to(DEV), w.to(DEV))
    for x, y in ((q, got[0]), (k, got[1])):
        _close(y, *norm_rope(x, w, table, pos, 1e-6, False), "rows")
        assert y[[2, 3, 5]].isnan().all()
    raw = torch.empty((6, 3 * 65 + 1), dtype=torch.float16, device=DEV)
    odd = raw[:, 1:].unflatten(1, (3, 65))[..., :64]
    odd.copy_(q)
    got3 = qk_norm_rope(odd, k.to(DEV), table.to(DEV), pos.to(DEV), w.to(DEV), w.to(DEV))
    _close(got3[0], *norm_rope(q, w, table, pos, 1e-6, False), "unaligned")


def _append(t, kv, q_lens, past, H, KH, D, PS, rot, norm, inter, seed, layout=None, tail=0, drop=(), positions=None,
            with_q=True, top=None):
    gen = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(q_lens, past)]
    P, table = make_table(lens, PS, gen)
    for b, i in drop:
        table[b, i] = -1 if i % 2 else P
    L, layer = 2, 1
    pool, scales, vals = make_pool(kv, P, L, KH, PS, D, gen, layout)
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    n, N = int(cu[-1]), int(cu[-1]) + tail
    qkv = (torch.randn((N, H + 2 * KH, D), generator=gen) * 1.5).to(FLOAT[t])
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=gen) for _ in range(2)) if norm else (None, None))
    angles = rope_angles(top or max(lens) + 1, rot) if rot else None
    own = torch.cat([torch.arange(p, p + a) for a, p in zip(q_lens, past)])
    pos = own if positions is None else positions
    gp, gs = to_gpu(pool, scales)
    g = qkv.to(DEV)
    out = torch.full((N, H, D), 7.0, dtype=FLOAT[t], device=DEV)
    got = rope_append(g[:, :H] if with_q else None, g[:, H:H + KH], g[:, H + KH:], gp, table.to(DEV),
                      torch.tensor(lens, dtype=torch.int32, device=DEV), cu.to(DEV), layer, _gpu(angles), kv_scales=gs,
                      positions=None if positions is None else torch.cat([positions, torch.zeros(tail)]).long().to(DEV),
                      q_weight=_gpu(qw) if with_q else None, k_weight=_gpu(kw), eps=1e-6, interleaved=inter,
                      query_out=out if with_q else None)
    torch.cuda.synchronize()
    if with_q:
        assert got is out and (out[n:] == 7).all()
        _close(out[:n], *norm_rope(qkv[:n, :H], qw, angles, pos, 1e-6, inter), "query")
    else:
        assert got is None
    k, k_size = norm_rope(qkv[:n, H:H + KH], kw, angles, pos, 1e-6, inter)
    v = qkv[:n, H + KH:].double()
    written = torch.zeros((P, PS), dtype=torch.bool)
    rows = {}
    # a page's earlier tokens end at its first new one, whether that is dropped
    # (its slot then holds no token: what was there before the call was none)
    entered = {}
    for b, (a, p) in enumerate(zip(q_lens, past)):
        for i in range(a):
            pid = int(table[b, (p + i) // PS])
            r = int(cu[b]) + i
            entered.setdefault(pid, (p + i) % PS)
            if 0 <= pid < P and (not rot or 0 <= int(pos[r]) < angles.shape[0]):
                written[pid, (p + i) % PS] = True
                rows[pid, (p + i) % PS] = r
    where = list(rows)
    ids, slots = (torch.tensor([w[j] for w in where], dtype=torch.long) for j in (0, 1))
    src = torch.tensor([rows[w] for w in where], dtype=torch.long)
    if kv in FLOAT:
        after = gp.cpu()
        for j, (x, size) in enumerate(((k, k_size), (v, v.abs()))):
            if where:
                _close(after[ids, layer, j, :, slots], x[src], size[src], "K" if j == 0 else "V")
        after[ids, layer, :, :, slots] = pool[ids, layer, :, :, slots]
        assert torch.equal(after, pool), "other rows of the pool changed"
        return
    every = torch.arange(P, dtype=torch.int32, device=DEV)
    deq = kv_quant.dequantize_pages(gp, gs, layer, every).cpu().double()
    other = kv_quant.dequantize_pages(gp, gs, 0, every).cpu().double()
    assert (other - vals[:, 0]).abs().max() <= 2.0 ** -22 * vals.abs().max(), "another layer changed"
    sc = gs.cpu().double()[:, layer]
    old_sc = scales.double()[:, layer]
    old = vals[:, layer]
    for j, (x, size) in enumerate(((k, k_size), (v, v.abs()))):
        x, size = x[src], size[src]  # [M, KH, D]
        room = F32 * size.amax(-1, keepdim=True)
        if kv == "int8":
            s = sc[ids, j, :, slots]
            assert ((s - x.abs().amax(-1) / 127).abs() <= F32 * size.amax(-1) / 64).all(), "scales"
            assert ((deq[ids, j, :, slots] - x).abs() <= s[..., None] * (0.5 + 2e-4) + room).all(), "codes"
            keep = ~written[:, None, :, None].expand(P, old.shape[2], PS, D)
            assert ((deq[:, j] - old[:, j]).abs()[keep] <= 2.0 ** -22 * old.abs().max()).all(), "other rows"
            continue
        want_s = old_sc[:, j].clone()  # [P, KH]
        for pid in set(int(i) for i in ids):
            mine = ids == pid
            big = x[mine].abs().amax((0, 2)) / 448
            want_s[pid] = big if entered[pid] == 0 else torch.maximum(big, old_sc[pid, j])
        assert ((sc[:, j] - want_s).abs() <= 2.0 ** -18 * (want_s + 1e-3)).all(), "page scales"
        step = lambda y, s: torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * s) * (1 + 2.0 ** -12)  # noqa: E731
        assert ((deq[ids, j, :, slots] - x).abs() <= step(x, sc[ids, j][..., None]) + room).all(), "codes"
        for pid in range(P):
            first = entered.get(pid, PS)
            grown = (sc[pid, j] > old_sc[pid, j])[:, None, None]
            a, b = deq[pid, j, :, :first], old[pid, j, :, :first]
            tol = torch.where(grown, step(b, sc[pid, j][:, None, None]), 2.0 ** -20 * b.abs())
            assert ((a - b).abs() <= tol).all(), "earlier tokens of a page"


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16", "int8", "fp8"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_lens,past,H,KH,D,PS,rot,norm,inter", [
    ([33, 1, 20], [100, 47, 0], 10, 2, 128, 16, 128, True, False),
    ([1] * 9, list(range(9, 18)), 4, 4, 64, 16, 64, False, False),
    ([0, 40, 0, 3], [5, 30, 0, 16], 3, 1, 80, 32, 32, True, True),
    ([5], [0], 2, 2, 256, 4, 256, True, False)])
def test_append(t, kv, q_lens, past, H, KH, D, PS, rot, norm, inter):
    _say(f"append {t} into {kv} q={q_lens[:4]} D={D} PS={PS}")
    _append(t, kv, q_lens, past, H, KH, D, PS, rot, norm, inter, seed=D + PS, tail=3)


@pytest.mark.parametrize("t,kv,D,PS,rot", [("bf16", "bf16", 30, 5, 20), ("f16", "f16", 33, 3, 32), ("f32", "f16", 1, 1, 0),
                                           ("bf16", "int8", 48, 12, 20), ("f32", "fp8", 16, 20, 10),
                                           ("f16", "fp8", 144, 40, 144), ("bf16", "int8", 240, 24, 0),
                                           ("f16", "fp8", 64, 64, 64)])
def test_append_odd_sizes(t, kv, D, PS, rot):
    _say(f"append {t} into {kv} D={D} PS={PS} rot={rot}")
    _append(t, kv, [70, 1, 5], [7, 3, 0], 3, 2, D, PS, rot, True, False, seed=D)


@pytest.mark.parametrize("layout", ["plain", "inline"])
@pytest.mark.parametrize("kv", ["int8", "fp8"])
def test_append_layouts(kv, layout):
    _say(f"append into {kv} {layout}")
    _append("bf16", kv, [33, 1, 20], [100, 47, 0], 10, 2, 128, 16, 128, True, False, seed=2, layout=layout)


@pytest.mark.parametrize("kv", ["f16", "int8", "fp8"])
def test_append_drops_and_positions(kv):
    _say(f"append into {kv}: absent pages, positions, no query")
    _append("f16", kv, [40, 9], [20, 5], 3, 2, 64, 16, 64, True, False, seed=3, drop=[(0, 2), (1, 0)], tail=1)
    _append("f16", kv, [40, 9], [20, 5], 3, 2, 64, 16, 64, True, False, seed=4, with_q=False)
    pos = torch.arange(49) * 3
    pos[[0, 7, 41]] = torch.tensor([-1, 200, 500])
    _append("f16", kv, [40, 9], [20, 5], 3, 2, 64, 16, 64, False, True, seed=5, positions=pos, tail=2, top=150)


def test_append_matches_quantize_append():
    """Single tokens without norm or rotation: the pools that
    kv_quant.quantize_append leaves, bit for bit."""
    _say("append of single tokens vs quantize_append")
    for codec in ("int8", "fp8"):
        gen = torch.Generator().manual_seed(8)
        B, KH, D, PS = 5, 2, 128, 16
        lens = [1, 16, 17, 40, 64]
        P, table = make_table(lens, PS, gen)
        pool, scales, _ = make_pool(codec, P, 1, KH, PS, D, gen)
        k, v = (torch.randn((B, KH, D), generator=gen).bfloat16().to(DEV) for _ in range(2))
        a, b = to_gpu(pool, scales), to_gpu(pool, scales)
        pos = torch.tensor(lens) - 1
        pid = table[torch.arange(B), pos // PS]
        kv_quant.quantize_append(*a, 0, pid.to(DEV), (pos % PS).to(DEV), k, v)
        rope_append(None, k, v, b[0], table.to(DEV), torch.tensor(lens, device=DEV),
                    torch.arange(B + 1, device=DEV), 0, kv_scales=b[1])
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)), codec
        assert torch.equal(a[1], b[1]), codec


@pytest.mark.parametrize("D,rot", [(128, 128), (80, 32), (30, 10)])
def test_in_place(D, rot):
    _say(f"rotation in place D={D} rot={rot}")
    gen = torch.Generator().manual_seed(D)
    q, k = (torch.randn((37, h, D), generator=gen).to(torch.bfloat16).to(DEV) for h in (9, 3))
    w = torch.randn(D, generator=gen).to(DEV)
    pos = torch.randint(0, 50, (37,), generator=gen).to(DEV)
    table = rope_table(50, rot, device=DEV)
    want = qk_norm_rope(q, k, table, pos, w, w)
    got = qk_norm_rope(q, k, table, pos, w, w, query_out=q, key_out=k)
    assert got[0] is q and got[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp8"])
def test_append_past_32_bits(kv):
    """Pages past 4 GiB of a pool take what the same pages of a small one do."""
    _say(f"append past 32 bits {kv}")
    gen = torch.Generator().manual_seed(3)
    lens = [70, 33]
    P, table = make_table(lens, 16, gen)
    pool, scales, _ = make_pool(kv, P, 1, 8, 16, 128, gen, None if kv == "bf16" else "plain")
    pool, scales = pool.to(DEV), _gpu(scales)
    far = (1 << 32) // (2 * 8 * 16 * 128 * pool.element_size()) + 3
    big = torch.empty((far + P, *pool.shape[1:]), dtype=pool.dtype, device=DEV)
    big[far:] = pool
    big_scales = None
    if scales is not None:
        big_scales = torch.zeros((far + P, *scales.shape[1:]), device=DEV)
        big_scales[far:] = scales
    k, v = (torch.randn((43, 8, 128), generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    batch = (torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor([0, 40, 43], dtype=torch.int32, device=DEV), 0)
    rope_append(None, k, v, pool, table.to(DEV), *batch, kv_scales=scales)
    rope_append(None, k, v, big, torch.where(table >= 0, table + far, table).to(torch.int32).to(DEV), *batch,
                kv_scales=big_scales)
    assert torch.equal(big[far:].view(torch.uint8), pool.view(torch.uint8))
    assert scales is None or torch.equal(big_scales[far:], scales)
