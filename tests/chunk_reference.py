"""Plain forms in 64 bits of the operators over a chunk of new tokens, on the
CPU, and the batches that their tests share."""
import math

import torch

from oracle import kv_codecs

FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of rounding to each type, relative
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make_table(lens, PS, gen, spare=3):
    """Shuffled pages for sequences of these lengths: (P, table [B, width])."""
    pages = [max(0, -(-n // PS)) for n in lens]
    P = sum(pages) + spare
    perm = torch.randperm(P, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(1, max(pages, default=1)) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return P, table


def make_pool(kind, P, L, KH, PS, D, gen, layout=None):
    """(pool, scales, values): a filled pool on the CPU in its stored layout,
    and the float64 values [P, L, 2, KH, PS, D] it stands for."""
    x = torch.randn((P, L, 2, KH, PS, D), generator=gen)
    if kind in FLOAT:
        pool = x.to(FLOAT[kind])
        return pool, None, pool.double()
    from vramancer_amd import kv_quant

    pool, scales = kv_quant.allocate_pool(P, L, KH, D, {"int8": "int8", "fp8": "fp8"}[kind], PS, "cpu", layout=layout)
    if kind == "int8":
        s = x.abs().amax(-1) / 127
        codes = torch.round(x / s[..., None]).to(torch.int8)
        vals = codes.double() * s.double()[..., None]
    else:
        s = x.abs().amax((-1, -2)) / 448
        codes = (x / s[..., None, None]).to(torch.float8_e4m3fn)
        vals = codes.double() * s.double()[..., None, None]
    raw, cr = pool.view(torch.uint8), codes.view(torch.uint8)
    raw[:, :, 0] = cr[:, :, 0]
    raw[:, :, 1] = tile_v(cr[:, :, 1])
    scales.copy_(s)
    return pool, scales, vals


def tile_v(v):
    """Token-major V slices [.., PS, D] as the quantized pools store them."""
    *lead, PS, D = v.shape
    return v.reshape(*lead, PS // 4, 4, D // 16, 16).transpose(-1, -3).reshape(v.shape)


def to_gpu(pool, scales, dev="cuda:0"):
    """The pair on the GPU in the same layout (inline pairs share a buffer)."""
    if scales is None:
        return pool.to(dev), None
    if pool.is_contiguous():
        return pool.to(dev), scales.to(dev)
    buf = pool.untyped_storage()
    raw = torch.empty(0, dtype=torch.uint8).set_(buf).to(dev)
    return (raw.view(pool.dtype).as_strided(pool.shape, pool.stride()),
            raw.view(torch.float32).as_strided(scales.shape, scales.stride(), storage_offset=scales.storage_offset()))


def attend(q, vals, table, lens, cu, layer, scale=None, causal=True, window=None):
    """(out, lse, reach): float64 attention by the definition, row by row, and
    per row and head sum_t p_t |v_t|, the size its rounding errors go by."""
    N, H, D = q.shape
    P, _, _, KH, PS, _ = vals.shape
    G = H // KH
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros((N, H, D), dtype=torch.float64)
    reach = torch.zeros((N, H, D), dtype=torch.float64)
    lse = torch.full((N, H), -math.inf, dtype=torch.float64)
    for b in range(len(lens)):
        r0, r1, ctx = int(cu[b]), int(cu[b + 1]), min(int(lens[b]), table.shape[1] * PS)
        if r1 <= r0:
            continue
        pages = [(int(table[b, t // PS]), t % PS) for t in range(max(ctx, 0))]
        there = torch.tensor([0 <= p < P for p, _ in pages], dtype=torch.bool)
        ids = torch.tensor([max(0, min(P - 1, p)) for p, _ in pages], dtype=torch.long)
        slots = torch.tensor([s for _, s in pages], dtype=torch.long)
        k, v = vals[ids, layer, 0, :, slots], vals[ids, layer, 1, :, slots]  # [ctx, KH, D]
        pos = int(lens[b]) - (r1 - r0) + torch.arange(r1 - r0)
        t = torch.arange(max(ctx, 0))
        see = there[None].expand(r1 - r0, -1).clone()
        if causal:
            see &= t[None] <= pos[:, None]
        if window:
            see &= t[None] > pos[:, None] - window
        for h in range(H):
            any_ = see.any(1)
            if not any_.any():
                continue
            s = q[r0:r1, h].double() @ k[:, h // G].T * scale
            s = s.masked_fill(~see, -math.inf)[any_]
            rows = torch.arange(r0, r1)[any_]
            p = torch.softmax(s, -1)
            vz = v[:, h // G]
            if vz.isfinite().all():
                out[rows, h] = p @ vz
                reach[rows, h] = p @ vz.abs()
            else:  # a token that a row does not see has no part in it, whatever it holds
                part = torch.where(see[any_][:, :, None], p[:, :, None] * vz[None], 0.0)
                out[rows, h] = part.sum(1)
                reach[rows, h] = part.abs().sum(1)
            lse[rows, h] = torch.logsumexp(s, -1)
    return out, lse, reach


def rope_angles(top, rot, base=10000.0):
    """[top, rot] float32 as rope_table computes it, from its definition."""
    freq = torch.tensor([base ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    a = torch.arange(top, dtype=torch.float64)[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def norm_rope(x, w, table, positions, eps, interleaved):
    """(y, size): float64 norm and rotation of [N, heads, D] rows, and the
    magnitude that each element's float32 rounding errors go by."""
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = y.abs().clone()
    out = y.clone()
    if table is not None:
        rot = table.shape[1]
        half = rot // 2
        a = torch.arange(half) * (2 if interleaved else 1)
        b = a + (1 if interleaved else half)
        known = (positions >= 0) & (positions < table.shape[0])
        cs = table[positions.clamp(0, table.shape[0] - 1).long()].double()[:, None]
        c, s = cs[..., :half], cs[..., half:]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., b] * c + y[..., a] * s
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
        out[~known] = math.nan
    return out, size
