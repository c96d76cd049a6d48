"""Operators between a prompt and the decode, timed one call at a time: how a
chunk of new tokens enters a paged cache and attends it.

``kind`` names the call:

  rotate   rope.qk_norm_rope: RMS norm of every query and key head and the
           rotation by position, in one pass
  append   paged_chunk.rope_append: the same with the new tokens' keys and
           values written into their pages (float, int8 or fp8 pools)
  attend   paged_chunk.paged_attention_chunk: attention of each sequence's
           new tokens over its pages, causal, in some cases within a window

The batch is ragged: sequence b has ``q_b`` new tokens after ``past_b`` tokens
in its pages.  Of ``B`` sequences the last ``ones`` have one new token, the
others between ``qlo`` and ``qhi``; pasts lie between ``plo`` and ``phi``.
``lens_seed`` draws both; values and page tables follow the seed given to
``prepare``.

Where ``own`` is false ``run`` computes the plain forms: elementary torch
operations in float32 over padded batches, rounded once at the end.
"""
import math
import random

import torch

own = False

DEVICE = "cuda:0"
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "int8": 1, "fp8": 1}
EPS = 1e-6


def listed():
    return [
        # queries and keys of a decode batch of 16 requests, small heads: latency
        dict(name="rotate-step", kind="rotate", N=16, H=16, KH=8, D=64, rot=64, t="f16", norm=True, inter=False,
             top=8192),
        # queries and keys of four prompts of about 2000 tokens, 14B heads
        dict(name="rotate-prompts", kind="rotate", N=8011, H=40, KH=8, D=128, rot=128, t="bf16", norm=True,
             inter=False, top=131072),
        # one new token for each of 32 requests, 7B heads, bf16 cache: latency
        dict(name="append-step", kind="append", t="bf16", kv="bf16", H=28, KH=4, D=128, PS=16, B=32, ones=32,
             qlo=1, qhi=1, plo=1024, phi=8192, rot=128, norm=False, inter=False, lens_seed=0),
        # prompts entering the int8 cache of a 14B model, with q / k norms
        dict(name="append-int8", kind="append", t="bf16", kv="int8", H=40, KH=8, D=128, PS=16, B=4, ones=0,
             qlo=1800, qhi=2200, plo=0, phi=300, rot=128, norm=True, inter=False, lens_seed=1),
        # a mixed batch entering an fp8 cache: chunks of prompts beside single
        # tokens; half of each head rotated, in adjacent pairs
        dict(name="append-fp8", kind="append", t="f16", kv="fp8", H=64, KH=8, D=128, PS=16, B=40, ones=36,
             qlo=200, qhi=700, plo=0, phi=1000, rot=64, norm=False, inter=True, lens_seed=2),
        # the follow-up question of one chat over its f16 cache: latency
        dict(name="attend-chat", kind="attend", t="f16", kv="f16", H=28, KH=4, D=128, PS=16, B=1, ones=0,
             qlo=17, qhi=17, plo=1531, phi=1531, window=0, lens_seed=0),
        # a 14B batch verifying four drafted tokens per request: cache bound
        dict(name="attend-verify", kind="attend", t="bf16", kv="int8", H=40, KH=8, D=128, PS=16, B=64, ones=0,
             qlo=4, qhi=4, plo=4000, phi=4092, window=0, lens_seed=0),
        # a long prompt of a 7B model in one chunk: matrix bound
        dict(name="attend-prompt", kind="attend", t="bf16", kv="bf16", H=28, KH=4, D=128, PS=16, B=1, ones=0,
             qlo=8192, qhi=8192, plo=0, phi=0, window=0, lens_seed=0),
        # one chunk deep in a long document, fp8 cache
        dict(name="attend-document", kind="attend", t="bf16", kv="fp8", H=64, KH=8, D=128, PS=16, B=1, ones=0,
             qlo=256, qhi=256, plo=130816, phi=130816, window=0, lens_seed=0),
        # a continuous batch: one prompt's chunk beside decoding requests
        dict(name="attend-mixed", kind="attend", t="bf16", kv="bf16", H=28, KH=4, D=128, PS=16, B=16, ones=15,
             qlo=509, qhi=509, plo=200, phi=4000, window=0, lens_seed=3),
        # two prompts of odd lengths within a window, head_dim 96
        dict(name="attend-window", kind="attend", t="f16", kv="f16", H=32, KH=8, D=96, PS=16, B=2, ones=0,
             qlo=1500, qhi=2100, plo=300, phi=900, window=1000, lens_seed=4),
        # float32 throughout, heads of 64, no grouping
        dict(name="attend-f32", kind="attend", t="f32", kv="f32", H=12, KH=12, D=64, PS=16, B=4, ones=0,
             qlo=100, qhi=160, plo=200, phi=512, window=0, lens_seed=5),
    ]


# ---------------------------------------------------------------------------
# Drawn cases
# ---------------------------------------------------------------------------

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(40, 8), (28, 4), (64, 8), (32, 8), (16, 8), (12, 12), (20, 4)]


def draw(rng):
    kind = rng.choices(["attend", "append", "rotate"], [5, 3, 2])[0]
    H, KH = rng.choice(HEADS)
    D = rng.choice([64, 80, 96, 128, 128, 128, 256])
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    rot = rng.choice([D, D, D, D // 2])
    if kind == "rotate":
        return dict(kind=kind, N=_log_int(rng, 1, 8000), H=H, KH=KH, D=D if H * D < 10000 else 64,
                    rot=rot if H * D < 10000 else 64, t=t, norm=rng.random() < 0.6, inter=rng.random() < 0.25,
                    top=rng.choice([4096, 32768, 131072]))
    case = dict(kind=kind, t=t, kv=rng.choice([t, t, "int8", "fp8"]), H=H, KH=KH, D=D, PS=rng.choice([16, 16, 16, 32]),
                lens_seed=rng.randrange(1 << 30))
    if kind == "append":
        case["B"] = B = _log_int(rng, 1, 64)
        case["qhi"] = hi = _log_int(rng, 1, min(2200, 8000 // B))
        case["phi"] = _log_int(rng, 1, 2000)
        case.update(rot=rot, norm=rng.random() < 0.5, inter=rng.random() < 0.25)
    else:
        case["B"] = B = _log_int(rng, 1, 64)
        # the padded scores of the plain form, and the bytes of queries and cache
        case["qhi"] = hi = _log_int(rng, 1, max(1, min(4096, 60_000_000 // (B * H * D * BYTES[t]))))
        top = min(1_000_000_000 // (B * H * hi), 400_000_000 // (B * KH * (2 * D * BYTES[case["kv"]] + 8)), 100_000)
        case["phi"] = _log_int(rng, 16, max(17, top - hi))
        case["window"] = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    case["qlo"] = max(1, hi // rng.choice([1, 2, 4]))
    case["plo"] = case["phi"] // rng.choice([1, 2, 8])
    case["ones"] = rng.choice([0, 0, B // 2])
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lens(case):
    """(new tokens, past tokens) of each sequence."""
    r = random.Random(case["lens_seed"])
    B = case["B"]
    q = [r.randint(case["qlo"], case["qhi"]) if b < B - case["ones"] else 1 for b in range(B)]
    return q, [r.randint(case["plo"], case["phi"]) for _ in range(B)]


def _gen(seed, device=DEVICE):
    return torch.Generator(device=device).manual_seed(int(seed))


def _table(case, seed):
    """Shuffled physical pages, a tenth of them spare."""
    q, past = _lens(case)
    PS = case["PS"]
    pages = [-(-(a + b) // PS) for a, b in zip(q, past)]
    P = max(1, math.ceil(sum(pages) * 1.1))
    perm = torch.randperm(P, generator=_gen(seed, "cpu")).to(torch.int32)
    table = torch.full((len(q), max(pages)), -1, dtype=torch.int32)
    touched, at = [], 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        touched.append(table[b, past[b] // PS:n])
        at += n
    return P, table.to(DEVICE), torch.cat(touched).to(DEVICE)


def _rope_table(top, rot):
    """[top, rot]: cosines, then sines, of position x frequency."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE) / rot)
    angle = torch.arange(top, dtype=torch.float64, device=DEVICE)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _pool(case, P, L, layer, gen):
    """(codes, scales) of a filled pool: dense for float and fp8 pools, codes
    and scales of a kv-head side by side, layer by layer, for int8."""
    KH, D, PS, kv = case["KH"], case["D"], case["PS"], case["kv"]
    std = 0.5 if kv in ("bf16", "f16") else 1.0
    shape = (P, 2, KH, PS, D)
    if kv in FLOAT:
        pool = torch.zeros((P, L, 2, KH, PS, D), dtype=FLOAT[kv], device=DEVICE)
        pool[:, layer] = torch.randn(shape, generator=gen, device=DEVICE) * std
        return pool, None
    x = torch.randn(shape, generator=gen, device=DEVICE)
    if kv == "int8":
        head = PS * (2 * D + 8)
        slab = KH * head
        buf = torch.zeros(P * L * slab, dtype=torch.uint8, device=DEVICE)
        pool = buf.view(torch.int8).as_strided((P, L, 2, KH, PS, D), (slab, P * slab, PS * D, head, D, 1))
        scales = buf.view(torch.float32).as_strided((P, L, 2, KH, PS), (slab // 4, P * slab // 4, PS, head // 4, 1),
                                                    storage_offset=2 * PS * D // 4)
        x[..., [3, D // 2 + 1]] *= 20.0
        s = x.abs().amax(-1) / 127
        pool[:, layer] = torch.round(x / s[..., None]).clamp(-127, 127).to(torch.int8)
    else:
        pool = torch.zeros((P, L, 2, KH, PS, D), dtype=torch.uint8, device=DEVICE).view(torch.float8_e4m3fn)
        scales = torch.zeros((P, L, 2, KH), dtype=torch.float32, device=DEVICE)
        s = x.abs().amax((-1, -2)) / 448
        pool.view(torch.uint8)[:, layer] = (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[:, layer] = s
    return pool, scales


def prepare(case, seed):
    gen = _gen(seed + 1)
    H, KH, D, dtype = case["H"], case["KH"], case["D"], FLOAT[case["t"]]
    s = {"case": case}
    if case["kind"] == "rotate":
        N = case["N"]
        s["positions"] = torch.randint(0, case["top"], (N,), generator=gen, device=DEVICE)
        s["table"] = _rope_table(case["top"], case["rot"])
    else:
        q, past = _lens(case)
        N = sum(q)
        P, s["pages"], s["touched"] = _table(case, seed)
        cu = [0]
        for n in q:
            cu.append(cu[-1] + n)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE)
        s["lens"] = torch.tensor([a + b for a, b in zip(q, past)], dtype=torch.int32, device=DEVICE)
        s["most"] = max(q)
        L, s["layer"] = 2, 1
        s["pool"], s["scales"] = _pool(case, P, L, s["layer"], gen)
    if case["kind"] == "attend":
        s["q"] = (torch.randn((N, H, D), generator=gen, device=DEVICE) * 2.0).to(dtype)
        return s
    # queries, keys and values are slices of one projection's output
    qkv = torch.randn((N, (H + 2 * KH) * D), generator=gen, device=DEVICE)
    qkv.view(N, H + 2 * KH, D)[..., 3] *= 4.0
    qkv = qkv.to(dtype)
    s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, KH * D, KH * D], 1))
    s["qw"] = s["kw"] = None
    if case["norm"]:
        s["qw"], s["kw"] = ((1 + 0.3 * torch.randn((D,), generator=gen, device=DEVICE)).to(dtype) for _ in range(2))
    if case["kind"] == "append":
        s["table"] = _rope_table(max(a + b for a, b in zip(*_lens(case))) + 1, case["rot"])
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotate": _own_rotate, "append": _own_append, "attend": _own_attend}[kind](state)
    return {"rotate": _rotate, "append": _append, "attend": _attend}[kind](state)


def _own_rotate(s):
    from vramancer_amd.rope import qk_norm_rope

    return qk_norm_rope(s["q"], s["k"], s["table"], s["positions"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                        interleaved=s["case"]["inter"])


def _own_append(s):
    from vramancer_amd import kv_quant
    from vramancer_amd.paged_chunk import rope_append

    q = rope_append(s["q"], s["k"], s["v"], s["pool"], s["pages"], s["lens"], s["cu"], s["layer"], s["table"],
                    kv_scales=s["scales"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                    interleaved=s["case"]["inter"])
    if s["scales"] is None:
        return q, s["pool"]
    return q, kv_quant.dequantize_pages(s["pool"], s["scales"], s["layer"], s["touched"]).bfloat16()


def _own_attend(s):
    from vramancer_amd.paged_chunk import paged_attention_chunk

    return paged_attention_chunk(s["q"], s["pool"], s["pages"], s["lens"], s["cu"], s["layer"],
                                 kv_scales=s["scales"], window=s["case"]["window"] or None)


def _norm_rope(x, w, cos_sin, case):
    """[N, heads, D] float32: RMS norm (where there is a weight), then the
    rotation of the first ``rot`` dims by each row's cosines and sines."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    r = case["rot"]
    cos, sin = (t[:, None] for t in cos_sin.split(r // 2, 1))
    if case["inter"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., r:]], -1)


def _rotate(s):
    cs = s["table"][s["positions"]]
    return tuple(_norm_rope(s[a].float(), s[b], cs, s["case"]).to(s[a].dtype) for a, b in (("q", "qw"), ("k", "kw")))


def _places(s):
    """(position, page, slot) of every new token."""
    cu, lens, PS = s["cu"].long(), s["lens"].long(), s["case"]["PS"]
    n = torch.arange(s["k"].shape[0], device=DEVICE)
    b = torch.searchsorted(cu, n, right=True) - 1
    pos = lens[b] - cu[b + 1] + n
    return pos, s["pages"][b, pos // PS].long(), pos % PS


def _v_cell(t, d, D):
    """(row, column) of the quantized V slice that holds token slot t, dim d."""
    at = ((t // 4 * 16 + d % 16) * (D // 16) + d // 16) * 4 + t % 4
    return at // D, at % D


def _logical_v(codes):
    """V slices [.., PS, D] as stored -> token-major."""
    *lead, PS, D = codes.shape
    return codes.reshape(*lead, PS // 4, 16, D // 16, 4).transpose(-1, -3).reshape(codes.shape)


def _stored_v(codes):
    *lead, PS, D = codes.shape
    return codes.reshape(*lead, PS // 4, 4, D // 16, 16).transpose(-1, -3).reshape(codes.shape)


def _append(s):
    case, layer, pool, scales = s["case"], s["layer"], s["pool"], s["scales"]
    D, KH, PS = case["D"], case["KH"], case["PS"]
    pos, page, slot = _places(s)
    cs = s["table"][pos]
    q = _norm_rope(s["q"].float(), s["qw"], cs, case).to(s["q"].dtype)
    k, v = _norm_rope(s["k"].float(), s["kw"], cs, case), s["v"].float()
    heads = torch.arange(KH, device=DEVICE)[None]
    if case["kv"] in FLOAT:
        pool[page[:, None], layer, 0, heads, slot[:, None]] = k.to(pool.dtype)
        pool[page[:, None], layer, 1, heads, slot[:, None]] = v.to(pool.dtype)
        return q, pool
    if case["kv"] == "int8":
        row, col = _v_cell(slot[:, None], torch.arange(D, device=DEVICE)[None], D)
        ks, vs = k.abs().amax(-1) / 127, v.abs().amax(-1) / 127
        kc, vc = (torch.round(x / t.clamp(min=1e-30)[..., None]).clamp(-127, 127).to(torch.int8)
                  for x, t in ((k, ks), (v, vs)))
        pool[page[:, None], layer, 0, heads, slot[:, None]] = kc
        pool[page[:, None, None], layer, 1, heads[..., None], row[:, None], col[:, None]] = vc
        scales[page[:, None], layer, 0, heads, slot[:, None]] = ks
        scales[page[:, None], layer, 1, heads, slot[:, None]] = vs
        both = pool[s["touched"].long(), layer]
        both = torch.stack([both[:, 0], _logical_v(both[:, 1])], 1)
        return q, (both.float() * scales[s["touched"].long(), layer][..., None]).bfloat16()
    # fp8: one scale per page and head, which only grows
    touched, raw, P = s["touched"].long(), pool.view(torch.uint8), pool.shape[0]
    where = torch.zeros(P, dtype=torch.int64, device=DEVICE)
    where[touched] = torch.arange(touched.numel(), device=DEVICE)
    first = torch.full((touched.numel(),), PS, device=DEVICE).scatter_reduce(0, where[page], slot, "amin")
    out = []
    for kv, x in ((0, k), (1, v)):
        amax = torch.zeros((touched.numel(), KH), device=DEVICE).scatter_reduce(
            0, where[page][:, None].expand(-1, KH), x.abs().amax(-1), "amax")
        old = scales[touched, layer, kv] * (first > 0)[:, None]
        new = torch.maximum(old, amax / 448)
        codes = raw[touched, layer, kv]
        vals = (codes if kv == 0 else _logical_v(codes)).view(torch.float8_e4m3fn).float()
        ratio = torch.where(new > old, old / new.clamp(min=1e-30), 1.0)[..., None, None]
        early = (torch.arange(PS, device=DEVICE)[None] < first[:, None])[:, None, :, None]
        vals = torch.where(early, vals * ratio, vals)
        vals[where[page][:, None], heads, slot[:, None]] = x / new[where[page]].clamp(min=1e-30)[..., None]
        codes = vals.to(torch.float8_e4m3fn)
        scales[touched, layer, kv] = new
        raw[touched, layer, kv] = (codes.view(torch.uint8) if kv == 0 else _stored_v(codes.view(torch.uint8)))
        out.append(codes.float() * new[..., None, None])
    return q, torch.stack(out, 1).bfloat16()


def _cache(s):
    """Keys and values of every sequence's pages, [B, KH, tokens, D] float32,
    and which of them are there, [B, tokens]."""
    case, layer, pages = s["case"], s["layer"], s["pages"]
    B, width = pages.shape
    KH, D, PS = case["KH"], case["D"], case["PS"]
    at = pages.long().clamp(min=0)
    raw = s["pool"].view(torch.uint8) if case["kv"] == "fp8" else s["pool"]
    got = []
    for kv in (0, 1):
        x = raw[at, layer, kv]
        if s["scales"] is not None:
            x = x if kv == 0 else _logical_v(x)
            x = (x.view(torch.float8_e4m3fn) if case["kv"] == "fp8" else x).float()
            t = s["scales"][at, layer, kv]
            x = x * (t[..., None, None] if case["kv"] == "fp8" else t[..., None])
        got.append(x.float().transpose(1, 2).reshape(B, KH, width * PS, D))
    t = torch.arange(width * PS, device=DEVICE)
    there = (t[None] < s["lens"][:, None]) & (pages >= 0).repeat_interleave(PS, 1)
    return got[0], got[1], there


def _attend(s):
    case, cu, most, q = s["case"], s["cu"].long(), s["most"], s["q"]
    N, H, D = q.shape
    KH = case["KH"]
    B, G = cu.numel() - 1, H // KH
    k, v, there = _cache(s)
    i = torch.arange(most, device=DEVICE)[None]
    n = cu[:-1, None] + i
    real = n < cu[1:, None]
    pos = s["lens"].long()[:, None] - (cu[1:] - cu[:-1])[:, None] + i
    x = q[n.clamp(max=N - 1)].float().reshape(B, most, KH, G, D).permute(0, 2, 1, 3, 4).reshape(B, KH, most * G, D)
    scores = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(D)).view(B, KH, most, G, -1)
    t = torch.arange(k.shape[2], device=DEVICE)[None, None]
    seen = there[:, None] & (t <= pos[..., None])
    if case["window"]:
        seen &= t > pos[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KH, most * G, -1), v).view(B, KH, most, G, D) / total.clamp(min=1e-30)
    out = torch.zeros((N, H, D), dtype=q.dtype, device=DEVICE)
    out[n[real]] = o.permute(0, 2, 1, 3, 4).reshape(B, most, H, D)[real].to(q.dtype)
    return out


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    H, KH, D, size = case["H"], case["KH"], case["D"], BYTES[case["t"]]
    if case["kind"] == "rotate":
        N = case["N"]
        return {"bytes": N * (2 * (H + KH) * D * size + 4 * case["rot"] + 8), "flops": N * (H + KH) * D * 7}
    q, past = _lens(case)
    N = sum(q)
    per = KH * 2 * D * BYTES[case["kv"]] + (KH * 8 if case["kv"] == "int8" else 0)  # cache bytes of a token
    table = sum(-(-(a + b) // case["PS"]) for a, b in zip(q, past)) * 4
    if case["kind"] == "append":
        return {"bytes": N * ((2 * H + 2 * KH) * D * size + 4 * case["rot"] + per), "flops": N * (H + 2 * KH) * D * 7}
    w = case["window"] or 1 << 40
    pairs = seen = 0
    for a, b in zip(q, past):
        # row i attends min(b + i + 1, w) tokens
        full = max(0, min(a, w - b))
        pairs += full * b + full * (full + 1) // 2 + (a - full) * min(w, 1 << 32)
        seen += min(a + b, w + a - 1)
    return {"bytes": 2 * N * H * D * size + seen * per + table, "flops": 4 * H * D * pairs}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend":
        return _exact_attend(s, case)
    q, past = _lens(case) if case["kind"] == "append" else (None, None)
    if q is None:
        pos = s["positions"]
    else:
        pos = torch.cat([torch.arange(b, a + b) for a, b in zip(q, past)]).to(DEVICE)
    angle = s["table"][pos].double()
    half = case["rot"] // 2

    def turn(x, w):
        y = x.double().clone()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * w.double()
        z = y.clone()
        first = torch.arange(half, device=DEVICE) * (2 if case["inter"] else 1)
        second = first + (1 if case["inter"] else half)
        c, sn = angle[:, None, :half], angle[:, None, half:]
        z[..., first] = y[..., first] * c - y[..., second] * sn
        z[..., second] = y[..., first] * sn + y[..., second] * c
        return z

    qr, kr = turn(s["q"], s["qw"]), turn(s["k"], s["kw"])
    if q is None:
        return qr, kr
    PS, layer, D = case["PS"], s["layer"], case["D"]
    vr = s["v"].double()
    if case["kv"] in FLOAT:
        pool = s["pool"].double()
        at = 0
        for b, (a, p) in enumerate(zip(q, past)):
            t = torch.arange(p, p + a, device=DEVICE)
            page = s["pages"][b, t // PS].long()
            for kv, x in ((0, kr), (1, vr)):
                pool[page, layer, kv, :, t % PS] = x[at:at + a]
            at += a
        return qr, pool
    tile = torch.arange(PS * D, device=DEVICE).view(PS // 4, 16, D // 16, 4)
    order = tile.permute(0, 3, 2, 1).reshape(-1)  # stored place of logical (t, d)
    vals = []
    at = 0
    for b, (a, p) in enumerate(zip(q, past)):
        first = p // PS
        ids = s["pages"][b, first:-(-(a + p) // PS)].long()
        n, lead = ids.numel(), p - first * PS
        for kv, x in ((0, kr), (1, vr)):
            codes = s["pool"].view(torch.uint8)[ids, layer, kv]  # [n, KH, PS, D]
            if kv:
                codes = codes.flatten(2)[:, :, order].view(codes.shape)
            codes = codes.view(torch.int8 if case["kv"] == "int8" else torch.float8_e4m3fn).double()
            codes = codes.transpose(0, 1).reshape(case["KH"], n * PS, D)
            rows = x[at:at + a].transpose(0, 1)
            sc = s["scales"][ids, layer, kv].double()
            if case["kv"] == "int8":
                sc = sc.transpose(0, 1).reshape(case["KH"], n * PS)
                sc[:, lead:lead + a] = rows.abs().amax(-1) / 127
                codes[:, lead:lead + a] = (rows / sc[:, lead:lead + a, None].clamp(min=1e-300)).round()
                val = codes * sc[..., None]
            else:
                old = sc.transpose(0, 1).clone()  # [KH, n]
                old[:, 1 if lead else 0:] = 0
                amax = torch.zeros((case["KH"], n * PS), dtype=torch.float64, device=DEVICE)
                amax[:, lead:lead + a] = rows.abs().amax(-1)
                new = torch.maximum(old, amax.view(-1, n, PS).amax(-1) / 448)
                per = new.repeat_interleave(PS, 1)[..., None].clamp(min=1e-300)
                codes[:, :lead] = (codes[:, :lead] * old[:, :1, None] / per[:, :lead]).to(torch.float8_e4m3fn).double()
                codes[:, lead:lead + a] = (rows / per[:, lead:lead + a]).to(torch.float8_e4m3fn).double()
                val = codes * per
            vals.append(val.view(case["KH"], n, PS, D).transpose(0, 1))
        at += a
    pages = [torch.stack(vals[i:i + 2], 1) for i in range(0, len(vals), 2)]
    return qr, torch.cat(pages)


def _exact_attend(s, case):
    q, past = _lens(case)
    H, KH, D, PS, layer = case["H"], case["KH"], case["D"], case["PS"], s["layer"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    tile = torch.arange(PS * D, device=DEVICE).view(PS // 4, 16, max(1, D // 16), 4) if s["scales"] is not None else None
    at = 0
    for b, (a, p) in enumerate(zip(q, past)):
        n = a + p
        ids = s["pages"][b, :-(-n // PS)].long()
        t = torch.arange(n, device=DEVICE)
        pos = torch.arange(p, n, device=DEVICE)
        hide = t[None] > pos[:, None]
        if case["window"]:
            hide |= t[None] <= pos[:, None] - case["window"]
        for kvh in range(KH):
            kv = []
            for j in (0, 1):
                if s["scales"] is None:
                    x = s["pool"][ids, layer, j, kvh].double()
                else:
                    x = s["pool"].view(torch.uint8)[ids, layer, j, kvh]
                    if j:
                        x = x.flatten(1)[:, tile.permute(0, 3, 2, 1).reshape(-1)].view(x.shape)
                    x = x.view(torch.int8 if case["kv"] == "int8" else torch.float8_e4m3fn).double()
                    sc = s["scales"][ids, layer, j, kvh].double()
                    x = x * sc.reshape(*sc.shape, *([1] * (x.dim() - sc.dim())))
                kv.append(x.reshape(-1, D)[:n])
            for h in range(kvh * (H // KH), (kvh + 1) * (H // KH)):
                for r in range(0, a, 1024):
                    sc = s["q"][at + r:at + min(a, r + 1024), h].double() @ kv[0].t() / math.sqrt(D)
                    sc.masked_fill_(hide[r:r + 1024], -math.inf)
                    out[at + r:at + min(a, r + 1024), h] = torch.softmax(sc, -1) @ kv[1]
        at += a
    return out
