"""Operators at the end and the start of a serving step, timed one call at a
time: how logits become tokens, and how lengths become the next step's tables.

``kind`` names the call:

  draw     sampling.sample_tokens: a token per row of logits, by temperature,
           top_k and top_p from a given random number, in some cases with the
           distribution it was drawn from
  verify   sampling.verify_drafts: drafted tokens against the target's
           probabilities, and the token that follows the accepted ones
  tables   paged_chunk.chunk_tables: page table, lengths, offsets and the
           place of every new token of a ragged batch, from the requests'
           lengths and a resident block table

Logits are a normal bulk with a few tokens far above it, as a language model's
are.  Where ``own`` is false ``run`` computes the plain forms: elementary torch
operations, in float64, since a token is an answer in whole numbers and follows
sums over the vocabulary next to borders.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the first token of one prompt, top_k and top_p: latency
        dict(name="draw-one", kind="draw", N=1, V=131072, t="f32", temp=0.8, k=50, p=0.95, probs=False),
        # one step of 16 requests, temperature only, some greedy: latency
        dict(name="draw-step", kind="draw", N=16, V=32000, t="f32", temp=1.0, k=0, p=1.0, probs=False),
        # one step of 64 requests with a nucleus, a large vocabulary
        dict(name="draw-nucleus", kind="draw", N=64, V=152000, t="bf16", temp=1.0, k=0, p=0.9, probs=False),
        # a draft model's step for 512 requests, its distribution kept for the verification
        dict(name="draw-drafts", kind="draw", N=512, V=131072, t="f16", temp=0.9, k=0, p=0.95, probs=True),
        # drafts looked up in the prompt (no distribution), 8 requests of 3: latency
        dict(name="verify-lookup", kind="verify", B=8, K=3, V=32000, t="f32", temp=0.7, k=0, p=1.0, q=False,
             ragged=False, lens_seed=1),
        # four drafted tokens for each of 64 requests
        dict(name="verify-64", kind="verify", B=64, K=4, V=152000, t="bf16", temp=1.0, k=0, p=1.0, q=True,
             ragged=False, lens_seed=2),
        # drafts of different lengths under top_k and top_p, an odd vocabulary
        dict(name="verify-ragged", kind="verify", B=37, K=7, V=100003, t="f16", temp=0.8, k=100, p=0.95, q=True,
             ragged=True, lens_seed=3),
        # a large batch of a throughput server
        dict(name="verify-large", kind="verify", B=160, K=5, V=131072, t="bf16", temp=1.0, k=0, p=1.0, q=True,
             ragged=False, lens_seed=4),
        # one new token for each of 32 requests: latency
        dict(name="tables-step", kind="tables", R=64, B=32, W=512, PS=16, plo=16, phi=8000, clo=1, chi=1, spare=0,
             lens_seed=5),
        # prompts and chunks beside decoding requests
        dict(name="tables-prompts", kind="tables", R=100, B=61, W=2051, PS=16, plo=0, phi=30000, clo=1, chi=2000,
             spare=301, lens_seed=6),
        # drafts for a thousand requests of long contexts
        dict(name="tables-large", kind="tables", R=1500, B=1024, W=8192, PS=16, plo=1000, phi=131000, clo=1, chi=8,
             spare=64, lens_seed=7),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["draw", "draw", "verify", "verify", "tables"])
    seed = rng.randrange(1 << 30)
    if kind == "tables":
        B = _log_int(rng, 1, 1024)
        PS = rng.choice([4, 16, 16, 32, 64])
        W = _log_int(rng, 4, 8192)
        chi = min(_log_int(rng, 1, max(1, min(2000, 64000 // B))), W * PS // 2)
        phi = W * PS - chi
        return dict(kind=kind, R=B + rng.randrange(0, B + 1), B=B, W=W, PS=PS, plo=rng.randrange(0, phi), phi=phi,
                    clo=rng.choice([0, 1, 1]), chi=chi, spare=rng.choice([0, 0, 1, 77]), lens_seed=seed)
    V = _log_int(rng, 1000, 160000)
    c = dict(kind=kind, V=V, t=rng.choice(["f32", "f16", "bf16", "bf16"]), temp=round(rng.uniform(0.4, 1.5), 3),
             k=rng.choice([0, 0, 1, 20, 50, 1000]), p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]))
    if kind == "draw":
        c.update(N=_log_int(rng, 1, min(512, 60_000_000 // V)), probs=rng.choice([False, False, True]))
    else:
        K = rng.randrange(1, 9)
        c.update(B=_log_int(rng, 1, min(256, 60_000_000 // (V * (K + 1)))), K=K, q=rng.choice([False, True, True]),
                 ragged=rng.choice([False, True]), lens_seed=seed)
    return c


def _counts(case):
    """Drafts of each sequence of a verify case."""
    rng = random.Random(case["lens_seed"])
    return [rng.randint(0, case["K"]) if case["ragged"] else case["K"] for _ in range(case["B"])]


def _lens(case):
    """(requests of the batch, tokens stored of every request, new tokens of each sequence) of a tables case."""
    rng = random.Random(case["lens_seed"])
    return (rng.sample(range(case["R"]), case["B"]), [rng.randint(case["plo"], case["phi"]) for _ in range(case["R"])],
            [rng.randint(case["clo"], case["chi"]) for _ in range(case["B"])])


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _logits(N, V, gen):
    """[N, V] float32: a normal bulk, and 40 tokens that stand above it by up to 12."""
    x = torch.randn((N, V), generator=gen, device=DEVICE) * 2.0 - 4.0
    each = V // 40
    hot = torch.randint(0, each, (N, 40), generator=gen, device=DEVICE) + torch.arange(40, device=DEVICE) * each
    up = torch.rand((N, 1), generator=gen, device=DEVICE) * 6.0 + 6.0
    up = up - torch.rand((N, 40), generator=gen, device=DEVICE) * 12.0
    return x.scatter_(1, hot, up)


def prepare(case, seed):
    gen = _gen(seed)
    s = {"case": case, "kind": case["kind"]}
    if case["kind"] == "tables":
        reqs, past, counts = _lens(case)
        i32 = dict(dtype=torch.int32, device=DEVICE)
        pages = case["R"] * case["W"]
        s.update(table=torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32).view(case["R"], case["W"]),
                 past=torch.tensor(past, **i32), counts=torch.tensor(counts, **i32), requests=torch.tensor(reqs, **i32),
                 rows=max(1, sum(counts) + case["spare"]))
        return s
    V = case["V"]
    if case["kind"] == "draw":
        N = B = case["N"]
        x = _logits(N, V, gen)
        some = x[5::16]  # requests held to a grammar: few tokens are allowed
        allowed = torch.rand(some.shape, generator=gen, device=DEVICE) < 0.01
        allowed[:, 0] = True
        some.masked_fill_(~allowed, -math.inf)
        s["logits"] = x.to(FLOAT[case["t"]])
        s["u"] = torch.rand(N, generator=gen, device=DEVICE)
    else:
        B, K, n = case["B"], case["K"], _counts(case)
        N = sum(n) + B
        x = _logits(N, V, gen)
        s["logits"] = x.to(FLOAT[case["t"]])
        cu = np.concatenate([[0], np.cumsum(np.array(n) + 1)])
        row = torch.tensor(cu[:-1], device=DEVICE)[:, None] + torch.arange(K, device=DEVICE)
        row = row.clamp(max=N - 1)
        if not case["ragged"]:
            s["logits"] = s["logits"].view(B, K + 1, V)
        s["cu"] = torch.tensor(cu, dtype=torch.int32, device=DEVICE) if case["ragged"] else None
        if case["q"]:  # a draft model near the target; its drafts are drawn from its own distribution
            q = torch.empty((B, K, V), device=DEVICE)
            for i in range(K):
                y = x[row[:, i]] + torch.randn((B, V), generator=gen, device=DEVICE) * 0.7
                q[:, i] = torch.softmax(y / case["temp"], -1)
            e = torch.rand((B, K, V), generator=gen, device=DEVICE).clamp_(min=1e-30).log_().neg_()
            s["drafts"], s["q"] = (q / e).argmax(-1), q
        else:  # tokens found in the prompt: the likely one or any other
            likely = x.argmax(-1)[row]
            other = torch.randint(0, V, (B, K), generator=gen, device=DEVICE)
            s["drafts"] = torch.where(torch.rand((B, K), generator=gen, device=DEVICE) < 0.8, likely, other)
            s["q"] = None
        s["ua"] = torch.rand((B, K), generator=gen, device=DEVICE)
        s["u"] = torch.rand(B, generator=gen, device=DEVICE)
    temp = torch.full((B,), case["temp"], device=DEVICE)
    temp[3::8] = 0.0  # a greedy request among the others
    s["temp"] = temp
    s["k"] = torch.full((B,), case["k"], dtype=torch.int32, device=DEVICE) if case["k"] else None
    s["p"] = torch.full((B,), case["p"], device=DEVICE) if case["p"] < 1 else None
    return s


def run(state):
    return (_own if own else _plain)[state["kind"]](state)


def _own_draw(s):
    from vramancer_amd import sampling

    logits = s["logits"]
    probs = torch.empty(logits.shape, device=logits.device) if s["case"]["probs"] else None
    tokens = sampling.sample_tokens(logits, s["u"], temperature=s["temp"], top_k=s["k"], top_p=s["p"], probs=probs)
    return [tokens] if probs is None else [tokens, probs]


def _own_verify(s):
    from vramancer_amd import sampling

    return list(sampling.verify_drafts(s["logits"], s["drafts"], s["ua"], s["u"], draft_probs=s["q"],
                                       cu_seqlens=s["cu"], temperature=s["temp"], top_k=s["k"], top_p=s["p"]))


def _own_tables(s):
    from vramancer_amd import paged_chunk

    t = paged_chunk.chunk_tables(s["table"], s["past"], s["counts"], s["rows"], s["case"]["PS"],
                                 requests=s["requests"])
    return [t.page_table, t.context_lens, t.cu_seqlens, t.positions, t.page_ids, t.slots, t.sequences]


def _weights(logits, temp, k, p):
    """[N, V] float64 weights of the tokens that may be drawn, zero for the others; not normed."""
    x = logits.double()
    temp = temp.double()[:, None]
    top = x.amax(-1, keepdim=True)
    w = torch.exp((x - top) / torch.where(temp > 0, temp, 1.0))
    first = torch.zeros_like(w).scatter_(1, x.argmax(-1, keepdim=True), 1.0)
    w = torch.where(temp > 0, w, first)
    if k is None and p is None:
        return w
    order = x.sort(dim=-1, descending=True, stable=True).indices
    sw = w.gather(1, order)
    rank = torch.arange(w.shape[1], device=w.device)
    if k is not None:
        sw = torch.where((rank < k[:, None]) | (k[:, None] <= 0), sw, 0.0)
    if p is not None:
        c = sw.cumsum(-1)
        p = p.double()[:, None]
        sw = torch.where((c - sw < p * c[:, -1:]) | (rank == 0) | (p >= 1), sw, 0.0)
    return torch.zeros_like(w).scatter_(1, order, sw)


def _pick(w, u):
    """The lowest index whose running sum passes u of the whole."""
    c = w.cumsum(-1)
    return (c <= u.double()[:, None] * c[:, -1:]).sum(-1)


def _plain_draw(s):
    w = _weights(s["logits"], s["temp"], s["k"], s["p"])
    tokens = _pick(w, s["u"])
    if not s["case"]["probs"]:
        return [tokens]
    return [tokens, (w / w.sum(-1, keepdim=True)).float()]


def _plain_verify(s):
    case, dev = s["case"], s["logits"].device
    B, K, V = case["B"], case["K"], case["V"]
    logits = s["logits"].reshape(-1, V)
    cu = s["cu"].long() if s["cu"] is not None else torch.arange(B + 1, device=dev) * (K + 1)
    n = cu[1:] - cu[:-1] - 1
    seq = torch.repeat_interleave(torch.arange(B, device=dev), n + 1, output_size=logits.shape[0])
    w = _weights(logits, s["temp"][seq], s["k"][seq] if s["k"] is not None else None,
                 s["p"][seq] if s["p"] is not None else None)
    z = w.sum(-1)
    i = torch.arange(K, device=dev)
    there = i < n[:, None]
    row = torch.where(there, cu[:-1, None] + i, 0)
    x = s["drafts"]
    px = w[row, x] / z[row]
    qx = s["q"].gather(2, x[..., None])[..., 0].double() if s["q"] is not None else torch.ones_like(px)
    ok = there & (s["ua"].double() * qx < px)
    accepted = ok.long().cumprod(-1).sum(-1)
    last = cu[:-1] + accepted
    pr = w[last] / z[last, None]
    refused = accepted < n
    at = accepted.clamp(max=K - 1)
    b = torch.arange(B, device=dev)
    if s["q"] is not None:
        rest = (pr - s["q"][b, at].double()).clamp(min=0.0)
    else:
        rest = pr.scatter(1, x[b, at][:, None], 0.0)
    rest = torch.where(refused[:, None] & (rest.sum(-1, keepdim=True) > 0), rest, pr)
    token = _pick(rest, s["u"])
    out = torch.nn.functional.pad(torch.where(i < accepted[:, None], x, -1), (0, 1), value=-1)
    out.scatter_(1, accepted[:, None], token[:, None])
    return [out, accepted.int()]


def _plain_tables(s):
    PS, N, dev = s["case"]["PS"], s["rows"], s["table"].device
    reqs, W = s["requests"].long(), s["table"].shape[1]
    past, counts = s["past"][reqs].long(), s["counts"].long()
    B = counts.shape[0]
    cu = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
    ctx = past + counts
    used = torch.arange(W, device=dev) * PS < ctx[:, None]
    pages = torch.where(used, s["table"][reqs], -1)
    r = torch.arange(N, device=dev)
    seq = torch.searchsorted(cu[1:], r, right=True)
    there = seq < B
    seq = seq.clamp(max=B - 1)
    pos = past[seq] + r - cu[seq]
    page = pages[seq, (pos // PS).clamp(max=W - 1)]
    return [pages, ctx.int(), cu.int(), torch.where(there, pos, 0).int(), torch.where(there, page, -1),
            torch.where(there, pos % PS, -1).int(), torch.where(there, seq, -1).int()]


_own = {"draw": _own_draw, "verify": _own_verify, "tables": _own_tables}
_plain = {"draw": _plain_draw, "verify": _plain_verify, "tables": _plain_tables}


def work(case):
    if case["kind"] == "tables":
        reqs, past, counts = _lens(case)
        used = sum(min(case["W"], -(-(past[r] + c) // case["PS"])) for r, c in zip(reqs, counts))
        N, B = max(1, sum(counts) + case["spare"]), case["B"]
        return {"bytes": 4 * (used + 3 * B) + 4 * (B * case["W"] + 2 * B + 1 + 4 * N), "flops": 4 * N + B * case["W"]}
    V, e = case["V"], BYTES[case["t"]]
    if case["kind"] == "draw":
        N = case["N"]
        return {"bytes": N * (V * e + 12 + 8) + (4 * N * V if case["probs"] else 0),
                "flops": N * V * (5 if case["probs"] else 4)}
    B, K = case["B"], case["K"]
    N = sum(_counts(case)) + B
    return {"bytes": N * V * e + (4 * B * V if case["q"] else 0) + B * (K * 16 + K * 8 + 24),
            "flops": 4 * N * V + 3 * B * V}


def exact(case, seed):
    if case["kind"] == "tables":
        return _exact_tables(case, prepare(case, seed))
    s = prepare(case, seed)
    logits = s["logits"].reshape(-1, case["V"]).float().cpu().numpy()
    temp = s["temp"].double().cpu().numpy()
    u = s["u"].double().cpu().numpy()
    if case["kind"] == "draw":
        if logits.size > 100_000_000:
            return None
        tokens, probs = [], []
        for r in range(case["N"]):
            p = _distribution(logits[r], temp[r], s["k"] is not None and int(s["k"][r]),
                              float(s["p"][r]) if s["p"] is not None else 1.0)
            tokens.append(_invert(p, u[r]))
            probs.append(p)
        tokens = torch.tensor(tokens)
        return [tokens, torch.from_numpy(np.stack(probs))] if case["probs"] else [tokens]
    n = _counts(case)
    first = np.concatenate([[0], np.cumsum(np.array(n) + 1)])
    drafts, ua = s["drafts"].cpu().numpy(), s["ua"].double().cpu().numpy()
    out = np.full((case["B"], case["K"] + 1), -1, dtype=np.int64)
    accepted = np.zeros(case["B"], dtype=np.int32)
    for b in range(case["B"]):
        k = int(s["k"][b]) if s["k"] is not None else 0
        top_p = float(s["p"][b]) if s["p"] is not None else 1.0
        for i in range(n[b] + 1):
            p = _distribution(logits[first[b] + i], temp[b], k, top_p)
            if i == n[b]:
                break
            x = drafts[b, i]
            q = np.zeros(case["V"])
            if s["q"] is not None:
                q = s["q"][b, i].double().cpu().numpy()
            else:
                q[x] = 1.0
            if not ua[b, i] * q[x] < p[x]:
                rest = np.maximum(p - q, 0.0)
                if s["q"] is None:
                    rest[x] = 0.0
                p = rest if rest.sum() > 0 else p
                break
            out[b, i] = x
            accepted[b] += 1
        out[b, accepted[b]] = _invert(p, u[b])
    return [torch.from_numpy(out), torch.from_numpy(accepted)]


def _distribution(row, temp, k, top_p):
    """Probabilities of one row of logits in 64 bits."""
    row = row.astype(np.float64)
    if not temp > 0:
        p = np.zeros(row.size)
        p[int(np.argmax(row))] = 1.0
        return p
    x = row / temp
    p = np.exp(x - x.max())
    if k and k > 0 or top_p < 1:
        order = np.argsort(-row, kind="stable")
        kept = order[:k] if k and k > 0 else order
        if top_p < 1:
            run = np.cumsum(p[kept])
            kept = kept[:int(np.searchsorted(run, top_p * run[-1], side="left")) + 1]
        only = np.zeros(row.size)
        only[kept] = p[kept]
        p = only
    return p / math.fsum(p) if p.size < 2000 else p / p.sum()


def _invert(p, u):
    run = np.cumsum(p)
    return int(np.searchsorted(run, u * run[-1], side="right"))


def _exact_tables(case, s):
    reqs, past, counts = _lens(case)
    table = s["table"].cpu().numpy()
    PS, N = case["PS"], s["rows"]
    pages = np.full((case["B"], case["W"]), -1, dtype=np.int32)
    pos, page, slot, seq = (np.full(N, v, dtype=np.int32) for v in (0, -1, -1, -1))
    cu = [0]
    for b, (r, c) in enumerate(zip(reqs, counts)):
        held = -(-(past[r] + c) // PS)
        pages[b, :held] = table[r, :held]
        for t in range(past[r], past[r] + c):
            at = cu[-1] + t - past[r]
            pos[at], page[at], slot[at], seq[at] = t, table[r, t // PS], t % PS, b
        cu.append(cu[-1] + c)
    ctx = np.array([past[r] + c for r, c in zip(reqs, counts)], dtype=np.int32)
    return [torch.from_numpy(a) for a in (pages, ctx, np.array(cu, dtype=np.int32), pos, page, slot, seq)]
