"""The chunk operators together, as a serving program uses them: prompts in
chunks through a Hugging Face model, drafted tokens, and layer steps that norm,
rotate, append, attend and decode.

Bars: logits as in test_gpu_paged_batch.py (2e-2 + 2e-2 |ref| for float pools,
5e-2 / 0.15 absolute on top of 2e-2 |ref| for int8 / fp8), since the same
products are taken of the same cached values.  Layer steps are held to the
operators' own tolerances in test_gpu_paged_chunk.py and test_gpu_rope.py; here
a decode over a cache filled by chunks must agree with a chunk of one token
over the same cache within float32 rounding of the decode (2e-3 + 1e-2 |ref|,
the decode's bar).
"""
import copy

import pytest
import torch
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

from chunk_reference import attend, norm_rope, rope_angles
from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_batch import (PagedChunkCache, chunk_step, decode_step, enable_paged_attention, prefill,
                                       prefill_chunked)
from vramancer_amd.paged_chunk import chunk_workspace, paged_attention_chunk, rope_append
from vramancer_amd.rope import rope_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {"float32": 2e-2, "float16": 2e-2, "bfloat16": 2e-2, "int8": 5e-2, "fp8": 0.15}


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _manager(dtype, max_pages=64, heads=2, D=128, layers=2, **kw):
    return PagedKVCacheManager(PagedKVConfig(page_size=16, num_layers=layers, num_kv_heads=heads, head_dim=D,
                                             max_pages=max_pages, device=DEV, dtype=dtype, **kw))


@pytest.fixture(scope="module")
def setting():
    cfg = LlamaConfig(vocab_size=256, hidden_size=512, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=128, max_position_embeddings=512)
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).eval()
    gen = torch.Generator().manual_seed(9)
    ids = torch.randint(0, 256, (1, 90), generator=gen)
    with torch.no_grad():
        ref = model(ids, past_key_values=DynamicCache(), use_cache=True).logits[0]
    gpu = copy.deepcopy(model).to(DEV)
    enable_paged_attention(gpu)
    return gpu, ids, ref


def _close(got, want, atol, what):
    err = (got.float().cpu() - want).abs()
    assert (err <= atol + 2e-2 * want.abs()).all(), f"{what}: max err {float(err.max()):.3e}"


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("chunk", [7, 32, 200])
def test_prefill_in_chunks_then_decode(setting, dtype, chunk):
    model, ids, ref = setting
    _say(f"prefill in chunks of {chunk}, pool {dtype}")
    mgr = _manager(dtype)
    with torch.no_grad():
        got = prefill_chunked(model, mgr, "r", ids[:, :70].to(DEV), chunk)
        _close(got[0], ref[69], TOL[dtype], "prompt")
        for t in range(70, 74):  # decode steps over the same pages
            _close(decode_step(model, mgr, ["r"], ids[0, t:t + 1].to(DEV))[0], ref[t], TOL[dtype], f"token {t}")
        # and a chunk of drafted tokens after them
        _close(chunk_step(model, mgr, ["r"], ids[:, 74:80].to(DEV))[0], ref[74:80], TOL[dtype], "drafted")
    assert list(mgr.token_counts(["r"])) == [80] and len(mgr._page_tables["r"].pages) == 5


def test_batch_of_drafts(setting):
    """Requests at different positions verify drafted tokens in one step."""
    model, ids, ref = setting
    _say("drafts of a batch")
    mgr = _manager("float32")
    with torch.no_grad():
        for rid, n in (("a", 11), ("b", 48), ("c", 33)):
            mgr.allocate(rid)
            prefill(model, mgr, rid, ids[:, :n].to(DEV))
        cache = PagedChunkCache(mgr, ["a", "b", "c"])
        toks = torch.stack([ids[0, n:n + 4] for n in (11, 48, 33)]).to(DEV)
        got = chunk_step(model, mgr, ["a", "b", "c"], toks, cache)
    for row, n in zip(got, (11, 48, 33)):
        _close(row, ref[n:n + 4], 2e-2, f"at {n}")


def test_refusals_of_steps(setting):
    model, ids, _ = setting
    mgr = _manager("float16", max_pages=3)
    mgr.allocate("x")
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="no page left"):
            prefill_chunked(model, mgr, "x", ids[:, :60].to(DEV), 64)
        assert list(mgr.token_counts(["x"])) == [0] and len(mgr._free_pages) == 3
        with pytest.raises(RuntimeError, match="empty prompt"):
            prefill_chunked(model, mgr, "x", ids[:, :0].to(DEV))
        prefill_chunked(model, mgr, "x", ids[:, :5].to(DEV))
        mgr.fork("x", "y")
        with pytest.raises(RuntimeError, match="share the page"):
            chunk_step(model, mgr, ["x", "y"], torch.zeros((2, 3), dtype=torch.long, device=DEV))
    with pytest.raises(KeyError):
        mgr.append_chunk(["nobody"], [1])
    with pytest.raises(RuntimeError, match="once only"):
        mgr.append_chunk(["x", "x"], [1, 1])
    with pytest.raises(RuntimeError, match="negative"):
        mgr.append_chunk(["x"], [-1])
    chunk = mgr.append_chunk(["x", "y"], [0, 0])
    assert chunk.num_tokens == 0
    q = torch.zeros((0, 4, 128), dtype=torch.float16, device=DEV)
    assert mgr.compute_attention_chunk(q, chunk, 0).shape == q.shape


@pytest.mark.parametrize("dtype,t", [("bfloat16", torch.bfloat16), ("int8", torch.bfloat16), ("fp8", torch.float16),
                                     ("float32", torch.float32)])
def test_layer_steps(dtype, t):
    """Three ragged chunks through one layer: rotated queries attend what the
    pool holds, and the last token decodes to the same."""
    _say(f"layer steps, pool {dtype}")
    H, KH, D = 10, 2, 128
    mgr = _manager(dtype, heads=KH, D=D, layers=1)
    gen = torch.Generator().manual_seed(3)
    table = rope_table(200, D, device=DEV)
    qw, kw = (1 + 0.2 * torch.randn(D, generator=gen) for _ in range(2))
    for rid in ("a", "b", "c"):
        mgr.allocate(rid)
    done = {"a": 0, "b": 0, "c": 0}
    for counts in ([40, 0, 3], [1, 70, 20], [5, 1, 33]):
        chunk = mgr.append_chunk(["a", "b", "c"], counts)
        n = sum(counts)
        qkv = (torch.randn((n, H + 2 * KH, D), generator=gen)).to(t)
        g = qkv.to(DEV)
        q = mgr.write_chunk(0, chunk, g[:, H:H + KH], g[:, H + KH:], g[:, :H], table, q_weight=qw.to(DEV),
                            k_weight=kw.to(DEV))
        pos = torch.cat([torch.arange(done[r], done[r] + c) for r, c in zip(done, counts)])
        want, size = norm_rope(qkv[:, :H], qw, rope_angles(200, D), pos, 1e-6, False)
        u = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[t]
        assert ((q.cpu().double() - want).abs() <= u * want.abs() + 2.0 ** -19 * size + 2.0 ** -25).all()
        out = mgr.compute_attention_chunk(q, chunk, 0)
        for r, c in zip(done, counts):
            done[r] += c
        # float64 attention over what the pages hold
        at = 0
        for r, c in zip(done, counts):
            if c:
                k, v = (x.double().cpu() for x in mgr.read_kv(r, 0))  # [KH, tokens, D]
                m = k.shape[1]
                vals = torch.stack([k, v])[None, None]  # one page of m tokens
                ref, _, reach = attend(q[at:at + c].cpu(), vals, torch.zeros((1, 1), dtype=torch.int32), [m],
                                       [0, c], 0)
                tol = u * (ref.abs() + reach) + 2.0 ** -16 * reach + 2.0 ** -25
                assert ((out[at:at + c].cpu().double() - ref).abs() <= tol).all(), (r, counts)
            at += c
    last = torch.randn((3, H, D), generator=gen).to(t).to(DEV)
    dec = mgr.compute_attention_decode(last.float(), ["a", "b", "c"], 0)
    one = paged_attention_chunk(last, mgr.gpu_pool, *mgr._block_table(["a", "b", "c"], DEV),
                                torch.arange(4, dtype=torch.int32, device=DEV), 0, kv_scales=mgr._kv_scales).float()
    assert ((dec - one).abs() <= 2e-3 + 1e-2 * dec.abs()).all()


def test_chunks_fill_turboquant_pages():
    """Rows written by a chunk are compressed like rows written one by one."""
    _say("chunks with TurboQuant compression")
    outs = []
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn((21, 2, 64), generator=gen).half().to(DEV) for _ in range(2))
    q = torch.randn((4, 64), generator=gen).to(DEV)
    for chunked in (True, False):
        torch.manual_seed(7)
        mgr = _manager("float16", heads=2, D=64, layers=1, kv_compression="turboquant")
        mgr.allocate("r")
        if chunked:
            for a, b in ((0, 5), (5, 20), (20, 21)):
                mgr.write_chunk(0, mgr.append_chunk(["r"], [b - a]), k[a:b], v[a:b])
        else:
            for i in range(21):
                mgr.write_kv("r", 0, *mgr.append_token("r"), k[i], v[i])
        mgr.flush_compression()
        outs.append(mgr.compute_attention_turbo(q, "r", 0))
    assert torch.equal(outs[0], outs[1])


def test_captured_steps_and_streams():
    """Append and attention captured into a graph with a padded batch: every
    replay equals the eager call on what the buffers then hold, and rows behind
    the batch are left alone; then the same calls on another stream."""
    _say("captured append and attention")
    H, KH, D, PS, N, B = 8, 2, 128, 16, 48, 3
    gen = torch.Generator().manual_seed(5)
    mk = lambda *s: torch.randn(s, generator=gen).bfloat16().to(DEV)  # noqa: E731
    q, k, v = mk(N, H, D), mk(N, KH, D), mk(N, KH, D)
    pool = torch.zeros((40, 1, 2, KH, PS, D), dtype=torch.bfloat16, device=DEV)
    table = torch.randperm(40, generator=gen)[:36].reshape(B, 12).int().to(DEV)
    angles = rope_table(256, D, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    q_out, out = torch.zeros_like(q), torch.zeros_like(q)
    ws = chunk_workspace(q, pool, B, 12)

    def both(q_out, out, pool, ws):
        rope_append(q, k, v, pool, table, lens, cu, 0, angles, query_out=q_out)
        paged_attention_chunk(q_out, pool, table, lens, cu, 0, out=out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(q_out, out, pool, ws)  # empty batch: nothing is written
    torch.cuda.synchronize()
    assert not out.any() and not pool.any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(q_out, out, pool, ws)
    total = torch.zeros(B, dtype=torch.int64)
    for step, counts in enumerate(([40, 1, 0], [1, 1, 1], [0, 20, 28], [16, 16, 16], [2, 0, 0])):
        total += torch.tensor(counts)
        q.copy_(mk(N, H, D)), k.copy_(mk(N, KH, D)), v.copy_(mk(N, KH, D))
        lens.copy_(total.int()), cu.copy_(torch.tensor([0] + counts).cumsum(0).int())
        pool2, q2, out2 = pool.clone(), q_out.clone(), out.clone()
        q_out.fill_(3.0), out.fill_(3.0), q2.fill_(3.0), out2.fill_(3.0)
        ws.fill_(255)
        graph.replay()
        both(q2, out2, pool2, None)
        torch.cuda.synchronize()
        assert torch.equal(out, out2) and torch.equal(q_out, q2) and torch.equal(pool, pool2), f"replay {step}"
        assert (out[sum(counts):] == 3).all() and (q_out[sum(counts):] == 3).all()
        with torch.cuda.stream(side):
            q3, out3, pool3 = torch.empty_like(q), torch.empty_like(q), pool.clone()
            q3.fill_(3.0), out3.fill_(3.0)
            both(q3, out3, pool3, None)
        torch.cuda.synchronize()
        assert torch.equal(out3, out)
