"""A step or prompt that fails leaves its requests, and the pool's books, as
they were.

Bars of logits: 2e-2 + 2e-2 |ref| as in test_gpu_chunk_steps.py.
"""
import copy

import pytest
import torch
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM, MistralConfig, MistralForCausalLM

from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_batch import (PagedBatchCache, PagedChunkCache, chunk_step, decode_step, enable_paged_attention,
                                       prefill_chunked)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = dict(vocab_size=256, hidden_size=256, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, max_position_embeddings=256)


def _manager(dtype="float32", max_pages=8, **kw):
    return PagedKVCacheManager(PagedKVConfig(page_size=16, num_layers=2, num_kv_heads=2, head_dim=64,
                                             max_pages=max_pages, device=DEV, dtype=dtype, **kw))


@pytest.fixture(scope="module")
def setting():
    cfg = LlamaConfig(**SIZES)
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).eval()
    ids = torch.randint(0, 256, (1, 90), generator=torch.Generator().manual_seed(9))
    with torch.no_grad():
        ref = model(ids, past_key_values=DynamicCache(), use_cache=True).logits[0]
    gpu = copy.deepcopy(model).to(DEV)
    enable_paged_attention(gpu)
    return gpu, ids, ref


def _close(got, want):
    err = (got.float().cpu() - want).abs()
    assert (err <= 2e-2 + 2e-2 * want.abs()).all(), f"max err {float(err.max()):.3e}"


def _state(mgr):
    return (sorted((rid, e.num_tokens, tuple(e.pages)) for rid, e in mgr._page_tables.items()), list(mgr._free_pages),
            [(p.allocated, p.ref_count) for p in mgr._pages], len(mgr._pending_compress))


@pytest.mark.parametrize("dtype", ["float32", "float16", "int8", "fp8"])
@pytest.mark.parametrize("had", [0, 5, 16])
def test_pool_that_runs_out_in_a_later_chunk(setting, dtype, had):
    model, ids, ref = setting
    print(f"[case] prefill out of pages in its second chunk, {dtype}, {had} tokens before", flush=True)
    mgr = _manager(dtype, max_pages=5)
    with torch.no_grad():
        if had:
            prefill_chunked(model, mgr, "x", ids[:, :had].to(DEV))
        before = _state(mgr)
        with pytest.raises(RuntimeError, match="no page left"):
            prefill_chunked(model, mgr, "x", ids[:, had:90].to(DEV), 32)
        assert _state(mgr) == before
        if dtype in ("float32", "float16"):  # and the rest of the prompt, as far as it fits
            _close(prefill_chunked(model, mgr, "x", ids[:, had:70].to(DEV), 32)[0], ref[69])
            _close(decode_step(model, mgr, ["x"], ids[0, 70:71].to(DEV))[0], ref[70])


@pytest.mark.parametrize("compression", [None, "turboquant"])
def test_model_that_raises(setting, compression):
    """A layer that raises after the first has written: the step's tokens are
    taken back, and the same step then gives what it should."""
    model, ids, ref = setting
    print(f"[case] raising model, compression {compression}", flush=True)
    mgr = _manager("float32", max_pages=16, kv_compression=compression)

    def stop(*args):
        raise ValueError("stop")

    with torch.no_grad():
        for rid, n in (("a", 11), ("b", 32)):
            prefill_chunked(model, mgr, rid, ids[:, :n].to(DEV))
        cache = PagedChunkCache(mgr, ["a", "b"])
        toks = torch.stack([ids[0, n:n + 9] for n in (11, 32)]).to(DEV)
        before = _state(mgr)
        hook = model.model.layers[1].register_forward_pre_hook(stop)
        try:
            for c in (None, cache):
                with pytest.raises(ValueError, match="stop"):
                    chunk_step(model, mgr, ["a", "b"], toks, c)
                assert _state(mgr) == before
            with pytest.raises(ValueError, match="stop"):
                prefill_chunked(model, mgr, "new", ids[:, :40].to(DEV), 16)
            assert _state(mgr) == before
        finally:
            hook.remove()
        for row, n in zip(chunk_step(model, mgr, ["a", "b"], toks, cache), (11, 32)):
            _close(row, ref[n:n + 9])
        mgr.flush_compression()


def test_model_with_a_sliding_window():
    """Its attention is refused in layer 0, after that layer's append."""
    print("[case] sliding window model", flush=True)
    torch.manual_seed(0)
    model = MistralForCausalLM(MistralConfig(**SIZES, sliding_window=32)).eval().to(DEV)
    enable_paged_attention(model)
    mgr = _manager()
    mgr.allocate("a")
    before = _state(mgr)
    with torch.no_grad():
        with pytest.raises(NotImplementedError, match="sliding"):
            prefill_chunked(model, mgr, "a", torch.zeros((1, 40), dtype=torch.long, device=DEV), 16)
        assert _state(mgr) == before
        with pytest.raises(NotImplementedError, match="sliding"):
            chunk_step(model, mgr, ["a"], torch.zeros((1, 4), dtype=torch.long, device=DEV))
    assert _state(mgr) == before


def test_caches_that_do_not_fit_the_step(setting):
    """A cache of another manager, or for single tokens, is not used."""
    model, ids, ref = setting
    print("[case] caches of another kind", flush=True)
    mgr, other = _manager(), _manager()
    with torch.no_grad():
        for m in (mgr, other):
            prefill_chunked(model, m, "a", ids[:, :11].to(DEV))
        before = _state(other)
        _close(chunk_step(model, mgr, ["a"], ids[:, 11:20].to(DEV), PagedChunkCache(other, ["a"]))[0], ref[11:20])
        _close(chunk_step(model, mgr, ["a"], ids[:, 20:25].to(DEV), PagedBatchCache(mgr, ["a"]))[0], ref[20:25])
    assert _state(other) == before and list(mgr.token_counts(["a"])) == [25]


def test_tokens_taken_back():
    """Tokens taken back one chunk after the other leave the pool's books as
    they were; a chunk whose requests have changed since is refused whole."""
    print("[case] take back", flush=True)
    mgr = _manager(max_pages=12)
    for rid in "ab":
        mgr.allocate(rid)
    states = [_state(mgr)]
    chunks = []
    for counts in ([5, 20], [0, 12], [40, 1]):
        chunks.append(mgr.append_chunk(["a", "b"], counts))
        states.append(_state(mgr))
    with pytest.raises(RuntimeError, match="append_chunk"):
        mgr._take_back(chunks[0])
    assert _state(mgr) == states[-1]
    for chunk, state in zip(chunks[::-1], states[-2::-1]):
        mgr._take_back(chunk)
        assert _state(mgr) == state
        with pytest.raises(RuntimeError, match="append_chunk"):
            mgr._take_back(chunk)
    chunk = mgr.append_chunk(["a"], [5])
    mgr.fork("a", "c")  # shares the page: it stays with the fork
    mgr._take_back(chunk)
    assert list(mgr.token_counts(["a", "c"])) == [0, 5] and len(mgr._free_pages) == 11
    assert mgr.append_chunk(["a"], [1]).places[0][0] != mgr._page_tables["c"].pages[0]


def test_block_table_after_tokens_taken_back():
    """A decode between an append and its undoing kept the pages that went
    back: the next one must not read them."""
    print("[case] block table after take back", flush=True)
    mgr = _manager(max_pages=6)
    gen = torch.Generator().manual_seed(2)
    for rid in "ab":
        mgr.allocate(rid)
    chunk = mgr.append_chunk(["a"], [20])
    q = torch.randn((1, 4, 64), generator=gen).to(DEV)
    mgr.compute_attention_decode(q, ["a"], 0)
    mgr._take_back(chunk)
    for rid, n in (("b", 16), ("a", 20)):
        k, v = (torch.randn((n, 2, 64), generator=gen).to(DEV) for _ in range(2))
        mgr.write_chunk(0, mgr.append_chunk([rid], [n]), k, v)
    want = torch.nn.functional.scaled_dot_product_attention(  # of a's 20 tokens
        q[0, :, None].cpu(), k.cpu().transpose(0, 1).repeat_interleave(2, 0), v.cpu().transpose(0, 1).repeat_interleave(2, 0))
    got = mgr.compute_attention_decode(q, ["a"], 0)[0].cpu()
    assert ((got - want[:, 0]).abs() <= 2e-3 + 1e-2 * want[:, 0].abs()).all()
