"""Steps that draw their tokens and fail, through a Hugging Face model: the same
step afterwards gives what it would have given without the failure (tokens and
pages are equal, kernels and inputs being the same)."""
import copy

import pytest
import torch
from transformers import LlamaConfig, LlamaForCausalLM

from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_batch import PagedBatchCache, enable_paged_attention, prefill, sample_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = dict(vocab_size=256, hidden_size=256, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, max_position_embeddings=256)


def _manager(dtype="float32", max_pages=40, PS=8, **kw):
    torch.manual_seed(7)  # (the compressor's signs)
    return PagedKVCacheManager(PagedKVConfig(page_size=PS, num_layers=2, num_kv_heads=2, head_dim=64,
                                             max_pages=max_pages, device=DEV, dtype=dtype, **kw))


@pytest.fixture(scope="module")
def model():
    cfg = LlamaConfig(**SIZES)
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    gpu = copy.deepcopy(LlamaForCausalLM(cfg).eval()).to(DEV)
    enable_paged_attention(gpu)
    return gpu


def _state(mgr):
    return (sorted((rid, e.num_tokens, tuple(e.pages)) for rid, e in mgr._page_tables.items()),
            list(mgr._free_pages), [(p.allocated, p.ref_count) for p in mgr._pages], len(mgr._pending_compress))


@pytest.mark.parametrize("compression", [None, "turboquant"])
@pytest.mark.parametrize("keep", [False, True])
def test_a_draw_that_fails_changes_nothing(model, compression, keep):
    ids = torch.randint(0, 256, (1, 16), generator=torch.Generator().manual_seed(9)).to(DEV)
    mgrs = [_manager("float16" if compression else "float32", kv_compression=compression) for _ in range(2)]
    rids = ["a", "b"]
    u = torch.tensor([0.3, 0.8], device=DEV)
    out = []
    with torch.no_grad():
        for disturbed, mgr in enumerate(mgrs):
            for rid, n in zip(rids, (5, 16)):
                mgr.allocate(rid)
                prefill(model, mgr, rid, ids[:, :n])
            cache = PagedBatchCache(mgr, rids) if keep else None
            pending = torch.tensor([1, 2], device=DEV)
            for step in range(3):
                before = _state(mgr)
                for bad in (dict(uniforms=u[:1]), dict(top_p=torch.rand(3, device=DEV)), dict(temperature="warm"),
                            dict(probs=torch.empty((2, 255), device=DEV)), dict(top_k=u)) if disturbed else ():
                    with pytest.raises((RuntimeError, ValueError)):
                        sample_step(model, mgr, rids, pending, cache=cache, **{"uniforms": u, **bad})
                    assert _state(mgr) == before
                pending = sample_step(model, mgr, rids, pending, u, temperature=0.9, top_p=0.9, cache=cache)
                out.append(pending.tolist())
            out.append(_state(mgr))
            mgr.flush_compression()
            out += [t.cpu().tolist() for r in rids for t in mgr.read_kv(r, 1)]
            out.append(None if compression is None else mgr._tq_slots.tolist())
    assert out[:len(out) // 2] == out[len(out) // 2:]
