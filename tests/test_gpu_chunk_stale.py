"""Batches of append_chunk whose requests have changed since are refused: their
pages may be another request's."""
import pytest
import torch

from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _manager():
    return PagedKVCacheManager(PagedKVConfig(page_size=16, num_layers=2, num_kv_heads=2, head_dim=64, max_pages=8,
                                             device=DEV, dtype="float32"))


def _rows(n):
    return tuple(torch.randn((n, h, 64), device=DEV) for h in (4, 2, 2))


@pytest.mark.parametrize("change", ["free", "freed and back", "append", "decode", "fork over", "another manager"])
def test_changed_requests_are_refused(change):
    print(f"[case] stale chunk: {change}", flush=True)
    mgr = _manager()
    for rid in "abc":
        mgr.allocate(rid)
    chunk = mgr.append_chunk(["a", "b"], [5, 20])
    q, k, v = _rows(25)
    mgr.write_chunk(0, chunk, k, v)
    mgr.append_chunk(["c"], [3])  # another request's change does not matter
    mgr.write_chunk(1, chunk, k, v)
    mgr.compute_attention_chunk(q, chunk, 1)
    user = mgr
    if change.startswith("free"):
        mgr.free("b")
    if change == "freed and back":
        mgr.allocate("b", 20)
    if change == "append":
        mgr.append_chunk(["a"], [1])
    if change == "decode":
        mgr.append_tokens(["b"])
    if change == "fork over":
        mgr.fork("c", "a")
    if change == "another manager":
        user = _manager()
        for rid in "abc":
            user.allocate(rid)
        user.append_chunk(["a", "b"], [5, 20])
        user.append_chunk(["c"], [3])
    before = user.gpu_pool.clone()
    with pytest.raises(RuntimeError, match="append_chunk"):
        user.write_chunk(0, chunk, k, v)
    with pytest.raises(RuntimeError, match="append_chunk"):
        user.compute_attention_chunk(q, chunk, 0)
    assert torch.equal(user.gpu_pool, before)


def test_batches_made_by_hand():
    """They have no manager to ask: the pages are the caller's concern."""
    mgr = _manager()
    mgr.allocate("a")
    made = mgr.append_chunk(["a"], [5])
    by_hand = type(made)(made.request_ids, made.counts, made.page_table, made.context_lens, made.cu_seqlens, made.places)
    q, k, v = _rows(5)
    mgr.append_chunk(["a"], [1])
    mgr.write_chunk(0, by_hand, k, v)
    assert mgr.compute_attention_chunk(q, by_hand, 0).isfinite().all()
