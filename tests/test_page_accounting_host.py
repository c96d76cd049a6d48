"""The page manager's books when tokens are taken back, on the host: whose
pages they are, and that what is refused changes nothing.

The managers have a pool of one number, on the host, to put their tables
beside; no call here reaches a GPU.
"""
import pytest
import torch

from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig


def _mgr(PS=8, max_pages=8, **kw):
    m = PagedKVCacheManager(PagedKVConfig(page_size=PS, num_layers=2, num_kv_heads=2, head_dim=64, max_pages=max_pages,
                                          device="cpu", **kw))
    m._gpu_pool = torch.zeros(1)
    return m


def _state(m):
    return (sorted((rid, e.num_tokens, tuple(e.pages)) for rid, e in m._page_tables.items()), list(m._free_pages),
            [(p.allocated, p.ref_count) for p in m._pages], len(m._pending_compress))


def _refused(m, *calls, match="has changed"):
    before = _state(m)
    for call in calls:
        with pytest.raises(RuntimeError, match=match):
            call()
        assert _state(m) == before


@pytest.mark.parametrize("more", [0, 3, 7, 20])
def test_tokens_behind_which_pages_were_reserved_stay(more):
    """9 tokens on two pages of 8: up to 7 more fit the second one, and a
    reservation for them (or for none) takes no page.  Its table names the
    batch's own pages, and its lengths count the batch's tokens."""
    m = _mgr()
    m.allocate("a"), m.allocate("b")
    chunk = m.append_chunk(["a", "b"], [9, 3])
    table, past = m.reserve(["a"], [more])
    assert past.tolist() == [9] and table[0, :2].tolist() == m._page_tables["a"].pages[:2]
    _refused(m, lambda: m.keep_chunk(chunk, [1, 3]), lambda: m.keep_chunk(chunk, [8, 0]), lambda: m._take_back(chunk))
    m.keep_chunk(chunk, [9, 2])  # (b was not reserved for)
    assert list(m.token_counts(["a", "b"])) == [9, 2]


def test_tokens_in_reserved_pages_stay_behind_a_second_reservation():
    m = _mgr()
    m.allocate("a")
    m.reserve(["a"], [40])
    chunk = m.append_chunk(["a"], [9])  # (no page is added for them)
    _, past = m.reserve(["a"], [20])
    assert past.tolist() == [9]
    _refused(m, lambda: m.keep_chunk(chunk, [2]), lambda: m._take_back(chunk))
    m.keep_chunk(chunk, [9])
    held = list(m._page_tables["a"].pages)
    chunk = m.append_chunk(["a"], [9])
    m.keep_chunk(chunk, [2])  # (reserved before it, not since)
    assert m._page_tables["a"].pages == held and list(m.token_counts(["a"])) == [11]


def test_a_reservation_that_is_refused_changes_nothing():
    m = _mgr()
    m.allocate("a"), m.allocate("b")
    chunk = m.append_chunk(["a", "b"], [9, 3])
    for ids, counts in ((["a", "b"], [100, 1]), (["a", "a"], [1, 1]), (["a"], [-1])):
        _refused(m, lambda: m.reserve(ids, counts), match=".")
    m.keep_chunk(chunk, [1, 3])
    assert list(m.token_counts(["a", "b"])) == [1, 3] and len(m._page_tables["a"].pages) == 1
