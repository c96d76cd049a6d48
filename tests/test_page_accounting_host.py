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


@pytest.mark.parametrize("had", [0, 2])
@pytest.mark.parametrize("kept", [0, 1, 3])
def test_tokens_that_a_fork_has_stay(kept, had):
    """A fork has the batch's tokens and shares their page: the request's next
    token must not go over them."""
    m = _mgr()
    m.allocate("a", had), m.allocate("b")
    chunk = m.append_chunk(["a", "b"], [4, 4])
    m.fork("a", "f")
    page = m._page_tables["a"].pages[0]
    if kept + had == 0:  # (all tokens of a page that came with them: it is the fork's alone then)
        m.keep_chunk(chunk, [kept, 4])
        assert m._page_tables["a"].pages == [] and m._page_tables["f"].pages == [page]
        assert m.append_token("a")[0] != page
        return
    _refused(m, lambda: m.keep_chunk(chunk, [kept, 4]))
    if had:
        _refused(m, lambda: m._take_back(chunk))
    m.keep_chunk(chunk, [4, kept])
    assert list(m.token_counts(["a", "b", "f"])) == [had + 4, kept, had + 4]
    assert m.append_token("a") == (page, had + 4)  # behind the fork's last token


@pytest.mark.parametrize("kept,fits", [(16, True), (9, False), (8, True), (3, False), (0, True)])
def test_tokens_of_whole_pages_go(kept, fits):
    m = _mgr()
    m.allocate("a", 16)
    chunk = m.append_chunk(["a"], [20])  # three pages of its own
    m.fork("a", "f")
    if not fits:
        _refused(m, lambda: m.keep_chunk(chunk, [kept]))
        return
    held = list(m._page_tables["a"].pages)
    m.keep_chunk(chunk, [kept])
    assert m._page_tables["a"].pages == held[:2 + kept // 8] and m._page_tables["f"].pages == held
    assert m.append_token("a")[0] not in held and len(m._free_pages) == 2


def test_pages_that_were_there_before_the_tokens():
    """Reserved pages stay the request's when their tokens are taken back, so
    that a fork must not have those."""
    m = _mgr()
    m.allocate("a")
    m.reserve(["a"], [16])
    chunk = m.append_chunk(["a"], [16])
    m.fork("a", "f")
    _refused(m, lambda: m.keep_chunk(chunk, [8]), lambda: m.keep_chunk(chunk, [0]), lambda: m._take_back(chunk))
    m.free("f")
    m.keep_chunk(chunk, [8])  # (nobody else has them any more)
    assert list(m.token_counts(["a"])) == [8] and len(m._page_tables["a"].pages) == 2


def test_forks_made_before():
    m = _mgr()
    m.allocate("a", 8)
    m.fork("a", "f")
    chunk = m.append_chunk(["a", "f"], [3, 4])  # (a page of its own for each)
    m.keep_chunk(chunk, [1, 2])
    assert list(m.token_counts(["a", "f"])) == [9, 10]
    chunk = m.append_chunk(["f"], [2])
    m.fork("f", "g")
    _refused(m, lambda: m.keep_chunk(chunk, [1]))
    assert m.fork("missing", "h") is None


def test_a_fork_of_pages_that_are_taken_back_whole():
    m = _mgr(PS=16, max_pages=12)
    m.allocate("a")
    chunk = m.append_chunk(["a"], [5])
    m.fork("a", "c")
    m._take_back(chunk)
    assert list(m.token_counts(["a", "c"])) == [0, 5] and len(m._free_pages) == 11
    assert m.append_chunk(["a"], [1]).places[0][0] != m._page_tables["c"].pages[0]


def test_no_reservations_with_compression():
    """What steps over reserved pages store does not enter the compression
    queue: refused before there are such pages, not when they are counted."""
    m = _mgr(kv_compression="turboquant")
    m.allocate("a")
    for n in (0, 3, 9):
        _refused(m, lambda: m.reserve(["a"], [n]), match="kv_compression")
    _refused(m, lambda: m.commit(["a"], [1]), match="kv_compression")
    assert m.append_chunk(["a"], [9]).places[0][1] == 0


def test_prefixes_once_no_reserved_page_is_left():
    """A prefix can follow when the reserved pages hold tokens, however those
    came; until then it is refused, and a fork does not get the empty ones."""
    m = _mgr()
    m.allocate("a")
    m.reserve(["a"], [8])
    _refused(m, lambda: m.try_prefix_cache("a", list(range(8))), match="reserved pages")
    assert m.fork("a", "f").pages == []
    chunk = m.append_chunk(["a"], [8])
    m.keep_chunk(chunk, [0])
    _refused(m, lambda: m.try_prefix_cache("a", list(range(8))), match="reserved pages")
    m.commit(["a"], [0])
    assert m.fork("a", "g").pages == []
    m.append_chunk(["a"], [5])
    assert m.fork("a", "h").pages == m._page_tables["a"].pages
    assert m.try_prefix_cache("a", list(range(8))) == 0 and list(m.token_counts(["a"])) == [16]
    for _ in range(2):
        m.allocate("b")
        m.reserve(["b"], [8])
        for t in range(8):
            m.append_token("b")
        assert m.try_prefix_cache("b", list(range(8))) == 8  # (a's page)
        m.free("b")


def test_commit_leaves_reserved_pages_reserved_while_tokens_can_be_taken_back():
    m = _mgr()
    m.allocate("a")
    m.reserve(["a"], [8])
    chunk = m.append_chunk(["a"], [8])
    m.commit(["a"], [0])  # (no reserved page is left at the moment)
    m.keep_chunk(chunk, [0])
    assert m.fork("a", "f").pages == []
    _refused(m, lambda: m.try_prefix_cache("a", list(range(8))), match="reserved pages")


@pytest.mark.parametrize("tokens,pages", [(1, 1), (8, 1), (9, 2), (24, 3)])
def test_turbo_attention_compresses_pages_with_tokens_only(tokens, pages, monkeypatch):
    """Pages behind a request's last token hold nothing to compress: codes made
    of them would stay when rows are stored there."""
    m = _mgr(kv_compression="turboquant")
    held = list(m.allocate("a", 24).pages)
    m._page_tables["a"].num_tokens = tokens
    seen = []
    monkeypatch.setattr(m, "_ensure_compressed", lambda ids, layer: seen.append(("made", list(ids), layer)))
    monkeypatch.setattr(m, "_turbo_decode", lambda q, lists, n, layer, scale: seen.append((lists, n)) or [q[0]])
    m.compute_attention_turbo(torch.zeros((4, 64)), "a", 1)
    assert seen == [("made", held[:pages], 1), ([held[:pages]], [tokens])]
