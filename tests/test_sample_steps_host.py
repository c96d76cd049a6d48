"""Decode and speculative steps around a model that is a plain function, on the
host: what they leave behind when they fail, and what the model gets.

The managers have a pool of one number, on the host; no call here reaches a
GPU, so that drawing a token always fails unless the test answers for it.
"""
import pytest
import torch

from vramancer_amd import sampling
from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_batch import PagedBatchCache, PagedChunkCache, decode_step, sample_step, speculative_step

V = 50


def _mgr(**kw):
    m = PagedKVCacheManager(PagedKVConfig(page_size=8, num_layers=2, num_kv_heads=2, head_dim=64, max_pages=8,
                                          device="cpu", **kw))
    m._gpu_pool = torch.zeros(1)
    for rid, n in (("a", 5), ("b", 8), ("c", 0)):
        m.allocate(rid, n)
    return m


class Model:
    """Begins the step in its cache as layer 0 does, keeps its ids, gives logits."""

    def __init__(self):
        self.seen, self.fail = [], None
        self.embeddings = torch.nn.Embedding(V, 4)

    def get_input_embeddings(self):
        return self.embeddings

    def __call__(self, ids, position_ids, past_key_values, use_cache):
        if self.fail == "early":
            raise ValueError("early")
        self.seen.append(ids.clone())
        if isinstance(past_key_values, PagedChunkCache):
            past_key_values._begin_chunk(ids.shape[1])
        else:
            past_key_values._begin_step()
        if self.fail == "late":
            raise ValueError("late")
        return (torch.zeros((*ids.shape, V)),)


def _state(m):
    return (sorted((rid, e.num_tokens, tuple(e.pages)) for rid, e in m._page_tables.items()), list(m._free_pages),
            [(p.allocated, p.ref_count) for p in m._pages], len(m._pending_compress))


@pytest.mark.parametrize("own_cache", [None, PagedBatchCache, PagedChunkCache])
@pytest.mark.parametrize("ids", [["a", "b", "c"], ["b"], ["c", "a"]])
def test_a_draw_that_fails_leaves_the_requests_as_they_were(ids, own_cache):
    m, model = _mgr(), Model()
    cache = own_cache and own_cache(m, ids)
    before = _state(m)
    for fail, text in ((None, "run on the GPU"), ("early", "early"), ("late", "late"), (None, "run on the GPU")):
        model.fail = fail
        with pytest.raises((RuntimeError, ValueError), match=text):
            sample_step(model, m, ids, torch.arange(len(ids)), torch.zeros(len(ids)), cache=cache)
        assert _state(m) == before
    model.fail = None
    decode_step(model, m, ids, torch.arange(len(ids)), cache)
    after = _state(m)
    assert after != before
    model.fail = "early"  # (the step before is no concern of this one)
    with pytest.raises(ValueError):
        sample_step(model, m, ids, torch.arange(len(ids)), torch.zeros(len(ids)), cache=cache)
    assert _state(m) == after


def test_a_step_that_answers_keeps_its_tokens(monkeypatch):
    m, model = _mgr(), Model()
    monkeypatch.setattr(sampling, "sample_tokens", lambda logits, u, **kw: torch.ones(3, dtype=torch.int64))
    cache = PagedBatchCache(m, ["a", "b", "c"])
    for step in range(1, 4):
        assert sample_step(model, m, ["a", "b", "c"], torch.arange(3), torch.zeros(3), cache=cache).tolist() == [1] * 3
        assert m.token_counts(["a", "b", "c"]).tolist() == [5 + step, 8 + step, step]


def test_a_request_that_changed_meanwhile_keeps_its_tokens(monkeypatch):
    m, model = _mgr(), Model()

    def draw(logits, u, **kw):
        m.append_token("a")
        raise RuntimeError("no")

    monkeypatch.setattr(sampling, "sample_tokens", draw)
    with pytest.raises(RuntimeError, match="no"):
        sample_step(model, m, ["a", "b"], torch.arange(2), torch.zeros(2))
    assert m.token_counts(["a", "b"]).tolist() == [7, 9]


def test_a_request_twice_in_a_step():
    m, model = _mgr(), Model()
    before = _state(m)
    with pytest.raises(RuntimeError, match="run on the GPU"):
        sample_step(model, m, ["a", "b", "a"], torch.arange(3), torch.zeros(3))
    assert _state(m) == before


def test_requests_without_a_token_do_not_reach_the_embeddings(monkeypatch):
    """A row of nothing but -inf or NaN gives token -1, which the loop hands to
    the next step: an index outside the embeddings ends a GPU process."""
    m, model = _mgr(), Model()
    none = torch.full((3,), -1, dtype=torch.int64)
    monkeypatch.setattr(sampling, "sample_tokens", lambda logits, u, **kw: none)
    pending = torch.tensor([4, -1, 0])
    pending = sample_step(model, m, ["a", "b", "c"], pending, torch.zeros(3))
    sample_step(model, m, ["a", "b", "c"], pending, torch.zeros(3))
    assert [x.flatten().tolist() for x in model.seen] == [[4, 0, 0], [0, 0, 0]]

    asked = []

    def verify(logits, drafts, *args, **kw):
        asked.append(drafts.tolist())
        return torch.full((3, 3), -1, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)

    monkeypatch.setattr(sampling, "verify_drafts", verify)
    drafts = torch.tensor([[1, V], [-1, 2], [3, 1 << 40]])
    for dtype in (torch.int64, torch.int32):
        tokens, accepted = speculative_step(model, m, ["a", "b", "c"], torch.tensor([-1, 7, -1], dtype=dtype), drafts, None,
                                            None)
        pending = tokens.gather(1, accepted.long()[:, None])[:, 0]
        assert pending.tolist() == [-1] * 3
        assert model.seen[-1].tolist() == [[0, 1, V - 1], [7, 0, 2], [0, 3, V - 1]] and model.seen[-1].dtype == dtype
    assert asked == [drafts.tolist()] * 2
