"""The operators of a speculative step together: drafts through a Hugging Face
model and the page manager, and a captured step that makes its tables from
lengths that it advances itself.

Tokens are compared with the host reference on the logits that the step itself
gives (a token is a whole number), and logits with the model's own over the
whole text: 2e-2 + 2e-2 |ref|, as in test_gpu_chunk_steps.py."""
import copy

import pytest
import torch
from transformers import DynamicCache, LlamaConfig, LlamaForCausalLM

from sampling_reference import sample, verify
from vramancer_amd import paged_batch
from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_batch import (PagedChunkCache, chunk_step, decode_step, enable_paged_attention, prefill,
                                       sample_step, speculative_step)
from vramancer_amd.paged_chunk import chunk_tables, paged_attention_chunk, rope_append
from vramancer_amd.rope import rope_table
from vramancer_amd.sampling import sample_tokens, verify_drafts

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = dict(vocab_size=256, hidden_size=256, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
             num_key_value_heads=2, head_dim=64, max_position_embeddings=256)


def _manager(dtype="float32", max_pages=40, PS=8, **kw):
    return PagedKVCacheManager(PagedKVConfig(page_size=PS, num_layers=2, num_kv_heads=2, head_dim=64,
                                             max_pages=max_pages, device=DEV, dtype=dtype, **kw))


@pytest.fixture(scope="module")
def setting():
    cfg = LlamaConfig(**SIZES)
    cfg._attn_implementation = "eager"
    torch.manual_seed(0)
    model = LlamaForCausalLM(cfg).eval()
    gpu = copy.deepcopy(model).to(DEV)
    enable_paged_attention(gpu)
    ids = torch.randint(0, 256, (1, 60), generator=torch.Generator().manual_seed(9))
    return model, gpu, ids


def _state(mgr):
    return (sorted((rid, e.num_tokens, tuple(e.pages)) for rid, e in mgr._page_tables.items()),
            list(mgr._free_pages), [(p.allocated, p.ref_count) for p in mgr._pages], len(mgr._pending_compress))


def _texts(setting, mgr, lens):
    model, gpu, ids = setting
    texts = {}
    for rid, n in lens.items():
        mgr.allocate(rid)
        prefill(gpu, mgr, rid, ids[:, :n].to(DEV))
        texts[rid] = ids[0, :n].tolist()
    return texts


def test_speculative_steps(setting, monkeypatch):
    """Steps whose drafts are the model's greedy ones up to a point: the pages
    hold exactly the text, whatever was refused before."""
    model, gpu, ids = setting
    mgr = _manager()
    rids = ["a", "b", "c"]
    texts = _texts(setting, mgr, {"a": 5, "b": 16, "c": 23})
    pending = torch.tensor([7, 8, 9], device=DEV)
    gen = torch.Generator().manual_seed(3)
    cache = PagedChunkCache(mgr, rids)
    seen = {}
    real = paged_batch.chunk_step

    def spy(*args):
        seen["logits"] = real(*args)
        return seen["logits"]

    monkeypatch.setattr(paged_batch, "chunk_step", spy)
    all_accepted = []
    with torch.no_grad():
        for step in range(6):
            K = (3, 1, 4, 2, 0, 5)[step]
            drafts = torch.randint(0, 256, (3, K), generator=gen)
            for b, rid in enumerate(rids):  # some right drafts
                text = texts[rid] + [int(pending[b])]
                for i in range(min(K, (step + b) % 4)):
                    drafts[b, i] = int(model(torch.tensor([text])).logits[0, -1].argmax())
                    text.append(int(drafts[b, i]))
            ua, u = torch.rand((3, K), generator=gen), torch.rand(3, generator=gen)
            temp = torch.tensor([0.0, 0.3, 0.0])
            tokens, accepted = speculative_step(gpu, mgr, rids, pending, drafts.to(DEV), ua.to(DEV), u.to(DEV),
                                                temperature=temp.to(DEV), top_k=40, cache=cache)
            want = verify(seen["logits"], drafts, ua, u, temperature=temp, top_k=40)
            assert tokens.cpu().tolist() == want[0].tolist() and accepted.cpu().tolist() == want[1].tolist()
            all_accepted += accepted.tolist()
            for b, rid in enumerate(rids):
                n = int(accepted[b])
                full = texts[rid] + [int(pending[b])] + drafts[b].tolist()
                ref = model(torch.tensor([full])).logits[0, len(texts[rid]):]
                err = (seen["logits"][b].cpu() - ref).abs()
                assert (err <= 2e-2 + 2e-2 * ref.abs()).all()
                texts[rid] = full[:len(texts[rid]) + 1 + n]
            pending = tokens.gather(1, accepted.long()[:, None])[:, 0]
            assert list(mgr.token_counts(rids)) == [len(texts[r]) for r in rids]
            assert [len(mgr._page_tables[r].pages) for r in rids] == [-(-len(texts[r]) // 8) for r in rids]
        got = decode_step(gpu, mgr, rids, pending)
    assert max(all_accepted) >= 3 and min(all_accepted) == 0
    for b, rid in enumerate(rids):
        ref = model(torch.tensor([texts[rid] + [int(pending[b])]])).logits[0, -1]
        err = (got[b].cpu() - ref).abs()
        assert (err <= 2e-2 + 2e-2 * ref.abs()).all()


def test_sample_step(setting):
    model, gpu, _ = setting
    mgr = _manager()
    _texts(setting, mgr, {"a": 5, "b": 16})
    other = _manager()
    _texts(setting, other, {"a": 5, "b": 16})
    u = torch.tensor([0.3, 0.8], device=DEV)
    probs = torch.empty((2, 256), device=DEV)
    ids = torch.tensor([1, 2], device=DEV)
    with torch.no_grad():
        got = sample_step(gpu, mgr, ["a", "b"], ids, u, temperature=0.9, top_p=0.8, probs=probs)
        logits = decode_step(gpu, other, ["a", "b"], ids)
    want, rows = sample(logits, u, temperature=0.9, top_p=0.8)
    assert got.cpu().tolist() == want.tolist()
    assert ((probs[0].cpu() > 0).numpy() == (rows[0] > 0)).all()


def test_a_step_that_fails_changes_nothing(setting):
    _, gpu, _ = setting
    mgr = _manager()
    _texts(setting, mgr, {"a": 5, "b": 16})
    before = _state(mgr)
    ids, drafts = torch.tensor([1, 2], device=DEV), torch.zeros((2, 9), dtype=torch.long, device=DEV)
    good = dict(accept_uniforms=torch.rand((2, 9), device=DEV), draw_uniforms=torch.rand(2, device=DEV))
    with torch.no_grad():
        for bad in (dict(accept_uniforms=torch.rand((2, 8), device=DEV)), dict(top_p=torch.rand(3, device=DEV)),
                    dict(draft_probs=torch.rand((2, 9, 100), device=DEV))):
            with pytest.raises(RuntimeError):
                speculative_step(gpu, mgr, ["a", "b"], ids, drafts, **{**good, **bad})
            assert _state(mgr) == before
        with pytest.raises(RuntimeError, match="drafts must be"):
            speculative_step(gpu, mgr, ["a", "b"], ids, drafts[:1], **good)
        # drafts outside the vocabulary end the list
        drafts[:, 1] = -1
        drafts[:, 2] = 256
        tokens, accepted = speculative_step(gpu, mgr, ["a", "b"], ids, drafts, **good)
    assert int(accepted.max()) <= 1 and (tokens.gather(1, accepted.long()[:, None]) >= 0).all()


@pytest.mark.parametrize("counts,kept", [([3, 0, 9], [1, 0, 1]), ([8, 8, 8], [0, 8, 3]), ([1, 1, 1], [0, 0, 0]),
                                         ([2, 5, 17], [2, 5, 17])])
def test_keep_chunk(counts, kept):
    """As if the refused tokens had never been appended: tokens and pages of each
    request (which pages they are goes by the order in which they were taken),
    the number of free ones, the compression queue; the pool holds what was
    kept."""
    gen = torch.Generator().manual_seed(1)
    states, codes = [], []
    rows = torch.randn((sum(counts), 2, 64), generator=gen).half().to(DEV)
    at = [0, counts[0], counts[0] + counts[1]]
    for keep in (True, False):
        torch.manual_seed(7)
        mgr = _manager("float16", kv_compression="turboquant")
        for rid, n in (("a", 5), ("b", 8), ("c", 15)):
            mgr.allocate(rid, n)
        if keep:
            chunk = mgr.append_chunk(["a", "b", "c"], counts)
            for layer in range(2):
                mgr.write_chunk(layer, chunk, rows, rows + 1)
            mgr.keep_chunk(chunk, kept)
            if kept != counts:
                with pytest.raises(RuntimeError, match="has changed"):
                    mgr.write_chunk(0, chunk, rows, rows)
        else:
            chunk = mgr.append_chunk(["a", "b", "c"], kept)
            pick = torch.tensor([a + i for a, k in zip(at, kept) for i in range(k)], dtype=torch.long, device=DEV)
            for layer in range(2):
                mgr.write_chunk(layer, chunk, rows[pick], rows[pick] + 1)
        lists = {r: list(mgr._page_tables[r].pages) for r in "abc"}
        used = sum(lists.values(), [])
        assert sorted(used + mgr._free_pages) == list(range(40)) and len(set(used)) == len(used)
        assert all(mgr._pages[p].ref_count == 1 for p in used) and not any(mgr._pages[p].allocated for p in mgr._free_pages)
        states.append([(r, mgr._page_tables[r].num_tokens, len(lists[r])) for r in "abc"] + [len(mgr._pending_compress)])
        mgr.flush_compression()
        assert not mgr._tq_slots[mgr._free_pages].any()
        codes.append([mgr._tq_slots[lists[r]].tolist() for r in "abc"])
        reads = [mgr.read_kv(r, 1) for r in "abc"]
        states.append([(k.cpu().tolist(), v.cpu().tolist()) for k, v in reads])
    assert states[0] == states[2] and states[1] == states[3] and codes[0] == codes[1]


def test_keep_chunk_refusals():
    mgr, other = _manager(), _manager()
    mgr.allocate("a"), other.allocate("a")
    chunk = mgr.append_chunk(["a"], [4])
    before = _state(mgr)
    for bad in ([5], [-1], [1, 1], []):
        with pytest.raises(RuntimeError, match="keep_chunk takes a number"):
            mgr.keep_chunk(chunk, bad)
    with pytest.raises(RuntimeError, match="this manager"):
        other.keep_chunk(chunk, [1])
    assert _state(mgr) == before
    mgr.append_token("a")
    with pytest.raises(RuntimeError, match="has changed"):
        mgr.keep_chunk(chunk, [1])
    with pytest.raises(RuntimeError, match="has changed"):
        mgr.keep_chunk(chunk, [4])


def test_keep_chunk_after_a_reservation():
    """Pages that reserve gave out behind a chunk's stay the request's."""
    mgr = _manager()
    mgr.allocate("a"), mgr.allocate("b")
    chunk = mgr.append_chunk(["a", "b"], [9, 3])
    table, past = mgr.reserve(["a"], [20])
    assert past.tolist() == [9] and table.tolist() == [mgr._page_tables["a"].pages]
    before = _state(mgr)
    for call in (lambda: mgr.keep_chunk(chunk, [1, 3]), lambda: mgr._take_back(chunk)):
        with pytest.raises(RuntimeError, match="has changed"):
            call()
        assert _state(mgr) == before
    mgr.keep_chunk(chunk, [9, 3])  # (takes nothing back)
    assert _state(mgr) == before
    held = list(mgr._page_tables["a"].pages)
    chunk = mgr.append_chunk(["a"], [9])  # into reserved pages: none of its own to give back
    mgr.keep_chunk(chunk, [2])
    assert mgr._page_tables["a"].pages == held and list(mgr.token_counts(["a"])) == [11]


def test_reserve_and_commit():
    mgr = _manager(max_pages=10)
    for rid, n in (("a", 5), ("b", 16)):
        mgr.allocate(rid, n)
    before = _state(mgr)
    for ids, counts, kind in ((["a", "x"], [1, 1], KeyError), (["a", "a"], [1, 1], RuntimeError),
                              (["a"], [-1], RuntimeError), (["a", "b"], [40, 40], RuntimeError),
                              (["a"], [1, 2], RuntimeError)):
        with pytest.raises(kind):
            mgr.reserve(ids, counts)
        assert _state(mgr) == before
    table, past = mgr.reserve(["b", "a"], [9, 2])
    assert past.tolist() == [16, 5] and list(mgr.token_counts(["a", "b"])) == [5, 16]
    pages = {r: mgr._page_tables[r].pages for r in "ab"}
    assert [len(pages["a"]), len(pages["b"])] == [1, 4]
    assert table.tolist() == [pages["b"], pages["a"] + [-1] * 3]
    with pytest.raises(RuntimeError, match="prefix"):
        mgr.try_prefix_cache("b", list(range(8)))
    fork = mgr.fork("b", "f")
    assert fork.pages == pages["b"][:2] and mgr._pages[pages["b"][2]].ref_count == 1
    with pytest.raises(RuntimeError, match="pages for 16 more"):
        mgr.commit(["a", "b"], [1, 17])
    with pytest.raises(KeyError):
        mgr.commit(["a", "x"], [1, 1])
    assert list(mgr.token_counts(["a", "b"])) == [5, 16]
    mgr.commit(["a", "b"], [3, 4])
    assert list(mgr.token_counts(["a", "b"])) == [8, 20]
    assert mgr.append_token("b") == (pages["b"][2], 4)  # reserved pages are the next ones
    chunk = mgr.append_chunk(["b"], [13])
    assert chunk.places[-1] == (mgr._page_tables["b"].pages[4], 1) and len(mgr._page_tables["b"].pages) == 5
    assert mgr.free("f") == 0 and mgr.free("b") == 5 and mgr.free("a") == 1
    assert sorted(mgr._free_pages) == list(range(10))


def test_captured_speculative_layer():
    """One captured step of one layer: tables from lengths, append, attention,
    logits, verification, lengths advanced by what was accepted.  Every replay
    equals the same step made with host tables, through another manager."""
    H, KH, D, PS, V, K, B = 4, 2, 64, 8, 300, 3, 3
    gen = torch.Generator().manual_seed(5)
    mk = lambda *s: torch.randn(s, generator=gen).to(DEV)  # noqa: E731
    emb, wk, wv, wq, head = mk(V, H * D), mk(H * D, KH * D) / 16, mk(H * D, KH * D) / 16, mk(H * D, H * D) / 16, mk(H * D, V)
    rids = ["a", "b", "c"]
    mgr, host = _manager(max_pages=40, PS=PS), _manager(max_pages=40, PS=PS)
    for m in (mgr, host):
        for r in rids:
            m.allocate(r)
    steps = 5
    table, past = mgr.reserve(rids, [steps * (K + 1)] * B)
    angles = rope_table(128, D, device=DEV)
    N = B * (K + 1)
    ids = torch.zeros((B, K + 1), dtype=torch.long, device=DEV)
    ua, u = torch.zeros((B, K), device=DEV), torch.zeros(B, device=DEV)
    counts = torch.full((B,), K + 1, dtype=torch.int32, device=DEV)

    def layer(pool, page_table, context_lens, cu):
        x = emb[ids.view(-1)]
        q = rope_append((x @ wq).view(N, H, D), (x @ wk).view(N, KH, D), (x @ wv).view(N, KH, D), pool, page_table,
                        context_lens, cu, 0, angles)
        y = paged_attention_chunk(q, pool, page_table, context_lens, cu, 0)
        logits = (y.view(N, H * D) @ head).view(B, K + 1, V)
        return verify_drafts(logits, ids[:, 1:], ua, u, temperature=0.7, top_k=50)

    tables = chunk_tables(table, past, counts, N, PS)

    def step():
        chunk_tables(table, past, counts, N, PS, out=tables)
        tokens, accepted = layer(mgr.gpu_pool, tables.page_table, tables.context_lens, tables.cu_seqlens)
        past.add_(accepted + 1)
        return tokens, accepted

    step()  # (warm, on what the replays start from: undone below)
    past.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, accepted = step()
    torch.cuda.synchronize()
    mgr.gpu_pool.zero_()
    past.zero_()
    pending = torch.tensor([5, 6, 7], device=DEV)
    total = torch.zeros(B, dtype=torch.long)
    for i in range(steps):
        ids[:, 0] = pending
        ids[:, 1:] = torch.randint(0, V, (B, K), generator=gen).to(DEV)
        if i % 2:  # drafts that the layer is likely to accept: those of the last step
            ids[:, 1:] = tokens[:, :K].clamp(min=0)
        ua.copy_(torch.rand((B, K), generator=gen) * 0.02)
        u.copy_(torch.rand(B, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        chunk = host.append_chunk(rids, [K + 1] * B)
        want, kept = layer(host.gpu_pool, chunk.page_table, chunk.context_lens, chunk.cu_seqlens)
        assert torch.equal(tokens, want) and torch.equal(accepted, kept), f"replay {i}"
        host.keep_chunk(chunk, [1 + n for n in kept.tolist()])
        total += kept.cpu().long() + 1
        assert past.tolist() == total.tolist() == list(host.token_counts(rids))
        pending = tokens.gather(1, accepted.long()[:, None])[:, 0]
    mgr.commit(rids, total.tolist())
    for r in rids:
        for layer_kv in zip(mgr.read_kv(r, 0), host.read_kv(r, 0)):
            assert torch.equal(*layer_kv)
    # the draft's own draws, from the same kind of logits
    assert sample_tokens(emb[:2] @ head, u[:2]).shape == (2,)
    assert chunk_step is paged_batch.chunk_step
