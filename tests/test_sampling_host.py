"""Refusals and sizes of the sampling operators and of chunk_tables on the
host: no call here reaches a GPU."""
import numpy as np
import pytest
import torch

from sampling_reference import distribution, pick, verify
from vramancer_amd import _lib
from vramancer_amd.paged_chunk import ChunkTables, chunk_tables
from vramancer_amd.sampling import _param, _params, sample_tokens, verify_drafts


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _sample(lib, **kw):
    a = dict(logits=16, dt=_lib.VRM_SRC_F32, stride=1000, u=16, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0,
             probs=None, tokens=16, ws=16, wsb=1 << 33, N=4, V=1000)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.vrm_sample_tokens(*a.values(), None)


def _verify(lib, **kw):
    a = dict(logits=16, dt=_lib.VRM_SRC_BF16, stride=1000, cu=None, drafts=16, db=8, q=16, qb=3000, qk=1000, ua=16, u=16,
             t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0, tokens=16, accepted=16, ws=16, wsb=1 << 33, N=8, B=2,
             K=3, V=1000)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.vrm_verify_drafts(*a.values(), None)


def _tables(lib, **kw):
    a = dict(table=16, stride=8, R=4, W=8, past=16, counts=16, requests=16, B=2, N=5, PS=16, pt=16, max_pp=8, cl=16, cu=16,
             pos=16, page=16, slot=16, seq=16)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.vrm_chunk_tables(*a.values(), None)


@pytest.mark.parametrize("bad,rc,text", [
    (dict(logits=None), -1, b"null"), (dict(u=None), -1, b"null"), (dict(tokens=None), -1, b"null"),
    (dict(N=-1), -1, b"sizes"), (dict(V=0), -1, b"sizes"), (dict(stride=-1), -1, b"sizes"), (dict(dt=3), -1, b"dtype"),
    (dict(V=(1 << 24) + 1), -2, b"above"), (dict(N=1 << 28), -2, b"too many"), (dict(ws=None), -3, b"workspace"),
    (dict(wsb=8), -3, b"workspace"), (dict(ws=8), -1, b"aligned")])
def test_sample_refusals(lib, bad, rc, text):
    assert _sample(lib, **bad) == rc and text in lib.vrm_last_error()


@pytest.mark.parametrize("bad,rc,text", [
    (dict(logits=None), -1, b"null"), (dict(drafts=None), -1, b"null"), (dict(ua=None), -1, b"null"),
    (dict(u=None), -1, b"null"), (dict(tokens=None), -1, b"null"), (dict(accepted=None), -1, b"null"),
    (dict(N=7), -1, b"rows"), (dict(N=-1, cu=16), -1, b"rows"), (dict(db=2), -1, b"bytes"), (dict(qk=-1), -1, b"stride"),
    (dict(K=-1), -1, b"sizes"), (dict(B=-1), -1, b"sizes"), (dict(V=0), -1, b"sizes"), (dict(dt=7), -1, b"dtype"),
    (dict(B=1 << 20, K=1 << 20, cu=16), -2, b"too many"), (dict(wsb=64), -3, b"workspace")])
def test_verify_refusals(lib, bad, rc, text):
    assert _verify(lib, **bad) == rc and text in lib.vrm_last_error()


@pytest.mark.parametrize("bad,rc,text", [
    (dict(table=None), -1, b"null"), (dict(past=None), -1, b"null"), (dict(counts=None), -1, b"null"),
    (dict(pt=None), -1, b"null"), (dict(cl=None), -1, b"null"), (dict(cu=None), -1, b"null"), (dict(pos=None), -1, b"null"),
    (dict(page=None), -1, b"null"), (dict(slot=None), -1, b"null"), (dict(seq=None), -1, b"null"),
    (dict(PS=0), -1, b"sizes"), (dict(N=-1), -1, b"sizes"), (dict(B=-1), -1, b"sizes"), (dict(R=-1), -1, b"sizes"),
    (dict(max_pp=-1), -1, b"sizes"), (dict(stride=-8), -1, b"sizes"), (dict(B=5, requests=None), -1, b"requests"),
    (dict(B=1 << 30, max_pp=1 << 20), -2, b"too many")])
def test_tables_refusals(lib, bad, rc, text):
    assert _tables(lib, **bad) == rc and text in lib.vrm_last_error()


_MB = 1 << 20  # (distinct places for every argument of a call that never runs)


@pytest.mark.parametrize("over", [
    dict(probs=_MB), dict(probs=_MB + 15996), dict(probs=_MB - 12), dict(tokens=_MB + 8), dict(tokens=2 * _MB),
    dict(tokens=3 * _MB - 16, t=3 * _MB), dict(tokens=3 * _MB, k=3 * _MB), dict(probs=3 * _MB, p=3 * _MB + 8),
    dict(ws=_MB + 1024), dict(ws=2 * _MB)])
def test_sample_outputs_on_inputs(lib, over):
    a = dict(logits=_MB, u=2 * _MB, tokens=5 * _MB, ws=6 * _MB, wsb=_MB)
    assert _sample(lib, **{**a, **over}) == -1 and b"overlap" in lib.vrm_last_error()


@pytest.mark.parametrize("over", [
    dict(tokens=2 * _MB), dict(tokens=2 * _MB - 8), dict(tokens=_MB), dict(tokens=3 * _MB + 23996), dict(tokens=4 * _MB),
    dict(accepted=5 * _MB + 4), dict(accepted=9 * _MB + 8, cu=9 * _MB), dict(accepted=9 * _MB, t=9 * _MB + 4),
    dict(accepted=9 * _MB, k=9 * _MB), dict(accepted=9 * _MB, p=9 * _MB), dict(ws=2 * _MB)])
def test_verify_outputs_on_inputs(lib, over):
    a = dict(logits=_MB, drafts=2 * _MB, q=3 * _MB, ua=4 * _MB, u=5 * _MB, tokens=6 * _MB, accepted=7 * _MB, ws=8 * _MB,
             wsb=_MB)
    assert _verify(lib, **{**a, **over}) == -1 and b"overlap" in lib.vrm_last_error()


@pytest.mark.parametrize("over", [
    dict(cl=2 * _MB), dict(cl=2 * _MB - 4), dict(pt=_MB), dict(pt=_MB + 124), dict(cu=3 * _MB), dict(pos=2 * _MB + 12),
    dict(page=4 * _MB + 4), dict(slot=3 * _MB + 4), dict(seq=4 * _MB - 16)])
def test_tables_outputs_on_inputs(lib, over):
    a = dict(table=_MB, past=2 * _MB, counts=3 * _MB, requests=4 * _MB, pt=5 * _MB, cl=6 * _MB, cu=7 * _MB, pos=8 * _MB,
             page=9 * _MB, slot=10 * _MB, seq=11 * _MB)
    assert _tables(lib, **{**a, **over}) == -1 and b"overlap" in lib.vrm_last_error()


def test_nothing_to_do(lib):
    assert _sample(lib, N=0, logits=None, tokens=None, u=None, ws=None) == 0
    assert _verify(lib, B=0, N=0, logits=None, tokens=None, u=None, ws=None) == 0


def test_workspaces_grow_with_the_call(lib):
    sample, ver = lib.vrm_sample_workspace_bytes, lib.vrm_verify_workspace_bytes
    assert 0 < sample(1, 1, 0, 0) <= sample(1, 1, 0, 1) <= sample(1, 1, 1, 1)
    for V in (1000, 8192, 8193, 200000):
        assert sample(64, V, 1, 1) >= sample(64, V, 0, 0) > sample(63, V, 0, 0) - 256
        assert ver(64, 4, V, 1) > ver(64, 4, V, 0) >= ver(64, 3, V, 0)
    assert sample(4, (1 << 24) + 1, 1, 1) == 0 and ver(-1, 2, 10, 0) == 0


@pytest.mark.parametrize("B,K,V", [(5000, 3, 8000), (9000, 3, 1000), (1 << 20, 1, 17), (3, 4, 8192), (3, 4, 8193),
                                   (300, 1, 150000)])
def test_a_workspace_with_filters_is_enough_without(lib, B, K, V):
    sample, ver = lib.vrm_sample_workspace_bytes, lib.vrm_verify_workspace_bytes
    assert ver(B, K, V, 1) >= ver(B, K, V, 0) >= ver(B, K, V - 1, 0) and ver(B, K, V, 1) >= ver(B, K, V - 1, 1)
    assert sample(B, V, 1, 1) >= max(sample(B, V, 0, 1), sample(B, V, 1, 0), sample(B, V - 1, 1, 1))


def test_python_refusals():
    x, u = torch.zeros((2, 5)), torch.zeros(2)
    with pytest.raises(RuntimeError, match="run on the GPU"):
        sample_tokens(x, u)
    with pytest.raises(RuntimeError, match="run on the GPU"):
        verify_drafts(torch.zeros((2, 3, 5)), torch.zeros((2, 2), dtype=torch.int64), torch.zeros((2, 2)), u)
    table, lens = torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="run on the GPU"):
        chunk_tables(table, lens, lens, 3, 16)
    for bad in (dict(num_rows=-1), dict(page_size=0), dict(max_pages=-1)):
        with pytest.raises(RuntimeError, match="must not be negative"):
            chunk_tables(table, lens, lens, **{"num_rows": 3, "page_size": 16, **bad})
    with pytest.raises(RuntimeError, match="block_table must be int32"):
        chunk_tables(table.long(), lens, lens, 3, 16)
    with pytest.raises(RuntimeError, match="past_lens must be"):
        chunk_tables(table, lens[:2], lens, 3, 16)
    with pytest.raises(RuntimeError, match="counts must be integers"):
        chunk_tables(table, lens, lens.float(), 3, 16)
    with pytest.raises(RuntimeError, match="requests must be"):
        chunk_tables(table, lens, lens, 3, 16, requests=lens[:2])
    with pytest.raises(RuntimeError, match="requests must be"):
        chunk_tables(table, lens, lens, 3, 16, requests=lens[0])
    with pytest.raises(RuntimeError, match="counts must be"):
        chunk_tables(table, lens, lens[None], 3, 16)
    short = ChunkTables(table, lens, lens, lens, lens, lens, lens)
    with pytest.raises(RuntimeError, match="out.cu_seqlens"):
        chunk_tables(table, lens, lens, 3, 16, out=short)


def test_parameters():
    assert _param("t", None, 3, torch.float32, 1.0) == (None, 1.0)
    assert _param("k", 1 << 40, 3, torch.int32, 0) == (None, 0x7fffffff)
    assert _param("k", -4, 3, torch.int32, 0) == (None, 0)
    k, _ = _param("k", torch.tensor([1 << 40, -1, 7]), 3, torch.int32, 0)
    assert k.dtype == torch.int32 and k.tolist() == [0x7fffffff, 0, 7]
    for bad in (torch.zeros(2), torch.zeros((3, 1)), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.bool)):
        with pytest.raises(RuntimeError, match="t must be"):
            _param("t", bad, 3, torch.float32, 1.0)
    with pytest.raises(RuntimeError, match="k must be"):
        _param("k", torch.zeros(3), 3, torch.int32, 0)
    assert _params(None, None, None, 2, 10)[-1] is False
    assert _params(0.5, 10, 1.0, 2, 10)[-1] is False and _params(0.5, 9, 1.0, 2, 10)[-1] is True
    assert _params(0.5, 0, 0.9, 2, 10)[-1] is True


def test_reference_by_hand():
    p = distribution(np.log([4.0, 1.0, 3.0, 2.0]))
    assert np.allclose(p, [0.4, 0.1, 0.3, 0.2], rtol=1e-15)
    assert np.allclose(distribution(np.log([4.0, 1.0, 3.0, 2.0]), top_k=2), [4 / 7, 0, 3 / 7, 0])
    assert np.allclose(distribution(np.log([4.0, 1.0, 3.0, 2.0]), top_p=0.65), [4 / 7, 0, 3 / 7, 0])
    assert np.allclose(distribution(np.log([4.0, 1.0, 3.0, 2.0]), top_p=0.71), [4 / 9, 0, 3 / 9, 2 / 9])
    assert np.allclose(distribution([1.0, 1.0, 1.0], top_k=2), [0.5, 0.5, 0])
    assert distribution([0.0, 5.0, 5.0], temperature=0.0).tolist() == [0, 1, 0]
    assert [pick(p, u) for u in (0.0, 0.39, 0.41, 0.75, 0.85, 1.0)] == [0, 0, 1, 2, 3, 3]
    # q = (1/4 each), p = (0.4, 0.1, 0.3, 0.2): draft 1 passes below 0.4, and what is left then is (0.15, 0, 0.05, 0)
    x = torch.tensor(np.log([[[4.0, 1.0, 3.0, 2.0]] * 2]))
    q = torch.full((1, 1, 4), 0.25)
    d = torch.tensor([[1]])
    run = lambda a, u: verify(x, d, torch.tensor([[a]]), torch.tensor([u]), q)[0].tolist()  # noqa: E731
    assert run(0.39, 0.45) == [[1, 1]] and run(0.41, 0.74) == [[0, -1]] and run(0.41, 0.76) == [[2, -1]]
