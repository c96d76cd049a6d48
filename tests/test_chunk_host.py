"""Refusals and sizes of the chunk operators on the host: no call here reaches
a GPU."""
import numpy as np
import pytest
import torch

from chunk_reference import make_pool, rope_angles
from vramancer_amd import _lib
from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_chunk import check_batch, check_pool, paged_attention_chunk, rope_append
from vramancer_amd.rope import check_positions, check_table, check_weights, qk_norm_rope, rope_table

SC = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _attend(lib, **kw):
    a = dict(q=16, qt=_lib.VRM_SRC_BF16, qn=1024, qh=128, pool=16, sc=None, pt=16, cl=16, cu=16, out=16, lse=None, ws=16,
             wsb=1 << 33, N=4, B=2, H=8, KH=2, D=128, PS=16, L=1, P=4, max_pp=64, layer=0, scale=0.1, causal=1, window=0,
             dt=_lib.VRM_KV_BF16)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.vrm_paged_chunk_attention(*a.values(), None)


def _append(lib, **kw):
    a = dict(q=16, qn=1024, qh=128, k=16, kn=256, kh=128, v=16, vn=256, vh=128, src=_lib.VRM_SRC_BF16, cs=16, rot=128,
             top=64, pos=None, pb=4, qw=None, kw=None, wt=0, eps=1e-6, inter=0, qo=16, pool=16, sc=None,
             dt=_lib.VRM_KV_BF16, pt=16, cl=16, cu=16, N=4, B=2, H=8, KH=2, D=128, PS=16, L=1, P=4, max_pp=2, layer=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.vrm_rope_append(*a.values(), None)


def _rope(lib, **kw):
    a = dict(q=16, qn=1024, qh=128, k=16, kn=256, kh=128, src=_lib.VRM_SRC_BF16, cs=16, rot=128, top=64, pos=16, pb=8,
             qw=None, kw=None, wt=0, eps=1e-6, inter=0, qo=16, ko=16, N=4, H=8, KH=2, D=128)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.vrm_qk_norm_rope(*a.values(), None)


@pytest.mark.parametrize("bad,rc,text", [
    (dict(q=None), -1, b"null"), (dict(cu=None), -1, b"null"), (dict(pt=None), -1, b"null"), (dict(H=7), -1, b"multiple"),
    (dict(layer=1), -1, b"layer_idx"), (dict(layer=-1), -1, b"layer_idx"), (dict(D=257), -2, b"head_dim"),
    (dict(D=0), -1, b"sizes"), (dict(window=-1), -1, b"window"), (dict(scale=float("nan")), -1, b"scale"),
    (dict(scale=float("inf")), -1, b"scale"), (dict(qt=9), -1, b"query dtype"), (dict(dt=99), -1, b"kv_dtype"),
    (dict(dt=_lib.VRM_KV_I8), -1, b"kv_scales"), (dict(sc=SC), -1, b"kv_scales"),
    (dict(dt=_lib.VRM_KV_I8, sc=SC, D=100), -2, b"head_dim"), (dict(dt=_lib.VRM_KV_FP8E4M3, sc=SC, PS=6), -2, b"page_size"),
    (dict(dt=_lib.VRM_KV_I8_INLINE, sc=SC), -1, b"inline"), (dict(wsb=16), -3, b"workspace"), (dict(ws=None), -3, b"workspace"),
    (dict(ws=8), -3, b"workspace"), (dict(N=1 << 30), -2, b"too many")])
def test_attention_refusals(lib, bad, rc, text):
    assert _attend(lib, **bad) == rc and text in lib.vrm_last_error()


@pytest.mark.parametrize("bad,rc,text", [
    (dict(q=None), -1, b"null"), (dict(k=None), -1, b"null"), (dict(v=None), -1, b"null"), (dict(cl=None), -1, b"null"),
    (dict(layer=2), -1, b"layer_idx"), (dict(D=300), -2, b"head_dim"), (dict(src=7), -1, b"source dtype"),
    (dict(qw=16, wt=5), -1, b"weight dtype"), (dict(rot=127), -1, b"rotary_dim"), (dict(rot=130), -1, b"rotary_dim"),
    (dict(top=0), -1, b"rotary_dim"), (dict(pos=16, pb=2), -1, b"positions"), (dict(eps=-1.0), -1, b"sizes"),
    (dict(dt=12), -1, b"kv_dtype"), (dict(dt=_lib.VRM_KV_FP8E4M3), -1, b"kv_scales"), (dict(sc=SC), -1, b"kv_scales"),
    (dict(dt=_lib.VRM_KV_I8, sc=SC, D=24, rot=8), -2, b"head_dim"), (dict(dt=_lib.VRM_KV_I8, sc=SC, PS=2), -2, b"page_size"),
    (dict(dt=_lib.VRM_KV_I8, sc=SC, pool=24), -1, b"aligned"), (dict(dt=_lib.VRM_KV_I8, sc=64), -1, b"inside"),
    (dict(N=1 << 29), -2, b"too many"), (dict(KH=0), -1, b"sizes")])
def test_append_refusals(lib, bad, rc, text):
    assert _append(lib, **bad) == rc and text in lib.vrm_last_error()


@pytest.mark.parametrize("bad,rc,text", [
    (dict(q=None), -1, b"null"), (dict(ko=None), -1, b"null"), (dict(pos=None), -1, b"null"), (dict(pb=3), -1, b"positions"),
    (dict(D=257, rot=2), -2, b"head_dim"), (dict(rot=0), -1, b"rotary_dim"), (dict(N=-1), -1, b"sizes"),
    (dict(src=3), -1, b"source dtype"), (dict(N=1 << 30), -2, b"too many")])
def test_rotation_refusals(lib, bad, rc, text):
    assert _rope(lib, **bad) == rc and text in lib.vrm_last_error()


def test_nothing_to_do(lib):
    """Empty calls return before they look at a pointer."""
    assert _attend(lib, N=0, q=None) == 0 and _attend(lib, B=0, cu=None) == 0
    assert _append(lib, N=0, k=None) == 0 and _append(lib, B=0, cu=None) == 0
    assert _rope(lib, N=0, q=None) == 0 and _rope(lib, H=0, KH=0) == 0


def test_workspace_bytes(lib):
    """None where every tile has a workgroup anyway, bounded elsewhere, 0 for a
    call that would be refused."""
    f = lib.vrm_paged_chunk_workspace_bytes
    bf, kv = _lib.VRM_SRC_BF16, _lib.VRM_KV_BF16
    assert f(100000, 4, 40, 8, 128, 16, 8192, bf, kv) == 0
    small = f(17, 1, 28, 4, 128, 16, 97, bf, kv)
    assert 0 < small < 1 << 28
    assert f(17, 1, 28, 4, 128, 16, 4, bf, kv) == 0  # a context of one block is not cut
    assert f(17, 1, 28, 5, 128, 16, 97, bf, kv) == 0 and f(17, 1, 28, 4, 300, 16, 97, bf, kv) == 0
    assert f(17, 1, 28, 4, 128, 16, 97, bf, 77) == 0
    for n, b in ((1, 1), (64, 64), (500, 3), (4096, 1), (300, 257)):
        for wide in (_lib.VRM_SRC_F32, bf):
            got = f(n, b, 32, 8, 128, 16, 100000, wide, kv)
            assert got < 1 << 30


def test_python_refuses_cpu_tensors_and_shapes():
    q, k = torch.zeros(4, 8, 64), torch.zeros(4, 2, 64)
    with pytest.raises(RuntimeError, match="CPU tensor"):
        qk_norm_rope(q, k, None, None)
    pool, _, _ = make_pool("bf16", 4, 1, 2, 16, 64, torch.Generator())
    t = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CPU tensor"):
        paged_attention_chunk(q, pool, t, t[0, :1], t[0], 0)
    with pytest.raises(RuntimeError, match="CPU tensor"):
        rope_append(None, k, k, pool, t, t[0, :1], t[0], 0)
    with pytest.raises(RuntimeError, match="page_table"):
        check_batch(t[0], t[0], t[0])
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        check_batch(t, t[0, :1], t[0, :1])
    with pytest.raises(RuntimeError, match="integers"):
        check_batch(t.float(), t[0, :1], t[0])
    assert check_batch(t.long(), t[0, :1], t[0])[0].dtype == torch.int32
    with pytest.raises(RuntimeError, match="head_dim"):
        check_pool(pool, None, 32)
    with pytest.raises(RuntimeError, match="kv_scales"):
        check_pool(pool, torch.zeros(1), 64)
    with pytest.raises(RuntimeError, match="contiguous"):
        check_pool(pool.transpose(3, 4), None, 64)  # (KH and PS exchanged: a strided view)
    p8, s8, _ = make_pool("int8", 4, 2, 2, 16, 64, torch.Generator())
    assert check_pool(p8, s8, 64) == _lib.VRM_KV_I8_INLINE
    with pytest.raises(RuntimeError, match="kv_scales"):
        check_pool(p8, None, 64)
    with pytest.raises(RuntimeError, match="allocate_pool"):
        check_pool(p8, s8.contiguous(), 64)
    with pytest.raises(RuntimeError, match="rotary_dim"):
        check_table(torch.zeros(4, 66), 64)
    with pytest.raises(RuntimeError, match="cos_sin"):
        check_table(torch.zeros(4, 64).double(), 64)
    with pytest.raises(RuntimeError, match="positions"):
        check_positions(torch.zeros(3), 3)
    with pytest.raises(RuntimeError, match="k_weight"):
        check_weights(torch.zeros(64), torch.zeros(64).half(), 64)


def test_rope_table_on_the_host():
    assert (rope_table(300, 32, device="cpu") - rope_angles(300, 32)).abs().max() <= 2.0 ** -24
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(max_positions=0), dict(inv_freq=np.ones(3))):
        with pytest.raises(RuntimeError):
            rope_table(**{**dict(max_positions=8, rotary_dim=8, device="cpu"), **bad})


def test_host_only_manager_refuses_chunks():
    mgr = PagedKVCacheManager(PagedKVConfig(device="cpu", max_pages=4))
    mgr.allocate("a")
    with pytest.raises(RuntimeError, match="GPU pool"):
        mgr.append_chunk(["a"], [1])
