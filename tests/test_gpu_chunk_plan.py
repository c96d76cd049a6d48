"""Chunk attention with either size of tiles, by what the caller says of the
contexts and by the window: always over all of context_lens.

Tolerances are those of test_gpu_paged_chunk.py.
"""
import pytest
import torch

from chunk_reference import FLOAT, attend, make_pool, make_table, to_gpu
from test_gpu_paged_chunk import _tolerance
from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_chunk import paged_attention_chunk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("window", [None, 60, 1100])
@pytest.mark.parametrize("qt,kv", [("bf16", "bf16"), ("f16", "int8"), ("f32", "f32")])
@pytest.mark.parametrize("q_lens,past", [([40, 1, 90], [1500, 20, 0]), ([150], [1300])])
def test_expected_context(qt, kv, q_lens, past, window):
    print(f"[case] expected context {qt} over {kv} q={q_lens} window={window}", flush=True)
    gen = torch.Generator().manual_seed(sum(q_lens))
    lens = [a + b for a, b in zip(q_lens, past)]
    P, table = make_table(lens, 16, gen)
    table = torch.cat([table, torch.full((len(lens), 8000), -1, dtype=torch.int32)], 1)
    pool, scales, vals = make_pool(kv, P, 1, 2, 16, 64, gen)
    cu = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    q = torch.randn((int(cu[-1]), 8, 64), generator=gen).to(FLOAT[qt])
    lens = torch.tensor(lens, dtype=torch.int32)
    gp, gs = to_gpu(pool, scales)
    want, _, reach = attend(q, vals, table[:, :200], lens, cu, 0, window=window)
    tol = _tolerance(want, reach, q.dtype, qt == "f32", 64, kv == "int8")
    for expected in (None, 1, 500, 1 << 40):
        got = paged_attention_chunk(q.to(DEV), gp, table.to(DEV), lens.to(DEV), cu.to(DEV), 0, kv_scales=gs, window=window,
                                    expected_context=expected)
        assert ((got.cpu().double() - want).abs() <= tol).all(), expected
    with pytest.raises(RuntimeError, match="expected_context"):
        paged_attention_chunk(q.to(DEV), gp, table.to(DEV), lens.to(DEV), cu.to(DEV), 0, kv_scales=gs, expected_context=0)


def test_manager_knows_its_contexts():
    mgr = PagedKVCacheManager(PagedKVConfig(page_size=16, num_layers=1, num_kv_heads=2, head_dim=64, max_pages=40,
                                            device=DEV, dtype="float16"))
    mgr.allocate("a"), mgr.allocate("b")
    assert mgr.append_chunk(["a"], [300]).expected_context == 300
    assert mgr.append_chunk(["a", "b"], [1, 9]).expected_context == 39  # (301 + 9 x 9) / 10, rounded up
    assert mgr.append_chunk(["a", "b"], [0, 0]).expected_context is None
