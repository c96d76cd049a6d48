"""Chunk attention over quantized pools at head dims below the padded width of
its tiles: what a workgroup's shared memory held before the call has no part
in the results."""
import math

import pytest
import torch

from chunk_reference import FLOAT, make_pool, make_table, to_gpu
from vramancer_amd.paged_chunk import paged_attention_chunk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _say(msg):
    print(f"[case] {msg}", flush=True)


def _fill_shared_memory(x, wide_rows):
    """A call over a bf16 (and a float32) pool of x, in workgroups on every CU."""
    for t in (torch.bfloat16, torch.float32):
        pool = torch.full((8, 1, 2, 1, 16, 128), x, dtype=t, device=DEV)
        n = 512 * (256 if wide_rows else 128)
        table = torch.full((1, 4096 if wide_rows else 8), -1, dtype=torch.int32, device=DEV)
        table[0, :8] = torch.arange(8)
        q = torch.zeros((n, 1, 128), dtype=t, device=DEV)
        paged_attention_chunk(q, pool, table, torch.tensor([128], dtype=torch.int32, device=DEV),
                              torch.tensor([0, n], dtype=torch.int32, device=DEV), 0, causal=False)


@pytest.mark.parametrize("qt,kv,D", [("bf16", "int8", 80), ("f16", "fp8", 48), ("bf16", "fp8", 112), ("bf16", "int8", 144),
                                     ("f32", "int8", 80), ("f32", "fp8", 16)])
@pytest.mark.parametrize("wide", [False, True], ids=["tight", "wide"])
def test_leftovers_in_shared_memory(qt, kv, D, wide):
    """A row whose block of tokens is finite takes the ordinary path, though a
    later token that other rows of its tile see is infinite: its bits do not
    depend on the calls before."""
    _say(f"leftovers {qt} over {kv} D={D} wide={wide}")
    gen = torch.Generator().manual_seed(D)
    B, KH, n = 64, 8, 256  # (tiles enough that none is cut along its keys)
    P, table = make_table([n] * B, 16, gen)
    pool, scales, _ = make_pool(kv, P, 1, KH, 16, D, gen, "plain")
    for b in range(B):
        pid, slot = int(table[b, 100 // 16]), 100 % 16
        if kv == "int8":
            scales[pid, 0, 1, :, slot] = math.inf
        else:
            at = slot // 4 * 16 * (D // 16) * 4 + slot % 4  # of dim 0
            pool.view(torch.uint8)[pid, 0, 1].view(KH, -1)[:, at] = 0x7f  # NaN
    if wide:
        table = torch.cat([table, torch.full((B, 4096), -1, dtype=torch.int32)], 1)
    pool, scales = to_gpu(pool, scales)
    q = torch.randn((B * n, KH, D), generator=gen).to(FLOAT[qt]).to(DEV)
    batch = (table.to(DEV), torch.full((B,), n, dtype=torch.int32, device=DEV),
             (torch.arange(B + 1) * n).to(torch.int32).to(DEV), 0)
    got = []
    for x in (0.0, math.nan, 0.0):
        _fill_shared_memory(x, wide)
        got.append(paged_attention_chunk(q, pool, *batch, kv_scales=scales).view(B, n, KH, D))
    assert got[0][:, :100].isfinite().all() and not got[0][:, 100:].isfinite().all()
    for y in got[1:]:
        assert torch.equal(y.nan_to_num(9.0), got[0].nan_to_num(9.0))
