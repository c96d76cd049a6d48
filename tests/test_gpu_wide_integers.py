"""chunk_tables of int64 arguments past 32 bits: the batch of those that fit."""
import pytest
import torch

from vramancer_amd.paged_chunk import chunk_tables

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_requests_and_counts_past_32_bits():
    table = torch.arange(4 * 6, dtype=torch.int32, device=DEV).view(4, 6)
    past = torch.tensor([3, 9, 0, 20], device=DEV)
    counts = torch.tensor([2, 5, 1, 3, 1 << 33], device=DEV)
    requests = torch.tensor([1, 1 << 32, (1 << 32) + 2, -(1 << 32), 0], device=DEV)
    got = chunk_tables(table, past, counts, 12, 4, requests=requests)
    want = chunk_tables(table, past.int(), torch.tensor([2, 5, 1, 3, 0x7fffffff], dtype=torch.int32, device=DEV), 12, 4,
                        requests=torch.tensor([1, 4, 4, -1, 0], dtype=torch.int32, device=DEV))
    for name in ("page_table", "context_lens", "cu_seqlens", "positions", "page_ids", "slots", "sequences"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    assert got.cu_seqlens.tolist() == [0, 2, 2, 2, 2, 12] and got.sequences.tolist() == [0] * 2 + [4] * 10
