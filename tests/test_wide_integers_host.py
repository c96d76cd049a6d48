"""Integers past 32 bits in the arguments of chunk_tables and of the sampling
operators, on the host: no call here reaches a GPU."""
import pytest
import torch

from vramancer_amd import paged_chunk

I64 = torch.tensor([0, 1, -1, -7, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 1, 1 << 62, -(1 << 31), -(1 << 32), -(1 << 62)])


def test_wide_integers_do_not_wrap():
    """A request of 2^32 is no request (and not request 0), a count of 2^32 more
    than any batch holds (and not none)."""
    got = paged_chunk._ints("requests", I64, len(I64))
    most = (1 << 31) - 1
    assert got.dtype == torch.int32 and got.is_contiguous()
    assert got[:5].tolist() == [0, 1, -1, -7, most]
    assert got[5:9].tolist() == [most] * 4 and (got[9:] < 0).all()
    strided = torch.stack([I64, I64]).t()[:, 0]
    assert paged_chunk._ints("requests", strided, None).tolist() == got.tolist()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.int8, torch.uint8])
def test_narrow_integers_stay(dtype):
    t = torch.tensor([0, 1, 100], dtype=dtype)
    assert paged_chunk._ints("counts", t, 3).tolist() == [0, 1, 100]
