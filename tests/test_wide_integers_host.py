"""Integers past 32 bits in the arguments of chunk_tables and of the sampling
operators, on the host: no call here reaches a GPU."""
import pytest
import torch

from vramancer_amd import paged_chunk, sampling

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


@pytest.mark.parametrize("bad", [dict(num_rows=1 << 31), dict(num_rows=(1 << 32) + 3), dict(page_size=(1 << 32) + 16),
                                 dict(max_pages=1 << 32)])
def test_sizes_past_32_bits(bad):
    table, lens = torch.zeros((3, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="2\\^31"):
        paged_chunk.chunk_tables(table, lens, lens, **{"num_rows": 3, "page_size": 16, **bad})


class Rows:
    """A tensor's face of more rows than 32 bits count."""

    is_cuda, dtype = True, torch.float16

    def __init__(self, *shape):
        self.shape = torch.Size(shape)

    def dim(self):
        return len(self.shape)

    def get_device(self):
        return 0


@pytest.mark.parametrize("N", [1 << 31, 1 << 32, (1 << 32) + 5])
def test_rows_past_32_bits(N, monkeypatch):
    monkeypatch.setattr(sampling._lib, "require_cuda", lambda *t: None)
    with pytest.raises(RuntimeError, match="2\\^31"):
        sampling.sample_tokens(Rows(N, 1), torch.zeros(1))
    with pytest.raises(RuntimeError, match="2\\^31"):
        sampling.verify_drafts(Rows(N, 1), torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 1)), torch.zeros(1),
                               cu_seqlens=torch.zeros(2, dtype=torch.int32))
