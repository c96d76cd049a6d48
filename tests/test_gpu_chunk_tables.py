"""chunk_tables against the definition, token by token on the host."""
import pytest
import torch

from vramancer_amd.paged_chunk import ChunkTables, chunk_tables

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAMES = ("page_table", "context_lens", "cu_seqlens", "positions", "page_ids", "slots", "sequences")


def reference(table, past, counts, N, PS, requests=None, max_pages=None):
    R, W = table.shape
    B = len(counts)
    requests = list(range(B)) if requests is None else requests
    width = W if max_pages is None else max_pages
    out = {"page_table": torch.full((B, width), -1), "context_lens": torch.zeros(B), "cu_seqlens": torch.zeros(B + 1),
           "positions": torch.zeros(N), "page_ids": torch.full((N,), -1), "slots": torch.full((N,), -1),
           "sequences": torch.full((N,), -1)}
    out = {k: v.int() for k, v in out.items()}
    at = 0
    for b, (r, n) in enumerate(zip(requests, counts)):
        there = 0 <= r < R
        stored = max(past[r], 0) if there else 0
        n = min(max(n, 0), N - at, 0x7fffffff - stored) if there else 0
        for i in range(n):
            t = stored + i
            out["positions"][at + i], out["slots"][at + i], out["sequences"][at + i] = t, t % PS, b
            if t // PS < W:
                out["page_ids"][at + i] = table[r, t // PS]
        at += n
        out["cu_seqlens"][b + 1] = at
        out["context_lens"][b] = stored + n
        if there:
            held = min(-(-(stored + n) // PS), W, width)
            out["page_table"][b, :held] = table[r, :held]
    return out


def run(table, past, counts, N, PS, requests=None, dtype=torch.int32, **kw):
    as_dev = lambda v: torch.tensor(v, dtype=dtype, device=DEV)  # noqa: E731
    return chunk_tables(table.to(DEV) if not table.is_cuda else table, as_dev(past), as_dev(counts), N, PS,
                        requests=None if requests is None else as_dev(requests), **kw)


def check(table, past, counts, N, PS, requests=None, **kw):
    got = run(table, past, counts, N, PS, requests, **kw)
    kw.pop("dtype", None)
    kw.pop("out", None)
    want = reference(table.cpu(), past, counts, N, PS, requests, **kw)
    for name in NAMES:
        t = getattr(got, name)
        assert t.dtype == torch.int32 and torch.equal(t.cpu(), want[name]), name
    return got


def table_of(R, W, seed=0):
    return torch.randperm(R * W, generator=torch.Generator().manual_seed(seed)).int().view(R, W)


@pytest.mark.parametrize("B,W,PS,top", [(1, 1, 1, 1), (3, 5, 4, 3), (17, 40, 16, 60), (64, 300, 5, 9), (300, 7, 16, 4),
                                        (2500, 3, 2, 2)])
def test_batches(B, W, PS, top):
    g = torch.Generator().manual_seed(B)
    R = B + 3
    past = torch.randint(0, max(1, W * PS - top), (R,), generator=g).tolist()
    counts = torch.randint(0, top + 1, (B,), generator=g).tolist()
    requests = torch.randperm(R, generator=g)[:B].tolist()
    N = sum(counts)
    for rows in sorted({N, N + 9, max(0, N - 2), 0}):
        check(table_of(R, W), past, counts, rows, PS, requests)
    check(table_of(R, W), past, counts, N, PS)  # the first B requests


def test_offsets_of_a_large_batch():
    # more sequences than a workgroup has threads, long rows of the table
    B, W = 3001, 1030
    g = torch.Generator().manual_seed(1)
    past = torch.randint(0, 16000, (B,), generator=g)
    counts = torch.randint(0, 4, (B,), generator=g)
    table = table_of(B, W)
    got = run(table, past.tolist(), counts.tolist(), 8000, 16)
    cu = torch.nn.functional.pad(counts.cumsum(0), (1, 0)).clamp(max=8000)
    assert torch.equal(got.cu_seqlens.cpu().long(), cu)
    ctx = past + cu[1:] - cu[:-1]
    assert torch.equal(got.context_lens.cpu().long(), ctx)
    held = torch.arange(W)[None] * 16 < ctx[:, None]
    assert torch.equal(got.page_table.cpu(), torch.where(held, table, -1))
    n = int(cu[-1])
    seq = torch.repeat_interleave(torch.arange(B), cu[1:] - cu[:-1])
    pos = past[seq] + torch.arange(n) - cu[seq]
    assert torch.equal(got.sequences.cpu()[:n].long(), seq) and torch.equal(got.positions.cpu()[:n].long(), pos)
    assert torch.equal(got.page_ids.cpu()[:n], table[seq, pos // 16])
    assert (got.sequences[n:] == -1).all() and (got.page_ids[n:] == -1).all()


def test_requests_that_are_not_there():
    check(table_of(4, 6), [3, 0, 9, 20], [2, 5, 1, 3, 4], 20, 4, [1, -1, 3, 4, 0])


def test_a_request_twice():
    check(table_of(3, 6), [3, 8, 0], [2, 2, 3], 10, 4, [1, 1, 2])


def test_lengths_past_the_table():
    check(table_of(3, 2), [7, 40, 0], [5, 3, 9], 17, 4)         # pages that are not there
    check(table_of(3, 2), [-5, 2, 1], [-3, 1, 2], 5, 4)         # negative lengths and counts
    check(table_of(2, 2), [0x7fffffff, 0x7ffffff0], [3, 40], 30, 16)  # positions stay below 2^31
    check(table_of(2, 2), [1, 2], [0x7fffffff, 0x7fffffff], 6, 16)


@pytest.mark.parametrize("width", [0, 1, 5, 11, 2000])
def test_other_widths(width):
    check(table_of(5, 9), [3, 30, 0, 17, 35], [1, 2, 0, 4, 1], 11, 4, max_pages=width)


def test_strides_and_types():
    wide = table_of(6, 33).to(DEV)
    check(wide[:, 2:20], [5, 60, 0, 9, 1, 2], [1, 2, 3, 4, 5, 6], 21, 4, dtype=torch.int64)
    check(wide[1:4], [5, 60, 0], [1, 2, 3], 6, 4, [2, 0, 1], dtype=torch.int16)
    check(wide.t()[:8, :4], [1, 2, 3, 4, 0, 0, 0, 0], [1] * 8, 8, 4)
    check(wide[:1].expand(4, 33), [1, 2, 3, 4], [1] * 4, 4, 4)


def test_no_sequences_no_rows():
    got = run(table_of(3, 4), [1, 2, 3], [], 5, 4, requests=[])
    assert got.cu_seqlens.tolist() == [0] and (got.sequences == -1).all() and (got.positions == 0).all()
    check(table_of(3, 4), [1, 2, 3], [1, 1, 1], 0, 4)
    got = chunk_tables(torch.zeros((0, 4), dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV),
                       torch.zeros(0, dtype=torch.int32, device=DEV), 2, 16)
    assert got.cu_seqlens.tolist() == [0] and got.page_ids.tolist() == [-1, -1]


def test_captured():
    """A graph that makes its tables from lengths that it changes itself, with
    eager calls between the replays."""
    R, W, PS, N = 6, 12, 4, 9
    table = table_of(R, W).to(DEV)
    past = torch.tensor([3, 9, 0, 5, 2, 11], dtype=torch.int32, device=DEV)
    counts = torch.tensor([1, 3, 2], dtype=torch.int32, device=DEV)
    reqs = torch.tensor([4, 0, 5], dtype=torch.int32, device=DEV)
    out = chunk_tables(table, past, counts, N, PS, requests=reqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chunk_tables(table, past, counts, N, PS, requests=reqs, out=out)
        past.index_add_(0, reqs.long(), counts)
    assert got is out and isinstance(out, ChunkTables)
    host = past.tolist()
    for step in range(4):
        n = [1 + step % 2, 3 - step % 3, step % 3]
        counts.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = reference(table.cpu(), host, n, N, PS, [4, 0, 5])
        for name in NAMES:
            assert torch.equal(getattr(out, name).cpu(), want[name]), (step, name)
        for r, c in zip([4, 0, 5], n):
            host[r] += c
        assert past.tolist() == host
        check(table, host, n, N, PS, [4, 0, 5])
