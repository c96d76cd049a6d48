"""Batches with as many rows as sequences that do not hold one token each: idle
sequences beside longer ones, as a batch padded to a fixed size has them.

Tolerances are those of test_gpu_rope.py and test_gpu_paged_chunk.py.
"""
import pytest
import torch

from chunk_reference import HALF, attend, norm_rope, rope_angles
from test_gpu_rope import _append, _close
from vramancer_amd.paged_attention import PagedKVCacheManager, PagedKVConfig
from vramancer_amd.paged_chunk import chunk_workspace, paged_attention_chunk, rope_append
from vramancer_amd.rope import qk_norm_rope, rope_table

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.mark.parametrize("q_lens,tail", [([0, 2], 0), ([1, 0, 2], 0), ([0, 3, 0], 0), ([1, 0, 1, 1], 1), ([2, 0, 0, 1], 1),
                                         ([1, 1, 1], 0), ([1], 0), ([0, 0, 0], 3)],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, list) else f"t{v}")
@pytest.mark.parametrize("kv,D,rot", [("f16", 64, 64), ("bf16", 30, 20), ("int8", 64, 64), ("fp8", 64, 32)])
def test_rows_as_many_as_sequences(kv, D, rot, q_lens, tail):
    _say(f"append into {kv} D={D} q={q_lens} and {tail} rows of none")
    assert sum(q_lens) + tail == len(q_lens)
    _append("f16", kv, q_lens, [5 + 17 * b for b in range(len(q_lens))], 6, 2, D, 16, rot, True, False, seed=len(q_lens) + D,
            tail=tail)


@pytest.mark.parametrize("dtype", ["float16", "int8", "fp8"])
def test_manager_with_an_idle_request(dtype):
    """Two steps of [1, 0, 2] tokens through the manager: what is attended is
    what was written, and the queries are the rotated ones."""
    _say(f"manager, counts [1, 0, 2], pool {dtype}")
    H, KH, D = 4, 2, 64
    mgr = PagedKVCacheManager(PagedKVConfig(page_size=16, num_layers=1, num_kv_heads=KH, head_dim=D, max_pages=16,
                                            device=DEV, dtype=dtype))
    for rid in "abc":
        mgr.allocate(rid)
    gen = torch.Generator().manual_seed(6)
    table = rope_table(64, D, device=DEV)
    done = [0, 0, 0]
    keys = [torch.empty((0, KH, D), dtype=torch.float64) for _ in done]
    for counts in ([1, 0, 2], [1, 0, 2], [0, 3, 0]):
        chunk = mgr.append_chunk(list("abc"), counts)
        qkv = torch.randn((3, H + 2 * KH, D), generator=gen).half()
        g = qkv.to(DEV)
        q = mgr.write_chunk(0, chunk, g[:, H:H + KH], g[:, H + KH:], g[:, :H], table)
        pos = torch.cat([torch.arange(d, d + c) for d, c in zip(done, counts)])
        want, size = norm_rope(qkv[:, :H], None, rope_angles(64, D), pos, 1e-6, False)
        _close(q, want, size, "query")
        k, _ = norm_rope(qkv[:, H:H + KH], None, rope_angles(64, D), pos, 1e-6, False)
        out, at = mgr.compute_attention_chunk(q, chunk, 0), 0
        for b, (rid, c) in enumerate(zip("abc", counts)):
            done[b] += c
            keys[b] = torch.cat([keys[b], k[at:at + c]])
            if c:
                kk, vv = (x.double().cpu() for x in mgr.read_kv(rid, 0))
                # stored keys: half a step of fp16, of int8 (amax / 254) or of e4m3
                step = {"float16": 2.0 ** -11, "int8": 1 / 254, "fp8": 2.0 ** -4}[dtype]
                big = keys[b].abs().amax()
                assert ((kk.transpose(0, 1) - keys[b]).abs() <= 2 * step * big + 2.0 ** -18 * big).all(), (rid, counts)
                ref, _, reach = attend(q[at:at + c].cpu(), torch.stack([kk, vv])[None, None],
                                       torch.zeros((1, 1), dtype=torch.int32), [done[b]], [0, c], 0)
                tol = HALF[torch.float16] * (ref.abs() + reach) + 2.0 ** -16 * reach + 2.0 ** -25
                assert ((out[at:at + c].cpu().double() - ref).abs() <= tol).all(), (rid, counts)
            at += c


def test_captured_batch_padded_to_its_sequences():
    """A graph over N = B rows, replayed with idle sequences in any place:
    every replay equals the formula and the eager call."""
    _say("captured append of a padded batch")
    H, KH, D, PS, B = 4, 2, 64, 16, 5
    gen = torch.Generator().manual_seed(8)
    q, k, v = (torch.zeros((B, h, D), dtype=torch.bfloat16, device=DEV) for h in (H, KH, KH))
    pool = torch.zeros((12, 1, 2, KH, PS, D), dtype=torch.bfloat16, device=DEV)
    table = torch.randperm(12, generator=gen)[:10].reshape(B, 2).int().to(DEV)
    angles = rope_table(64, D, device=DEV)
    lens, cu = torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    q_out, out = torch.zeros_like(q), torch.zeros_like(q)
    ws = chunk_workspace(q, pool, B, 2)

    def both(q_out, out, pool, ws):
        rope_append(q, k, v, pool, table, lens, cu, 0, angles, query_out=q_out)
        paged_attention_chunk(q_out, pool, table, lens, cu, 0, out=out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(q_out, out, pool, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both(q_out, out, pool, ws)
    total = torch.zeros(B, dtype=torch.int64)
    for step, counts in enumerate(([1, 1, 1, 1, 1], [1, 0, 1, 1, 1], [0, 1, 1, 0, 1], [0, 0, 5, 0, 0], [0, 0, 0, 0, 2])):
        total += torch.tensor(counts)
        n = sum(counts)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=gen))
        lens.copy_(total.int()), cu.copy_(torch.tensor([0] + counts).cumsum(0).int())
        pool2 = pool.clone()
        q_out.fill_(3.0), out.fill_(3.0)
        graph.replay()
        q2, out2 = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
        both(q2, out2, pool2, None)
        torch.cuda.synchronize()
        assert torch.equal(q_out, q2) and torch.equal(out, out2) and torch.equal(pool, pool2), step
        assert (q_out[n:] == 3).all() and (out[n:] == 3).all()
        pos = torch.cat([torch.arange(int(t) - c, int(t)) for t, c in zip(total, counts)])
        want, size = norm_rope(q[:n].cpu(), None, rope_angles(64, D), pos, 1e-6, False)
        _close(q_out[:n], want, size, f"query {step}")
        want, _, reach = attend(q_out[:n].cpu(), pool.double().cpu(), table.cpu(), lens.cpu(), cu.cpu(), 0)
        tol = HALF[torch.bfloat16] * (want.abs() + reach) + 2.0 ** -16 * reach + 1e-30
        assert ((out[:n].cpu().double() - want).abs() <= tol).all(), step


def test_more_rows_than_a_grid_dimension_holds():
    """More than 2^26 rows, a wavefront to each: more than 2^32 threads."""
    N, D = 34_000_000, 2
    _say(f"norms of 2 x {N} rows")
    q = torch.randn((N, 1, D), device=DEV).bfloat16()
    w = torch.full((D,), 0.75, device=DEV)
    got = qk_norm_rope(q, q, None, None, w, w)
    x = q.double()
    want = 0.75 * x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    for y in got:  # half a step of bf16, and the float32 terms
        assert ((y.double() - want).abs() <= (HALF[torch.bfloat16] + 2.0 ** -19) * want.abs() + 1e-30).all()
