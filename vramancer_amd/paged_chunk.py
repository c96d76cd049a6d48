"""A chunk of new tokens over the paged KV cache: how it enters its pages and
attends them.

The decode attends one token per sequence.  Prompts, chunks of prompts,
drafted tokens to verify and batches that mix them with decoding requests have
several.  ``rope_append`` norms and rotates their queries and keys and writes
keys and values into the pages in one pass; ``paged_attention_chunk`` attends
them straight from the pages.  The reference has no counterpart: its prompts
run through the model's own attention, and ``from_hf_cache`` stores the result
(core/paged_attention.py:716-805).

A batch is ragged and described by three int32 device tensors:

* ``cu_seqlens`` [B + 1]: sequence b's new tokens are rows ``cu_seqlens[b] ..
  cu_seqlens[b + 1]`` of the N given.  Rows from ``cu_seqlens[B]`` on belong to
  no sequence: they are neither read nor written, so that N can stay fixed
  while a captured graph is replayed over smaller batches;
* ``context_lens`` [B]: tokens in the cache, the new ones included, so that new
  token i of q is at position ``context_lens[b] - q + i``;
* ``page_table`` [B, max_pages] as the decode takes it.

``chunk_tables`` makes them, and the place of every new token, from lengths
that are on the device: a step whose lengths follow from the one before it
(``sampling.verify_drafts``) needs no copy to the host.

Everything else is decided on the device; no call reads a tensor back.  Like
the decode these are forward only: outputs carry no gradient.
"""
from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import Any, Optional

import torch

from . import _lib, kv_quant
from .rope import check_heads, check_out, check_positions, check_table, check_weights, launch, src_code

__all__ = ["rope_append", "paged_attention_chunk", "chunk_workspace", "chunk_tables", "ChunkTables"]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(N: int, B: int, H: int, KH: int, D: int, PS: int, max_pp: int, q_code: int, kv_code: int) -> int:
    return _lib.load().vrm_paged_chunk_workspace_bytes(N, B, H, KH, D, PS, max_pp, q_code, kv_code)


def chunk_workspace(query, kv_pool, batch: int, max_pages_per_seq: int):
    """The workspace that a ``paged_attention_chunk`` call needs for a query
    and a pool of these shapes and types, for callers that keep one
    (``workspace=``)."""
    N, H, D = query.shape
    KH, PS = kv_pool.shape[3], kv_pool.shape[4]
    nbytes = _workspace_bytes(N, batch, H, KH, D, PS, max_pages_per_seq, src_code(query.dtype),
                              _lib.kv_dtype_code(kv_pool.dtype))
    return torch.empty(nbytes, dtype=torch.uint8, device=query.device)


def check_pool(kv_pool, kv_scales, D: int):
    """The kv_dtype code of a pool as the C ABI takes it."""
    if kv_pool.dim() != 6:
        raise RuntimeError(f"kv_pool must be [P, L, 2, KH, PS, D], got shape {tuple(kv_pool.shape)}")
    P, L, two, KH, PS, Dp = kv_pool.shape
    if two != 2 or Dp != D:
        raise RuntimeError(f"kv_pool shape {tuple(kv_pool.shape)} does not match head_dim {D}")
    code = _lib.kv_dtype_code(kv_pool.dtype)
    if code not in (_lib.VRM_KV_I8, _lib.VRM_KV_FP8E4M3):
        if kv_scales is not None:
            raise RuntimeError("kv_scales is only meaningful for int8 / float8_e4m3fn pools")
        if not kv_pool.is_contiguous():
            raise RuntimeError("a float kv_pool must be contiguous")
        return code
    want = (P, L, 2, KH, PS) if code == _lib.VRM_KV_I8 else (P, L, 2, KH)
    if kv_scales is None or tuple(kv_scales.shape) != want or kv_scales.dtype != torch.float32:
        raise RuntimeError(f"{kv_pool.dtype} pool needs float32 kv_scales of shape {want}")
    code = kv_quant.pool_dtype_code(kv_pool, kv_scales)
    if code is None:
        raise RuntimeError("kv_pool and kv_scales must be dense arrays or the two views allocate_pool returns")
    return code


def check_batch(page_table, context_lens, cu_seqlens):
    """(page_table, context_lens, cu_seqlens, B) as contiguous int32 tensors."""
    if page_table.dim() != 2 or context_lens.dim() != 1 or page_table.shape[0] != context_lens.shape[0]:
        raise RuntimeError(f"page_table must be [B, max_pages] and context_lens [B], got {tuple(page_table.shape)} and "
                           f"{tuple(context_lens.shape)}")
    B = context_lens.shape[0]
    if tuple(cu_seqlens.shape) != (B + 1,):
        raise RuntimeError(f"cu_seqlens must be [B + 1 = {B + 1}], got {tuple(cu_seqlens.shape)}")
    out = []
    for t in (page_table, context_lens, cu_seqlens):
        if t.dtype != torch.int32:
            if t.dtype not in (torch.int64, torch.int16, torch.int8, torch.uint8):
                raise RuntimeError(f"page_table, context_lens and cu_seqlens must be integers, got {t.dtype}")
            t = t.to(torch.int32)
        out.append(t.contiguous())
    return out[0], out[1], out[2], B


def rope_append(
    query: Any,         # [N, H, D] float32 / float16 / bfloat16, or None: only keys and values
    key: Any,           # [N, KH, D]
    value: Any,         # [N, KH, D]
    kv_pool: Any,       # [P, L, 2, KH, PS, D] float32 / float16 / bfloat16 / int8 / float8_e4m3fn
    page_table: Any,    # [B, max_pages]
    context_lens: Any,  # [B], the new tokens included
    cu_seqlens: Any,    # [B + 1]
    layer_idx: int,
    cos_sin: Any = None,  # [max_positions, rotary_dim] float32 (rope.rope_table), or None: no rotation
    kv_scales: Any = None,
    positions: Any = None,  # [N] int32 / int64; default: the tokens' own
    q_weight: Any = None,
    k_weight: Any = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    query_out: Any = None,
) -> Any:
    """Norms and rotates the new tokens' queries and keys as
    ``rope.qk_norm_rope`` does, writes keys and values into their pages, and
    returns the queries, [N, H, D] in their dtype (``None`` without queries).

    Keys go from float32 straight to the pool's type: rounded to nearest even,
    or to ``kv_quant``'s int8 codes and per-token scales.  An fp8 page's scale
    becomes the larger of its own (0 if it is entered at slot 0) and
    amax / 448 over its new tokens, and codes already in it are re-encoded once
    when it grows.

    ``positions`` change the rotation only, not the places.  Keys and values
    for absent pages (entries < 0 or >= P), negative positions or positions
    outside the rotation table are dropped; in the last case the query row is
    NaN.  Rows from ``cu_seqlens[B]`` on are left as they were.  Sequences of
    one call must not write the same slots, nor, in an fp8 pool, the same page.
    """
    _lib.require_cuda(key, query, value, kv_pool, page_table, context_lens, cu_seqlens, cos_sin, kv_scales, positions,
                      q_weight, k_weight, query_out)
    key = check_heads("key", key, None, None, None)
    N, KH, D = key.shape
    value = check_heads("value", value, N, D, key.dtype)
    src = src_code(key.dtype)
    code = check_pool(kv_pool, kv_scales, D)
    P, L, _, pool_heads, PS, _ = kv_pool.shape
    if KH != pool_heads or value.shape[1] != KH:
        raise RuntimeError(f"key and value must have the pool's {pool_heads} heads, got {KH} and {value.shape[1]}")
    H = 0
    if query is not None:
        query = check_heads("query", query, N, D, key.dtype)
        H = query.shape[1]
        query_out = check_out("query_out", query_out, query)
    elif query_out is not None:
        raise RuntimeError("query_out without a query")
    page_table, context_lens, cu_seqlens, B = check_batch(page_table, context_lens, cu_seqlens)
    rot, top = check_table(cos_sin, D)
    if positions is not None:
        positions = check_positions(positions, N)
    q_weight, k_weight, w_code = check_weights(q_weight, k_weight, D)
    ptr = _lib.ptr
    q_n, q_h = query.stride()[:2] if H else (0, 0)
    (k_n, k_h, _), (v_n, v_h, _) = key.stride(), value.stride()
    rc = launch(key, _lib.load().vrm_rope_append, ptr(query), q_n, q_h, key.data_ptr(), k_n, k_h, value.data_ptr(), v_n,
                v_h, src, ptr(cos_sin), rot, top, ptr(positions),
                positions.element_size() if positions is not None else 4, ptr(q_weight), ptr(k_weight), w_code,
                float(eps), 1 if interleaved else 0, ptr(query_out), kv_pool.data_ptr(), ptr(kv_scales), code,
                page_table.data_ptr(), context_lens.data_ptr(), cu_seqlens.data_ptr(), N, B, H, KH, D, PS, L, P,
                page_table.shape[1], int(layer_idx))
    _lib.check(rc, "rope_append")
    return query_out


def paged_attention_chunk(
    query: Any,         # [N, H, D] float32 / float16 / bfloat16, last dim contiguous
    kv_pool: Any,       # [P, L, 2, KH, PS, D] float32 / float16 / bfloat16 / int8 / float8_e4m3fn
    page_table: Any,    # [B, max_pages]
    context_lens: Any,  # [B], the new tokens included
    cu_seqlens: Any,    # [B + 1]
    layer_idx: int,
    scale: Optional[float] = None,
    kv_scales: Any = None,
    causal: bool = True,
    window: Optional[int] = None,
    out: Any = None,
    lse: Any = None,
    workspace: Any = None,
    expected_context: Optional[int] = None,
) -> Any:
    """Attention of each sequence's new tokens over its pages; the new tokens'
    keys and values are in the cache already.

    Row n attends the tokens of its sequence up to its own position (all of
    them with ``causal=False``), the last ``window`` of those when given.
    Tokens of absent pages (entries < 0 or >= P) are skipped; a row that sees
    nothing gives zeros.  ``scale`` defaults to 1 / sqrt(D).  Returns [N, H, D]
    in the query's dtype (``out`` when given; rows past ``cu_seqlens[B]`` are
    left as they were, undefined in an output allocated here).  ``lse``
    optionally takes ln sum exp of the scaled scores, [N, H] float32, for
    ``combine_attention``.

    ``expected_context`` is about how many tokens a sequence has (their mean
    over the new tokens), for callers that know it and whose table is wider
    than that, as one of a fixed width for a captured graph is.  It chooses the
    kernel's tiles for such contexts; what is attended does not depend on it.

    Calls may run at once on several streams if they share neither output nor
    ``workspace``; results do not depend on what a workspace held before, and
    are the same from call to call.
    """
    _lib.require_cuda(query, kv_pool, page_table, context_lens, cu_seqlens, kv_scales, out, lse, workspace)
    if query.dim() != 3:
        raise RuntimeError(f"query must be [N, H, D], got shape {tuple(query.shape)}")
    N, H, D = query.shape
    q_code = src_code(query.dtype)
    code = check_pool(kv_pool, kv_scales, D)
    P, L, _, KH, PS, _ = kv_pool.shape
    page_table, context_lens, cu_seqlens, B = check_batch(page_table, context_lens, cu_seqlens)
    if window is not None and not 0 < window < 1 << 31:
        raise RuntimeError(f"window must be a positive number of tokens, got {window}")
    if expected_context is not None and expected_context <= 0:
        raise RuntimeError(f"expected_context must be a positive number of tokens, got {expected_context}")
    if query.stride(2) != 1 and D > 1:
        query = query.contiguous()
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != query.shape or out.dtype != query.dtype or not out.is_contiguous():
        raise RuntimeError(f"out must be a contiguous {query.dtype} [{N}, {H}, {D}] tensor, got {out.dtype} "
                           f"{tuple(out.shape)}")
    if lse is not None and (tuple(lse.shape) != (N, H) or lse.dtype != torch.float32 or not lse.is_contiguous()):
        raise RuntimeError(f"lse must be a contiguous float32 [{N}, {H}] tensor")
    max_pp = page_table.shape[1]
    need = _workspace_bytes(N, B, H, KH, D, PS, max_pp, q_code, code) if H % KH == 0 else 0
    if workspace is None:
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=query.device)
    elif not workspace.is_contiguous():
        raise RuntimeError("workspace must be contiguous")
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    ptr = _lib.ptr
    q_n, q_h, _ = query.stride()
    rc = launch(query, _lib.load().vrm_paged_chunk_attention_expecting, query.data_ptr(), q_code, q_n, q_h,
                kv_pool.data_ptr(), ptr(kv_scales), page_table.data_ptr(), context_lens.data_ptr(),
                cu_seqlens.data_ptr(), out.data_ptr(), ptr(lse), ptr(workspace), ws_bytes, N, B, H, KH, D, PS, L, P,
                max_pp, int(layer_idx), 1.0 / math.sqrt(D) if scale is None else float(scale), 1 if causal else 0,
                window or 0, min(int(expected_context or 0), 0x7fffffff), code)
    _lib.check(rc, "paged_attention_chunk")
    return out


@dataclass
class ChunkTables:
    """A ragged batch of new tokens (``chunk_tables``), int32 on the device."""

    page_table: Any    # [B, max_pages]
    context_lens: Any  # [B], the new tokens included
    cu_seqlens: Any    # [B + 1]
    positions: Any     # [N] position of every new token, 0 behind the last sequence
    page_ids: Any      # [N] its page, -1 where there is none
    slots: Any         # [N] its slot there, -1 behind the last sequence
    sequences: Any     # [N] its sequence, -1 behind the last one


def _ints(name: str, t, n: Optional[int]):
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        raise RuntimeError(f"{name} must be [{'B' if n is None else n}], got shape {tuple(t.shape)}")
    if t.dtype != torch.int32:
        if t.dtype not in (torch.int64, torch.int16, torch.int8, torch.uint8):
            raise RuntimeError(f"{name} must be integers, got {t.dtype}")
        if t.dtype == torch.int64:  # (the nearest value of 32 bits)
            t = t.clamp(-0x80000000, 0x7fffffff)
        t = t.to(torch.int32)
    return t.contiguous()


def chunk_tables(
    block_table: Any,  # [R, W] int32, rows may be strided
    past_lens: Any,    # [R] tokens stored
    counts: Any,       # [B] new tokens
    num_rows: int,     # N
    page_size: int,
    requests: Any = None,  # [B] rows of block_table; default: the first B
    max_pages: Optional[int] = None,
    out: Optional[ChunkTables] = None,
) -> ChunkTables:
    """What ``rope_append``, ``paged_attention_chunk`` and
    ``PagedKVCacheManager.write_kv_batch`` take, for ``counts[b]`` new tokens of
    each request ``requests[b]``, from a block table that stays on the device
    and holds the pages of the new tokens already
    (``PagedKVCacheManager.reserve``).

    ``num_rows`` is the N of the batch's tensors: tokens past it get no place
    (``cu_seqlens`` ends at it), rows behind the last token belong to no
    sequence.  ``max_pages`` (default W) is the page table's width; a row holds
    the pages up to its last token's, -1 behind them.  A request outside
    [0, R) and a negative count have no tokens.  ``out`` takes the tensors of
    an earlier call of the same sizes, for a captured graph that reads them;
    none of them may be an input too (lengths move on in a tensor of their own,
    not from ``context_lens`` of one call into the next one's ``out``)."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32:
        raise RuntimeError(f"block_table must be int32 [R, W], got {block_table.dtype} {tuple(block_table.shape)}")
    R, W = block_table.shape
    N, PS = int(num_rows), int(page_size)
    max_pp = W if max_pages is None else int(max_pages)
    if N < 0 or PS < 1 or max_pp < 0:
        raise RuntimeError(f"num_rows and max_pages must not be negative and page_size positive, got {N}, {max_pp}, "
                           f"{PS}")
    if max(R, W, N, PS, max_pp) > 0x7fffffff:
        raise RuntimeError(f"sizes must be below 2^31, got {R} rows of {W} pages, num_rows {N}, page_size {PS} and "
                           f"max_pages {max_pp}")
    if block_table.stride(1) != 1 and W > 1:
        block_table = block_table.contiguous()
    past_lens = _ints("past_lens", past_lens, R)
    counts = _ints("counts", counts, None)
    B = counts.shape[0]
    if requests is not None:
        requests = _ints("requests", requests, B)
    if out is None:
        _lib.require_cuda(block_table, past_lens, counts, requests)
        sizes = (B * max_pp, B, B + 1, N, N, N, N)
        parts = torch.empty(sum(sizes), dtype=torch.int32, device=block_table.device)
        at = parts.data_ptr()
        ptrs = []
        for n in sizes:
            ptrs.append(at)
            at += 4 * n
        # (the views need no gradients: this form takes 1.6 us, split_with_sizes 2.0)
        table, ctx, cu, pos, page, slot, seq = torch.unsafe_split_with_sizes(parts, sizes)
        out = ChunkTables(table.view(B, max_pp), ctx, cu, pos, page, slot, seq)
    else:
        for name, shape in (("page_table", (B, max_pp)), ("context_lens", (B,)), ("cu_seqlens", (B + 1,)),
                            ("positions", (N,)), ("page_ids", (N,)), ("slots", (N,)), ("sequences", (N,))):
            t = getattr(out, name)
            if tuple(t.shape) != shape or t.dtype != torch.int32 or not t.is_contiguous():
                raise RuntimeError(f"out.{name} must be a contiguous int32 {list(shape)} tensor, got {t.dtype} "
                                   f"{tuple(t.shape)}")
        tensors = (out.page_table, out.context_lens, out.cu_seqlens, out.positions, out.page_ids, out.slots,
                   out.sequences)
        _lib.require_cuda(block_table, past_lens, counts, requests, *tensors)
        ptrs = [t.data_ptr() for t in tensors]
    rc = launch(block_table, _lib.load().vrm_chunk_tables, block_table.data_ptr(), block_table.stride(0), R, W,
                past_lens.data_ptr(), counts.data_ptr(), None if requests is None else requests.data_ptr(), B, N, PS,
                ptrs[0], max_pp, *ptrs[1:])
    _lib.check(rc, "chunk_tables")
    return out
