"""From logits to tokens, on the GPU: a token per row by temperature, top_k and
top_p, and drafted tokens verified against the target's probabilities.

The decode and chunk steps (``paged_batch.decode_step``, ``chunk_step``) return
logits.  ``sample_tokens`` draws a token from each row; ``verify_drafts`` takes
the logits of a chunk whose tokens after the first are drafts, accepts as many
of them as the target's distribution allows and draws the token that follows.
Random numbers are inputs, so that a program owns its generators, a captured
graph draws anew from numbers written into the same tensor, and every call can
be repeated; numbers outside [0, 1] are taken into it, NaN as 0.  Weights and
sums are float64.  The reference draws on the host from its batcher's logits.

Rows of logits are float32, float16 or bfloat16; a row's token i has the weight
exp((l_i - max l) / temperature).  ``top_k`` keeps the k first in the order
(logit descending, index ascending), ``top_p`` of those the shortest prefix
whose weights reach top_p times the sum of theirs.  A temperature of 0 (or
below) keeps the arg max alone, the first of equal ones.  -inf and NaN are
tokens that cannot be drawn; a row of nothing else gives token -1.

``temperature``, ``top_k`` and ``top_p`` are a number for all sequences or a
tensor [B] with one for each (k <= 0, p >= 1: all tokens); temperatures and
top_p are taken as float32.  No call reads a tensor back.  An output that lies
on an input's memory is refused.
"""
from __future__ import annotations

import functools
from typing import Any, Optional, Tuple

import torch

from . import _lib
from .rope import launch, src_code

__all__ = ["sample_tokens", "verify_drafts", "sample_workspace", "verify_workspace"]


@functools.lru_cache(maxsize=256)
def _sample_bytes(N: int, V: int, filtered: bool, with_probs: bool) -> int:
    return _lib.load().vrm_sample_workspace_bytes(N, V, filtered, with_probs)


@functools.lru_cache(maxsize=256)
def _verify_bytes(B: int, K: int, V: int, filtered: bool) -> int:
    return _lib.load().vrm_verify_workspace_bytes(B, K, V, filtered)


def sample_workspace(rows: int, vocab: int, filtered: bool = True, with_probs: bool = True, device: Any = "cuda"):
    """A workspace for ``sample_tokens`` calls of up to these sizes, for
    callers that keep one; ``filtered``: whether top_k or top_p is given,
    ``with_probs``: whether ``probs`` is."""
    return torch.empty(_sample_bytes(rows, vocab, bool(filtered), bool(with_probs)), dtype=torch.uint8, device=device)


def verify_workspace(batch: int, drafts: int, vocab: int, filtered: bool = True, device: Any = "cuda"):
    """A workspace for ``verify_drafts`` calls of up to these sizes."""
    return torch.empty(_verify_bytes(batch, drafts, vocab, bool(filtered)), dtype=torch.uint8, device=device)


def _param(name: str, value, B: int, dtype, none):
    """(tensor or None, number) of a parameter given as a number or as [B]."""
    if value is None:
        return None, none
    if isinstance(value, torch.Tensor):
        if value.dim() != 1 or value.shape[0] != B:
            raise RuntimeError(f"{name} must be a number or a tensor [{B}], got shape {tuple(value.shape)}")
        if value.dtype != dtype:
            if value.dtype.is_floating_point != dtype.is_floating_point or value.dtype == torch.bool:
                raise RuntimeError(f"{name} must be {dtype}, got {value.dtype}")
            if value.dtype == torch.int64:  # (a k past 32 bits is "all tokens")
                value = value.clamp(0, 0x7fffffff)
            value = value.to(dtype)
        return value.contiguous(), none
    return None, (float(value) if dtype is torch.float32 else min(max(int(value), 0), 0x7fffffff))


def _params(temperature, top_k, top_p, B: int, V: int):
    t, t_all = _param("temperature", temperature, B, torch.float32, 1.0)
    k, k_all = _param("top_k", top_k, B, torch.int32, 0)
    p, p_all = _param("top_p", top_p, B, torch.float32, 1.0)
    return t, t_all, k, k_all, p, p_all, k is not None or 0 < k_all < V or p is not None or p_all < 1.0


def _uniforms(name: str, u, shape):
    if tuple(u.shape) != shape or u.dtype != torch.float32:
        raise RuntimeError(f"{name} must be float32 {list(shape)}, got {u.dtype} {tuple(u.shape)}")
    return u.contiguous()


def _out(name: str, out, shape, dtype, device):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(out.shape) != shape or out.dtype != dtype or not out.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous {dtype} {list(shape)} tensor, got {out.dtype} "
                           f"{tuple(out.shape)}")
    return out


def _workspace(workspace, need: int, device):
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if not workspace.is_contiguous():
        raise RuntimeError("workspace must be contiguous")
    return workspace


def _check_sizes(*sizes) -> None:
    if max(sizes) > 0x7fffffff:
        raise RuntimeError(f"rows, drafts and vocabulary must be below 2^31, got {sizes}")


def sample_tokens(
    logits: Any,    # [N, V] float32 / float16 / bfloat16
    uniforms: Any,  # [N] float32 in [0, 1)
    temperature: Any = None,
    top_k: Any = None,
    top_p: Any = None,
    probs: Any = None,  # [N, V] float32, filled with the distributions
    out: Any = None,
    workspace: Any = None,
) -> Any:
    """A token for each row: the lowest index whose running sum of kept
    weights passes ``uniforms[n]`` of their whole, int64 [N] (``out`` when
    given).

    ``probs`` takes the distribution that was drawn from, zero for the tokens
    that are not kept: what ``verify_drafts`` needs of a draft model.  Rows may
    be strided (a slice of a longer vocabulary, every last row of a chunk).
    Calls may run at once on several streams if they share neither outputs nor
    ``workspace``."""
    _lib.require_cuda(logits, uniforms, probs, out, workspace,
                      *(v for v in (temperature, top_k, top_p) if isinstance(v, torch.Tensor)))
    if logits.dim() != 2:
        raise RuntimeError(f"logits must be [N, V], got shape {tuple(logits.shape)}")
    code = src_code(logits.dtype)
    N, V = logits.shape
    _check_sizes(N, V)
    if V < 1:
        raise RuntimeError("logits must have at least one token")
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    uniforms = _uniforms("uniforms", uniforms, (N,))
    t, t_all, k, k_all, p, p_all, filtered = _params(temperature, top_k, top_p, N, V)
    if probs is not None:
        probs = _out("probs", probs, (N, V), torch.float32, logits.device)
    out = _out("out", out, (N,), torch.int64, logits.device)
    if N == 0:
        return out
    workspace = _workspace(workspace, _sample_bytes(N, V, filtered, probs is not None), logits.device)
    ptr = _lib.ptr
    rc = launch(logits, _lib.load().vrm_sample_tokens, logits.data_ptr(), code, logits.stride(0), uniforms.data_ptr(),
                ptr(t), t_all, ptr(k), k_all, ptr(p), p_all, ptr(probs), out.data_ptr(), workspace.data_ptr(),
                workspace.numel() * workspace.element_size(), N, V)
    _lib.check(rc, "sample_tokens")
    return out


def verify_drafts(
    logits: Any,           # [B, K + 1, V], or [N, V] with cu_seqlens
    drafts: Any,           # [B, K] int32 / int64
    accept_uniforms: Any,  # [B, K] float32 in [0, 1)
    draw_uniforms: Any,    # [B] float32 in [0, 1)
    draft_probs: Any = None,  # [B, K, V] float32, or None: certain drafts
    cu_seqlens: Any = None,   # [B + 1]
    temperature: Any = None,
    top_k: Any = None,
    top_p: Any = None,
    out: Any = None,       # [B, K + 1] int64
    accepted: Any = None,  # [B] int32
    workspace: Any = None,
) -> Tuple[Any, Any]:
    """Verifies each sequence's drafted tokens: (tokens [B, K + 1] int64,
    accepted [B] int32).

    Row i of a sequence's logits is the target's distribution p of what
    follows its draft i - 1 (row 0: what follows the token before the drafts),
    under the sequence's temperature, top_k and top_p.  Draft i is accepted if
    all before it are and ``accept_uniforms[b, i] * q(x) < p(x)``, q its
    ``draft_probs[b, i]`` or, for drafts that were not drawn at random (looked
    up, an arg max), 1.  The token after the accepted ones is drawn with
    ``draw_uniforms[b]``: from p of the last row where all were accepted,
    otherwise from max(p - q, 0) of the refused one's row, so that tokens are
    distributed as if the target had drawn them.  ``tokens`` holds the accepted
    drafts, that token, and -1 behind it.

    A ragged batch has its rows as ``paged_chunk`` has them: sequence b's are
    ``cu_seqlens[b] .. cu_seqlens[b + 1]``, one more than its drafts, of which
    the first min(K, rows - 1) of ``drafts[b]`` count; a sequence without rows
    has -1 throughout.  A draft outside the vocabulary (-1 behind a short list)
    ends the drafts: the next token is p's own."""
    _lib.require_cuda(logits, drafts, accept_uniforms, draw_uniforms, draft_probs, cu_seqlens, out, accepted, workspace,
                      *(v for v in (temperature, top_k, top_p) if isinstance(v, torch.Tensor)))
    if drafts.dim() != 2 or drafts.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"drafts must be int32 or int64 [B, K], got {drafts.dtype} {tuple(drafts.shape)}")
    code = src_code(logits.dtype)
    B, K = drafts.shape
    V = logits.shape[-1] if logits.dim() else 0
    if cu_seqlens is None:
        if logits.dim() != 3 or tuple(logits.shape[:2]) != (B, K + 1):
            raise RuntimeError(f"logits must be [{B}, {K + 1}, V] without cu_seqlens, got shape {tuple(logits.shape)}")
        logits = logits.reshape(B * (K + 1), V)
    else:
        if logits.dim() != 2:
            raise RuntimeError(f"logits must be [N, V] with cu_seqlens, got shape {tuple(logits.shape)}")
        if tuple(cu_seqlens.shape) != (B + 1,) or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f"cu_seqlens must be int32 or int64 [B + 1 = {B + 1}], got {cu_seqlens.dtype} "
                               f"{tuple(cu_seqlens.shape)}")
        cu_seqlens = cu_seqlens.to(torch.int32).contiguous()
    _check_sizes(logits.shape[0], B, K, V)
    if V < 1:
        raise RuntimeError("logits must have at least one token")
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    drafts = drafts.contiguous()
    accept_uniforms = _uniforms("accept_uniforms", accept_uniforms, (B, K))
    draw_uniforms = _uniforms("draw_uniforms", draw_uniforms, (B,))
    q_b = q_k = 0
    if draft_probs is not None:
        if tuple(draft_probs.shape) != (B, K, V) or draft_probs.dtype != torch.float32:
            raise RuntimeError(f"draft_probs must be float32 [{B}, {K}, {V}], got {draft_probs.dtype} "
                               f"{tuple(draft_probs.shape)}")
        if draft_probs.stride(2) != 1 and V > 1:
            draft_probs = draft_probs.contiguous()
        q_b, q_k, _ = draft_probs.stride()
        if K == 0:
            draft_probs = None
    t, t_all, k, k_all, p, p_all, filtered = _params(temperature, top_k, top_p, B, V)
    out = _out("out", out, (B, K + 1), torch.int64, logits.device)
    accepted = _out("accepted", accepted, (B,), torch.int32, logits.device)
    if B == 0:
        return out, accepted
    workspace = _workspace(workspace, _verify_bytes(B, K, V, filtered), logits.device)
    ptr = _lib.ptr
    rc = launch(logits, _lib.load().vrm_verify_drafts, logits.data_ptr(), code, logits.stride(0), ptr(cu_seqlens),
                drafts.data_ptr(), drafts.element_size(), ptr(draft_probs), q_b, q_k, accept_uniforms.data_ptr(),
                draw_uniforms.data_ptr(), ptr(t), t_all, ptr(k), k_all, ptr(p), p_all, out.data_ptr(),
                accepted.data_ptr(), workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                logits.shape[0], B, K, V)
    _lib.check(rc, "verify_drafts")
    return out, accepted
