"""RMS norms of query and key heads and the rotation by position, in one pass.

Models that norm their query and key heads and rotate them by position spend
several passes over both on it; ``qk_norm_rope`` reads and writes them once.
``paged_chunk.rope_append`` does the same and puts the keys and values into
their cache pages on the way.  The reference leaves both to the model.

Angles come from a table that a program computes once per model
(``rope_table``): far positions need 64 bits, and a table serves every
frequency scaling.  Forward only: outputs carry no gradient.
"""
from __future__ import annotations

from typing import Any, Optional, Tuple

import torch

from . import _lib

__all__ = ["rope_table", "qk_norm_rope"]


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, inv_freq: Any = None,
               attention_scaling: float = 1.0, device: Any = "cuda") -> Any:
    """[max_positions, rotary_dim] float32: the cosines, then the sines, of
    position x frequency, computed in float64.

    Frequencies are base^(-2 i / rotary_dim), or ``inv_freq`` [rotary_dim / 2]
    (a model's scaled ones); cosines and sines are multiplied by
    ``attention_scaling``."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if max_positions <= 0:
        raise RuntimeError(f"max_positions must be positive, got {max_positions}")
    if inv_freq is None:
        freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    else:
        freq = torch.as_tensor(inv_freq).to(device=device, dtype=torch.float64).reshape(-1)
        if freq.numel() != rotary_dim // 2:
            raise RuntimeError(f"inv_freq must hold rotary_dim / 2 = {rotary_dim // 2} values, got {freq.numel()}")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat([angle.cos(), angle.sin()], 1) * attention_scaling).to(torch.float32)


def launch(t, fn, *args) -> int:
    """fn(*args, stream) on t's device and its current stream."""
    index = t.get_device()
    if torch.cuda.current_device() == index:
        return fn(*args, _lib.stream_of(t))
    with torch.cuda.device(index):
        return fn(*args, _lib.stream_of(t))


_SRC_CODES = {torch.float32: _lib.VRM_SRC_F32, torch.float16: _lib.VRM_SRC_F16, torch.bfloat16: _lib.VRM_SRC_BF16}


def src_code(dtype) -> int:
    code = _SRC_CODES.get(dtype)
    return _lib.src_dtype_code(dtype) if code is None else code  # (raises)


def check_heads(name: str, t, N: Optional[int], D: Optional[int], dtype):
    """A [N, heads, D] tensor whose last dim is contiguous (copied if not)."""
    if t.dim() != 3 or (N is not None and t.shape[0] != N) or (D is not None and t.shape[2] != D):
        want = "[N, heads, D]" if N is None else f"[{N}, heads, {D}]"
        raise RuntimeError(f"{name} must be {want}, got shape {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"query, key and value must share a dtype, got {t.dtype} and {dtype}")
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def check_table(cos_sin, D: int) -> Tuple[int, int]:
    """(rotary_dim, max_positions) of a rotation table, (0, 0) without one."""
    if cos_sin is None:
        return 0, 0
    if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous():
        raise RuntimeError("cos_sin must be a contiguous float32 [max_positions, rotary_dim] table (rope_table)")
    top, rot = cos_sin.shape
    if rot % 2 or not 0 < rot <= D or top < 1:
        raise RuntimeError(f"cos_sin {tuple(cos_sin.shape)}: rotary_dim must be even and at most head_dim {D}")
    return rot, top


def check_positions(positions, N: int):
    """Contiguous int32 / int64 [N] positions."""
    if positions.dim() != 1 or positions.shape[0] != N or positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"positions must be an int32 or int64 [{N}] tensor, got {positions.dtype} "
                           f"{tuple(positions.shape)}")
    return positions.contiguous()


def check_weights(q_weight, k_weight, D: int):
    """(q_weight, k_weight, dtype code), each [D] of one dtype or None."""
    first = q_weight if q_weight is not None else k_weight
    if first is None:
        return None, None, _lib.VRM_SRC_F32
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.dim() != 1 or w.shape[0] != D or w.dtype != first.dtype):
            raise RuntimeError(f"{name} must be [{D}], both weights of one dtype; got {w.dtype} {tuple(w.shape)}")
    return (None if q_weight is None else q_weight.contiguous(), None if k_weight is None else k_weight.contiguous(),
            src_code(first.dtype))


def check_out(name: str, out, like):
    """A contiguous output shaped like `like`, allocated where not given."""
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if out.shape != like.shape or out.dtype != like.dtype or not out.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous {like.dtype} {tuple(like.shape)} tensor, got {out.dtype} "
                           f"{tuple(out.shape)}")
    return out


def qk_norm_rope(
    query: Any,      # [N, H, D] float32 / float16 / bfloat16, last dim contiguous
    key: Any,        # [N, KH, D]
    cos_sin: Any,    # [max_positions, rotary_dim] float32 (rope_table), or None
    positions: Any,  # [N] int32 / int64, or None without a table
    q_weight: Any = None,
    k_weight: Any = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    query_out: Any = None,
    key_out: Any = None,
) -> Tuple[Any, Any]:
    """RMS norm of every query and key head (where its weight [D] is given),
    then the rotation of its first ``rotary_dim`` dims by the token's position.

    Pairs are (d, d + rotary_dim / 2), or (2 d, 2 d + 1) with ``interleaved``.
    Everything is float32 until the result is rounded to the inputs' dtype.
    Inputs may be slices of one projection's output (any token and head
    strides); outputs are dense, and may be the inputs where those are.  A
    position outside the table gives a row of NaN.  Returns (query, key).
    """
    _lib.require_cuda(query, key, cos_sin, positions, q_weight, k_weight, query_out, key_out)
    query = check_heads("query", query, None, None, None)
    N, H, D = query.shape
    key = check_heads("key", key, N, D, query.dtype)
    KH = key.shape[1]
    code = src_code(query.dtype)
    rot, top = check_table(cos_sin, D)
    if cos_sin is not None:
        if positions is None:
            raise RuntimeError("positions are needed with a rotation table")
        positions = check_positions(positions, N)
    q_weight, k_weight, w_code = check_weights(q_weight, k_weight, D)
    query_out = check_out("query_out", query_out, query)
    key_out = check_out("key_out", key_out, key)
    (q_n, q_h, _), (k_n, k_h, _) = query.stride(), key.stride()
    ptr = _lib.ptr
    rc = launch(query, _lib.load().vrm_qk_norm_rope, query.data_ptr(), q_n, q_h, key.data_ptr(), k_n, k_h, code,
                ptr(cos_sin), rot, top, ptr(positions), positions.element_size() if positions is not None else 4,
                ptr(q_weight), ptr(k_weight), w_code, float(eps), 1 if interleaved else 0, query_out.data_ptr(),
                key_out.data_ptr(), N, H, KH, D)
    _lib.check(rc, "qk_norm_rope")
    return query_out, key_out
