"""Norms of queries and keys per head and the rotation by their positions, in one pass.

The step of an attention layer right before ``update_and_fetch``: the
reference's layers rotate queries and keys there (llama.py:90-91), and models
with query and key norms take those first.  Positions may have several axes
(time, height, width), each frequency reading the one it belongs to.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch

from . import _lib, ops
from .affine import _device_guard, _same_device

__all__ = ["norm_rope"]

PAIRS = ("half", "adjacent")


@functools.lru_cache(maxsize=1024)
def _plan(q_shape, q_dtype, k_shape, k_dtype, pos_shape, pos_stride, pos_dtype, inv_shape, axis_shape, axis_dtype,
          qw_shape, kw_shape, pairs):
    """What a call's shapes and types come to, once they fit: (Hk, dtype code, rotated coordinates, axes, position
    bytes, position strides over (axis, b, l))."""
    if len(q_shape) != 4 or len(k_shape) != 4 or q_dtype != k_dtype:
        raise ValueError(f"queries {tuple(q_shape)} {q_dtype} and keys {tuple(k_shape)} {k_dtype} must be "
                         "(B, H, L, D) of one dtype")
    B, Hq, L, D = q_shape
    Hk = k_shape[1]
    if k_shape != (B, Hk, L, D):
        raise ValueError(f"keys {tuple(k_shape)} do not match queries {tuple(q_shape)}")
    if pairs not in PAIRS:
        raise ValueError(f"pairs must be one of {PAIRS}, got {pairs!r}")
    rot = 0
    if inv_shape is not None:
        if len(inv_shape) != 1 or 2 * inv_shape[0] > D:
            raise ValueError(f"inv_freq of shape {tuple(inv_shape)} for a head dim of {D}")
        rot = 2 * inv_shape[0]
    if axis_shape is not None and (axis_shape != (rot // 2,) or axis_dtype != torch.int32):
        raise ValueError(f"axis must be int32 ({rot // 2},), got {axis_dtype} {tuple(axis_shape)}")
    for shape, what in ((qw_shape, "q"), (kw_shape, "k")):
        if shape is not None and shape != (D,):
            raise ValueError(f"{what}_weight of shape {tuple(shape)}: ({D},) is needed")
    code = _lib.torch_dtype_code(q_dtype)
    if pos_shape is None:
        if axis_shape is not None:
            raise ValueError("several axes need a positions tensor (axes, L) or (axes, B, L)")
        return Hk, code, rot, 1, 0, (0, 0, 0)
    if pos_dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {pos_dtype}")
    lead = 0 if axis_shape is None else 1
    if len(pos_shape) not in (1 + lead, 2 + lead):
        raise ValueError(f"positions of shape {tuple(pos_shape)} are not " +
                         ("(axes, L) or (axes, B, L)" if lead else "(L,) or (B, L)"))
    rows = len(pos_shape) == 2 + lead
    axes = pos_shape[0] if lead else 1
    if axes < 1 or pos_shape[-1] != L or (rows and pos_shape[lead] not in (1, B)):
        raise ValueError(f"positions of shape {tuple(pos_shape)} for {B} sequences of {L} tokens")
    sb = pos_stride[lead] if rows and pos_shape[lead] == B else 0
    return Hk, code, rot, axes, 4 if pos_dtype == torch.int32 else 8, (pos_stride[0] if lead else 0, sb, pos_stride[-1])


def norm_rope(queries: torch.Tensor, keys: torch.Tensor, positions: Union[int, torch.Tensor],
              inv_freq: Optional[torch.Tensor], axis: Optional[torch.Tensor] = None,
              q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
              eps: float = 1e-6, pairs: str = "half", factor: float = 1.0,
              _direct: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Normed and rotated copies of queries (B, Hq, L, D) and keys (B, Hk, L, D).

    ``q_weight`` / ``k_weight`` (D,): RMS norm over each head's vector times
    the weight; a side without weight keeps its vectors.  ``inv_freq`` (rot/2,)
    f32 on the device: frequency i turns coordinates (i, i + rot/2)
    (``pairs="half"``) or (2i, 2i + 1) (``"adjacent"``) by position *
    inv_freq[i], times ``factor``; coordinates from rot on stay, and None turns
    none.  ``positions``: the first token's position, or integers (L,) or
    (B, L); with ``axis`` (rot/2,) int32, which names the axis that each
    frequency reads, (axes, L) or (axes, B, L).

    Computed in f32 (angles in 64 bits), rounded once; the results are
    contiguous, whatever the inputs' strides.  There is no backward pass.
    """
    if not _direct and torch.compiler.is_compiling():
        tensor = isinstance(positions, torch.Tensor)
        return torch.ops.kaplumba.norm_rope(queries, keys, positions if tensor else None,
                                            0 if tensor else positions, inv_freq, axis, q_weight, k_weight,
                                            float(eps), pairs, float(factor))
    pos = positions if isinstance(positions, torch.Tensor) else None
    given = [t for t in (inv_freq, axis, q_weight, k_weight, pos) if t is not None]
    _same_device(queries, keys, *given)
    if torch.is_grad_enabled() and any([t.requires_grad for t in (queries, keys, *given)]):
        raise NotImplementedError("norm_rope has no backward pass: call it under torch.no_grad()")
    Hk, dtype, rot, axes, pos_bytes, pos_strides = _plan(
        queries.shape, queries.dtype, keys.shape, keys.dtype, *((pos.shape, pos.stride(), pos.dtype) if pos is not None
                                                                else (None, None, None)),
        inv_freq.shape if inv_freq is not None else None, *((axis.shape, axis.dtype) if axis is not None else (None, None)),
        q_weight.shape if q_weight is not None else None, k_weight.shape if k_weight is not None else None, pairs)
    start = 0 if pos is not None else int(positions)
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous()):
        inv_freq = inv_freq.to(torch.float32).contiguous()
    if axis is not None:
        axis = axis.contiguous()
    wtype = 0
    if q_weight is not None:
        q_weight = q_weight.contiguous()
        wtype = q_weight.dtype
    if k_weight is not None:
        k_weight = k_weight.contiguous()
        if wtype and k_weight.dtype != wtype:
            q_weight, k_weight = q_weight.float(), k_weight.float()
        wtype = k_weight.dtype
    if wtype:
        wtype = _lib.torch_dtype_code(wtype)
    if queries.stride(-1) != 1:
        queries = queries.contiguous()
    if keys.stride(-1) != 1:
        keys = keys.contiguous()
    B, Hq, L, D = queries.shape
    q_out = torch.empty_like(queries, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(keys, memory_format=torch.contiguous_format)

    with _device_guard(queries):
        rc = _lib.load().tq_norm_rope(
            queries.data_ptr(), keys.data_ptr(), dtype, B, Hq, Hk, L, D, *queries.stride()[:3], *keys.stride()[:3],
            q_weight.data_ptr() if q_weight is not None else None,
            k_weight.data_ptr() if k_weight is not None else None, wtype, float(eps), rot,
            1 if pairs == "adjacent" else 0, inv_freq.data_ptr() if inv_freq is not None else None, float(factor),
            axis.data_ptr() if axis is not None else None, axes, pos.data_ptr() if pos is not None else None, pos_bytes,
            start, *pos_strides, q_out.data_ptr(), k_out.data_ptr(), ops._stream(queries))
    _lib.check(rc, "tq_norm_rope")
    return q_out, k_out
