"""Norms of queries and keys per head and the rotation by their positions, in one pass.

The step of an attention layer right before ``update_and_fetch``: the
reference's layers rotate queries and keys there (llama.py:90-91), and models
with query and key norms take those first.  Positions may have several axes
(time, height, width), each frequency reading the one it belongs to.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib, ops
from .affine import _device_guard, _same_device

__all__ = ["norm_rope"]

PAIRS = ("half", "adjacent")


def _positions(positions, axis, B: int, L: int, device):
    """(tensor or None, start, strides over (axis, b, l), number of axes)."""
    if not isinstance(positions, torch.Tensor):
        if axis is not None:
            raise ValueError("several axes need a positions tensor (axes, L) or (axes, B, L)")
        return None, int(positions), (0, 0, 0), 1
    p = positions
    if p.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {p.dtype}")
    if p.device != device:
        raise ValueError(f"positions are on {p.device}, the vectors on {device}")
    lead = 0 if axis is None else 1
    if p.dim() not in (1 + lead, 2 + lead):
        raise ValueError(f"positions of shape {tuple(p.shape)} are not " +
                         ("(axes, L) or (axes, B, L)" if lead else "(L,) or (B, L)"))
    axes = p.shape[0] if lead else 1
    if axes < 1 or p.shape[-1] != L or (p.dim() == 2 + lead and p.shape[lead] not in (1, B)):
        raise ValueError(f"positions of shape {tuple(p.shape)} for {B} sequences of {L} tokens")
    sa = p.stride(0) if lead else 0
    sb = p.stride(lead) if p.dim() == 2 + lead and p.shape[lead] == B else 0
    return p, 0, (sa, sb, p.stride(-1)), axes


def _weight(w, dim: int, device, what: str):
    if w is None:
        return None
    if w.shape != (dim,) or w.device != device:
        raise ValueError(f"{what}_weight of shape {tuple(w.shape)} on {w.device}: ({dim},) on {device} is needed")
    return w.contiguous()


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
    given = [t for t in (inv_freq, axis, q_weight, k_weight) if t is not None]
    _same_device(queries, keys, *given)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (queries, keys, *given)):
        raise NotImplementedError("norm_rope has no backward pass: call it under torch.no_grad()")
    if queries.dim() != 4 or keys.dim() != 4 or queries.dtype != keys.dtype:
        raise ValueError(f"queries {tuple(queries.shape)} {queries.dtype} and keys {tuple(keys.shape)} {keys.dtype} "
                         "must be (B, H, L, D) of one dtype")
    B, Hq, L, D = queries.shape
    Hk = keys.shape[1]
    if keys.shape != (B, Hk, L, D):
        raise ValueError(f"keys {tuple(keys.shape)} do not match queries {tuple(queries.shape)}")
    if pairs not in PAIRS:
        raise ValueError(f"pairs must be one of {PAIRS}, got {pairs!r}")
    rot = 0
    if inv_freq is not None:
        if inv_freq.dim() != 1 or 2 * inv_freq.numel() > D:
            raise ValueError(f"inv_freq of shape {tuple(inv_freq.shape)} for a head dim of {D}")
        inv_freq = inv_freq.to(torch.float32).contiguous()
        rot = 2 * inv_freq.numel()
    if axis is not None:
        if axis.shape != (rot // 2,) or axis.dtype != torch.int32:
            raise ValueError(f"axis must be int32 ({rot // 2},), got {axis.dtype} {tuple(axis.shape)}")
        axis = axis.contiguous()
    pos, start, (sa, sb, sl), axes = _positions(positions, axis, B, L, queries.device)
    q_weight = _weight(q_weight, D, queries.device, "q")
    k_weight = _weight(k_weight, D, queries.device, "k")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        q_weight, k_weight = q_weight.float(), k_weight.float()
    w = q_weight if q_weight is not None else k_weight
    dtype = _lib.torch_dtype_code(queries.dtype)
    wtype = _lib.torch_dtype_code(w.dtype) if w is not None else 0
    if queries.stride(-1) != 1:
        queries = queries.contiguous()
    if keys.stride(-1) != 1:
        keys = keys.contiguous()
    q_out = torch.empty((B, Hq, L, D), dtype=queries.dtype, device=queries.device)
    k_out = torch.empty((B, Hk, L, D), dtype=keys.dtype, device=keys.device)

    def ptr(t):
        return t.data_ptr() if t is not None else None

    with _device_guard(queries):
        rc = _lib.load().tq_norm_rope(
            queries.data_ptr(), keys.data_ptr(), dtype, B, Hq, Hk, L, D, queries.stride(0), queries.stride(1),
            queries.stride(2), keys.stride(0), keys.stride(1), keys.stride(2), ptr(q_weight), ptr(k_weight), wtype,
            float(eps), rot, 1 if pairs == "adjacent" else 0, ptr(inv_freq), float(factor), ptr(axis), axes,
            ptr(pos), pos.element_size() if pos is not None else 0, start, sa, sb, sl, q_out.data_ptr(),
            k_out.data_ptr(), ops._stream(queries))
    _lib.check(rc, "tq_norm_rope")
    return q_out, k_out
