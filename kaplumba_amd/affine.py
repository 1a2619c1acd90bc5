"""The group-affine cache's kernels: quantized write, read back, attention.

A row of ``dim`` coordinates is kept as 4- or 8-bit codes with a scale and a
bias for each group of 32, 64 or 128 coordinates (coordinate i stands for
``scale * code_i + bias``): the form of the reference's affine caches
(mixed_quant_cache.py: 8-bit keys, 4-bit values), next to the rotated
codebook indices of ``TurboQuantKVCache``.

An ``AffineState`` holds the codes and the (scale, bias) pairs; its head dim
and bit width follow from its shapes and the group size.  Functions check
their arguments on the host, run on torch's current stream of the tensors'
device and raise as the other wrappers of this package do.

What follows from shapes, strides and types alone (the checks, the layout, the
workspace's size) is worked out once for each such set and remembered: a short
decode step waits for the host (one call 20 -> 11 us of it).
"""
from __future__ import annotations

import contextlib
import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib, ops

__all__ = ["AffineState", "affine_state", "append_affine_kv", "dequantize_affine", "attention_affine"]

GROUP_SIZES = (32, 64, 128)
BITS = (4, 8)
MAX_DIM = 512


class AffineState(NamedTuple):
    """codes (B, H, T, dim * bits / 32) uint32 and params (B, H, T, dim / group_size, 2):
    the (scale, bias) pairs, in the dtype of the vectors."""

    codes: torch.Tensor
    params: torch.Tensor


_NO_GUARD = contextlib.nullcontext()


def _device_guard(t: torch.Tensor):
    """Makes t's device the current one where it is not: a kernel is launched on
    the current device, whatever stream it is given."""
    if torch._C._cuda_getDevice() == t.device.index:
        return _NO_GUARD
    return torch.cuda.device(t.device)


def _check_group(group_size: int) -> int:
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size!r}")
    return int(group_size)


def _check_bits(bits) -> int:
    if bits not in BITS:
        raise ValueError(f"affine codes have 4 or 8 bits, got {bits!r}")
    return int(bits)


def _check_dim(dim: int, group_size: int, what: str) -> int:
    if dim % group_size or not 0 < dim <= MAX_DIM:
        raise ValueError(f"{what} dim {dim} is not a multiple of group_size {group_size} up to {MAX_DIM}")
    return dim


def affine_state(B: int, H: int, capacity: int, dim: int, bits: int, group_size: int, dtype, device) -> AffineState:
    """Zeroed buffers for ``capacity`` tokens of (B, H, ., dim) vectors."""
    _check_dim(dim, _check_group(group_size), "head")
    return AffineState(
        torch.zeros((B, H, capacity, dim * _check_bits(bits) // 32), dtype=torch.uint32, device=device),
        torch.zeros((B, H, capacity, dim // group_size, 2), dtype=dtype, device=device))


def _same_device(*ts: torch.Tensor) -> None:
    """Raises unless all tensors are on one ROCm device."""
    try:
        d = ts[0].get_device()
        same = d >= 0
        for t in ts:
            same &= t.get_device() == d
    except AttributeError:  # not a tensor
        same = False
    if not same:
        ops._require_device(*ts)
        raise ValueError(f"tensors are on different devices: {[str(t.device) for t in ts]}")


@functools.lru_cache(maxsize=1024)
def _layout(c_shape, c_stride, c_dtype, p_shape, p_stride, group_size: int, what: str) -> Tuple[int, int, int]:
    """(dim, bits, capacity) of a state that views a token range of contiguous
    (B, H, cap, ...) buffers, from its shapes and strides."""
    _check_group(group_size)
    if len(c_shape) != 4 or len(p_shape) != 5 or p_shape[4] != 2 or c_shape[:3] != p_shape[:3]:
        raise ValueError(f"{what} state of shapes {tuple(c_shape)} / {tuple(p_shape)} is not "
                         "(B, H, T, words) codes and (B, H, T, groups, 2) params")
    if c_dtype != torch.uint32:
        raise ValueError(f"{what} codes must be uint32, got {c_dtype}")
    B, H, T, pw = c_shape
    dim = _check_dim(p_shape[3] * group_size, group_size, what)
    bits = next((b for b in BITS if pw * 32 == dim * b), None)
    if bits is None:
        raise ValueError(f"{what} rows of {pw} words hold no {dim} codes of 4 or 8 bits")
    pg = 2 * p_shape[3]
    cap = c_stride[1] // pw if H > 1 else c_stride[0] // pw if B > 1 else max(T, 1)
    if B * H * T > 0:
        ok = c_stride[3] == 1 and p_stride[4] == 1 and (p_shape[3] == 1 or p_stride[3] == 2) and cap >= T
        ok = ok and (T <= 1 or (c_stride[2] == pw and p_stride[2] == pg))
        if H > 1:
            ok = ok and c_stride[1] == cap * pw and p_stride[1] == cap * pg
        if B > 1:
            ok = ok and c_stride[0] == H * cap * pw and p_stride[0] == H * cap * pg
        if not ok:
            raise ValueError(f"{what} state must view one token range of contiguous (B, H, cap, {pw}) codes and "
                             f"(B, H, cap, {p_shape[3]}, 2) params")
    return dim, bits, cap


def _check_aligned(st: AffineState, what: str) -> None:
    """Rows of codes are whole 16-byte pieces; a (scale, bias) pair is loaded at once."""
    codes, params = st
    if codes.data_ptr() & 15 or params.data_ptr() % (2 * params.element_size()):
        raise ValueError(f"{what} state is not aligned (16 bytes of codes, a pair of params)")


def _is_contiguous(shape, stride) -> bool:
    want = 1
    for n, st in zip(reversed(shape), reversed(stride)):
        if n != 1 and st != want:
            return False
        want *= max(n, 1)
    return True


def _vectors(x: torch.Tensor) -> torch.Tensor:
    """x with a contiguous, 16-byte aligned last axis (compacted where it has none)."""
    sb, sh, sl, sd = x.stride()
    if sd != 1 or (x.data_ptr() | (sb | sh | sl) * x.element_size()) & 15:
        return x.clone(memory_format=torch.contiguous_format)  # a contiguous x may start off 16 bytes too
    return x


@functools.lru_cache(maxsize=1024)
def _append_plan(k_shape, v_shape, k_dtype, v_dtype, kc_shape, kc_stride, kc_dtype, kp_shape, kp_stride, kp_dtype,
                 vc_shape, vc_stride, vc_dtype, vp_shape, vp_stride, vp_dtype, group_size):
    """(key bits, value bits, capacity) of an append whose shapes and types fit."""
    _check_group(group_size)
    if len(k_shape) != 4 or len(v_shape) != 4 or v_shape[:3] != k_shape[:3]:
        raise ValueError(f"keys {tuple(k_shape)} and values {tuple(v_shape)} must share (B, H, L)")
    bits = []
    for shape, dtype, cs, ct, cd, ps, pt, pd, what in (
            (k_shape, k_dtype, kc_shape, kc_stride, kc_dtype, kp_shape, kp_stride, kp_dtype, "key"),
            (v_shape, v_dtype, vc_shape, vc_stride, vc_dtype, vp_shape, vp_stride, vp_dtype, "value")):
        dim, b, _ = _layout(cs, ct, cd, ps, pt, group_size, what)
        if shape[3] != dim:
            raise ValueError(f"{what} head dim {shape[3]} != the state's {dim}")
        if dtype != pd or dtype != k_dtype:
            raise ValueError(f"{what}s of {dtype} for a state of {pd} and keys of {k_dtype}")
        if not (_is_contiguous(cs, ct) and _is_contiguous(ps, pt)):
            raise ValueError("cache buffers must be contiguous")
        if cs[:2] != k_shape[:2] or cs[2] != kc_shape[2]:
            raise ValueError(f"{what} buffers {tuple(cs)} do not match ({k_shape[0]}, {k_shape[1]}, capacity)")
        bits.append(b)
    _lib.torch_dtype_code(k_dtype)
    return bits[0], bits[1], kc_shape[2]


def append_affine_kv(k: torch.Tensor, v: torch.Tensor, k_state: AffineState, v_state: AffineState, offset: int,
                     group_size: int = 64, _direct: bool = False) -> None:
    """Quantize keys (B, H, L, Dk) and values (B, H, L, Dv) into rows offset..offset+L
    of the states' capacity buffers, in one launch.

    Each side's bit width is that of its state; both share dtype, B, H, L,
    capacity and group size.  A group's bias is its least value, its scale a
    (2^bits - 1)-th of its range rounded to the dtype; a group that holds an
    infinity or NaN stands for NaN.
    """
    if not _direct and torch.compiler.is_compiling():
        return torch.ops.kaplumba.append_affine_kv(k, v, *k_state, *v_state, offset, group_size)
    kc, kp = k_state
    vc, vp = v_state
    _same_device(k, v, kc, kp, vc, vp)
    kb, vb, cap = _append_plan(k.shape, v.shape, k.dtype, v.dtype, kc.shape, kc.stride(), kc.dtype, kp.shape, kp.stride(),
                               kp.dtype, vc.shape, vc.stride(), vc.dtype, vp.shape, vp.stride(), vp.dtype, group_size)
    _check_aligned(k_state, "key")
    _check_aligned(v_state, "value")
    B, H, L, Dk = k.shape
    if not 0 <= offset <= cap - L:
        raise ValueError(f"rows {offset}..{offset + L} are outside the capacity of {cap}")
    k, v = _vectors(k), _vectors(v)
    with _device_guard(k):
        rc = _lib.load().tq_append_affine_kv(
            k.data_ptr(), v.data_ptr(), _lib.torch_dtype_code(k.dtype), B, H, L, Dk, v.shape[-1],
            *k.stride()[:3], *v.stride()[:3], kb, vb, group_size, kc.data_ptr(), kp.data_ptr(), vc.data_ptr(),
            vp.data_ptr(), cap, offset, ops._stream(k))
    _lib.check(rc, "tq_append_affine_kv")


def dequantize_affine(state: AffineState, group_size: int = 64, dtype: Optional[torch.dtype] = None,
                      _direct: bool = False) -> torch.Tensor:
    """(B, H, T, dim) values ``scale * code + bias`` of a state (a token range of its
    buffers), computed in f32 and rounded once to ``dtype`` (default: the state's)."""
    c, p = state
    dtype = dtype or p.dtype
    if not _direct and torch.compiler.is_compiling():
        return torch.ops.kaplumba.dequantize_affine(c, p, group_size, dtype)
    _same_device(c, p)
    dim, bits, cap = _layout(c.shape, c.stride(), c.dtype, p.shape, p.stride(), group_size, "cache")
    B, H, T, _ = c.shape
    out = torch.empty((B, H, T, dim), dtype=dtype, device=c.device)
    code_in, code_out = _lib.torch_dtype_code(p.dtype), _lib.torch_dtype_code(dtype)
    if B * H * T == 0:
        return out
    _check_aligned(state, "cache")
    with _device_guard(out):
        rc = _lib.load().tq_dequantize_affine(c.data_ptr(), p.data_ptr(), code_in, B, H, T, dim, bits, group_size, cap,
                                              out.data_ptr(), code_out, ops._stream(out))
    _lib.check(rc, "tq_dequantize_affine")
    return out


@functools.lru_cache(maxsize=1024)
def _attention_plan(q_shape, q_dtype, kc_shape, kc_stride, kc_dtype, kp_shape, kp_stride, kp_dtype, vc_shape, vc_stride,
                    vc_dtype, vp_shape, vp_stride, vp_dtype, group_size):
    """What an attention call's shapes and types come to, once they fit:
    (Hkv, T, Dv, key bits, value bits, capacity, dtype code, workspace bytes)."""
    _check_group(group_size)
    if len(q_shape) != 4:
        raise ValueError(f"queries must be (B, Hq, L, D), got {tuple(q_shape)}")
    B, Hq, L, Dk = q_shape
    dim, kb, cap = _layout(kc_shape, kc_stride, kc_dtype, kp_shape, kp_stride, group_size, "key")
    Dv, vb, vcap = _layout(vc_shape, vc_stride, vc_dtype, vp_shape, vp_stride, group_size, "value")
    Hkv, T = kc_shape[1], kc_shape[2]
    if dim != Dk:
        raise ValueError(f"query head dim {Dk} != key head dim {dim}")
    if kc_shape[0] != B or vc_shape[:3] != kc_shape[:3]:
        raise ValueError(f"queries of batch {B}, keys {tuple(kc_shape[:3])} and values {tuple(vc_shape[:3])} must share "
                         "(B, Hkv, T)")
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads are not a multiple of {Hkv} kv heads")
    if not q_dtype == kp_dtype == vp_dtype:
        raise ValueError(f"queries of {q_dtype} over states of {kp_dtype} and {vp_dtype}")
    code = _lib.torch_dtype_code(q_dtype)
    if B * Hq * L * T and vcap != cap:
        raise ValueError("key and value buffers must share a capacity")
    ws = _lib.load().tq_attention_affine_workspace_size(B, Hq, Hkv, L, Dk, Dv, T)
    return Hkv, T, Dv, kb, vb, cap, code, ws


def attention_affine(queries: torch.Tensor, k_state: AffineState, v_state: AffineState, group_size: int = 64,
                     scale: float = 1.0, causal: bool = False, seq_lens=None, seq_starts=None, mask=None,
                     _direct: bool = False) -> torch.Tensor:
    """Attention of queries (B, Hq, L, Dk) straight from the states' codes; the
    output is (B, Hq, L, Dv) in the queries' dtype, which is the states' too.

    ``causal``, ``seq_lens`` and ``seq_starts`` as in ``ops.attention_packed``;
    ``mask`` is a boolean or additive array broadcast against (B, Hq, L, T)
    (``ops.prepare_mask``).  A row that sees no key weighs all its tokens
    alike; one whose every score is -inf, and a sequence without tokens, give
    zeros.  There is no backward pass.
    """
    if not _direct and torch.compiler.is_compiling():
        return torch.ops.kaplumba.attention_affine(
            queries, *k_state, *v_state, group_size, float(scale), bool(causal),
            ops._opt_tensor(seq_lens, torch.int32), ops._opt_tensor(seq_starts, torch.int32),
            ops._opt_tensor(mask, None))
    kc, kp = k_state
    vc, vp = v_state
    _same_device(queries, kc, kp, vc, vp)
    if queries.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("attention_affine has no backward pass: call it under torch.no_grad()")
    Hkv, T, Dv, kb, vb, cap, dtype, ws_bytes = _attention_plan(
        queries.shape, queries.dtype, kc.shape, kc.stride(), kc.dtype, kp.shape, kp.stride(), kp.dtype, vc.shape,
        vc.stride(), vc.dtype, vp.shape, vp.stride(), vp.dtype, group_size)
    B, Hq, L, Dk = queries.shape
    if Dv == Dk:
        out = torch.empty_like(queries, memory_format=torch.contiguous_format)
    else:
        out = queries.new_empty((B, Hq, L, Dv))
    if B * Hq * L * T == 0:
        return out.zero_()
    _check_aligned(k_state, "key")
    _check_aligned(v_state, "value")
    queries = _vectors(queries)
    seq_lens = ops._seq_array(seq_lens, B, queries.device)
    seq_starts = ops._seq_array(seq_starts, B, queries.device)
    mt, mkind, mstr = None, _lib.TQ_MASK_NONE, None
    if mask is not None:
        mt, mkind, mstr = ops.prepare_mask(mask, B, Hkv, Hq // Hkv, L, T, queries.device, grouped=False)
    with _device_guard(queries):
        ws = ops._workspace(queries.device, ws_bytes)
        rc = _lib.load().tq_attention_affine(
            queries.data_ptr(), dtype, B, Hq, Hkv, L, Dk, Dv, *queries.stride()[:3], float(scale), kc.data_ptr(),
            kp.data_ptr(), kb, vc.data_ptr(), vp.data_ptr(), vb, group_size, cap, T,
            seq_starts.data_ptr() if seq_starts is not None else None,
            seq_lens.data_ptr() if seq_lens is not None else None, 1 if causal else 0,
            mt.data_ptr() if mt is not None else None, mkind, mstr, out.data_ptr(), ws.data_ptr(), ws.numel(),
            ops._stream(queries))
    _lib.check(rc, "tq_attention_affine")
    return out
