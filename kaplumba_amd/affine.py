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
"""
from __future__ import annotations

import contextlib
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
    ops._require_device(*ts)
    if any(t.device != ts[0].device for t in ts[1:]):
        raise ValueError(f"tensors are on different devices: {[str(t.device) for t in ts]}")


def _shape_of(st: AffineState, group_size: int, what: str) -> Tuple[int, int]:
    """(dim, bits) of a state from its shapes."""
    c, p = st.codes, st.params
    if c.dim() != 4 or p.dim() != 5 or p.shape[4] != 2 or c.shape[:3] != p.shape[:3]:
        raise ValueError(f"{what} state of shapes {tuple(c.shape)} / {tuple(p.shape)} is not "
                         "(B, H, T, words) codes and (B, H, T, groups, 2) params")
    if c.dtype != torch.uint32:
        raise ValueError(f"{what} codes must be uint32, got {c.dtype}")
    dim = _check_dim(p.shape[3] * group_size, group_size, what)
    for bits in BITS:
        if c.shape[3] * 32 == dim * bits:
            return dim, bits
    raise ValueError(f"{what} rows of {c.shape[3]} words hold no {dim} codes of 4 or 8 bits")


def _check_aligned(st: AffineState, what: str) -> None:
    """Rows of codes are whole 16-byte pieces; a (scale, bias) pair is loaded at once."""
    if st.codes.data_ptr() & 15 or st.params.data_ptr() % (2 * st.params.element_size()):
        raise ValueError(f"{what} state is not aligned (16 bytes of codes, a pair of params)")


def _capacity(st: AffineState, what: str) -> int:
    """Token capacity of the contiguous (B, H, cap, ...) buffers that a state views a token range of."""
    c, p = st.codes, st.params
    B, H, T, pw = c.shape
    pg = 2 * p.shape[3]
    cap = c.stride(1) // pw if H > 1 else c.stride(0) // pw if B > 1 else max(T, 1)
    ok = c.stride(3) == 1 and p.stride(4) == 1 and (p.shape[3] == 1 or p.stride(3) == 2) and cap >= T
    ok = ok and (T <= 1 or (c.stride(2) == pw and p.stride(2) == pg))
    if H > 1:
        ok = ok and c.stride(1) == cap * pw and p.stride(1) == cap * pg
    if B > 1:
        ok = ok and c.stride(0) == H * cap * pw and p.stride(0) == H * cap * pg
    if not ok:
        raise ValueError(f"{what} state must view one token range of contiguous (B, H, cap, {pw}) codes and "
                         f"(B, H, cap, {p.shape[3]}, 2) params")
    _check_aligned(st, what)
    return cap


def _vectors(x: torch.Tensor) -> torch.Tensor:
    """x with a contiguous, 16-byte aligned last axis (compacted where it has none)."""
    if x.stride(-1) != 1:
        return x.contiguous()
    sb, sh, sl, _ = x.stride()
    if (x.data_ptr() | (sb | sh | sl) * x.element_size()) & 15:
        return x.contiguous()
    return x


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
    _same_device(k, v, *k_state, *v_state)
    _check_group(group_size)
    if k.dim() != 4 or v.shape[:3] != k.shape[:3] or v.dim() != 4:
        raise ValueError(f"keys {tuple(k.shape)} and values {tuple(v.shape)} must share (B, H, L)")
    B, H, L, Dk = k.shape
    sides = []
    for x, st, what in ((k, k_state, "key"), (v, v_state, "value")):
        dim, bits = _shape_of(st, group_size, what)
        if x.shape[-1] != dim:
            raise ValueError(f"{what} head dim {x.shape[-1]} != the state's {dim}")
        if x.dtype != st.params.dtype or x.dtype != k.dtype:
            raise ValueError(f"{what}s of {x.dtype} for a state of {st.params.dtype} and keys of {k.dtype}")
        if not (st.codes.is_contiguous() and st.params.is_contiguous()):
            raise ValueError("cache buffers must be contiguous")
        if st.codes.shape[:2] != (B, H) or st.codes.shape[2] != k_state.codes.shape[2]:
            raise ValueError(f"{what} buffers {tuple(st.codes.shape)} do not match ({B}, {H}, capacity)")
        _check_aligned(st, what)
        sides.append(bits)
    cap = k_state.codes.shape[2]
    if not 0 <= offset <= cap - L:
        raise ValueError(f"rows {offset}..{offset + L} are outside the capacity of {cap}")
    k, v = _vectors(k), _vectors(v)
    with _device_guard(k):
        rc = _lib.load().tq_append_affine_kv(
            k.data_ptr(), v.data_ptr(), _lib.torch_dtype_code(k.dtype), B, H, L, Dk, v.shape[-1],
            k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2), sides[0], sides[1],
            group_size, k_state.codes.data_ptr(), k_state.params.data_ptr(), v_state.codes.data_ptr(),
            v_state.params.data_ptr(), cap, offset, ops._stream(k))
    _lib.check(rc, "tq_append_affine_kv")


def dequantize_affine(state: AffineState, group_size: int = 64, dtype: Optional[torch.dtype] = None,
                      _direct: bool = False) -> torch.Tensor:
    """(B, H, T, dim) values ``scale * code + bias`` of a state (a token range of its
    buffers), computed in f32 and rounded once to ``dtype`` (default: the state's)."""
    dtype = dtype or state.params.dtype
    if not _direct and torch.compiler.is_compiling():
        return torch.ops.kaplumba.dequantize_affine(*state, group_size, dtype)
    _same_device(*state)
    dim, bits = _shape_of(state, _check_group(group_size), "cache")
    B, H, T = state.codes.shape[:3]
    out = torch.empty((B, H, T, dim), dtype=dtype, device=state.codes.device)
    code_in, code_out = _lib.torch_dtype_code(state.params.dtype), _lib.torch_dtype_code(dtype)
    if out.numel() == 0:
        return out
    cap = _capacity(state, "cache")
    with _device_guard(out):
        rc = _lib.load().tq_dequantize_affine(
            state.codes.data_ptr(), state.params.data_ptr(), code_in, B, H, T, dim, bits, group_size, cap,
            out.data_ptr(), code_out, ops._stream(out))
    _lib.check(rc, "tq_dequantize_affine")
    return out


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
    _same_device(queries, *k_state, *v_state)
    if torch.is_grad_enabled() and queries.requires_grad:
        raise NotImplementedError("attention_affine has no backward pass: call it under torch.no_grad()")
    _check_group(group_size)
    if queries.dim() != 4:
        raise ValueError(f"queries must be (B, Hq, L, D), got {tuple(queries.shape)}")
    B, Hq, L, Dk = queries.shape
    dim, kb = _shape_of(k_state, group_size, "key")
    Dv, vb = _shape_of(v_state, group_size, "value")
    Hkv, T = k_state.codes.shape[1], k_state.codes.shape[2]
    if dim != Dk:
        raise ValueError(f"query head dim {Dk} != key head dim {dim}")
    if k_state.codes.shape[0] != B or v_state.codes.shape[:3] != k_state.codes.shape[:3]:
        raise ValueError(f"queries of batch {B}, keys {tuple(k_state.codes.shape[:3])} and values "
                         f"{tuple(v_state.codes.shape[:3])} must share (B, Hkv, T)")
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads are not a multiple of {Hkv} kv heads")
    if not queries.dtype == k_state.params.dtype == v_state.params.dtype:
        raise ValueError(f"queries of {queries.dtype} over states of {k_state.params.dtype} and {v_state.params.dtype}")
    dtype = _lib.torch_dtype_code(queries.dtype)
    out = torch.empty((B, Hq, L, Dv), dtype=queries.dtype, device=queries.device)
    if out.numel() == 0:
        return out
    if T == 0:
        return out.zero_()
    cap = _capacity(k_state, "key")
    if _capacity(v_state, "value") != cap:
        raise ValueError("key and value buffers must share a capacity")
    queries = _vectors(queries)
    seq_lens = ops._seq_array(seq_lens, B, queries.device)
    seq_starts = ops._seq_array(seq_starts, B, queries.device)
    mt, mkind, mstr = None, _lib.TQ_MASK_NONE, None
    if mask is not None:
        mt, mkind, mstr = ops.prepare_mask(mask, B, Hkv, Hq // Hkv, L, T, queries.device, grouped=False)
    lib = _lib.load()
    with _device_guard(queries):
        ws = ops._workspace(queries.device, lib.tq_attention_affine_workspace_size(B, Hq, Hkv, L, Dk, Dv, T))
        rc = lib.tq_attention_affine(
            queries.data_ptr(), dtype, B, Hq, Hkv, L, Dk, Dv, queries.stride(0), queries.stride(1),
            queries.stride(2), float(scale), k_state.codes.data_ptr(), k_state.params.data_ptr(), kb,
            v_state.codes.data_ptr(), v_state.params.data_ptr(), vb, group_size, cap, T,
            seq_starts.data_ptr() if seq_starts is not None else None,
            seq_lens.data_ptr() if seq_lens is not None else None, 1 if causal else 0,
            mt.data_ptr() if mt is not None else None, mkind, mstr, out.data_ptr(), ws.data_ptr(), ws.numel(),
            ops._stream(queries))
    _lib.check(rc, "tq_attention_affine")
    return out
