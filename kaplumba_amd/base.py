"""SDPA dispatch of the model layer (models/base.py:160-226 of the reference).

TurboQuant layers attend straight from packed indices; the unquantized
(mixed-precision) layers use the same split-K kernel with plain fp16/bf16
loads, the group-affine ones read their codes.  All run on libkaplumba_tq.so;
there is no dequantize fallback.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .batch_cache import BatchKVCache, _LeftPadded
from .cache import _split_mask
from .rope import norm_rope


def scaled_dot_product_attention(queries: torch.Tensor, keys, values, cache, scale: float,
                                 mask, sinks: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Route attention by cache type, as models/base.py:160-226 does.

    Left-padded batch caches (BatchTurboQuantKVCache, BatchKVCache) attend
    over each row's tokens ``[left_padding[b], _idx)``; their ``make_mask``
    returns None / "causal" and the padding is skipped by the kernel.
    """
    if type(cache).__name__ in ("TurboQuantKVCache", "BatchTurboQuantKVCache"):
        if sinks is not None:
            raise ValueError("TurboQuant KV cache does not support attention sinks.")
        if queries.shape[-2] == 1:
            return cache.decode_attention(queries, keys_state=keys, values_state=values,
                                          scale=scale, mask=mask)
        return cache.prefill_attention(queries, keys_state=keys, values_state=values,
                                       scale=scale, mask=mask)
    if type(cache).__name__ == "QuantizedKVCache":
        if sinks is not None:
            raise ValueError("Quantized KV cache does not support attention sinks.")
        return cache.quantized_attention(queries, keys_state=keys, values_state=values, scale=scale, mask=mask)
    if sinks is not None:
        raise NotImplementedError("attention sinks are not supported by the HIP kernels")
    causal, arr = _split_mask(mask, queries.shape[-2])
    starts = cache._seq_starts(queries.device) if isinstance(cache, BatchKVCache) else None
    return ops.attention_plain(queries, keys, values, scale, causal, seq_starts=starts, mask=arr)


def attention_step(queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, cache, scale: float,
                   mask=None, *, inv_freq: Optional[torch.Tensor] = None, positions=None,
                   axis: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                   k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, pairs: str = "half",
                   factor: float = 1.0) -> torch.Tensor:
    """One attention layer from its projections to its output, over any cache of this package.

    Norms and rotates queries and keys (``norm_rope``), appends keys and values
    to the cache, and attends (llama.py:86-97 of the reference, with the
    norms).  ``positions`` defaults to the cache's own: the new tokens follow
    ``cache.offset``, per row in a left-padded batch cache.
    """
    if positions is None:
        if axis is not None:
            raise ValueError("several axes need positions")
        if isinstance(cache, _LeftPadded):
            at = cache.offset[:, None] + torch.arange(queries.shape[2])
            positions = at.to(device=queries.device, dtype=torch.int32)
        else:
            positions = cache.offset
    queries, keys = norm_rope(queries, keys, positions, inv_freq, axis=axis, q_weight=q_weight, k_weight=k_weight,
                              eps=eps, pairs=pairs, factor=factor)
    keys, values = cache.update_and_fetch(keys, values)
    return scaled_dot_product_attention(queries, keys, values, cache, scale, mask)
