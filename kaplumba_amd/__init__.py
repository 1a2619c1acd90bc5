"""kaplumba_amd -- MI355X-native TurboQuant KV-cache hot path.

A from-scratch HIP/gfx950 implementation of the TurboQuant KV cache of
zayutaha/kaplumba (mlx_lm/models/turboquant_cache.py), behind the same cache
API: append-time quantization, decode/verify attention straight from packed
indices, and the mixed-precision fp16-layer split; next to it a group-affine
cache (4- or 8-bit codes), and the norms and rotations of queries and keys
that come before either.
"""
from .cache import (  # noqa: F401
    KVCache,
    QuantizedKVCache,
    TurboQuantKVCache,
    TurboQuantMSEState,
    can_trim_prompt_cache,
    create_attention_mask,
    create_causal_mask,
    load_prompt_cache,
    make_prompt_cache,
    save_prompt_cache,
    trim_prompt_cache,
)
from .batch_cache import BatchKVCache, BatchTurboQuantKVCache  # noqa: F401
from .affine import AffineState, append_affine_kv, attention_affine, dequantize_affine  # noqa: F401
from .rope import norm_rope  # noqa: F401
from .base import attention_step, scaled_dot_product_attention  # noqa: F401

__version__ = "0.1.0"
