"""Wan 2.2 DiT around the in-context sparse attention (the reference's
model.py), for one denoising step on B200s with Ulysses sequence parallelism,
and the low-precision operators that it can run its projections and its
cross-attention in (4-bit linear layers, 8-bit key/value cache).
"""
from .lowp import (  # noqa: F401
    Fp4Tensor,
    Kv8Cache,
    fp4_dequantize,
    fp4_global_scale,
    fp4_linear,
    fp4_quantize,
    kv8_attention,
    kv8_dequantize,
    kv8_quantize,
)
from .model import WanDiT, WanDiTConfig, sinusoidal_embedding_1d  # noqa: F401
from .rope import head_dim_splits, rope_table, token_positions  # noqa: F401

__all__ = ["WanDiT", "WanDiTConfig", "sinusoidal_embedding_1d", "head_dim_splits", "rope_table", "token_positions",
           "Fp4Tensor", "Kv8Cache", "fp4_dequantize", "fp4_global_scale", "fp4_linear", "fp4_quantize",
           "kv8_attention", "kv8_dequantize", "kv8_quantize"]
