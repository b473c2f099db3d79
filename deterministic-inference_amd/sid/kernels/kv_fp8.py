"""The 8-bit KV pool: its format, its writer and its reader.

A K (or V) vector of one token's head, 128 elements, is stored as e4m3 codes c and one power of
two 2^e (an E8M0 byte): x ~ c 2^e with the smallest e for which max |x| <= 448 2^e, -117 <= e <=
119. A pool is three tensors:

    k_cache, v_cache   float8_e4m3fn   [slots, HKV, 128]
    kv_scales          float8_e8m0fnu  [slots, HKV, 2]     (K's scale, V's)

so that ``k_cache.float() * kv_scales[..., :1].float()`` is K: 2064 bytes a token of the Qwen3
shape instead of 4096. A vector that holds an infinity or a NaN is NaN as a whole. Pass
``kv_scales`` to qkv_post / rmsnorm_qkv_post (sid.kernels.ops), DecodeAttention.forward and
extend_attention_fwd to run them on such a pool; EngineConfig(kv_cache_dtype="fp8_e4m3") keeps the
engine's cache in it. The reference's pool is bf16 (sid/engine/kv_cache.py:33-40).
"""

from __future__ import annotations

import torch

from sid.kernels.jit import load_ext

HEAD_DIM = 128


def layer_scales(kv_cache, layer: int):
    """The scales of a KV cache's layer; None where its pools are bf16."""
    scales = getattr(kv_cache, "scales", None)
    return None if scales is None else scales(layer)


def alloc_cache_fp8(num_slots: int, num_kv_heads: int, device) -> tuple:
    """(k_cache, v_cache, kv_scales) of an empty pool: every vector zero."""
    shape = (num_slots, num_kv_heads, HEAD_DIM)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
            for _ in range(2))
    scales = torch.full((num_slots, num_kv_heads, 2), 127, dtype=torch.uint8, device=device)
    return k, v, scales.view(torch.float8_e8m0fnu)


def reshape_and_cache_fp8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                          v_cache: torch.Tensor, kv_scales: torch.Tensor,
                          slot_mapping: torch.Tensor) -> None:
    """Quantise bf16 rows k, v [T, HKV, 128] (any token stride) into slots slot_mapping[t]
    (int64). Slots outside the pool are skipped; a slot is named at most once."""
    load_ext().reshape_and_cache_fp8(k, v, k_cache, v_cache, kv_scales, slot_mapping)


def gather_cache_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scales: torch.Tensor,
                     slots: torch.Tensor) -> tuple:
    """The pool's rows of `slots` (int64) as bf16 k, v [N, HKV, 128], exactly; rows of slots
    outside the pool are zeros."""
    shape = k_cache.shape
    if len(shape) != 3:
        raise RuntimeError("k_cache must be [S, HKV, D]")
    n, hkv, d = slots.numel(), shape[1], shape[2]
    # one allocation for both (an eager call of a few rows is bound by the host)
    k, v = torch.empty((2, n, hkv, d), dtype=torch.bfloat16, device=slots.device).unbind(0)
    flat = slots if slots.dim() == 1 else slots.reshape(-1)
    load_ext().gather_cache_fp8(k_cache, v_cache, kv_scales, flat, k, v)
    return k, v
