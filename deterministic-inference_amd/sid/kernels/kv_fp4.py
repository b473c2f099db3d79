"""The 4-bit KV pool: its format, its writer and its reader.

A K (or V) vector of one token's head, 128 elements, is stored as four blocks of 32. A block is 32
e2m1 codes c (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one power of two 2^e (an E8M0
byte): x ~ c 2^e with the smallest e for which max |x| <= 6 2^e, -125 <= e <= 125. A pool is three
tensors:

    k_cache, v_cache   float4_e2m1fn_x2   [slots, HKV, 64]      (two codes a byte, the even
                                                                 element in the low half)
    kv_scales          float8_e8m0fnu     [slots, HKV, 2, 4]    (K's four blocks, V's four)

1088 bytes a token of the Qwen3 shape, where a bf16 pool takes 4096 and an 8-bit one 2064. A
vector that holds an infinity or a NaN is NaN as a whole (byte 255 in all four blocks). Pass
``kv_scales`` with such caches to qkv_post / rmsnorm_qkv_post (sid.kernels.ops),
DecodeAttention.forward and extend_attention_fwd to run them on such a pool;
EngineConfig(kv_cache_dtype="fp4_e2m1") keeps the engine's cache in it. The reference's pool is bf16
(sid/engine/kv_cache.py:33-40).
"""

from __future__ import annotations

import torch

from sid.kernels.jit import load_ext

HEAD_DIM = 128
BLOCK = 32
FP4 = torch.float4_e2m1fn_x2


def alloc_cache_fp4(num_slots: int, num_kv_heads: int, device) -> tuple:
    """(k_cache, v_cache, kv_scales) of an empty pool: every vector zero."""
    shape = (num_slots, num_kv_heads, HEAD_DIM // 2)
    k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(FP4) for _ in range(2))
    scales = torch.full((num_slots, num_kv_heads, 2, HEAD_DIM // BLOCK), 127, dtype=torch.uint8,
                        device=device)
    return k, v, scales.view(torch.float8_e8m0fnu)


def reshape_and_cache_fp4(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                          v_cache: torch.Tensor, kv_scales: torch.Tensor,
                          slot_mapping: torch.Tensor) -> None:
    """Quantise bf16 rows k, v [T, HKV, 128] (any token stride) into slots slot_mapping[t]
    (int64). Slots outside the pool are skipped; a slot is named at most once."""
    load_ext().reshape_and_cache_fp4(k, v, k_cache, v_cache, kv_scales, slot_mapping)


def gather_cache_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_scales: torch.Tensor,
                     slots: torch.Tensor) -> tuple:
    """The pool's rows of `slots` (int64) as bf16 k, v [N, HKV, 128], exactly; rows of slots
    outside the pool are zeros."""
    shape = k_cache.shape
    if len(shape) != 3:
        raise RuntimeError("k_cache must be [S, HKV, D / 2]")
    n, hkv = slots.numel(), shape[1]
    # one allocation for both (an eager call of a few rows is bound by the host)
    k, v = slots.new_empty((2, n, hkv, HEAD_DIM), dtype=torch.bfloat16).unbind(0)
    flat = slots if slots.dim() == 1 else slots.reshape(-1)
    load_ext().gather_cache_fp4(k_cache, v_cache, kv_scales, flat, k, v)
    return k, v
