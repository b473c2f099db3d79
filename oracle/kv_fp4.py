"""Oracles of the 4-bit KV pool (numpy, 64 bits).

e2m1_values     the 16 codes' values, from the format: sign, 2 exponent bits (bias 1), 1 mantissa
                bit, subnormals, neither infinity nor NaN.
store_ref       a vector's scale bytes and packed codes, block by block of 32: the smallest e with
                max |x| <= 6 2^e, clamped to [-125, 125]; the nearest code of x / 2^e, ties to the
                even code, by search over the table; a vector with an infinity or a NaN: byte 255
                in every block.
load_ref        what packed codes and scale bytes stand for.
Attention over such a pool: oracle/kv_fp8.py's attention_ref on load_ref's values.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
E_MIN, E_MAX = -125, 125


def e2m1_values() -> np.ndarray:
    c = np.arange(16)
    exp, man = (c >> 1) & 3, (c & 1).astype(np.float64)
    x = np.where(exp == 0, man * 0.5, (1 + man / 2) * 2.0 ** (exp - 1.0))
    return np.where(c & 8, -x, x)


def store_ref(x: np.ndarray) -> tuple:
    """(packed codes uint8 [..., D/2], scale bytes uint8 [..., D/32]) of float64 [..., D]."""
    x = np.asarray(x, dtype=np.float64)
    bad = ~np.isfinite(x).all(-1)
    safe = np.where(bad[..., None], 0.0, x).reshape(*x.shape[:-1], -1, BLOCK)
    top = np.abs(safe).max(-1)
    e = np.full(top.shape, E_MIN, dtype=np.int64)
    for cand in range(E_MIN, E_MAX):  # raise e while the next smaller one does not hold the maximum
        e = np.where(top > 6.0 * 2.0 ** cand, cand + 1, e)
    y = np.clip(safe / (2.0 ** e)[..., None], -6.0, 6.0)
    grid = e2m1_values()[:8]  # 0 .. 6, increasing
    hi = np.clip(np.searchsorted(grid, np.abs(y)), 1, 7)
    lo = hi - 1
    dl, dh = np.abs(y) - grid[lo], grid[hi] - np.abs(y)
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(y), code + 8, code)
    code = np.where(bad[..., None, None], 7, code).reshape(x.shape).astype(np.uint8)
    bytes_ = np.where(bad[..., None], 255, e + 127).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), bytes_


def load_ref(codes: np.ndarray, bytes_: np.ndarray) -> np.ndarray:
    """float64 [..., D] of packed codes [..., D/2] with scale bytes [..., D/32] (255: NaN)."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1, BLOCK)
    scale = np.where(bytes_ == 255, np.nan, 2.0 ** (bytes_.astype(np.float64) - 127.0))
    return (e2m1_values()[c] * scale[..., None]).reshape(*codes.shape[:-1], -1)
