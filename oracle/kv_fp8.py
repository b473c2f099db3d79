"""Oracles of the 8-bit KV pool (numpy, 64 bits).

e4m3_values     the 256 codes' values, from the format: sign, 4 exponent bits (bias 7), 3
                mantissa bits, subnormals, 0x7f / 0xff NaN, no infinity. Pinned by hand-computed
                codes and by torch's own conversion (tests/test_kv_fp8.py).
store_ref       a vector's scale byte and codes: the smallest e with max |x| <= 448 2^e, clamped
                to [-117, 119]; the nearest code of x / 2^e, ties to the code with an even
                mantissa, by search over the table; a vector with an infinity or a NaN: byte
                255, codes 0x7f.
load_ref        what codes and scale bytes stand for.
attention_ref   softmax attention in 64 bits with the error bounds' ingredients: the output, the
                same weights over |v|, and the largest sum |q| |k| of a visible pair.
"""

from __future__ import annotations

import numpy as np


def e4m3_values() -> np.ndarray:
    c = np.arange(256)
    exp, man = (c >> 3) & 15, (c & 7).astype(np.float64)
    x = np.where(exp == 0, man * 2.0 ** -9, (8 + man) * 2.0 ** (exp - 10.0))
    x = np.where(c & 128, -x, x)
    return np.where((c & 127) == 127, np.nan, x)


def store_ref(x: np.ndarray) -> tuple:
    """(codes uint8, scale bytes uint8 [...]) of float64 vectors x [..., D]."""
    x = np.asarray(x, dtype=np.float64)
    bad = ~np.isfinite(x).all(-1)
    safe = np.where(bad[..., None], 0.0, x)
    top = np.abs(safe).max(-1)
    e = np.full(top.shape, -117, dtype=np.int64)
    for cand in range(-117, 119):  # raise e while the next smaller one does not hold the maximum
        e = np.where(top > 448.0 * 2.0 ** cand, cand + 1, e)
    y = np.clip(safe / (2.0 ** e)[..., None], -448.0, 448.0)
    grid = e4m3_values()[:127]  # 0 .. 448, increasing
    hi = np.clip(np.searchsorted(grid, np.abs(y)), 1, 126)
    lo = hi - 1
    dl, dh = np.abs(y) - grid[lo], grid[hi] - np.abs(y)
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(y), code + 128, code)
    code = np.where(bad[..., None], 0x7f, code)
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def load_ref(codes: np.ndarray, bytes_: np.ndarray) -> np.ndarray:
    """float64 values of codes [..., D] with scale bytes [...]."""
    return e4m3_values()[codes] * (2.0 ** (bytes_.astype(np.float64) - 127.0))[..., None]


def attention_ref(q: np.ndarray, k: np.ndarray, v: np.ndarray, sm_scale: float,
                  first: int | None = None) -> tuple:
    """q [T, HQ, D], k and v [L, HKV, D] float64. first: query i sees keys 0 .. first + i; None:
    every key. (output, weights over |v| [T, HQ, D], max sum |q| |k| * sm_scale)."""
    t, hq, _ = q.shape
    n, hkv, _ = k.shape
    g = hq // hkv
    out, mag, top = np.zeros(q.shape), np.zeros(q.shape), 0.0
    if n == 0:
        return out, mag, top
    seen = np.ones((t, n), bool) if first is None else \
        np.arange(n)[None, :] <= first + np.arange(t)[:, None]
    for h in range(hq):
        s = q[:, h] @ k[:, h // g].T * sm_scale
        s = np.where(seen, s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h] = p @ v[:, h // g]
        mag[:, h] = p @ np.abs(v[:, h // g])
        top = max(top, float((np.abs(q[:, h]) @ np.abs(k[:, h // g]).T).max()) * sm_scale)
    return out, mag, top
