"""The 4-bit KV pool's oracle, pinned by hand-computed codes, and its operators' refusals (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.kv_fp4 import BLOCK, e2m1_values, load_ref, store_ref


def test_code_values():
    assert e2m1_values().tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6] + \
        [-0.0, -0.5, -1, -1.5, -2, -3, -4, -6]


def _block(*x):
    out = np.zeros(128)
    out[:len(x)] = x
    return out


@pytest.mark.parametrize("x,byte,codes", [
    # ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4
    ((6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), 127, (7, 0, 2, 2, 4, 4, 6, 6)),
    ((-6.0, -0.26, -0.74, 5.01, 4.99), 127, (15, 9, 9, 7, 6)),
    ((6.03125, 3.0), 128, (5, 3)),           # above 6: the next exponent; 3.0156 -> 3, 1.5
    ((0.75,), 124, (7,)),                    # 6 2^-3
    ((2.0 ** -127,), 2, (0,)),               # below the smallest exponent: a quarter of 2^-125
    ((3 * 2.0 ** -126,), 2, (3,)),           # 1.5 2^-125
    ((1.99 * 2.0 ** 127,), 252, (7,)),       # above the largest: 6 2^125
    ((float("nan"), 1.0), 255, (7, 7)),
    ((1.0, float("-inf")), 255, (7, 7)),
])
def test_store_by_hand(x, byte, codes):
    c, b = store_ref(_block(*x))
    assert b[0] == byte
    assert (b[1:] == (255 if byte == 255 else 2)).all()
    flat = np.stack([c & 15, c >> 4], -1).reshape(-1)
    assert flat[:len(codes)].tolist() == list(codes)


def test_stored_values_are_within_the_formats_rounding():
    """|x - c 2^e| is at most 2^e times 1/4 below 2, 1/2 below 4, 1 up to 6; every c 2^e is a bf16
    value; a block's neighbours do not matter."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(200, 128)) * np.exp(3 * rng.normal(size=(200, 1)))
    c, b = store_ref(x)
    y = load_ref(c, b)
    scale = np.repeat(2.0 ** (b.astype(float) - 127), BLOCK, -1)
    a = np.abs(x) / scale
    assert (a <= 6).all() and (a.reshape(200, -1, BLOCK).max(-1) > 3).all()
    assert (np.abs(x - y) <= scale * np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))).all()
    t = torch.from_numpy(y)
    assert torch.equal(t.to(torch.bfloat16).double(), t)
    c2, b2 = store_ref(x[:, :BLOCK])
    assert np.array_equal(c2, c[:, :BLOCK // 2]) and np.array_equal(b2[:, 0], b[:, 0])


def test_alloc_is_zeros():
    from sid.kernels.kv_fp4 import FP4, alloc_cache_fp4
    k, v, s = alloc_cache_fp4(3, 2, "cpu")
    assert k.shape == v.shape == (3, 2, 64) and k.dtype == v.dtype == FP4
    assert s.shape == (3, 2, 2, 4) and s.dtype == torch.float8_e8m0fnu
    assert not load_ref(k.view(torch.uint8).numpy(), s.view(torch.uint8)[:, :, 0].numpy()).any()


def _lib():
    from sid.kernels.jit import load_ext
    return load_ext().lib


def test_pool_entry_points_refuse_bad_arguments():
    """The library's own checks, before any device work (addresses are never looked at)."""
    lib = _lib()

    def store(k=16, ldk=1024, slots=16, t=1, hkv=8, d=128, s=4, kc=16, sc=16):
        return lib.sid_reshape_and_cache_fp4(k, ldk, 16, 1024, kc, 16, sc, slots, t, hkv, d, s, None)

    def load(k=16, n=1, hkv=8, d=128, s=4, kc=16):
        return lib.sid_gather_cache_fp4(kc, 16, 16, 16, k, 16, n, hkv, d, s, None)

    for call, text in ((lambda: store(t=-1), b"negative"), (lambda: store(d=64), b"head_dim"),
                       (lambda: store(k=0), b"null"), (lambda: store(slots=0), b"null"),
                       (lambda: store(ldk=1016), b"stride"), (lambda: store(ldk=1028), b"stride"),
                       (lambda: store(hkv=0), b"head count"), (lambda: store(s=0), b"empty"),
                       (lambda: store(kc=24), b"aligned"), (lambda: store(sc=8), b"aligned"),
                       (lambda: load(n=-3), b"negative"), (lambda: load(k=0), b"null"),
                       (lambda: load(d=256), b"head_dim"), (lambda: load(kc=8), b"aligned"),
                       (lambda: load(hkv=1 << 20), b"head count")):
        assert call() == 1 and text in lib.sid_last_error()
    assert store(t=0) == 0 and load(n=0) == 0


def test_operators_refuse_cpu_tensors():
    from sid.kernels.kv_fp4 import alloc_cache_fp4, gather_cache_fp4, reshape_and_cache_fp4
    pool = alloc_cache_fp4(4, 8, "cpu")
    x = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    at = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        reshape_and_cache_fp4(x, x, *pool, at)
    with pytest.raises(RuntimeError, match="GPU"):
        gather_cache_fp4(*pool, at)
