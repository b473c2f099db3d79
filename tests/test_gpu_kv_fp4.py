"""The 4-bit KV pool's writer and reader against their 64-bit oracle (oracle/kv_fp4.py), bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import HKV, HQ, D
from oracle.kv_fp4 import load_ref, store_ref

pytestmark = pytest.mark.gpu


def _say(*a):
    print(*a, flush=True)


def _u8(t):
    return t.view(torch.uint8).cpu().numpy()


def _rows(n, hkv=HKV, seed=0, spread=1.0):
    """bf16 [n, hkv, D] whose vectors and blocks differ in size, with larger channels."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, hkv, D, generator=g) * torch.exp(spread * torch.randn(n, hkv, 1, generator=g))
    x = x * torch.exp(0.5 * torch.randn(n, hkv, 4, generator=g)).repeat_interleave(32, -1)
    x[..., ::31] *= 5.0
    return x.to(torch.bfloat16).cuda()


def _empty(slots, hkv=HKV):
    from sid.kernels.kv_fp4 import alloc_cache_fp4
    return alloc_cache_fp4(slots, hkv, "cuda")


@pytest.mark.parametrize("t,hkv", [(1, 8), (1, 1), (3, 2), (37, 5), (100, 8), (513, 8), (70, 16)])
def test_store_matches_oracle(t, hkv):
    from sid.kernels.kv_fp4 import reshape_and_cache_fp4
    _say("store", t, hkv)
    k, v = _rows(t, hkv, 1, 3.0), _rows(t, hkv, 2, 3.0)
    kc, vc, sc = _empty(t + 20, hkv)
    slots = torch.randperm(t + 20, device="cuda")[:t]
    reshape_and_cache_fp4(k, v, kc, vc, sc, slots)
    at = slots.cpu().numpy()
    for i, (x, c) in enumerate(((k, kc), (v, vc))):
        codes, b = store_ref(x.double().cpu().numpy())
        assert np.array_equal(_u8(c)[at], codes)
        assert np.array_equal(_u8(sc)[at, :, i], b)
    rest = np.setdiff1d(np.arange(t + 20), at)
    assert not _u8(kc)[rest].any() and not _u8(vc)[rest].any() and (_u8(sc)[rest] == 127).all()


def test_store_every_edge_value():
    """Zeros, the exponents' borders (6 2^e and its neighbours), values that clamp at both ends, ties
    between codes, subnormal bf16, infinities and NaNs; a block at an edge beside ordinary ones."""
    from sid.kernels.kv_fp4 import reshape_and_cache_fp4
    rows = [torch.zeros(D), -torch.zeros(D)]
    g = torch.Generator().manual_seed(0)
    for e in list(range(-133, 128, 9)) + [-125, -126, -124, -123, 122, 123, 124, 125, 126, 127]:
        for m in (1.0, 1.5, 1.4921875, 1.5078125, 1.9921875):
            x = torch.randn(D, generator=g).clamp(-0.9, 0.9).double() * m * 2.0 ** e
            x[5] = m * 2.0 ** e
            rows.append(x.float())
            y = torch.randn(D, generator=g)
            y[32:64] = x[:32].float()
            rows.append(y)
    tie = torch.zeros(D)
    tie[0] = 6.0
    tie[1:8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    tie[32:64] = tie[:32] * 2.0 ** -100
    tie[64:96] = tie[:32] * 2.0 ** -123
    rows += [tie, -tie]
    sub = torch.arange(D).float() * 2.0 ** -133
    rows += [sub, -sub]
    for bad in (float("inf"), float("-inf"), float("nan")):
        for at in (0, 77, 127):
            x = torch.randn(D, generator=g)
            x[at] = bad
            rows.append(x)
    x = torch.stack(rows).to(torch.bfloat16)[:, None].repeat(1, HKV, 1).cuda()
    n = x.shape[0]
    kc, vc, sc = _empty(n)
    reshape_and_cache_fp4(x, -x, kc, vc, sc, torch.arange(n, device="cuda"))
    for i, (s, c) in enumerate(((1, kc), (-1, vc))):
        codes, b = store_ref(s * x.double().cpu().numpy())
        assert np.array_equal(_u8(sc)[..., i, :], b)
        got = _u8(c)
        bad = got != codes
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], codes[bad][:4])


def test_store_strided_rows_and_skipped_slots():
    """K and V as columns of a projection; padding (-1) and out-of-range slots; no rows at all."""
    from sid.kernels.kv_fp4 import reshape_and_cache_fp4
    t = 9
    proj = torch.randn(t, (HQ + 2 * HKV) * D, device="cuda").to(torch.bfloat16)
    k = proj[:, HQ * D:(HQ + HKV) * D].view(t, HKV, D)
    v = proj[:, (HQ + HKV) * D:].view(t, HKV, D)
    assert not k.is_contiguous()
    kc, vc, sc = _empty(12)
    slots = torch.tensor([3, -1, 0, 12, 11, -7, 5, 1 << 40, 4], device="cuda")
    reshape_and_cache_fp4(k, v, kc, vc, sc, slots)
    want = _empty(12)
    keep = (slots >= 0) & (slots < 12)
    reshape_and_cache_fp4(k[keep].contiguous(), v[keep].contiguous(), *want, slots[keep])
    for a, b in zip((kc, vc, sc), want):
        assert np.array_equal(_u8(a), _u8(b))
    assert _u8(kc)[3].any() and not _u8(kc)[1].any()
    reshape_and_cache_fp4(k[:0], v[:0], kc, vc, sc, slots[:0])
    with pytest.raises(RuntimeError, match="heads and dims"):
        reshape_and_cache_fp4(k.transpose(1, 2).contiguous().transpose(1, 2), v, kc, vc, sc, slots)


def test_load_every_code_and_scale():
    """All 16 codes under every scale byte that the writer stores, and under NaN's: exact."""
    from sid.kernels.kv_fp4 import gather_cache_fp4
    bytes_ = np.concatenate([np.arange(2, 253), [255]]).astype(np.uint8)
    n = len(bytes_)
    kc, vc, sc = _empty(n, 2)
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(4, 64), (n, 1, 1))
    kc.view(torch.uint8).copy_(torch.from_numpy(codes[:, :2]))
    vc.view(torch.uint8).copy_(torch.from_numpy(codes[:, 2:]))
    sc.view(torch.uint8).copy_(torch.from_numpy(bytes_)[:, None, None, None])
    order = torch.randperm(n, device="cuda")
    k, v = gather_cache_fp4(kc, vc, sc, order)
    at = order.cpu().numpy()
    for got, c in ((k, codes[:, :2]), (v, codes[:, 2:])):
        want = load_ref(c[at], np.broadcast_to(bytes_[at][:, None, None], (n, 2, 4)))
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)
    sc.view(torch.uint8)[7, 1, 0] = torch.tensor([9, 255, 130, 252], dtype=torch.uint8)
    k, _ = gather_cache_fp4(kc, vc, sc, torch.tensor([7], device="cuda"))
    want = load_ref(codes[7:8, 1], np.array([[9, 255, 130, 252]], dtype=np.uint8))
    assert np.array_equal(k[:, 1].double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("n,hkv", [(1, 8), (5, 3), (77, 8), (1000, 8)])
def test_store_then_load(n, hkv):
    from sid.kernels.kv_fp4 import gather_cache_fp4, reshape_and_cache_fp4
    k, v = _rows(n, hkv, 3), _rows(n, hkv, 4)
    pool = _empty(n + 5, hkv)
    slots = torch.randperm(n + 5, device="cuda")[:n]
    reshape_and_cache_fp4(k, v, *pool, slots)
    got = gather_cache_fp4(*pool, slots.view(1, -1))
    for x, y in zip((k, v), got):
        assert np.array_equal(y.double().cpu().numpy(), load_ref(*store_ref(x.double().cpu().numpy())))
    out = gather_cache_fp4(*pool, torch.tensor([-1, n + 5, 1 << 50, int(slots[0])], device="cuda"))
    assert not out[0][:3].any() and torch.equal(out[0][3], got[0][0]) and torch.equal(out[1][3], got[1][0])
    assert gather_cache_fp4(*pool, slots[:0])[0].shape == (0, hkv, D)


def test_rows_read_back_are_stored_again_unchanged():
    """What a pool stands for is stored as it is: moving a request's cache loses nothing."""
    from sid.kernels.kv_fp4 import gather_cache_fp4, reshape_and_cache_fp4
    n = 300
    pool, again = _empty(n), _empty(n)
    at = torch.arange(n, device="cuda")
    reshape_and_cache_fp4(_rows(n, seed=5, spread=4.0), _rows(n, seed=6), *pool, at)
    rows = gather_cache_fp4(*pool, at)
    reshape_and_cache_fp4(*rows, *again, at)
    for x, y in zip(rows, gather_cache_fp4(*again, at)):
        assert torch.equal(x, y)


def test_pool_refusals():
    from sid.kernels.kv_fp4 import gather_cache_fp4, reshape_and_cache_fp4
    x = _rows(2)
    kc, vc, sc = _empty(4)
    at = torch.arange(2, device="cuda")
    u8 = kc.view(torch.uint8)
    for args, text in (((x, x, u8, vc, sc, at), "k_cache must be"), ((x.float(), x, kc, vc, sc, at), "bf16"),
                       ((x, x[:1], kc, vc, sc, at), "k's shape"), ((x, x, kc, vc, sc, at[:1]), "T entries"),
                       ((x, x, kc, vc[:2], sc, at), "both be"), ((x, x, kc, vc, sc[:, :, :1], at), "contig"),
                       ((x, x, kc, vc, sc[..., 0].contiguous(), at), "kv_scales must be"),
                       ((x, x, kc, vc, sc, at.int()), "slot_mapping must be"),
                       ((x[:, :4], x[:, :4], kc, vc, sc, at), "matching the cache"),
                       ((x, x, kc, vc, sc.cpu(), at), "GPU")):
        with pytest.raises(RuntimeError, match=text):
            reshape_and_cache_fp4(*args)
    with pytest.raises(RuntimeError, match="kv_scales must be"):
        gather_cache_fp4(kc, vc, sc[:2], at)
    from sid.kernels.kv_fp8 import alloc_cache_fp8
    k8, v8, s8 = alloc_cache_fp8(4, HKV, "cuda")
    with pytest.raises(RuntimeError, match="k_cache"):
        reshape_and_cache_fp4(x, x, k8, v8, s8, at)


def test_store_and_load_on_another_stream_and_in_a_graph():
    from sid.kernels.kv_fp4 import gather_cache_fp4, reshape_and_cache_fp4
    n = 50
    x, y = _rows(n, seed=8), _rows(n, seed=9)
    want = [torch.from_numpy(load_ref(*store_ref(t.double().cpu().numpy()))) for t in (x, y)]
    pool, at = _empty(n), torch.arange(n, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        reshape_and_cache_fp4(x, y, *pool, at)
        got = gather_cache_fp4(*pool, at)
        graph = torch.cuda.CUDAGraph()
        kin, vin = torch.zeros_like(x), torch.zeros_like(y)
        reshape_and_cache_fp4(kin, vin, *pool, at)
        side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.double().cpu(), b)
    with torch.cuda.graph(graph):
        reshape_and_cache_fp4(kin, vin, *pool, at)
        out = gather_cache_fp4(*pool, at)
    for _ in range(3):
        kin.copy_(x)
        vin.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a.double().cpu(), b)
        kin.zero_()
        vin.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert not out[0].any() and not out[1].any()
