"""The 8-bit KV pool on the CPU: its oracle against torch's conversion and hand-computed codes,
and the entry points' refusals (all of which come before any device work)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle.kv_fp8 import e4m3_values, load_ref, store_ref


@pytest.fixture(scope="module")
def lib():
    from sid.kernels.jit import load_ext
    return load_ext().lib


def test_code_table():
    t = e4m3_values()
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, want, equal_nan=True)
    assert t[0x7e] == 448.0 and t[1] == 2.0 ** -9 and t[8] == 2.0 ** -6 and np.isnan(t[0x7f])


def test_store_ref_by_hand():
    x = np.zeros((6, 128))
    x[0, 0] = 448.0           # exactly 448 2^0
    x[1, 0] = 449.0           # just above: e = 1
    x[2, :3] = [1.0, 0.5, -0.25]
    x[3, 0] = 3.3e38          # above 448 2^119: saturates
    x[4, 0] = np.inf
    codes, b = store_ref(x)
    assert b.tolist()[:3] == [127, 128, 127 - 8]      # 1.0 <= 448 2^-8 = 1.75
    assert b[3] == 246 and codes[3, 0] == 0x7e
    assert b[4] == 255 and (codes[4] == 0x7f).all()
    assert b[5] == 10 and (codes[5] == 0).all()
    assert load_ref(codes, b)[2, :3].tolist() == [1.0, 0.5, -0.25]
    assert codes[1, 0] == 0x76  # 224.5 -> 224 = 1.75 2^7


def test_store_ref_rounds_like_torch():
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(400, 128, generator=g) * torch.exp(3 * torch.randn(400, 1, generator=g)))
    x = x.to(torch.bfloat16).double()
    codes, b = store_ref(x.numpy())
    y = (x * torch.exp2(127.0 - torch.from_numpy(b).double())[:, None]).float()
    assert np.array_equal(codes, y.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    # half a step of 3 mantissa bits: 2^-4 of a normal value, 2^-10 below
    err = np.abs(load_ref(codes, b) - x.numpy())
    assert (err <= np.maximum(2.0 ** -4 * x.abs().numpy(), 2.0 ** (b[:, None] - 127.0 - 10))).all()


F = ctypes.c_float(0.1)


def _err(lib):
    return lib.sid_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(d=64), "head_dim"), (dict(hkv=0), "head count"), (dict(k=None), "null"),
    (dict(sc=None), "null"), (dict(slots=0), "empty"), (dict(ldk=1000), "strides"),
    (dict(ldk=1028), "strides"), (dict(k=8), "aligned"), (dict(kc=24), "aligned"),
    (dict(t=-1), "negative"),
], ids=str)
def test_store_refusals(lib, change, text):
    a = dict(k=16, ldk=1024, v=16, ldv=1024, kc=16, vc=16, sc=16, map=16, t=4, hkv=8, d=128,
             slots=10)
    a.update(change)
    assert lib.sid_reshape_and_cache_fp8(*a.values(), None) == 1
    assert text in _err(lib)


@pytest.mark.parametrize("change,text", [
    (dict(d=96), "head_dim"), (dict(hkv=-1), "head count"), (dict(v=None), "null"),
    (dict(slots=0), "empty"), (dict(k=4), "aligned"), (dict(n=-2), "negative"),
], ids=str)
def test_gather_refusals(lib, change, text):
    a = dict(kc=16, vc=16, sc=16, idx=16, k=16, v=16, n=3, hkv=8, d=128, slots=10)
    a.update(change)
    assert lib.sid_gather_cache_fp8(*a.values(), None) == 1
    assert text in _err(lib)


DECODE = dict(q=16, kc=16, vc=16, sc=16, ptr=16, idx=16, ns=None, b=2, hq=16, hkv=8, d=128,
              slots=10, ms=4, fixed=0, seg=0, grid=4, variant=0, order=None, scale=F, po=16,
              pl=16, pb=2, ps=4, o=16, workers=0)


@pytest.mark.parametrize("change,text", [
    (dict(d=64), "head_dim"), (dict(hq=8), "q heads"), (dict(sc=None), "null"),
    (dict(q=None), "null"), (dict(variant=4), "variant"), (dict(variant=-1), "variant"),
    (dict(grid=0), "grid_slots"), (dict(grid=1025), "grid_slots"), (dict(ms=0), "max_splits"),
    (dict(fixed=-1), "fixed_split"), (dict(seg=-1), "segment_size"), (dict(po=None), "workspace"),
    (dict(ps=3), "workspace"), (dict(pb=1), "workspace"), (dict(workers=4), "order"),
    (dict(workers=-1), "workers"), (dict(slots=0), "empty"), (dict(kc=17), "aligned"),
    (dict(b=-1), "negative"),
], ids=str)
def test_decode_refusals(lib, change, text):
    assert lib.sid_flash_decode_fp8_fwd(*{**DECODE, **change}.values(), None) == 1
    assert text in _err(lib)


EXTEND = dict(q=16, kc=16, vc=16, sc=16, qo=16, ptr=16, idx=16, b=2, t=8, hq=16, hkv=8, d=128,
              slots=10, me=4, mk=100, scale=F, ws=None, wb=0, o=16)


@pytest.mark.parametrize("change,text", [
    (dict(d=64), "head_dim"), (dict(hq=24), "q heads"), (dict(sc=None), "null"),
    (dict(o=None), "null"), (dict(slots=0), "empty"), (dict(vc=8), "aligned"),
    (dict(b=70000), "grid"), (dict(t=-1), "negative"),
], ids=str)
def test_extend_refusals(lib, change, text):
    assert lib.sid_extend_attention_fp8_fwd(*{**EXTEND, **change}.values(), None) == 1
    assert text in _err(lib)


@pytest.mark.parametrize("batch,total,me,mk,fan", [
    (4, 128, 32, 2080, True), (16, 512, 32, 2080, True), (1, 256, 256, 8256, True),
    (8, 300, 64, 3064, True), (1, 1, 1, 4000, True), (1, 512, 512, 512, False),
    (1, 1024, 1024, 1024, False), (2, 1000, 500, 2500, False), (4, 8192, 2048, 2048, False),
    (64, 64, 1, 9000, False),
], ids=str)
def test_fan_out_rule(lib, batch, total, me, mk, fan):
    need = lib.sid_extend_attention_fp8_workspace_bytes(batch, total, 16, 8, me, mk)
    assert (need > 0) == fan
    assert need <= lib.sid_extend_attention_workspace_bytes(batch, total, 16, 8, me, mk)
    assert not fan or need == (-(-mk // 512) * 130 + 1) * total * 16 * 4


def test_fused_writers_refuse(lib):
    post = [16, None, 0, 4, 16, 8, 128, 16, 16, F, 16, 16, 100, 16, 16, 16, 16, None, 10, None]
    assert lib.sid_qkv_post_fp8(*post) == 1 and "null" in _err(lib)
    norm = [16, 0, 16, F, 16, 4, 1024, 16, 8, 128, 16, 16, 16, 16, 100, 16, 16, 16, 16, None, 10,
            None]
    assert lib.sid_rmsnorm_qkv_post_fp8(*norm) == 1 and "null" in _err(lib)


def test_no_work_is_a_success(lib):
    z = None
    assert lib.sid_reshape_and_cache_fp8(z, 0, z, 0, z, z, z, z, 0, 8, 128, 10, z) == 0
    assert lib.sid_gather_cache_fp8(z, z, z, z, z, z, 0, 8, 128, 10, z) == 0
    assert lib.sid_flash_decode_fp8_fwd(*{**DECODE, "b": 0}.values(), z) == 0
    assert lib.sid_extend_attention_fp8_fwd(*{**EXTEND, "t": 0}.values(), z) == 0


def test_engine_config_and_pool():
    from sid.config import EngineConfig, ModelConfig
    from sid.engine.kv_cache import KVCache
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        EngineConfig(kv_cache_dtype="int3")
    cfg = EngineConfig(kv_pool_tokens=64, max_reqs=2, max_seq_len=64, kv_cache_dtype="fp8_e4m3")
    kv = KVCache(cfg, ModelConfig(num_layers=2), "cpu")
    assert kv.layer(1)[0].dtype == torch.float8_e4m3fn and kv.scales(1).shape == (64, 8, 2)
    with pytest.raises(ValueError, match="head_dim"):
        KVCache(cfg, ModelConfig(num_layers=2, head_dim=64), "cpu")
    plain = KVCache(EngineConfig(kv_pool_tokens=64, max_reqs=2, max_seq_len=64),
                    ModelConfig(num_layers=2), "cpu")
    assert plain.layer(1)[0].dtype == torch.bfloat16 and plain.scales(1) is None


def test_native_forward_refuses_missing_scales(lib):
    from sid.model.native import Batch, Model, _bind
    _bind(lib)
    m, b = Model(), Batch()
    m.num_layers = 2
    none = (ctypes.c_void_p * 2)(16, None)
    assert lib.sid_qwen3_extend_forward_fp8(ctypes.byref(m), ctypes.byref(b), None, None, 0, None,
                                            None, None) == 1
    assert lib.sid_qwen3_extend_forward_fp8(ctypes.byref(m), ctypes.byref(b), none, None, 0, None,
                                            None, None) == 1
    assert "layer 1" in _err(lib)


def test_ops_reject_cpu_tensors():
    from sid.kernels.kv_fp8 import alloc_cache_fp8, gather_cache_fp8, reshape_and_cache_fp8
    k, v, s = alloc_cache_fp8(4, 8, "cpu")
    assert k.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu
    assert not k.float().any() and (s.float() == 1).all() and tuple(s.shape) == (4, 8, 2)
    x = torch.zeros(1, 8, 128, dtype=torch.bfloat16)
    at = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        reshape_and_cache_fp8(x, x, k, v, s, at)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        gather_cache_fp8(k, v, s, at)


# ---------------------------------------------------------------- decode plans (host)

PLAN_BATCHES = [[1], [1024], [300] * 4, [500] * 3, [8192], [2048] * 8, [512] * 16,
                list(range(128, 4097, 128)), [2048] * 64, [4096] * 128, [3000] * 160,
                [1024] * 256, list(range(20, 301)), [100000, 1, 1, 1], [1] * 300, [2_000_000]]


@pytest.mark.parametrize("lens", PLAN_BATCHES, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("bucketed", [False, True])
def test_decode_plan_covers_every_token(lens, bucketed):
    from sid.kernels.decode_attention import (length_bucket, plan_variant_fp8, segment_tokens,
                                              workspace_slots)
    bound = length_bucket(max(lens)) if bucketed else max(lens)
    (splits, seg, slots), variant = plan_variant_fp8(lens, bound, 256, 32)
    assert splits == 1 and variant in (2, 3) and seg % 32 == 0
    assert slots * seg >= bound and slots <= min(workspace_slots(bound, 32, 256), 1024)
    tokens = segment_tokens(lens, len(lens), splits, 0, seg, slots)
    assert tokens.sum(axis=0).tolist() == list(lens)
    if sum(lens) >= 256 * 512 and max(lens) <= 4096:
        # plenty of work: no CU is left more than a third above the mean
        from sid.kernels.decode_attention import _busiest_cu
        assert _busiest_cu(tokens.reshape(-1), 256) <= 1.34 * sum(lens) / 256


def test_decode_plan_of_small_and_empty_batches():
    from sid.kernels.decode_attention import plan_variant_fp8
    assert plan_variant_fp8([1024], 1024, 256, 32) == ((1, 32, 32), 2)  # spread out
    assert plan_variant_fp8([], 1, 256, 32)[0] == (1, 2048, 1)
    assert plan_variant_fp8([0, 0, 5], 5, 256, 32)[0][0] == 1
    assert plan_variant_fp8([0, 1024], 1024, 256, 32) == plan_variant_fp8([1024], 1024, 256, 32)
