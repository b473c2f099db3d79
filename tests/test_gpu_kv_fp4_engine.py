"""The engine over a 4-bit KV pool (EngineConfig.kv_cache_dtype "fp4_e2m1") and with scaled rotary
positions: what its fused paths put in the pool and compute equals the unfused ones, and the modes'
guarantees hold as with bf16."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from sid.config import Mode, ModelConfig, SamplingParams
from sid.engine.batch import build_prefill_batch
from sid.engine.engine import Engine
from sid.engine.model_runner import ModelRunner
from test_gpu_kv_fp8_engine import _hashes, _prompts, _requests, _run
from test_gpu_kv_fp8_engine import _cfg as _cfg8

pytestmark = pytest.mark.gpu

HQ, HKV, D = 16, 8, 128
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}


def _cfg(mode=Mode.NONDET, **kw):
    return _cfg8(mode, **{"kv_cache_dtype": "fp4_e2m1", **kw})


def _u8(t):
    return t.view(torch.uint8)


@pytest.mark.parametrize("scaling", [None, YARN], ids=["plain", "yarn"])
@pytest.mark.parametrize("t", [1, 5, 64, 129])
@pytest.mark.parametrize("form", ["qkv", "partials", "chain_bf16", "chain_fp32"])
def test_fused_writers_equal_write_of_unfused(t, form, scaling):
    """q and the pool of the fused epilogues: the bits of the bf16 epilogue's q, and of its K/V
    rows given to reshape_and_cache_fp4."""
    from sid.kernels import ops
    from sid.kernels.kv_fp4 import alloc_cache_fp4, reshape_and_cache_fp4
    from sid.kernels.rope import RotaryEmbedding
    print("fused", form, t, flush=True)
    g = torch.Generator().manual_seed(t)
    width = (HQ + 2 * HKV) * D
    rand = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    qn, kn = (1 + 0.2 * rand(D)).to(torch.bfloat16), (1 + 0.2 * rand(D)).to(torch.bfloat16)
    cs = RotaryEmbedding(D, 4096, 1e6, "cuda", scaling=scaling).cos_sin
    pos = torch.randint(0, 5000, (t,), generator=g).cuda()  # some beyond the table: not rotated
    slots = torch.randperm(t + 8, generator=g)[:t].cuda()
    if t > 3:
        slots[2], slots[3] = -1, t + 8
    if form in ("qkv", "partials"):
        x = rand(t, width).to(torch.bfloat16) if form == "qkv" else rand(4, t, width)
        if t > 3:  # a NaN and an infinity: their vectors are NaN as a whole
            x[..., 1, HQ * D + 130] = float("nan")
            x[..., 0, (HQ + HKV) * D + 700] = float("inf")
        call = lambda kc, vc, sc: ops.qkv_post(  # noqa: E731
            x, qn, kn, 1e-6, pos, cs, slots, kc, vc, HQ, kv_scales=sc)
    else:
        src = rand(t, 1024) if form == "chain_fp32" else rand(t, 1024).to(torch.bfloat16)
        nw = (1 + 0.1 * rand(1024)).to(torch.bfloat16)
        w = ops.pack_decode_weight((0.05 * rand(width, 1024)).to(torch.bfloat16))
        call = lambda kc, vc, sc: ops.rmsnorm_qkv_post(  # noqa: E731
            src, nw, 1e-6, w, qn, kn, pos, cs, slots, kc, vc, HQ, kv_scales=sc)
    n = t + 8
    kb = torch.zeros(n, HKV, D, dtype=torch.bfloat16, device="cuda")
    vb = torch.zeros_like(kb)
    q0 = call(kb, vb, None)
    pool, want = (alloc_cache_fp4(n, HKV, "cuda") for _ in range(2))
    for x4 in pool + want:
        _u8(x4).fill_(0x5a)  # rows that no token names stay
    q1 = call(*pool)
    keep = slots[(slots >= 0) & (slots < n)]
    reshape_and_cache_fp4(kb[keep], vb[keep], *want, keep)
    assert torch.equal(q0, q1)
    for a, b in zip(pool, want):
        assert torch.equal(_u8(a), _u8(b))


def test_fused_writers_refuse_other_pools():
    from sid.kernels import ops
    from sid.kernels.kv_fp4 import alloc_cache_fp4
    from sid.kernels.rope import RotaryEmbedding
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, (HQ + 2 * HKV) * D, generator=g).cuda().bfloat16()
    w = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    cs = RotaryEmbedding(D, 64, 1e6, "cuda").cos_sin
    pos = slots = torch.arange(2, device="cuda")
    k, v, s = alloc_cache_fp4(8, HKV, "cuda")
    run = lambda k, v, s: ops.qkv_post(x, w, w, 1e-6, pos, cs, slots, k, v, HQ, kv_scales=s)  # noqa: E731
    for bad in ((k, v, None), (k, v[:4], s), (k, v, s[:4]), (k, v, _u8(s)), (_u8(k), v, s),
                (k, v.cpu(), s), (k[:, ::2], v[:, ::2], s)):
        with pytest.raises((RuntimeError, ValueError)):
            run(*bad)


@pytest.mark.parametrize("n", [1, 7, 20])
def test_every_driver_gives_the_same_bits(n):
    """Graphs or eager, native executor or op by op, fused chain or separate launches."""
    prompts = _prompts(n, n)
    want = None
    for graphs, native, chain in ((True, True, True), (False, True, True), (False, False, True),
                                  (False, False, False), (False, True, False)):
        runner = ModelRunner(_cfg(use_graphs=graphs), "cuda")
        runner.model.native_extend = native
        runner.model.decode_chain = chain
        logits, pools, _ = _run(runner, prompts)
        if want is None:
            want = (logits, pools)
            assert all(x.isfinite().all() for x in logits)
            continue
        for a, b in zip(want[0] + want[1], logits + pools):
            assert torch.equal(a, b), (graphs, native, chain)


def test_first_layer_stores_the_bf16_pools_rows():
    """Layer 0's K/V depend on the prompt alone: the pool holds the bf16 engine's rows, quantised,
    and KVCache.read gives back what they stand for."""
    from sid.kernels.kv_fp4 import alloc_cache_fp4, gather_cache_fp4, reshape_and_cache_fp4
    prompts = _prompts(4, 3)
    a = ModelRunner(_cfg(), "cuda")
    b = ModelRunner(_cfg(kv_cache_dtype="bfloat16"), "cuda")
    _, _, reqs = _run(a, prompts, steps=0)
    other = _requests(b, prompts)
    b.forward(build_prefill_batch(other, b.kv_cache, "cuda", invariant=False))
    for r, o in zip(reqs, other):
        kb, vb = b.kv_cache.read(0, o.req_row, 0, o.prompt_len)
        pool = alloc_cache_fp4(r.prompt_len, 8, "cuda")
        at = torch.arange(r.prompt_len, device="cuda")
        reshape_and_cache_fp4(kb, vb, *pool, at)
        k, v = a.kv_cache.read(0, r.req_row, 0, r.prompt_len)
        k2, v2 = gather_cache_fp4(*pool, at)
        assert torch.equal(k, k2) and torch.equal(v, v2)
    k, v = a.kv_cache.read(2, reqs[0].req_row, 3, 3)
    assert k.shape == (0, 8, 128) and v.shape == (0, 8, 128)


@pytest.mark.parametrize("mode,temperature", [(Mode.DVR, 0.0), (Mode.DVR, 0.7),
                                              (Mode.BATCH_INVARIANT, 0.0),
                                              (Mode.BATCH_INVARIANT, 0.7)], ids=str)
def test_identical_across_batch_widths(mode, temperature):
    eng = Engine(_cfg(mode))
    assert len(_hashes(eng, temperature)) == 1


def test_extend_decode_backend_and_a_small_pool():
    """Decode through the chunk kernel, and more requests than the pool holds at once."""
    prompts = _prompts(12, 5)
    params = SamplingParams(max_new_tokens=20, ignore_eos=True)
    eng = Engine(_cfg(decode_backend="extend", use_graphs=False))
    assert all(len(o.token_ids) == 20 for o in eng.generate(prompts[:3], params))
    small = Engine(_cfg(Mode.BATCH_INVARIANT, kv_pool_tokens=512))
    big = Engine(_cfg(Mode.BATCH_INVARIANT))
    assert ([o.token_ids for o in small.generate(prompts, params)]
            == [o.token_ids for o in big.generate(prompts, params)])


def test_scaled_positions_reach_the_models_pool():
    """A model with rope_scaling stores keys turned by the scaled angles: layer 0's K of a prompt is
    that of the unscaled model turned back and on, within its bf16 roundings."""
    from sid.kernels.rope import scaled_frequencies
    from sid.model.loader import random_weights
    from sid.model.qwen3 import Qwen3Model
    prompt = _prompts(1, 9, 100, 120)
    out = {}
    for name, scaling in (("plain", None), ("yarn", YARN)):
        runner = ModelRunner(_cfg(kv_cache_dtype="bfloat16", use_graphs=False), "cuda")
        mcfg = dataclasses.replace(runner.mcfg, rope_scaling=scaling)
        runner.model = Qwen3Model(mcfg, random_weights(mcfg, "cuda", seed=7), "cuda")
        _, _, reqs = _run_plain(runner, prompt)
        out[name] = runner.kv_cache.read(0, reqs[0].req_row, 0, len(prompt[0]))[0].double().cpu()
    plain, yarn = out["plain"].numpy(), out["yarn"].numpy()
    half = D // 2
    pos = np.arange(plain.shape[0])[:, None, None]
    f0, g0 = scaled_frequencies(D, ModelConfig().rope_theta)
    f1, g1 = scaled_frequencies(D, ModelConfig().rope_theta, YARN)
    d = pos * (f1 - f0).numpy()[None, None]
    c, s = np.cos(d) * g1 / g0, np.sin(d) * g1 / g0
    a, b = plain[..., :half], plain[..., half:]
    want = np.concatenate([a * c - b * s, b * c + a * s], -1)
    mag = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1) * max(g1, 1.0)
    # half a bf16 step of each stored value, the table's fp32 angles' sines
    assert (np.abs(yarn - want) <= 2.0 ** -8 * (mag + np.abs(want)) + 2.0 ** -20 * mag).all()
    assert np.abs(yarn - plain).max() > 0.1
    # the engine's own setting is that model
    runner = ModelRunner(_cfg(kv_cache_dtype="bfloat16", use_graphs=False, rope_scaling=YARN), "cuda")
    assert runner.mcfg.rope_scaling == YARN
    _, _, reqs = _run_plain(runner, prompt)
    assert np.array_equal(runner.kv_cache.read(0, reqs[0].req_row, 0, len(prompt[0]))[0]
                          .double().cpu().numpy(), yarn)


def _run_plain(runner, prompts):
    reqs = _requests(runner, prompts)
    logits = runner.forward(build_prefill_batch(reqs, runner.kv_cache, "cuda", invariant=False))
    return logits, None, reqs
