"""The engine over an 8-bit KV pool (EngineConfig.kv_cache_dtype "fp8_e4m3"): what its fused paths
put there and compute equals the unfused ones, and the modes' guarantees hold as with bf16."""

from __future__ import annotations

import hashlib

import pytest
import torch

from sid.config import EngineConfig, Mode, SamplingParams
from sid.engine.batch import build_prefill_batch
from sid.engine.engine import Engine
from sid.engine.model_runner import ModelRunner
from sid.engine.request import Request

pytestmark = pytest.mark.gpu


def _cfg(mode=Mode.NONDET, **kw):
    base = dict(kv_pool_tokens=32768, max_reqs=64, max_seq_len=2048, max_decode_batch=64,
                num_layers=3, seed=7, kv_cache_dtype="fp8_e4m3")
    return EngineConfig(mode=mode, **{**base, **kw})


def _prompts(n, seed, lo=8, hi=120):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 151936, (int(torch.randint(lo, hi, (1,), generator=g)),),
                          generator=g).tolist() for _ in range(n)]


def _requests(runner, prompts):
    reqs = []
    for rid, p in enumerate(prompts):
        r = Request(rid, p, SamplingParams(max_new_tokens=64), runner.mcfg.eos_token_ids)
        r.req_row = runner.kv_cache.open_row()
        reqs.append(r)
    return reqs


def _bytes(kv):
    return [t.view(torch.uint8).clone() for ts in (kv.k_pools, kv.v_pools, kv.kv_scales) for t in ts]


def _run(runner, prompts, steps=3):
    """Logits of a prefill and of some decode steps, and the pools after them."""
    reqs = _requests(runner, prompts)
    fb = build_prefill_batch(reqs, runner.kv_cache, "cuda", invariant=False)
    logits = [runner.forward(fb).clone()]
    for r, t in zip(reqs, logits[0].argmax(-1).tolist()):
        r.output_ids.append(t)
    for _ in range(steps):
        fb = runner.prepare_decode(reqs, False)
        logits.append(runner.forward(fb).clone())
        for r, t in zip(reqs, logits[-1].argmax(-1).tolist()):
            r.output_ids.append(t)
    return logits, _bytes(runner.kv_cache), reqs


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
    from sid.kernels.kv_fp8 import alloc_cache_fp8, gather_cache_fp8, reshape_and_cache_fp8
    prompts = _prompts(4, 3)
    a = ModelRunner(_cfg(), "cuda")
    b = ModelRunner(_cfg(kv_cache_dtype="bfloat16"), "cuda")
    _, _, reqs = _run(a, prompts, steps=0)
    other = _requests(b, prompts)
    b.forward(build_prefill_batch(other, b.kv_cache, "cuda", invariant=False))
    for r, o in zip(reqs, other):
        kb, vb = b.kv_cache.read(0, o.req_row, 0, o.prompt_len)
        slots = torch.from_numpy(b.kv_cache.slot_range(o.req_row, 0, o.prompt_len)).cuda()
        assert torch.equal(kb, b.kv_cache.k_pools[0][slots])
        pool = alloc_cache_fp8(r.prompt_len, 8, "cuda")
        at = torch.arange(r.prompt_len, device="cuda")
        reshape_and_cache_fp8(kb, vb, *pool, at)
        k, v = a.kv_cache.read(0, r.req_row, 0, r.prompt_len)
        k2, v2 = gather_cache_fp8(*pool, at)
        assert torch.equal(k, k2) and torch.equal(v, v2)
    k, v = a.kv_cache.read(2, reqs[0].req_row, 3, 3)
    assert k.shape == (0, 8, 128) and v.shape == (0, 8, 128)


WIDTHS = (1, 4, 16)


def _hashes(engine, temperature, max_new=70):
    watched, fillers = _prompts(1, 100)[0], _prompts(16, 200)
    out = set()
    for width in WIDTHS:
        comp = [watched] + fillers[:width - 1]
        pos = {1: 0, 4: 2, 16: 11}[width]
        comp[0], comp[pos] = comp[pos], comp[0]
        params = [SamplingParams(max_new_tokens=max_new, temperature=temperature, seed=1234,
                                 top_p=0.95 if temperature > 0 else 1.0, is_deterministic=True,
                                 ignore_eos=True) for _ in comp]
        ids = engine.generate(comp, params)[pos].token_ids
        assert len(ids) == max_new
        out.add(hashlib.sha256(str(ids).encode()).hexdigest())
    return out


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
    out = eng.generate(prompts[:3], params)
    assert all(len(o.token_ids) == 20 for o in out)
    small = Engine(_cfg(Mode.BATCH_INVARIANT, kv_pool_tokens=512))
    big = Engine(_cfg(Mode.BATCH_INVARIANT))
    a = [o.token_ids for o in small.generate(prompts, params)]
    b = [o.token_ids for o in big.generate(prompts, params)]
    assert a == b
