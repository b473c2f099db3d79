"""A whole model over the 8-bit KV pool: its logits against those over a bf16 pool, with the pool's
rows quantised there too (what the attention kernels may differ by) and with them as they are (what
the format costs)."""

from __future__ import annotations

import pytest
import torch

from sid.engine.batch import build_prefill_batch
from sid.engine.model_runner import ModelRunner
from sid.kernels.kv_fp8 import alloc_cache_fp8, gather_cache_fp8, reshape_and_cache_fp8
from test_gpu_kv_fp8_engine import _cfg, _prompts, _requests

pytestmark = pytest.mark.gpu


def _quantise_rows_first(model):
    """Every attention finds its step's rows of the bf16 pool rounded to the 8-bit format's values."""
    attend = model._attend

    def with_quantised_rows(layer, q, fb, kv_cache, *rest):
        k, v = kv_cache.layer(layer)
        slots = fb.out_slots
        pool = alloc_cache_fp8(slots.numel(), k.shape[1], k.device)
        at = torch.arange(slots.numel(), device=k.device)
        reshape_and_cache_fp8(k[slots], v[slots], *pool, at)
        k[slots], v[slots] = gather_cache_fp8(*pool, at)
        return attend(layer, q, fb, kv_cache, *rest)
    model._attend = with_quantised_rows


def _logits(runner, prompts, tokens=None, steps=4):
    """Logits of a prefill and of decode steps; tokens: what the steps append (None: the argmax)."""
    reqs = _requests(runner, prompts)
    out = [runner.forward(build_prefill_batch(reqs, runner.kv_cache, "cuda", invariant=False)).clone()]
    for step in range(steps):
        new = out[-1].argmax(-1).tolist() if tokens is None else tokens[step]
        for r, t in zip(reqs, new):
            r.output_ids.append(t)
        out.append(runner.forward(runner.prepare_decode(reqs, False)).clone())
    return out


def _far(a, b):
    """The largest relative distance of two steps' rows."""
    return max(float(((x - y).norm(dim=-1) / y.norm(dim=-1)).max()) for x, y in zip(a, b))


@pytest.mark.parametrize("lo,hi", [(8, 120), (600, 900)], ids=["short", "long"])
def test_logits_equal_those_over_quantised_bf16_rows(lo, hi):
    """One layer: its K and V depend on the tokens alone, so both pools hold the same values and the
    attention outputs differ by their roundings (of p and of the result, 2^-8 of the mean |v| and
    2^-8 of themselves). The eight roundings to bf16 behind them (o, residual, norm, gate and up, the
    activation, down, residual, norm) may then fall either way, half a step, 2^-8, each: ten times
    2^-8 in all, below 2^-4."""
    prompts = _prompts(5, 11, lo, hi)
    a = _logits(ModelRunner(_cfg(num_layers=1), "cuda"), prompts)
    tokens = [x.argmax(-1).tolist() for x in a]
    b = ModelRunner(_cfg(num_layers=1, kv_cache_dtype="bfloat16", use_graphs=False), "cuda")
    b.model.native_extend = False
    _quantise_rows_first(b.model)
    far = _far(a, _logits(b, prompts, tokens))
    print("relative distance", far, flush=True)
    assert far <= 2.0 ** -4


@pytest.mark.parametrize("lo,hi", [(8, 120), (600, 900)], ids=["short", "long"])
def test_logits_near_those_over_bf16_rows(lo, hi):
    """A stored value is off by at most 2^-4 of itself, so an attention's output is off by about as
    much of its norm at most (the values' roundings are independent; a score's, a sum of 128 of them,
    is smaller beside 1). What each of the three layers adds to the residual stream is off by no more,
    and its norms keep ratios: 3 2^-4."""
    prompts = _prompts(5, 12, lo, hi)
    a = _logits(ModelRunner(_cfg(), "cuda"), prompts)
    tokens = [x.argmax(-1).tolist() for x in a]
    far = _far(a, _logits(ModelRunner(_cfg(kv_cache_dtype="bfloat16"), "cuda"), prompts, tokens))
    print("relative distance", far, flush=True)
    assert 0.0 < far <= 3 * 2.0 ** -4
