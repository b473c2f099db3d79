"""The 8-bit KV pool's attention where its inputs are unusual: queries and keys that are not numbers,
rows that no request covers, grids beyond one launch's limits. Where a kernel is shared with the
bf16 pool, its form is run too."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import HKV, HQ, D, SCALE
from test_gpu_kv_fp8 import (_batch, _bounded, _chunk, _chunk_batch, _decode, _i32, _pool, _say)

pytestmark = pytest.mark.gpu


def _queries(n, seed=0, hq=HQ):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, hq, D, generator=g).to(torch.bfloat16).cuda()


def _as_bf16(pool):
    """The same K and V (exact in bf16) as a bf16 pool."""
    return [torch.from_numpy(x).to(torch.bfloat16).cuda() for x in pool[3:5]]


def _decode_bf16(q, kv, ptr, idx, splits, fixed, seg, slots, variant):
    from sid.kernels.jit import load_ext
    po = torch.full((q.shape[0], HQ, slots, D), float("nan"), device="cuda")
    pl = torch.full((q.shape[0], HQ, slots), float("nan"), device="cuda")
    o = torch.full_like(q, float("nan"))
    load_ext().flash_decode_fwd(q, *kv, ptr, idx, None, splits, fixed, SCALE, po, pl, o,
                                segment_size=seg, grid_slots=slots, variant=variant)
    return o


def _fan_bytes(q, specs, hq=HQ, hkv=HKV, fp8=True):
    from sid.kernels.jit import load_ext
    return load_ext().extend_attention_workspace_bytes(
        len(specs), q.shape[0], hq, hkv, max(e for _, e in specs), max(p + e for p, e in specs),
        fp8=fp8)


# ---- queries that are not numbers -------------------------------------------------------------

@pytest.mark.parametrize("pool8", [True, False], ids=["fp8", "bf16"])
@pytest.mark.parametrize("lens,args", [([70], (1, 0, 0, 1)), ([70, 130], (1, 0, 32, 5)),
                                       ([1500], (1, 0, 32, 47)), ([70, 9, 130, 40, 64], (1, 0, 32, 5)),
                                       ([70, 9, 1500, 40, 64], (1, 0, 32, 47))],
                         ids=["one_slot", "latency", "latency_long", "fixed", "many_slots"])
def test_decode_nonfinite_queries_give_nan(pool8, lens, args):
    """A head whose query holds a NaN or an infinity has no softmax: NaN, whichever merge joins the
    slots, also where every score is minus infinity. The other heads keep their bits."""
    pool, ptr, idx, at = _batch(lens, seed=13)
    k = pool[3]
    kc = pool[0].view(torch.uint8)
    kc[:, 3, 9] = 0xb9             # kv head 3: element 9 of every key is negative
    k[:, 3, 9] = -1.125 * pool[2][:, 3, 0].double().cpu().numpy()
    kv = _as_bf16(pool)
    run = (lambda x, v: _decode(x, pool, ptr, idx, *args, v)) if pool8 else \
        (lambda x, v: _decode_bf16(x, kv, ptr, idx, *args, v))
    q = _queries(len(lens), 3)
    bad = q.clone()
    bad[0, 3, 77] = float("nan")
    bad[0, 7, 9] = float("inf")    # kv head 3: every score -inf
    bad[0, 6, 9] = float("-inf")   # and +inf
    bad[-1, 12, 0] = float("inf")
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    hit[0, [3, 6, 7]] = True
    hit[-1, 12] = True
    for variant in range(4):
        clean, o = run(q, variant), run(bad, variant)
        assert not clean.isnan().any()
        assert torch.equal(o[~hit], clean[~hit]), variant
        assert o[hit].isnan().all(), variant


@pytest.mark.parametrize("args", [(1, 0, 0, 1), (1, 0, 32, 4)], ids=["one_slot", "slots"])
@pytest.mark.parametrize("batch", [1, 5])
def test_decode_every_key_nan_gives_nan(args, batch):
    """A request all of whose keys are NaN: its rows are NaN, and no request's without keys are."""
    lens = [100] + [0, 60, 7, 90][:batch - 1]
    pool, ptr, idx, at = _batch(lens, seed=14)
    q = _queries(batch, 4)
    clean = _decode(q, pool, ptr, idx, *args, 2)
    slots = torch.from_numpy(at[0]).cuda()
    pool[0].view(torch.uint8)[slots, 2] = 0x7f
    pool[2].view(torch.uint8)[slots, 2, 0] = 255
    o = _decode(q, pool, ptr, idx, *args, 2)
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    hit[0, 4:6] = True
    assert o[hit].isnan().all()
    assert torch.equal(o[~hit], clean[~hit])
    if batch > 1:
        assert not o[1].any()


# ---- rows that no request covers ------------------------------------------------------------------

@pytest.mark.parametrize("pool8", [True, False], ids=["fp8", "bf16"])
@pytest.mark.parametrize("fill", [0, 1, 0x3f, 0xff])
def test_fanned_out_rows_behind_the_last_sequence_stay(pool8, fill):
    """With the splits fanned out, as without: rows past the last sequence are left as they were,
    whatever the workspace held."""
    from sid.kernels.jit import load_ext
    specs = [(2048, 32), (900, 5)]
    q, pool, qo, ptr, idx, at, _ = _chunk_batch(specs, seed=18)
    qq = torch.cat([q, q[:7]])
    kv, kw = (pool[:2], dict(kv_scales=pool[2])) if pool8 else (_as_bf16(pool), {})
    need = _fan_bytes(qq, specs, fp8=pool8)
    assert need > 0
    ws = torch.full((need,), fill, dtype=torch.uint8, device="cuda")
    got = []
    for w in (ws, None):
        o = torch.full_like(qq, 7.0)
        load_ext().extend_attention_fwd(qq, *kv, qo, ptr, idx, 32, SCALE, o, 2080, w, **kw)
        assert (o[q.shape[0]:] == 7.0).all()
        got.append(o)
    assert torch.equal(*got)


@pytest.mark.parametrize("pool8", [True, False], ids=["fp8", "bf16"])
@pytest.mark.parametrize("fill", [0, 1])
def test_fanned_out_rows_of_a_refused_request_stay(pool8, fill):
    """A request with fewer keys than new tokens is left out (its rows stay), with the fan-out too."""
    from sid.kernels.jit import load_ext
    specs = [(2048, 32), (0, 40), (700, 9)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=19)
    kv, kw = (pool[:2], dict(kv_scales=pool[2])) if pool8 else (_as_bf16(pool), {})
    lens = [2080, 39, 709]  # one key short
    flat = torch.cat([_i32(a[:n].tolist()) for a, n in zip(at, lens)])
    ptr = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
    need = _fan_bytes(q, specs, fp8=pool8)
    assert need > 0
    got = []
    for w in (torch.full((need,), fill, dtype=torch.uint8, device="cuda"), None):
        o = torch.full_like(q, 7.0)
        load_ext().extend_attention_fwd(q, *kv, qo, ptr, flat, 40, SCALE, o, 2080, w, **kw)
        assert (o[32:72] == 7.0).all()
        assert not o.isnan().any()
        got.append(o)
    assert torch.equal(*got)


# ---- bounds beyond one launch ----------------------------------------------------------------------

def test_chunk_one_long_prompt_among_thousands():
    """5000 requests, one of 4000 tokens: 5 million places for workgroups, nearly all of them empty."""
    rng = np.random.default_rng(1)
    specs = [(int(rng.integers(0, 4)), 1) for _ in range(5000)]
    specs[3210] = (0, 4000)
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=26)
    _say("thousands", q.shape[0])
    o = _chunk(q, pool, qo, ptr, idx, specs, workspace=False)
    assert not o.isnan().any()
    for i in (0, 1, 3209, 3210, 3211, 4999, *rng.integers(0, 5000, 6).tolist()):
        p, e = specs[i]
        a, b = int(qoh[i]), int(qoh[i + 1])
        one = _chunk(q[a:b].contiguous(), pool, _i32([0, e]), _i32([0, p + e]),
                     _i32(at[i].tolist()), [(p, e)], workspace=False)
        assert torch.equal(one, o[a:b]), i


def test_chunk_placed_by_key_count_beyond_one_grid_dimension():
    """200 ragged requests under a bound of 50000 new tokens: the places of the tiles that there are
    come first, over 2^18 in all."""
    from sid.kernels.jit import load_ext
    rng = np.random.default_rng(3)
    specs = [(int(rng.integers(0, 60)), int(rng.integers(1, 90))) for _ in range(200)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=28)
    got = []
    for bound in (50000, 89):
        o = torch.full_like(q, float("nan"))
        load_ext().extend_attention_fwd(q, pool[0], pool[1], qo, ptr, idx, bound, SCALE, o, 150,
                                        None, kv_scales=pool[2])
        assert not o.isnan().any()
        got.append(o)
    assert torch.equal(*got)


@pytest.mark.parametrize("pool8", [True, False], ids=["fp8", "bf16"])
def test_chunk_bound_of_keys_beyond_a_fanned_out_grid(pool8):
    """A bound of 17 million keys (no request has them) asks for more splits than a grid's third
    dimension holds: the keys are walked, with the same bits."""
    from sid.kernels.jit import load_ext
    hkv, specs, bound = 1, [(100, 64)], 17_000_000
    pool = _pool(300, hkv, seed=27)
    q = _queries(64, 27, 2)
    at = np.random.default_rng(2).permutation(300)[:164]
    qo, ptr, idx = _i32([0, 64]), _i32([0, 164]), _i32(at.tolist())
    kv, kw = (pool[:2], dict(kv_scales=pool[2])) if pool8 else (_as_bf16(pool), {})
    ext = load_ext()
    need = ext.extend_attention_workspace_bytes(1, 64, 2, hkv, 64, bound, fp8=pool8)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    o, want = torch.zeros_like(q), torch.zeros_like(q)
    ext.extend_attention_fwd(q, *kv, qo, ptr, idx, 64, SCALE, o, bound, ws, **kw)
    ext.extend_attention_fwd(q, *kv, qo, ptr, idx, 64, SCALE, want, 164, None, **kw)
    assert torch.equal(o, want)
    _bounded(o, q, pool[3][at], pool[4][at], first=100, chunk=True)
