"""Chunk attention over the 4-bit pool: a row's bits follow from its position and its keys alone, also
where its scores move the softmax's reference maximum.

A row keeps the reference maximum of a split's first 32 keys until a score is 24 octaves above it. The
rows of the first test have a score just there, where roundings decide, and one that is higher still
behind it; whether they moved shows in the last bits of p, and so of the output."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import HKV, HQ, D
from test_gpu_kv_fp4_attention import _batch, _chunk, _i32, _of_rows, _queries, _ramp, _say

pytestmark = pytest.mark.gpu

LN2 = float(np.float32(np.log(2)))  # as sm_scale: a score in octaves is q k itself, in fp32 too
EDGES = [0.5, 1.0, 1.5, 2.0, 3.0, 4.0]  # in units of 2^-21 (an ulp of 4)


def _edge_keys(n):
    """K rows (every value exact in the pool) and the queries of a row that stands at the edge and of
    one that is far past it: scores -20 at key 5, 4 + edge 2^-21 (30) at key 40, 4.625 (-96) at key
    70, -96 at all others."""
    k = np.zeros((n, HKV, D))
    k[:, :, [0, 64]], k[:, :, [1, 65]] = -64.0, -32.0
    k[5, :, [0, 64]], k[5, :, [1, 65]] = -16.0, -4.0
    k[40, :, 0], k[40, :, 1], k[40, :, 32] = 4.0, 0.0, 2.0 ** -15
    k[40, :, 64], k[40, :, 65] = 24.0, 6.0
    k[70, :, 0], k[70, :, 1], k[70, :, 33] = 4.0, 0.5, 0.125

    def edge(units):
        q = torch.zeros(HQ, D)
        q[:, [0, 1, 33]] = 1.0
        q[:, 32] = units * 2.0 ** -6
        return q
    past = torch.zeros(HQ, D)
    past[:, [64, 65]] = 1.0
    return k, edge, past


def _run(q, pool, specs, slots, workspace):
    """Chunks (prefix, n) over the keys that `slots` name for each."""
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.jit import load_ext
    qo = _i32(np.cumsum([0] + [e for _, e in specs]).tolist())
    ptr = _i32(np.cumsum([0] + [p + e for p, e in specs]).tolist())
    idx = _i32(np.concatenate([s[:p + e] for s, (p, e) in zip(slots, specs)]).tolist())
    args = (q, pool[0], pool[1], qo, ptr, idx, max(e for _, e in specs), LN2)
    keys = max(p + e for p, e in specs)
    if workspace:
        return extend_attention_fwd(*args, max_kv_len=keys, kv_scales=pool[2])
    o = torch.full_like(q, float("nan"))
    load_ext().extend_attention_fwd(*args, o, keys, None, kv_scales=pool[2])
    return o


@pytest.mark.parametrize("n,workspace", [(130, False), (2100, True), (2100, False)],
                         ids=["walked", "fanned_out", "walked_splits"])
def test_a_row_at_the_edge_does_not_see_its_neighbours(n, workspace):
    _say("edge", n, workspace)
    k, edge, past = _edge_keys(n)
    v = np.random.default_rng(n).normal(size=(n, HKV, D))
    pool = _of_rows((k, v))
    at = np.random.default_rng(1).permutation(n)
    pool = tuple(x.view(torch.uint8)[torch.from_numpy(np.argsort(at)).cuda()].view(x.dtype)
                 for x in pool[:3])  # key i lies in slot at[i]
    rows = [past] + [edge(u) for u in EDGES]
    q = torch.stack(rows).to(torch.bfloat16).cuda()
    first = n - len(rows)
    together = _run(q, pool, [(first, len(rows))], [at], workspace)
    for i, u in enumerate(EDGES, 1):
        alone = _run(q[i:i + 1].contiguous(), pool, [(first + i, 1)], [at], workspace)
        assert torch.equal(alone[0], together[i]), u
        with_others = _run(torch.cat([q[i:i + 1], q]), pool, [(first + i, 1), (first, len(rows))],
                           [at, at], workspace)
        assert torch.equal(with_others[0], together[i]) and torch.equal(with_others[1:], together), u
    # by the formula: what key 5 and the -96s hold is below 2^-24 of a weight
    w = np.exp2(np.array([[4.0 + u * 2.0 ** -21, 4.625] for u in EDGES]))
    w /= w.sum(1, keepdims=True)
    val = pool[1].view(torch.uint8)[torch.from_numpy(at[[40, 70]]).cuda()].cpu().numpy()
    byte = pool[2].view(torch.uint8)[torch.from_numpy(at[[40, 70]]).cuda()].cpu().numpy()[:, :, 1]
    from oracle.kv_fp4 import load_ref
    x = load_ref(val, byte).repeat(2, axis=1)  # [2, HQ, D]
    want = np.einsum("rk,khd->rhd", w, x)
    # p to bf16 (2^-8 of it), the output once more; the rest is fp32, and key 5's weight
    bound = np.einsum("rk,khd->rhd", w, np.abs(x)) * (2.0 ** -8 + 2.0 ** -20) + np.abs(want) * 2.0 ** -8 \
        + 2.0 ** -24 * np.abs(v).max() * 1.25
    assert (np.abs(together[1:].double().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("size", [8.0, 40.0], ids=["moves_now_and_then", "moves_at_most_tiles"])
def test_rising_scores_keep_bits(size):
    """With and without the workspace, alone and in a batch, a chunk cut off multiples of 16; rows of
    a wave differ in how often they move."""
    _say("rising", size)
    specs = [(0, 130), (700, 50), (1000, 40)]
    pool, ptr, idx, at, queries = _ramp([p + e for p, e in specs], 5, True)
    qoh = np.cumsum([0] + [e for _, e in specs])
    q = queries(int(qoh[-1]))
    g = torch.Generator().manual_seed(8)
    q = (q.float() * (torch.rand(q.shape[0], 1, 1, generator=g) * size).cuda()).to(torch.bfloat16)
    o = _chunk(q, pool, _i32(qoh.tolist()), ptr, idx, specs)
    assert torch.isfinite(o).all()
    assert torch.equal(o, _chunk(q, pool, _i32(qoh.tolist()), ptr, idx, specs, workspace=False))
    for i, (p, e) in enumerate(specs):
        a, b = int(qoh[i]), int(qoh[i + 1])
        cuts = [0, 1, 7, e // 2 + 1, e - 3, e]
        for lo, hi in [(0, e)] + list(zip(cuts, cuts[1:])):
            part = _chunk(q[a + lo:a + hi].contiguous(), pool, _i32([0, hi - lo]), _i32([0, p + hi]),
                          _i32(at[i][:p + hi].tolist()), [(p + lo, hi - lo)], workspace=lo % 2 == 0)
            assert torch.equal(part, o[a + lo:a + hi]), (i, lo, hi)


def test_decode_scales_of_either_sign():
    """q at -s is -q at s: the codes' signs alone differ."""
    from sid.kernels.jit import load_ext
    lens = [1, 70, 500, 1300]
    pool, ptr, idx, _ = _batch(lens, seed=4)
    q = _queries(len(lens), 4)

    def run(q, scale, slots):
        po = torch.full((len(lens), HQ, slots, D), float("nan"), device="cuda")
        pl = torch.full((len(lens), HQ, slots), float("nan"), device="cuda")
        o = torch.full_like(q, float("nan"))
        load_ext().flash_decode_fwd(q, pool[0], pool[1], ptr, idx, None, 1, 0, scale, po, pl, o,
                                    segment_size=256 if slots > 1 else 0, grid_slots=slots, variant=3,
                                    kv_scales=pool[2])
        return o
    for slots in (1, 6):
        o = run(q, 0.09, slots)
        assert torch.isfinite(o).all() and torch.equal(run(-q, -0.09, slots), o)
