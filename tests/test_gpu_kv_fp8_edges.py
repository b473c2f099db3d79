"""The 8-bit KV pool's attention where its inputs are unusual: queries that hold infinities, NaNs,
zeros or outliers, keys that are NaN, rows that no request covers, fanned-out windows behind whose mask
NaNs lie, other head counts, slots outside the pool, grids and bounds beyond one launch's limits. Where
a kernel is shared with the bf16 pool, its form is run too. Bounds: test_gpu_kv_fp8.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import HKV, HQ, D, SCALE
from oracle.kv_fp8 import attention_ref
from test_gpu_kv_fp8 import (_batch, _bounded, _check_decode, _chunk, _chunk_batch, _decode, _i32,
                             _pool, _say)

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


@pytest.mark.parametrize("workspace", [True, False])
def test_chunk_nonfinite_queries_give_nan(workspace):
    specs = [(1000, 70), (0, 40)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=15)
    assert _fan_bytes(q, specs) > 0
    clean = _chunk(q, pool, qo, ptr, idx, specs, workspace)
    bad = q.clone()
    bad[0, 3, 77] = float("nan")
    bad[17, 7, 9] = float("inf")
    bad[69, 0, 127] = float("-inf")
    bad[75, 15, 64] = float("inf")
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    for row, h in ((0, 3), (17, 7), (69, 0), (75, 15)):
        hit[row, h] = True
    o = _chunk(bad, pool, qo, ptr, idx, specs, workspace)
    assert not clean.isnan().any()
    assert o[hit].isnan().all()
    assert torch.equal(o[~hit], clean[~hit])


# ---- queries of zeros, tiny ones, and with outliers ---------------------------------------------

def test_zero_and_tiny_queries_take_the_mean():
    """A query of zeros weighs its keys alike, and so does one of bf16's smallest values."""
    specs = [(700, 40)]
    q, pool, qo, ptr, idx, at, _ = _chunk_batch(specs, seed=16)
    q[::2] = 0
    q[1::4] = 2.0 ** -133
    for ws in (True, False):
        _bounded(_chunk(q, pool, qo, ptr, idx, specs, ws), q, pool[3][at[0]], pool[4][at[0]],
                 first=700, chunk=True)
    pool, ptr, idx, at = _batch([90, 300], seed=16)
    q = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device="cuda")
    q[1, ::2] = -2.0 ** -133
    for args in ((1, 0, 0, 1), (1, 0, 64, 5)):
        _check_decode(_decode(q, pool, ptr, idx, *args, 2), q, pool, at)


def _outlier_case(ratio):
    """Queries with one element `ratio` times the others' size, over keys that are zero there: what
    is left of the scores is the small elements' alone."""
    specs = [(1000, 48)]
    q, pool, qo, ptr, idx, at, _ = _chunk_batch(specs, seed=17)
    assert _fan_bytes(q, specs) > 0
    dims = torch.randint(0, D, (q.shape[0], HQ), generator=torch.Generator().manual_seed(1)).cuda()
    dims = dims % 4 * 37  # four dims, so that the keys stay mostly as they are
    q.scatter_(2, dims[..., None], float(ratio))
    for d in (0, 37, 74, 111):
        pool[0].view(torch.uint8)[:, :, d] = 0
        pool[3][:, :, d] = 0.0
    return specs, q, pool, qo, ptr, idx, at[0]


@pytest.mark.parametrize("ratio", [2.0 ** 6, 2.0 ** 12, 2.0 ** 16, 2.0 ** 20])
def test_chunk_queries_with_outliers(ratio):
    """The chunk kernel splits a query into two e4m3 vectors of scale 2^e, 2^e < max |q| / 224: an
    element below 2^-6 2^e is off by up to 2^-14 2^e, and a score by the sum of that over |k|. That
    joins the bound of a score's own error (derivation: test_gpu_kv_fp8.py)."""
    specs, q, pool, qo, ptr, idx, at = _outlier_case(ratio)
    qd, k, v = q.double().cpu().numpy(), pool[3][at], pool[4][at]
    ref, mag, top = attention_ref(qd, k, v, SCALE, specs[0][0])
    n = k.shape[0]
    e = np.exp2(np.ceil(np.log2(np.abs(qd).max(-1) / 448.0)))        # [T, HQ]
    k1 = np.abs(k).sum(-1).max(0)                                    # [HKV]
    split = 2.0 ** -14 * e * k1.repeat(HQ // HKV)[None] * SCALE
    err_p = 136 * 2.0 ** -24 * top + 2.0 ** -20 + split[..., None]
    tol = 2.0 ** -8 * np.abs(ref) + 2 * err_p * np.abs(v).max() + (n + 64) * 2.0 ** -24 * mag \
        + 2.0 ** -8 * mag
    for ws in (True, False):
        o = _chunk(q, pool, qo, ptr, idx, specs, ws).double().cpu().numpy()
        assert np.isfinite(o).all()
        assert (np.abs(o - ref) <= tol).all()


@pytest.mark.parametrize("ratio", [2.0 ** 6, 2.0 ** 16])
def test_decode_queries_with_outliers(ratio):
    """Decode takes q as it is: outliers cost nothing."""
    _, q, pool, _, ptr, idx, at = _outlier_case(ratio)
    q = q[:1].contiguous()
    for args in ((1, 0, 0, 1), (1, 0, 64, 17)):
        _check_decode(_decode(q, pool, ptr, idx, *args, 2), q, pool, [at])


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


# ---- NaNs behind the mask of a fanned-out window ----------------------------------------------------

FAN_SPECS = [[(1000, 70)], [(2048, 32)] * 4, [(1526, 50)], [(505, 64), (2000, 17)]]


@pytest.mark.parametrize("which", [0, 1], ids=["nan_k", "nan_v"])
@pytest.mark.parametrize("specs", FAN_SPECS, ids=str)
def test_fanned_out_nan_reaches_only_rows_that_see_it(specs, which):
    """NaN keys at a sequence's first and last place, at tiles' and splits' first and last, in a split
    that only a workgroup's later rows reach: the rows that see the key are NaN, the others keep
    their bits. In every request in turn, both with the fan-out and without."""
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=20)
    assert _fan_bytes(q, specs) > 0
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    assert not clean.isnan().any()
    assert torch.equal(clean, _chunk(q, pool, qo, ptr, idx, specs, workspace=False))
    codes, sc = pool[which].view(torch.uint8), pool[2].view(torch.uint8)
    for i in {0, len(specs) - 1}:
        p, e = specs[i]
        keys = {0, 63, 64, 511, 512, 1023, 1024, 1535, 1536, 2047, 2048, p - 1, p, p + 1, p + 15,
                p + 16, p + 31, p + 32, p + e - 2, p + e - 1}
        for key in sorted(x for x in keys if 0 <= x < p + e):
            slot, head = int(at[i][key]), key % HKV
            kept = codes[slot, head].clone(), sc[slot, head].clone()
            codes[slot, head] = 0x7f
            sc[slot, head, which] = 255
            hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
            hit[int(qoh[i]) + max(0, key - p):int(qoh[i + 1]), 2 * head:2 * head + 2] = True
            for ws in (True, False):
                o = _chunk(q, pool, qo, ptr, idx, specs, ws)
                assert o[hit].isnan().all(), (i, key, ws)
                assert torch.equal(o[~hit], clean[~hit]), (i, key, ws)
            codes[slot, head], sc[slot, head] = kept


def test_fanned_out_slot_zero_and_unnamed_rows_of_nan():
    """Every slot that no request names, slot 0 among them, holds NaNs: nothing reaches a row."""
    specs = [(1000, 70), (2048, 3)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=22)
    assert _fan_bytes(q, specs) > 0
    used = np.concatenate(at)
    if 0 in used:  # give slot 0's row another place
        spare = int(np.setdiff1d(np.arange(pool[3].shape[0]), used)[-1])
        for t in pool[:3]:
            t.view(torch.uint8)[spare] = t.view(torch.uint8)[0]
        idx[idx == 0] = spare
        used = np.where(used == 0, spare, used)
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    free = torch.from_numpy(np.setdiff1d(np.arange(pool[3].shape[0]), used)).cuda()
    assert 0 in free
    for t, val in zip(pool[:3], (0x7f, 0x7f, 255)):
        t.view(torch.uint8)[free] = val
    for ws in (True, False):
        assert torch.equal(_chunk(q, pool, qo, ptr, idx, specs, ws), clean)


def test_fanned_out_alone_in_a_batch_and_walked_keep_bits():
    """Requests that fan out alone, in a batch that fans out and in one that walks."""
    specs = [(2048, 32), (1400, 1), (3001, 64), (530, 33)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=23)
    assert _fan_bytes(q, specs) > 0
    o = _chunk(q, pool, qo, ptr, idx, specs)
    assert torch.equal(o, _chunk(q, pool, qo, ptr, idx, specs, workspace=False))
    for i, (p, e) in enumerate(specs[:3]):
        a, b = int(qoh[i]), int(qoh[i + 1])
        assert _fan_bytes(q[a:b], [(p, e)]) > 0
        one = _chunk(q[a:b].contiguous(), pool, _i32([0, e]), _i32([0, p + e]),
                     _i32(at[i].tolist()), [(p, e)])
        assert torch.equal(one, o[a:b])


def test_fanned_out_chunk_in_a_graph():
    """A captured window whose splits fan out, replayed over other pools' contents and queries with
    eager work between the replays: as its eager run and as the walking kernel."""
    from sid.kernels.extend_attention import extend_attention_fwd
    specs = [(1000, 40), (2000, 8)]
    q, pool, qo, ptr, idx, at, _ = _chunk_batch(specs, seed=24)
    assert _fan_bytes(q, specs) > 0

    def run():
        return extend_attention_fwd(q, pool[0], pool[1], qo, ptr, idx, 40, SCALE, max_kv_len=2008,
                                    kv_scales=pool[2])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for step in range(4):
        q.copy_(_queries(q.shape[0], 50 + step))
        pool[0].view(torch.uint8)[step::5, step] ^= 0x80
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, run())
        assert torch.equal(got, _chunk(q, pool, qo, ptr, idx, specs, workspace=False))
        torch.zeros(1 << 20, device="cuda").sum().item()


# ---- other head counts, slots outside the pool ----------------------------------------------------

@pytest.mark.parametrize("hkv", [1, 2, 5, 16])
@pytest.mark.parametrize("specs", [[(1000, 70)], [(3, 90), (700, 1), (0, 33)], [(100, 1100)] * 3],
                         ids=["window", "ragged", "long"])
def test_chunk_other_head_counts(hkv, specs):
    from sid.kernels.jit import load_ext
    _say("heads", hkv, specs)
    lens = [p + e for p, e in specs]
    size = sum(lens) + 9
    pool = _pool(size, hkv, seed=hkv)
    rng = np.random.default_rng(hkv)
    at = np.split(rng.permutation(size)[:sum(lens)], np.cumsum(lens)[:-1])
    qoh = np.concatenate([[0], np.cumsum([e for _, e in specs])])
    q = _queries(int(qoh[-1]), hkv, 2 * hkv)
    qo, ptr = _i32(qoh.tolist()), _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
    idx = _i32(np.concatenate(at).tolist())
    o = _chunk(q, pool, qo, ptr, idx, specs)
    walked = torch.full_like(q, float("nan"))
    load_ext().extend_attention_fwd(q, pool[0], pool[1], qo, ptr, idx, max(e for _, e in specs),
                                    SCALE, walked, max(lens), None, kv_scales=pool[2])
    assert torch.equal(o, walked)
    for i, (p, e) in enumerate(specs):
        a = int(qoh[i])
        for j in sorted({0, e - 1, *rng.integers(0, e, 6).tolist()}):
            n = p + j + 1
            _bounded(o[a + j:a + j + 1], q[a + j:a + j + 1], pool[3][at[i][:n]],
                     pool[4][at[i][:n]], chunk=True)


@pytest.mark.parametrize("workspace", [True, False])
def test_chunk_bad_slots_read_slot_zero(workspace):
    specs = [(1000, 70), (5, 64)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=25)
    assert _fan_bytes(q, specs) > 0
    bad = idx.clone()
    size = pool[3].shape[0]
    places = [(0, 3, -4), (0, 999, 1 << 30), (0, 1069, size), (0, 64, -2 ** 31), (1, 0, 2 ** 31 - 1)]
    at0 = [a.copy() for a in at]
    for i, key, slot in places:
        bad[int(ptr[i]) + key] = slot
        at0[i][key] = 0
    o = _chunk(q, pool, qo, ptr, bad, specs, workspace)
    for i, (p, e) in enumerate(specs):
        a, b = int(qoh[i]), int(qoh[i + 1])
        _bounded(o[a:b], q[a:b], pool[3][at0[i]], pool[4][at0[i]], first=p, chunk=True)


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
