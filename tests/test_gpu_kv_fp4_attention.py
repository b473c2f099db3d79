"""Decode and chunk attention over the 4-bit pool against 64 bits of what the pool stands for, their
invariances, NaNs, odd inputs, and the operators together over a pool that grows. Bounds:
test_gpu_kv_fp8.py (the same roundings: scores and sums in fp32, p to bf16 in the chunk kernel)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import HKV, HQ, D, SCALE
from oracle.kv_fp4 import load_ref, store_ref
from oracle.kv_fp8 import attention_ref
from test_gpu_kv_fp8 import _bounded, _check_decode, _chunk, _decode, _i32, _say

pytestmark = pytest.mark.gpu
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _u8(t):
    return t.view(torch.uint8)


def _of_rows(rows):
    """(k, v, scales on the GPU, float64 K, V) of a pool that the oracle quantised from rows (k, v),
    float64 [slots, hkv, D]."""
    out, vals, bytes_ = [], [], []
    for x in rows:
        codes, b = store_ref(x)
        out.append(torch.from_numpy(codes).cuda().view(FP4))
        bytes_.append(b)
        vals.append(load_ref(codes, b))
    scales = torch.from_numpy(np.stack(bytes_, 2)).cuda().view(E8M0)
    return out[0], out[1], scales, vals[0], vals[1]


def _pool(slots, hkv=HKV, seed=0):
    rng = np.random.default_rng(seed)
    rows = []
    for _ in range(2):
        x = rng.normal(size=(slots, hkv, D)) * np.exp(0.7 * rng.normal(size=(slots, hkv, 1)))
        x *= np.repeat(np.exp(0.5 * rng.normal(size=(slots, hkv, 4))), 32, -1)
        x[..., ::31] *= 3.0
        rows.append(x)
    return _of_rows(rows)


def _batch(lens, seed=0, extra=32, page=None, hkv=HKV):
    """Shuffled slots (or whole pages) for requests of these lengths: (pool, indptr, idx, slots)."""
    rng = np.random.default_rng(seed)
    step = page or 1
    pages = [-(-n // step) for n in lens]
    size = (sum(pages) + (2 if page else extra)) * step
    perm = rng.permutation(size // step)
    first = np.cumsum([0] + pages)
    idx = [perm[f:f + p][np.arange(n) // step] * step + np.arange(n) % step
           for f, p, n in zip(first, pages, lens)]
    flat = np.concatenate(idx) if sum(lens) else np.zeros(1, int)
    return _pool(size, hkv, seed), _i32(np.cumsum([0] + list(lens)).tolist()), _i32(flat.tolist()), idx


def _queries(n, seed=0, hq=HQ):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, hq, D, generator=g).to(torch.bfloat16).cuda()


def _chunk_batch(specs, seed=0, page=None, hkv=HKV):
    pool, ptr, idx, at = _batch([p + e for p, e in specs], seed=seed, page=page, hkv=hkv)
    qo = np.cumsum([0] + [e for _, e in specs])
    return _queries(int(qo[-1]), seed, 2 * hkv), pool, _i32(qo.tolist()), ptr, idx, at, qo


def _fan_bytes(specs, hkv=HKV):
    from sid.kernels.jit import load_ext
    return load_ext().extend_attention_workspace_bytes(
        len(specs), sum(e for _, e in specs), 2 * hkv, hkv, max(e for _, e in specs),
        max(p + e for p, e in specs), fp4=True)


def _make_nan(pool, which, slot, head):
    _u8(pool[2])[slot, head, which] = 255


# ---- decode -----------------------------------------------------------------------------------

@pytest.mark.parametrize("lens", [[1], [2], [7, 8, 9], [31, 32, 33], [63, 64, 65], [255, 256, 257],
                                  [0, 5, 0], [1000, 32, 999], [17 * i + 1 for i in range(17)], [3001]],
                         ids=lambda s: f"b{len(s)}_max{max(s)}")
@pytest.mark.parametrize("variant", [0, 1, 2, 3])
@pytest.mark.parametrize("plan", ["one", "fixed256", "splits4_seg64"])
def test_decode_against_oracle(lens, variant, plan):
    _say("decode", lens, variant, plan)
    pool, ptr, idx, at = _batch(lens, seed=len(lens))
    q = _queries(len(lens), 1)
    longest = max(lens)
    if plan == "one":
        args = (1, 0, 0, 1)
    elif plan == "fixed256":
        args = (max(1, -(-longest // 256)), 256, 256, max(1, -(-longest // 256)))
    else:
        chunk = max(32, -(-(-(-longest // 4)) // 32) * 32)
        args = (4, 0, 64, 4 * -(-chunk // 64))
    _check_decode(_decode(q, pool, ptr, idx, *args, variant), q, pool, at)


@pytest.mark.parametrize("lens", [[1], [1024], [300] * 5 + [1], [2000, 64, 7, 900] * 8,
                                  [700 + i for i in range(96)], [40] * 256,
                                  [128 + 63 * i for i in range(64)]], ids=lambda s: f"b{len(s)}")
def test_decode_step_plan(lens):
    """The plan that a serving loop makes (shape, geometry, order, workers) over paged slots."""
    from sid.kernels.decode_attention import DecodeAttention
    _say("step plan", len(lens))
    pool, ptr, idx, at = _batch(lens, seed=3, page=16)
    q = _queries(len(lens), 2)
    attn = DecodeAttention(len(lens), HQ, HKV, D, 32, 256, 4096, "cuda")
    attn.part_o.fill_(float("nan"))
    attn.part_lse.fill_(float("nan"))
    plan = attn.step_plan(lens, kv_fp4=True)
    run = lambda: attn.forward(q, *pool[:2], ptr, idx, _i32(lens), max(lens), SCALE, False,  # noqa: E731
                               kv_scales=pool[2], **plan)
    o = run()
    for i in range(0, len(lens), max(1, len(lens) // 12)):
        _check_decode(o[i:i + 1], q[i:i + 1], pool, [at[i]])
    assert torch.equal(o, run())


def test_decode_workers_and_orders_keep_bits():
    from sid.kernels.decode_attention import segment_tokens, worker_order, workgroup_order
    lens = [900, 0, 33, 2500, 1, 400, 1300]
    pool, ptr, idx, _ = _batch(lens, seed=9)
    q = _queries(len(lens), 9)
    tok = segment_tokens(lens, len(lens), 0, 256, 256, 10)
    for variant in (2, 3):
        base = _decode(q, pool, ptr, idx, 10, 256, 256, 10, variant)
        o1 = _decode(q, pool, ptr, idx, 10, 256, 256, 10, variant,
                     order=torch.from_numpy(workgroup_order(tok, 256)).cuda())
        assert torch.equal(base, o1)
        for w in (1, 5, 64, 256):
            o2 = _decode(q, pool, ptr, idx, 10, 256, 256, 10, variant,
                         order=torch.from_numpy(worker_order(tok, w)).cuda(), workers=w)
            assert torch.equal(base, o2)


def test_decode_fixed_splits_do_not_depend_on_the_batch():
    from sid.kernels.decode_attention import DecodeAttention
    lens = [700, 1, 256, 3000, 513]
    pool, ptr, idx, at = _batch(lens, seed=5)
    q = _queries(len(lens), 5)
    attn = DecodeAttention(8, HQ, HKV, D, 32, 256, 4096, "cuda")
    o = attn.forward(q, *pool[:2], ptr, idx, _i32(lens), max(lens), SCALE, True, kv_scales=pool[2])
    for i, n in enumerate(lens):
        one = attn.forward(q[i:i + 1].contiguous(), *pool[:2], _i32([0, n]), _i32(at[i].tolist()),
                           _i32([n]), n, SCALE, True, kv_scales=pool[2])
        assert torch.equal(one[0], o[i])


def test_decode_bad_slots_and_nan_rows():
    """Slots outside the pool read slot 0; NaN rows that no request names reach nothing; a NaN key or
    value makes its own request's rows of its head NaN and no others."""
    lens = [70, 130]
    pool, ptr, idx, at = _batch(lens, seed=6)
    q = _queries(2, 6)
    for s in sorted(set(range(pool[3].shape[0])) - set(np.concatenate(at).tolist()) - {0}):
        _u8(pool[2])[s] = 255
    bad = idx.clone()
    bad[3], bad[100] = -4, 1 << 30
    at0 = [a.copy() for a in at]
    at0[0][3] = 0
    at0[1][30] = 0
    for variant in range(4):
        _check_decode(_decode(q, pool, ptr, bad, 4, 0, 64, 8, variant), q, pool, at0)
    for which in (0, 1):
        for key in (50, 69):  # (the last stands in for the positions past the end)
            slot, keep = int(at[0][key]), _u8(pool[2])[int(at[0][key])].clone()
            _make_nan(pool, which, slot, 3)
            for variant in range(4):
                for args in ((4, 0, 64, 8), (1, 0, 0, 1)):
                    o = _decode(q, pool, ptr, idx, *args, variant)
                    assert o[0, 6:8].isnan().all()
                    assert not o[0, :6].isnan().any() and not o[0, 8:].isnan().any()
                    assert not o[1].isnan().any()
            _u8(pool[2])[slot] = keep


@pytest.mark.parametrize("lens,args", [([70], (1, 0, 0, 1)), ([70, 130], (1, 0, 32, 5)),
                                       ([1500], (1, 0, 32, 47)), ([70, 9, 130, 40, 64], (1, 0, 32, 5)),
                                       ([70, 9, 1500, 40, 64], (1, 0, 32, 47))],
                         ids=["one_slot", "latency", "latency_long", "fixed", "many_slots"])
def test_decode_nonfinite_queries_give_nan(lens, args):
    """A head whose query holds a NaN or an infinity has no softmax: NaN, also where every score is
    minus infinity. The other heads keep their bits."""
    pool, ptr, idx, at = _batch(lens, seed=13)
    c = _u8(pool[0])
    c[:, 3, 4] = (c[:, 3, 4] & 0x0f) | 0xb0  # kv head 3: element 9 of every key is negative
    q = _queries(len(lens), 3)
    bad = q.clone()
    bad[0, 3, 77] = float("nan")
    bad[0, 7, 9] = float("inf")    # every score -inf
    bad[0, 6, 9] = float("-inf")   # and +inf
    bad[-1, 12, 0] = float("inf")
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    hit[0, [3, 6, 7]] = True
    hit[-1, 12] = True
    for variant in range(4):
        clean, o = (_decode(x, pool, ptr, idx, *args, variant) for x in (q, bad))
        assert not clean.isnan().any()
        assert torch.equal(o[~hit], clean[~hit]), variant
        assert o[hit].isnan().all(), variant


@pytest.mark.parametrize("args", [(1, 0, 0, 1), (1, 0, 32, 4)], ids=["one_slot", "slots"])
@pytest.mark.parametrize("batch", [1, 5])
def test_decode_every_key_nan_gives_nan(args, batch):
    lens = [100] + [0, 60, 7, 90][:batch - 1]
    pool, ptr, idx, at = _batch(lens, seed=14)
    q = _queries(batch, 4)
    clean = _decode(q, pool, ptr, idx, *args, 2)
    _u8(pool[2])[torch.from_numpy(at[0]).cuda(), 2, 0] = 255
    o = _decode(q, pool, ptr, idx, *args, 2)
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    hit[0, 4:6] = True
    assert o[hit].isnan().all() and torch.equal(o[~hit], clean[~hit])
    if batch > 1:
        assert not o[1].any()


@pytest.mark.parametrize("up", [100, -100, 60, -125])
def test_decode_extreme_scales_stay_in_their_heads(up):
    """A head whose keys and values have exponents near the format's ends beside ordinary ones: the
    others' results keep their bits."""
    lens = [300]
    pool, ptr, idx, at = _batch(lens, seed=15)
    q = _queries(1, 15)
    for args in ((1, 0, 0, 1), (1, 0, 64, 5)):
        for variant in (2, 3):
            clean = _decode(q, pool, ptr, idx, *args, variant)
            keep = _u8(pool[2])[:, 5].clone()
            _u8(pool[2])[:, 5] = 127 + up
            o = _decode(q, pool, ptr, idx, *args, variant)
            _u8(pool[2])[:, 5] = keep
            others = [h for h in range(HQ) if h // 2 != 5]
            assert torch.equal(o[:, others], clean[:, others])
            if up < 0:  # scores of next to nothing: the mean of next to nothing
                assert float(o[:, 10:12].abs().max()) <= 6 * 2.0 ** up


# ---- chunk ------------------------------------------------------------------------------------

@pytest.mark.parametrize("specs", [
    [(0, 1)], [(0, 2)], [(0, 32)], [(0, 33)], [(0, 65)], [(0, 500)], [(1, 1)], [(100, 32)],
    [(1000, 64)], [(100, 32), (0, 17), (999, 1), (5, 64)], [(31, 32), (32, 32), (33, 32), (256, 32)],
    [(7, 1), (100, 1), (2000, 1)], [(63, 65), (191, 1), (0, 129)], [(0, 0), (10, 5), (3, 0)],
], ids=str)
@pytest.mark.parametrize("workspace", [True, False])
def test_chunk_against_oracle(specs, workspace):
    _say("chunk", specs, workspace)
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=len(specs), page=16)
    o = _chunk(q, pool, qo, ptr, idx, specs, workspace)
    for i, (p, e) in enumerate(specs):
        if e:
            a, b = int(qoh[i]), int(qoh[i + 1])
            _bounded(o[a:b], q[a:b], pool[3][at[i]], pool[4][at[i]], first=p, chunk=True)


@pytest.mark.parametrize("specs", [[(0, 1100)], [(0, 1025), (500, 1100), (0, 1024), (3, 1500),
                                                 (0, 1300), (100, 1200)], [(0, 700), (0, 3), (0, 90)] * 6],
                         ids=["one", "wide", "ragged"])
def test_chunk_long_grids(specs):
    """Grids too large to fan out: both workgroup sizes, ragged batches; sampled rows."""
    _say("chunk grid", len(specs))
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=11, page=16)
    o = _chunk(q, pool, qo, ptr, idx, specs)
    assert not o.isnan().any()
    rng = np.random.default_rng(0)
    for i, (p, e) in enumerate(specs[:8]):
        a = int(qoh[i])
        for j in {0, e - 1, int(rng.integers(e)), int(rng.integers(e))}:
            n = p + j + 1
            _bounded(o[a + j:a + j + 1], q[a + j:a + j + 1], pool[3][at[i][:n]], pool[4][at[i][:n]],
                     chunk=True)


def test_chunk_fanout_and_batch_keep_bits():
    """With and without the workspace, alone and in a batch, whole or window by window, in a batch
    large enough for the wide workgroups."""
    specs = [(300, 64), (0, 40), (1023, 33), (2048, 32)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=2)
    o = _chunk(q, pool, qo, ptr, idx, specs)
    assert torch.equal(o, _chunk(q, pool, qo, ptr, idx, specs, workspace=False))
    for i, (p, e) in enumerate(specs):
        a, b = int(qoh[i]), int(qoh[i + 1])
        one = _chunk(q[a:b].contiguous(), pool, _i32([0, e]), _i32([0, p + e]),
                     _i32(at[i].tolist()), [(p, e)])
        assert torch.equal(one, o[a:b])
        cut = e // 3 + 1
        for lo, hi in ((0, cut), (cut, e)):
            part = _chunk(q[a + lo:a + hi].contiguous(), pool, _i32([0, hi - lo]),
                          _i32([0, p + hi]), _i32(at[i][:p + hi].tolist()), [(p + lo, hi - lo)])
            assert torch.equal(part, o[a + lo:a + hi])
    wide = [(0, 2100)] * 4
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(wide, seed=3)
    o = _chunk(q, pool, qo, ptr, idx, wide)
    for lo, hi in ((0, 40), (700, 800), (2068, 2100)):
        part = _chunk(q[lo:hi].contiguous(), pool, _i32([0, hi - lo]), _i32([0, hi]),
                      _i32(at[0][:hi].tolist()), [(lo, hi - lo)])
        assert torch.equal(part, o[lo:hi])


@pytest.mark.parametrize("batch,lo,hi,pre", [(2, 900, 2100, 700), (17, 1, 400, 900), (63, 1, 50, 300),
                                             (65, 20, 40, 5), (256, 0, 9, 40), (257, 1, 9, 40)])
def test_chunk_placement_covers_every_tile(batch, lo, hi, pre):
    _say("placement", batch)
    rng = np.random.default_rng(batch)
    specs = [(int(rng.integers(0, pre + 1)), int(rng.integers(lo, hi + 1))) for _ in range(batch)]
    specs[batch // 2] = (pre, hi)
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=batch)
    o = _chunk(q, pool, qo, ptr, idx, specs, workspace=False)
    assert not o.isnan().any()
    for i in sorted({0, 1, batch // 2, batch - 1, *rng.integers(0, batch, 6).tolist()}):
        p, e = specs[i]
        if e:
            one = _chunk(q[int(qoh[i]):int(qoh[i + 1])].contiguous(), pool, _i32([0, e]),
                         _i32([0, p + e]), _i32(at[i].tolist()), [(p, e)])
            assert torch.equal(one, o[int(qoh[i]):int(qoh[i + 1])]), i


@pytest.mark.parametrize("which", [0, 1], ids=["nan_k", "nan_v"])
@pytest.mark.parametrize("specs", [[(1000, 70)], [(2048, 32)] * 4, [(1526, 50)], [(505, 64), (2000, 17)]],
                         ids=str)
def test_fanned_out_nan_reaches_only_rows_that_see_it(specs, which):
    """NaN keys at sequences', tiles' and splits' first and last places: the rows that see the key are
    NaN, the others keep their bits, with the fan-out and without."""
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=20)
    assert _fan_bytes(specs) > 0
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    assert not clean.isnan().any()
    assert torch.equal(clean, _chunk(q, pool, qo, ptr, idx, specs, workspace=False))
    sc = _u8(pool[2])
    for i in {0, len(specs) - 1}:
        p, e = specs[i]
        keys = {0, 63, 64, 511, 512, 1024, 1535, 1536, 2047, 2048, p - 1, p, p + 15, p + 16, p + 31,
                p + 32, p + e - 2, p + e - 1}
        for key in sorted(x for x in keys if 0 <= x < p + e):
            slot, head = int(at[i][key]), key % HKV
            kept = sc[slot, head].clone()
            sc[slot, head, which] = 255
            hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
            hit[int(qoh[i]) + max(0, key - p):int(qoh[i + 1]), 2 * head:2 * head + 2] = True
            for ws in (True, False):
                o = _chunk(q, pool, qo, ptr, idx, specs, ws)
                assert o[hit].isnan().all(), (i, key, ws)
                assert torch.equal(o[~hit], clean[~hit]), (i, key, ws)
            sc[slot, head] = kept


@pytest.mark.parametrize("which", [0, 1], ids=["nan_k", "nan_v"])
@pytest.mark.parametrize("key", [5, 42, 512, 1023, 1204])
def test_wide_grid_nan_reaches_only_rows_that_see_it(key, which):
    specs = [(5, 1200)] * 6
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=21)
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    _make_nan(pool, which, int(at[0][key]), 3)
    o = _chunk(q, pool, qo, ptr, idx, specs)
    hit = torch.zeros(o.shape, dtype=torch.bool, device="cuda")
    hit[max(0, key - 5):int(qoh[1]), 6:8] = True
    assert o[hit].isnan().all() and torch.equal(o[~hit], clean[~hit])


def test_chunk_unnamed_rows_of_nan_reach_nothing():
    """Every slot that no request names, slot 0 among them, holds NaNs; rows past the last sequence
    stay, with the fan-out and without."""
    from sid.kernels.jit import load_ext
    specs = [(1000, 70), (2048, 3)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=22)
    used = np.concatenate(at)
    if 0 in used:  # give slot 0's row another place
        spare = int(np.setdiff1d(np.arange(pool[3].shape[0]), used)[-1])
        for t in pool[:3]:
            _u8(t)[spare] = _u8(t)[0]
        idx[idx == 0] = spare
        used = np.where(used == 0, spare, used)
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    _u8(pool[2])[torch.from_numpy(np.setdiff1d(np.arange(pool[3].shape[0]), used)).cuda()] = 255
    qq = torch.cat([q, q[:7]])
    need = load_ext().extend_attention_workspace_bytes(2, qq.shape[0], HQ, HKV, 70, 2051, fp4=True)
    assert need > 0
    for ws in (torch.full((need,), 0x3f, dtype=torch.uint8, device="cuda"), None):
        o = torch.full_like(qq, 7.0)
        load_ext().extend_attention_fwd(qq, pool[0], pool[1], qo, ptr, idx, 70, SCALE, o, 2051, ws,
                                        kv_scales=pool[2])
        assert torch.equal(o[:q.shape[0]], clean) and (o[q.shape[0]:] == 7.0).all()


@pytest.mark.parametrize("fill", [0, 1, 0xff])
def test_fanned_out_rows_of_a_refused_request_stay(fill):
    """A request with fewer keys than new tokens is left out (its rows stay), with the fan-out too."""
    from sid.kernels.jit import load_ext
    specs = [(2048, 32), (0, 40), (700, 9)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=19)
    lens = [2080, 39, 709]  # one key short
    flat = torch.cat([_i32(a[:n].tolist()) for a, n in zip(at, lens)])
    ptr = _i32(np.cumsum([0] + lens).tolist())
    got = []
    for w in (torch.full((_fan_bytes(specs),), fill, dtype=torch.uint8, device="cuda"), None):
        o = torch.full_like(q, 7.0)
        load_ext().extend_attention_fwd(q, pool[0], pool[1], qo, ptr, flat, 40, SCALE, o, 2080, w,
                                        kv_scales=pool[2])
        assert (o[32:72] == 7.0).all() and not o.isnan().any()
        got.append(o)
    assert torch.equal(*got)


@pytest.mark.parametrize("workspace", [True, False])
def test_chunk_nonfinite_queries_give_nan(workspace):
    specs = [(1000, 70), (0, 40)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=15)
    clean = _chunk(q, pool, qo, ptr, idx, specs, workspace)
    bad = q.clone()
    hit = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
    for row, h, d, x in ((0, 3, 77, "nan"), (17, 7, 9, "inf"), (69, 0, 127, "-inf"), (75, 15, 64, "inf")):
        bad[row, h, d] = float(x)
        hit[row, h] = True
    o = _chunk(bad, pool, qo, ptr, idx, specs, workspace)
    assert not clean.isnan().any()
    assert o[hit].isnan().all() and torch.equal(o[~hit], clean[~hit])


def test_zero_and_tiny_queries_take_the_mean():
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


@pytest.mark.parametrize("ratio", [2.0 ** 6, 2.0 ** 12, 2.0 ** 16, 2.0 ** 20])
def test_queries_with_outliers(ratio):
    """Queries with one element `ratio` times the others' size, over keys that are zero there: what is
    left of the scores is the small elements' alone. The chunk kernel splits a query into two e4m3
    vectors of scale 2^e, 2^e < max |q| / 224: an element below 2^-6 2^e is off by up to 2^-14 2^e,
    and a score by the sum of that over |k|, which joins the bound of a score's own error. The decode
    kernel's bound has the same term where its test says so."""
    specs = [(1000, 48)]
    q, pool, qo, ptr, idx, at, _ = _chunk_batch(specs, seed=17)
    dims = torch.randint(0, 4, (q.shape[0], HQ), generator=torch.Generator().manual_seed(1)).cuda() * 37
    q.scatter_(2, dims[..., None], float(ratio))
    c = _u8(pool[0])
    for d in (0, 37, 74, 111):
        c[:, :, d // 2] &= 0x0f if d % 2 else 0xf0
        pool[3][:, :, d] = 0.0
    qd, k, v = q.double().cpu().numpy(), pool[3][at[0]], pool[4][at[0]]
    ref, mag, top = attention_ref(qd, k, v, SCALE, 1000)
    n = k.shape[0]
    e = np.exp2(np.ceil(np.log2(np.abs(qd).max(-1) / 448.0)))
    split = 2.0 ** -14 * e * np.abs(k).sum(-1).max(0).repeat(2)[None] * SCALE
    err_p = 136 * 2.0 ** -24 * top + 2.0 ** -20 + split[..., None]
    tol = 2.0 ** -8 * np.abs(ref) + 2 * err_p * np.abs(v).max() + (n + 64) * 2.0 ** -24 * mag \
        + 2.0 ** -8 * mag
    for ws in (True, False):
        o = _chunk(q, pool, qo, ptr, idx, specs, ws).double().cpu().numpy()
        assert np.isfinite(o).all() and (np.abs(o - ref) <= tol).all()
    ref, mag, top = attention_ref(qd[:1], k, v, SCALE)
    err_p = 136 * 2.0 ** -24 * top + 2.0 ** -20 + split[:1, :, None]
    tol = 2.0 ** -8 * np.abs(ref) + 2 * err_p * np.abs(v).max() + (n + 64) * 2.0 ** -24 * mag
    for args in ((1, 0, 0, 1), (1, 0, 64, 17)):
        o = _decode(q[:1].contiguous(), pool, ptr, idx, *args, 2).double().cpu().numpy()
        assert (np.abs(o - ref) <= tol).all()


def _ramp(lens, seed, up):
    """A pool whose scores rise (or fall) by about 12 octaves of exp every 64 positions, and queries
    for it: every tile moves its rows' maxima (or none but the first does)."""
    g = torch.Generator().manual_seed(seed)
    _, ptr, idx, at = _batch(lens, seed=seed, page=16)
    size = int(idx.max()) + 17
    w = torch.randn(HKV, D, generator=g)
    x = torch.randn(2, size, HKV, D, generator=g)
    for a in at:
        pos = torch.arange(len(a), dtype=torch.float32)
        x[0, torch.from_numpy(a)] += (pos if up else -pos)[:, None, None] * w / 87.0
    pool = _of_rows([t.double().numpy() for t in x])

    def queries(n):
        q = torch.randn(n, HQ, D, generator=g) * 0.3 + w.repeat_interleave(2, 0)
        return q.to(torch.bfloat16).cuda()
    return pool, ptr, idx, at, queries


@pytest.mark.parametrize("up", [True, False], ids=["rising", "falling"])
def test_scores_that_move_every_tile(up):
    specs = [(0, 130), (700, 50), (1000, 40)]
    pool, ptr, idx, at, queries = _ramp([p + e for p, e in specs], 5, up)
    qoh = np.cumsum([0] + [e for _, e in specs])
    q = queries(int(qoh[-1]))
    for workspace in (True, False):
        o = _chunk(q, pool, _i32(qoh.tolist()), ptr, idx, specs, workspace)
        for i, (p, e) in enumerate(specs):
            a, b = int(qoh[i]), int(qoh[i + 1])
            _bounded(o[a:b], q[a:b], pool[3][at[i]], pool[4][at[i]], first=p, chunk=True)
    lens = [1, 70, 500, 1300]
    pool, ptr, idx, at, queries = _ramp(lens, 6, up)
    q = queries(len(lens))
    for variant in (2, 3):
        for args in ((1, 0, 0, 1), (1, 0, 256, 6)):
            _check_decode(_decode(q, pool, ptr, idx, *args, variant), q, pool, at)


@pytest.mark.parametrize("hkv", [1, 2, 5, 16])
@pytest.mark.parametrize("specs", [[(1000, 70)], [(3, 90), (700, 1), (0, 33)], [(100, 1100)] * 3],
                         ids=["window", "ragged", "long"])
def test_chunk_other_head_counts(hkv, specs):
    _say("heads", hkv, specs)
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=hkv, hkv=hkv)
    o = _chunk(q, pool, qo, ptr, idx, specs)
    assert torch.equal(o, _chunk(q, pool, qo, ptr, idx, specs, workspace=False))
    rng = np.random.default_rng(hkv)
    for i, (p, e) in enumerate(specs):
        a = int(qoh[i])
        for j in sorted({0, e - 1, *rng.integers(0, e, 6).tolist()}):
            n = p + j + 1
            _bounded(o[a + j:a + j + 1], q[a + j:a + j + 1], pool[3][at[i][:n]], pool[4][at[i][:n]],
                     chunk=True)


@pytest.mark.parametrize("workspace", [True, False])
def test_chunk_bad_slots_read_slot_zero(workspace):
    specs = [(1000, 70), (5, 64)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=25)
    bad, size = idx.clone(), pool[3].shape[0]
    at0 = [a.copy() for a in at]
    for i, key, slot in [(0, 3, -4), (0, 999, 1 << 30), (0, 1069, size), (0, 64, -2 ** 31),
                         (1, 0, 2 ** 31 - 1)]:
        bad[int(ptr[i]) + key] = slot
        at0[i][key] = 0
    o = _chunk(q, pool, qo, ptr, bad, specs, workspace)
    for i, (p, e) in enumerate(specs):
        a, b = int(qoh[i]), int(qoh[i + 1])
        _bounded(o[a:b], q[a:b], pool[3][at0[i]], pool[4][at0[i]], first=p, chunk=True)


def test_chunk_thousands_of_requests_and_large_bounds():
    """5000 requests, one of 4000 tokens; ragged requests under a bound of 50000 new tokens; a bound
    of 17 million keys: the same bits as with the bounds that they need."""
    from sid.kernels.jit import load_ext
    rng = np.random.default_rng(1)
    specs = [(int(rng.integers(0, 4)), 1) for _ in range(5000)]
    specs[3210] = (0, 4000)
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=26)
    o = _chunk(q, pool, qo, ptr, idx, specs, workspace=False)
    assert not o.isnan().any()
    for i in (0, 3209, 3210, 3211, 4999):
        p, e = specs[i]
        a, b = int(qoh[i]), int(qoh[i + 1])
        one = _chunk(q[a:b].contiguous(), pool, _i32([0, e]), _i32([0, p + e]), _i32(at[i].tolist()),
                     [(p, e)], workspace=False)
        assert torch.equal(one, o[a:b]), i
    for specs, bounds, keys in (([(int(rng.integers(0, 60)), int(rng.integers(1, 90))) for _ in range(200)],
                                 (50000, 89), (150, 150)), ([(100, 64)], (64, 64), (17_000_000, 164))):
        q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=28, hkv=1)
        got = []
        for bound, mk in zip(bounds, keys):
            o = torch.full_like(q, float("nan"))
            need = load_ext().extend_attention_workspace_bytes(len(specs), q.shape[0], 2, 1, bound, mk,
                                                               fp4=True)
            ws = torch.empty(need, dtype=torch.uint8, device="cuda") if 0 < need < 1 << 33 else None
            load_ext().extend_attention_fwd(q, pool[0], pool[1], qo, ptr, idx, bound, SCALE, o, mk, ws,
                                            kv_scales=pool[2])
            assert not o.isnan().any()
            got.append(o)
        assert torch.equal(*got)


def test_large_pool_addresses():
    """Slots whose byte offset is beyond 2^32 (codes) in all four operators."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.kv_fp4 import alloc_cache_fp4, gather_cache_fp4, reshape_and_cache_fp4
    kc, vc, sc = alloc_cache_fp4((1 << 23) + 5000, HKV, "cuda")  # 4.3e9 bytes of K codes
    n = 150
    at = torch.randperm(4000)[:n].sort()[0] + (1 << 23) + 500
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, HKV, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    reshape_and_cache_fp4(k, v, kc, vc, sc, at.cuda())
    k2, v2 = gather_cache_fp4(kc, vc, sc, at.cuda())
    kd, vd = (load_ref(*store_ref(x.double().cpu().numpy())) for x in (k, v))
    assert np.array_equal(k2.double().cpu().numpy(), kd) and np.array_equal(v2.double().cpu().numpy(), vd)
    q = _queries(1, 3)
    attn = DecodeAttention(1, HQ, HKV, D, 32, 256, 4096, "cuda")
    ptr, idx = _i32([0, n]), at.int().cuda()
    o = attn.forward(q, kc, vc, ptr, idx, _i32([n]), n, SCALE, False, kv_scales=sc)
    o2 = extend_attention_fwd(q, kc, vc, _i32([0, 1]), ptr, idx, 1, SCALE, kv_scales=sc)
    _bounded(o, q, kd, vd)
    _bounded(o2, q, kd, vd, chunk=True)


# ---- together ---------------------------------------------------------------------------------

def test_pool_that_grows_at_far_positions():
    """A projection's q and k rotated at positions of a stretched context, k and v written and
    attended to; then read back, then single tokens appended and decoded, then a window over
    everything: each step against 64 bits of what the pool stands for."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.kv_fp4 import alloc_cache_fp4, gather_cache_fp4, reshape_and_cache_fp4
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(D, 131072, 1e6, "cuda", scaling=dict(
        rope_type="yarn", factor=4.0, original_max_position_embeddings=32768))
    start, cap = [0, 100000, 40000], 260
    perm = torch.randperm(3 * cap, generator=torch.Generator().manual_seed(5))
    slots = [perm[i * cap:(i + 1) * cap] for i in range(3)]
    pool = alloc_cache_fp4(3 * cap, HKV, "cuda")
    vals = [(np.zeros((0, HKV, D)), np.zeros((0, HKV, D))) for _ in start]
    attn = DecodeAttention(3, HQ, HKV, D, 32, 256, 4096, "cuda")
    g = torch.Generator().manual_seed(6)

    def write(counts):
        """New tokens' rows into the pool; their rotated queries."""
        n = sum(counts)
        proj = torch.randn(n, HQ + 2 * HKV, D, generator=g).to(torch.bfloat16).cuda()
        pos = torch.cat([start[i] + torch.arange(len(vals[i][0]), len(vals[i][0]) + c)
                         for i, c in enumerate(counts)]).cuda()
        q, k = rope.rotate(proj[:, :HQ], proj[:, HQ:HQ + HKV], pos)
        v = proj[:, HQ + HKV:]
        at = torch.cat([slots[i][len(vals[i][0]):len(vals[i][0]) + c] for i, c in enumerate(counts)])
        reshape_and_cache_fp4(k, v, *pool, at.cuda())
        got = gather_cache_fp4(*pool, at.cuda())
        n = 0
        for i, c in enumerate(counts):
            new = [load_ref(*store_ref(x[n:n + c].double().cpu().numpy())) for x in (k, v)]
            for x, y in zip(got, new):
                assert np.array_equal(x[n:n + c].double().cpu().numpy(), y)
            vals[i] = tuple(np.concatenate([a, b]) for a, b in zip(vals[i], new))
            n += c
        return q

    def inputs():
        full = [len(v[0]) for v in vals]
        idx = torch.cat([slots[i][:n] for i, n in enumerate(full)])
        return full, _i32(np.cumsum([0] + full).tolist()), idx.int().cuda()

    def chunk(counts):
        q = write(counts)
        full, ptr, idx = inputs()
        qo = np.cumsum([0] + counts)
        o = _chunk(q, pool, _i32(qo.tolist()), ptr, idx, [(f - c, c) for f, c in zip(full, counts)])
        for i, c in enumerate(counts):
            a, b = int(qo[i]), int(qo[i + 1])
            _bounded(o[a:b], q[a:b], *vals[i], first=full[i] - c, chunk=True)

    chunk([40, 3, 129])
    for _ in range(4):
        q = write([1, 1, 1])
        full, ptr, idx = inputs()
        o = attn.forward(q, *pool[:2], ptr, idx, _i32(full), max(full), SCALE, False,
                         kv_scales=pool[2], **attn.step_plan(full, kv_fp4=True))
        for i in range(3):
            _bounded(o[i:i + 1], q[i:i + 1], *vals[i])
    chunk([70, 33, 64])


def test_graph_replays_on_another_stream():
    """rotate + store + decode + chunk + load captured twice over one pool and one DecodeAttention,
    replayed in turn with other inputs on a stream of their own, eager work between the replays."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.kv_fp4 import gather_cache_fp4, reshape_and_cache_fp4
    from sid.kernels.rope import RotaryEmbedding
    pool, _, _, at = _batch([900, 33, 400, 1, 2000], seed=4)
    kc, vc, sc = pool[:3]
    attn = DecodeAttention(5, HQ, HKV, D, 32, 256, 4096, "cuda")
    rope = RotaryEmbedding(D, 131072, 1e6, "cuda", rotary_dim=64, interleaved=True)

    def step(pick):
        lens = [len(at[i]) for i in pick]
        n = len(pick)
        ptr, idx = _i32(np.cumsum([0] + lens).tolist()), _i32(np.concatenate([at[i] for i in pick]).tolist())
        new = torch.tensor([int(at[i][-1]) for i in pick], device="cuda")
        pos = torch.tensor([70000 + x for x in lens], device="cuda")
        proj = torch.zeros(n, HQ + 2 * HKV, D, dtype=torch.bfloat16, device="cuda")
        seq, qo, plan = _i32(lens), _i32(list(range(n + 1))), attn.step_plan(lens, kv_fp4=True)

        def run():
            q, k = rope.rotate(proj[:, :HQ], proj[:, HQ:HQ + HKV], pos)
            reshape_and_cache_fp4(k, proj[:, HQ + HKV:], kc, vc, sc, new)
            o = attn.forward(q, kc, vc, ptr, idx, seq, max(lens), SCALE, False, kv_scales=sc, **plan)
            c = extend_attention_fwd(q, kc, vc, qo, ptr, idx, 1, SCALE, max_kv_len=max(lens), kv_scales=sc)
            return (q, o, c, *gather_cache_fp4(kc, vc, sc, new))

        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        return proj, run, graph, out

    steps = [step([0, 3, 4]), step([4, 2, 1, 0, 3]), step([1])]
    side, g = torch.cuda.Stream(), torch.Generator().manual_seed(7)
    for _ in range(3):
        for proj, run, graph, out in steps:
            proj.copy_(torch.randn(proj.shape, generator=g).to(torch.bfloat16))
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                graph.replay()
            side.synchronize()
            got = [x.clone() for x in out]
            with torch.cuda.stream(side):
                want = run()
            side.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            torch.zeros(1 << 20, device="cuda").sum().item()


# ---- refusals ---------------------------------------------------------------------------------

def test_refusals():
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.kv_fp4 import alloc_cache_fp4
    from sid.kernels.kv_fp8 import alloc_cache_fp8
    kc, vc, sc = alloc_cache_fp4(8, HKV, "cuda")
    k8, v8, s8 = alloc_cache_fp8(8, HKV, "cuda")
    x = torch.zeros(8, HKV, D, dtype=torch.bfloat16, device="cuda")

    def refused(match, fn, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*a, **kw)

    attn = DecodeAttention(2, HQ, HKV, D, 32, 256, 4096, "cuda")
    q = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device="cuda")
    ptr, idx, seq, qo = _i32([0, 2, 4]), _i32([1, 2, 3, 4]), _i32([2, 2]), _i32([0, 1, 2])
    for call in (lambda *p, **kw: attn.forward(q, *p, ptr, idx, seq, 2, SCALE, False, **kw),
                 lambda *p, **kw: extend_attention_fwd(q, *p, qo, ptr, idx, 1, SCALE, **kw)):
        refused("bfloat16", call, kc, vc)                       # codes without their scales
        refused("kv_scales must be", call, kc, vc, kv_scales=s8)  # another pool's scales
        refused("e2m1|float4", call, kc, v8, kv_scales=sc)
        refused("kv_scales must be", call, k8, v8, kv_scales=sc)
        refused("e8m0", call, kc, vc, kv_scales=sc.view(torch.uint8))
        refused("float8_e4m3fn", call, x, x, kv_scales=sc)
        refused("both be", call, kc, vc[:4], kv_scales=sc)
    refused("B\\+1", attn.forward, q, kc, vc, ptr[:2], idx, seq, 2, SCALE, False, kv_scales=sc)
    refused("int32", attn.forward, q, kc, vc, ptr.long(), idx, seq, 2, SCALE, False, kv_scales=sc)
    q4 = torch.zeros(2, 8, D, dtype=torch.bfloat16, device="cuda")
    refused("workspace|q heads", attn.forward, q4, kc, vc, ptr, idx, seq, 2, SCALE, False, kv_scales=sc)
    refused("q heads", extend_attention_fwd, q4, kc, vc, qo, ptr, idx, 1, SCALE, kv_scales=sc)


def test_chunk_scale_that_is_refused():
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch([(10, 5)], seed=1)
    from sid.kernels.extend_attention import extend_attention_fwd
    for bad in (-0.1, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="sm_scale"):
            extend_attention_fwd(q, *pool[:2], qo, ptr, idx, 5, bad, max_kv_len=15, kv_scales=pool[2])


def test_decode_two_workers_a_cu_keep_bits():
    """More segments than two a CU: the placement deals them to workers."""
    from sid.kernels.decode_attention import DecodeAttention, placement, stage1_workers_fp4
    lens = [9000 - 150 * i for i in range(40)]
    pool, ptr, idx, at = _batch(lens, seed=23, page=16)
    q = _queries(len(lens), 23)
    attn = DecodeAttention(len(lens), HQ, HKV, D, 32, 256, max(lens), "cuda")
    order, workers = placement(lens, len(lens), 1, 0, 256, 36, 3, attn.cu_count(),
                               workers_of=stage1_workers_fp4, kv_fp4=True)
    assert workers == 2 * attn.cu_count()
    plan = dict(geometry=(1, 256, 36), variant=3, wg_order=torch.from_numpy(order).cuda(),
                workers=workers)
    run = lambda **kw: attn.forward(q, *pool[:2], ptr, idx, _i32(lens), max(lens), SCALE, False,  # noqa: E731
                                    kv_scales=pool[2], **{**plan, **kw})
    attn.part_o.fill_(float("nan"))
    attn.part_lse.fill_(float("nan"))
    o = run()
    assert torch.equal(o, run(wg_order=None, workers=0))
    for i in (0, 17, 39):
        _check_decode(o[i:i + 1], q[i:i + 1], pool, [at[i]])
