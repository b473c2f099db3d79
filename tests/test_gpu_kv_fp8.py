"""The 8-bit KV pool's operators against 64-bit oracles (oracle/kv_fp8.py): the writer (plain and
fused into the qkv epilogues) and the reader bit for bit, decode and chunk attention within
bounds that count their roundings, their invariances, what hidden NaNs may not reach, and the
operators together over a paged pool that grows.

Attention bounds. The result is rounded once to bf16 (half a step: 2^-8 of it). A score is an fp32
sum of 128 products with a few more roundings, so it is off by at most 136 2^-24 S, S the largest
sum |q| |k| sm_scale; p = exp of it by at most that plus 2^-20 relative, and the quotient of two
sums of p by twice that, times max |v|, plus the fp32 sums' own (n + 64) 2^-24 of the mean of |v|
under the same weights (M). The chunk kernel rounds p to bf16: 2^-8 M more."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import HKV, HQ, D, SCALE
from oracle.kv_fp8 import attention_ref, load_ref, store_ref

pytestmark = pytest.mark.gpu
FP8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _say(*a):
    print(*a, flush=True)


def _u8(t):
    return t.view(torch.uint8).cpu().numpy()


def _rows(n, hkv=HKV, seed=0, spread=1.0):
    """bf16 [n, hkv, D] whose vectors differ in size, with larger channels."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, hkv, D, generator=g) * torch.exp(spread * torch.randn(n, hkv, 1, generator=g))
    x[..., ::31] *= 5.0
    return x.to(torch.bfloat16).cuda()


def _pool(slots, hkv=HKV, seed=0, spread=0.7):
    """A pool of random rows, quantised by the oracle: (k, v, scales on the GPU, float64 K, V)."""
    out, vals, bytes_ = [], [], []
    for s in (0, 1):
        x = _rows(slots, hkv, seed * 2 + s, spread).double().cpu().numpy()
        codes, b = store_ref(x)
        out.append(torch.from_numpy(codes).cuda().view(FP8))
        bytes_.append(b)
        vals.append(load_ref(codes, b))
    scales = torch.from_numpy(np.stack(bytes_, -1)).cuda().view(E8M0)
    return out[0], out[1], scales, vals[0], vals[1]


def _empty(slots, hkv=HKV):
    from sid.kernels.kv_fp8 import alloc_cache_fp8
    return alloc_cache_fp8(slots, hkv, "cuda")


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# ---- writer and reader ------------------------------------------------------------------------

@pytest.mark.parametrize("t,hkv", [(1, 8), (1, 1), (3, 2), (37, 5), (100, 8), (513, 8), (70, 16)])
def test_store_matches_oracle(t, hkv):
    from sid.kernels.kv_fp8 import reshape_and_cache_fp8
    _say("store", t, hkv)
    k, v = _rows(t, hkv, 1, 3.0), _rows(t, hkv, 2, 3.0)
    kc, vc, sc = _empty(t + 20, hkv)
    slots = torch.randperm(t + 20, device="cuda")[:t]
    reshape_and_cache_fp8(k, v, kc, vc, sc, slots)
    at = slots.cpu().numpy()
    for i, (x, c) in enumerate(((k, kc), (v, vc))):
        codes, b = store_ref(x.double().cpu().numpy())
        assert np.array_equal(_u8(c)[at], codes)
        assert np.array_equal(_u8(sc)[at, :, i], b)
    rest = np.setdiff1d(np.arange(t + 20), at)
    assert not _u8(kc)[rest].any() and not _u8(vc)[rest].any() and (_u8(sc)[rest] == 127).all()


def test_store_every_edge_value():
    """Zeros, the exponents' borders (448 2^e and its neighbours), values that clamp at both ends,
    ties between codes, subnormal bf16, infinities and NaNs."""
    from sid.kernels.kv_fp8 import reshape_and_cache_fp8
    rows = [torch.zeros(D)]
    g = torch.Generator().manual_seed(0)
    for e in list(range(-126, 128, 9)) + [-117, -118, -109, -108, 119, 120, 126, 127]:
        for m in (1.0, 1.75, 1.7421875, 1.7578125, 1.9921875):
            x = torch.randn(D, generator=g).clamp(-0.9, 0.9).double() * m * 2.0 ** e
            x[5] = m * 2.0 ** e
            rows.append(x.float())
    tie = torch.zeros(D)
    tie[0] = 448.0
    tie[1:17] = torch.arange(16) * 2.0 + 17.0      # half-way between neighbours from 16 up
    tie[17:25] = (torch.arange(8) + 0.5) * 2.0 ** -9  # and between subnormal codes
    rows += [tie, -tie]
    sub = torch.arange(D).float() * 2.0 ** -133
    rows += [sub, -sub]
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.randn(D, generator=g)
        x[77] = bad
        rows.append(x)
    x = torch.stack(rows).to(torch.bfloat16)[:, None].repeat(1, HKV, 1).cuda()
    n = x.shape[0]
    kc, vc, sc = _empty(n)
    reshape_and_cache_fp8(x, -x, kc, vc, sc, torch.arange(n, device="cuda"))
    for i, (s, c) in enumerate(((1, kc), (-1, vc))):
        codes, b = store_ref(s * x.double().cpu().numpy())
        assert np.array_equal(_u8(sc)[..., i], b)
        got = _u8(c)
        bad = got != codes
        assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], codes[bad][:4])


def test_store_strided_rows_and_skipped_slots():
    """K and V as columns of a projection; padding (-1) and out-of-range slots."""
    from sid.kernels.kv_fp8 import reshape_and_cache_fp8
    t = 9
    proj = torch.randn(t, (HQ + 2 * HKV) * D, device="cuda").to(torch.bfloat16)
    k = proj[:, HQ * D:(HQ + HKV) * D].view(t, HKV, D)
    v = proj[:, (HQ + HKV) * D:].view(t, HKV, D)
    assert not k.is_contiguous()
    kc, vc, sc = _empty(12)
    slots = torch.tensor([3, -1, 0, 12, 11, -7, 5, 1 << 40, 4], device="cuda")
    reshape_and_cache_fp8(k, v, kc, vc, sc, slots)
    want = _empty(12)
    keep = (slots >= 0) & (slots < 12)
    reshape_and_cache_fp8(k[keep].contiguous(), v[keep].contiguous(), *want, slots[keep])
    for a, b in zip((kc, vc, sc), want):
        assert np.array_equal(_u8(a), _u8(b))
    assert _u8(kc)[3].any() and not _u8(kc)[1].any()
    with pytest.raises(RuntimeError, match="heads and dims"):
        reshape_and_cache_fp8(k.transpose(1, 2).contiguous().transpose(1, 2), v, kc, vc, sc, slots)


def test_load_every_code_and_scale():
    """All 256 codes under every scale byte that the writer stores: exact bf16 values."""
    from sid.kernels.kv_fp8 import gather_cache_fp8
    bytes_ = np.arange(10, 247, dtype=np.uint8)
    n = bytes_.size
    codes = np.arange(256, dtype=np.uint8).reshape(2, D)
    pool = torch.from_numpy(np.tile(codes[None], (n, 1, 1))).cuda().view(FP8)  # 2 heads
    sc = torch.from_numpy(np.stack([np.tile(bytes_[:, None], (1, 2)),
                                    np.tile(bytes_[::-1, None], (1, 2))], -1).copy()).cuda()
    k, v = gather_cache_fp8(pool, pool.clone(), sc.view(E8M0), torch.arange(n, device="cuda"))
    for got, b in ((k, bytes_), (v, bytes_[::-1])):
        want = load_ref(np.tile(codes[None], (n, 1, 1)), np.tile(b[:, None], (1, 2)))
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("n", [1, 2, 77, 1000])
def test_load_order_repeats_and_range(n):
    from sid.kernels.kv_fp8 import gather_cache_fp8
    kc, vc, sc, kv, vv = _pool(300, seed=4)
    g = torch.Generator().manual_seed(n)
    slots = torch.randint(-5, 305, (n,), generator=g)
    if n > 4:
        slots[:4] = torch.tensor([0, 299, 300, -1])
    k, v = gather_cache_fp8(kc, vc, sc, slots.cuda())
    s = slots.numpy()
    ok = (s >= 0) & (s < 300)
    for got, val in ((k, kv), (v, vv)):
        want = np.where(ok[:, None, None], val[np.where(ok, s, 0)], 0.0)
        assert np.array_equal(got.double().cpu().numpy(), want)


def test_round_trip_bounds_and_nan():
    from sid.kernels.kv_fp8 import gather_cache_fp8, reshape_and_cache_fp8
    t = 200
    k, v = _rows(t, seed=7), _rows(t, seed=8)
    k[3, 2, 11] = float("nan")
    v[5, 1, 0] = float("inf")
    kc, vc, sc = _empty(t)
    at = torch.arange(t, device="cuda")
    reshape_and_cache_fp8(k, v, kc, vc, sc, at)
    k2, v2 = gather_cache_fp8(kc, vc, sc, at)
    assert k2[3, 2].isnan().all() and v2[5, 1].isnan().all()
    assert int(k2.isnan().sum()) == D and int(v2.isnan().sum()) == D
    # the stated format, in torch's own types
    assert torch.equal(k2.float().nan_to_num(), (kc.float() * sc.float()[..., :1]).nan_to_num())
    ok = ~k2.isnan()
    err = (k2.float() - k.float()).abs()[ok]
    top = k.float().abs().amax(-1, keepdim=True).expand_as(k)[ok]
    # half a step: 2^-4 of the value, and 2^-10 2^e below the normal codes, 2^e < 2 max / 448
    assert (err <= torch.maximum(2.0 ** -4 * k.float().abs()[ok], top * 2.0 ** -9 / 448)).all()


def test_large_pool_addresses():
    """Slots whose byte offset is beyond 2^32 (codes) in all four operators."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.kv_fp8 import gather_cache_fp8, reshape_and_cache_fp8
    slots = (1 << 22) + 5000  # 4.3e9 bytes of K codes
    kc, vc, sc = _empty(slots)
    n = 150
    at = torch.randperm(4000)[:n].sort()[0] + (1 << 22) + 500
    k, v = _rows(n, seed=1), _rows(n, seed=2)
    reshape_and_cache_fp8(k, v, kc, vc, sc, at.cuda())
    k2, v2 = gather_cache_fp8(kc, vc, sc, at.cuda())
    codes, b = store_ref(k.double().cpu().numpy())
    kd = load_ref(codes, b)
    assert np.array_equal(k2.double().cpu().numpy(), kd)
    vd = v2.double().cpu().numpy()
    q = torch.randn(1, HQ, D, device="cuda").to(torch.bfloat16)
    attn = DecodeAttention(1, HQ, HKV, D, 32, 256, 4096, "cuda")
    ptr, idx = _i32([0, n]), at.int().cuda()
    o = attn.forward(q, kc, vc, ptr, idx, _i32([n]), n, SCALE, False, kv_scales=sc)
    o2 = extend_attention_fwd(q, kc, vc, _i32([0, 1]), ptr, idx, 1, SCALE, kv_scales=sc)
    _bounded(o, q, kd, vd)
    _bounded(o2, q, kd, vd, chunk=True)


# ---- the fused writers ------------------------------------------------------------------------

@pytest.mark.parametrize("t", [1, 5, 64, 129])
@pytest.mark.parametrize("form", ["qkv", "partials", "chain_bf16", "chain_fp32"])
def test_fused_writers_equal_write_of_unfused(t, form):
    """q and the pool of the fused epilogues: the bits of the bf16 epilogue's q, and of its K/V
    rows given to reshape_and_cache_fp8."""
    from sid.kernels import ops
    from sid.kernels.kv_fp8 import reshape_and_cache_fp8
    from sid.kernels.rope import RotaryEmbedding
    _say("fused", form, t)
    g = torch.Generator().manual_seed(t)
    width = (HQ + 2 * HKV) * D
    rand = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    qn, kn = (1 + 0.2 * rand(D)).to(torch.bfloat16), (1 + 0.2 * rand(D)).to(torch.bfloat16)
    cs = RotaryEmbedding(D, 4096, 1e6, "cuda").cos_sin
    pos = torch.randint(0, 5000, (t,), generator=g).cuda()  # some beyond the table: not rotated
    slots = torch.randperm(t + 8, generator=g)[:t].cuda()
    if t > 3:
        slots[2] = -1
    if form in ("qkv", "partials"):
        x = rand(t, width).to(torch.bfloat16) if form == "qkv" else rand(4, t, width)
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
    pool = _empty(n)
    q1 = call(*pool)
    want = _empty(n)
    keep = slots[slots >= 0]
    reshape_and_cache_fp8(kb[keep], vb[keep], *want, keep)
    assert torch.equal(q0, q1)
    for a, b in zip(pool, want):
        assert np.array_equal(_u8(a), _u8(b))


# ---- decode -----------------------------------------------------------------------------------

def _bounded(o, q, k, v, first=None, chunk=False):
    ref, mag, top = attention_ref(q.double().cpu().numpy(), k, v, SCALE, first)
    n = k.shape[0]
    err_p = 136 * 2.0 ** -24 * top + 2.0 ** -20
    tol = 2.0 ** -8 * np.abs(ref) + 2 * err_p * np.abs(v).max() + (n + 64) * 2.0 ** -24 * mag
    if chunk:
        tol = tol + 2.0 ** -8 * mag
    err = np.abs(o.double().cpu().numpy() - ref)
    worst = float((err / np.maximum(tol, 1e-30)).max())
    assert worst <= 1.0, f"error is {worst:.2f} of its bound"


def _batch(lens, seed=0, extra=32, page=None):
    """Shuffled slots (or whole pages) for requests of these lengths: (pool, indptr, idx)."""
    rng = np.random.default_rng(seed)
    if page:
        pages = [-(-n // page) for n in lens]
        perm = rng.permutation(sum(pages) + 2)
        idx, at = [], 0
        for n, p in zip(lens, pages):
            pos = np.arange(n)
            idx.append(perm[at:at + p][pos // page] * page + pos % page)
            at += p
        size = (sum(pages) + 2) * page
    else:
        size = sum(lens) + extra
        idx = np.split(rng.permutation(size)[:sum(lens)], np.cumsum(lens)[:-1])
    flat = np.concatenate(idx) if sum(lens) else np.zeros(1, int)
    ptr = np.concatenate([[0], np.cumsum(lens)])
    return _pool(size, seed=seed), _i32(ptr.tolist()), _i32(flat.tolist()), idx


def _decode(q, pool, ptr, idx, splits, fixed, seg, slots, variant, order=None, workers=0):
    from sid.kernels.jit import load_ext
    b = q.shape[0]
    po = torch.full((b, HQ, slots, D), float("nan"), device="cuda")
    pl = torch.full((b, HQ, slots), float("nan"), device="cuda")
    o = torch.full_like(q, float("nan"))
    load_ext().flash_decode_fwd(q, pool[0], pool[1], ptr, idx, None, splits, fixed, SCALE, po, pl,
                                o, segment_size=seg, grid_slots=slots, variant=variant,
                                wg_order=order, workers=workers, kv_scales=pool[2])
    return o


def _check_decode(o, q, pool, idx):
    for i, at in enumerate(idx):
        if len(at) == 0:
            assert not o[i].any()
        else:
            _bounded(o[i:i + 1], q[i:i + 1], pool[3][at], pool[4][at])


DECODE_LENS = [[1], [2], [31, 32, 33], [255, 256, 257], [0, 5, 0], [1000, 32, 999],
               [17 * i + 1 for i in range(17)], [3001]]


@pytest.mark.parametrize("lens", DECODE_LENS, ids=lambda s: f"b{len(s)}_max{max(s)}")
@pytest.mark.parametrize("variant", [0, 1, 2, 3])
@pytest.mark.parametrize("plan", ["one", "fixed256", "splits4_seg64"])
def test_decode_against_oracle(lens, variant, plan):
    _say("decode", lens, variant, plan)
    pool, ptr, idx, at = _batch(lens, seed=len(lens))
    q = torch.randn(len(lens), HQ, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    longest = max(lens)
    if plan == "one":
        args = (1, 0, 0, 1)
    elif plan == "fixed256":
        args = (max(1, -(-longest // 256)), 256, 256, max(1, -(-longest // 256)))
    else:
        chunk = max(32, -(-(-(-longest // 4)) // 32) * 32)
        args = (4, 0, 64, 4 * -(-chunk // 64))
    o = _decode(q, pool, ptr, idx, *args, variant)
    _check_decode(o, q, pool, at)


@pytest.mark.parametrize("lens", [[1], [1024], [300] * 5 + [1], [2000, 64, 7, 900] * 8,
                                  [700 + i for i in range(96)], [40] * 256,
                                  [128 + 63 * i for i in range(64)]], ids=lambda s: f"b{len(s)}")
def test_decode_step_plan(lens):
    """The plan that a serving loop makes (shape, geometry, order, workers) over paged slots."""
    from sid.kernels.decode_attention import DecodeAttention
    _say("step plan", len(lens))
    pool, ptr, idx, at = _batch(lens, seed=3, page=16)
    q = torch.randn(len(lens), HQ, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    attn = DecodeAttention(len(lens), HQ, HKV, D, 32, 256, 4096, "cuda")
    attn.part_o.fill_(float("nan"))
    attn.part_lse.fill_(float("nan"))
    plan = attn.step_plan(lens, kv_fp8=True)
    o = attn.forward(q, *pool[:2], ptr, idx, _i32(lens), max(lens), SCALE, False,
                     kv_scales=pool[2], **plan)
    pick = range(0, len(lens), max(1, len(lens) // 12))
    for i in pick:
        _check_decode(o[i:i + 1], q[i:i + 1], pool, [at[i]])
    again = attn.forward(q, *pool[:2], ptr, idx, _i32(lens), max(lens), SCALE, False,
                         kv_scales=pool[2], **plan)
    assert torch.equal(o, again)


def test_decode_workers_and_orders_keep_bits():
    from sid.kernels.decode_attention import segment_tokens, worker_order, workgroup_order
    lens = [900, 0, 33, 2500, 1, 400, 1300]
    pool, ptr, idx, _ = _batch(lens, seed=9)
    q = torch.randn(len(lens), HQ, D, device="cuda").to(torch.bfloat16)
    slots = 10
    base = _decode(q, pool, ptr, idx, 10, 256, 256, slots, 2)
    tok = segment_tokens(lens, len(lens), 0, 256, 256, slots)
    o1 = _decode(q, pool, ptr, idx, 10, 256, 256, slots, 2,
                 order=torch.from_numpy(workgroup_order(tok, 256)).cuda())
    assert torch.equal(base, o1)
    for w in (1, 5, 64, 256):
        o2 = _decode(q, pool, ptr, idx, 10, 256, 256, slots, 2,
                     order=torch.from_numpy(worker_order(tok, w)).cuda(), workers=w)
        assert torch.equal(base, o2)


def test_decode_fixed_splits_do_not_depend_on_the_batch():
    from sid.kernels.decode_attention import DecodeAttention
    lens = [700, 1, 256, 3000, 513]
    pool, ptr, idx, at = _batch(lens, seed=5)
    q = torch.randn(len(lens), HQ, D, device="cuda").to(torch.bfloat16)
    attn = DecodeAttention(8, HQ, HKV, D, 32, 256, 4096, "cuda")
    o = attn.forward(q, *pool[:2], ptr, idx, _i32(lens), max(lens), SCALE, True, kv_scales=pool[2])
    for i, n in enumerate(lens):
        one = attn.forward(q[i:i + 1].contiguous(), *pool[:2], _i32([0, n]), _i32(at[i].tolist()),
                           _i32([n]), n, SCALE, True, kv_scales=pool[2])
        assert torch.equal(one[0], o[i])


def test_decode_bad_slots_read_slot_zero_and_neighbours_stay():
    """Slots outside the pool read slot 0; a NaN row that no request names reaches nothing; one
    request's NaN stays in its own rows and heads."""
    lens = [70, 130]
    pool, ptr, idx, at = _batch(lens, seed=6)
    kc, vc, sc, kd, vd = pool
    q = torch.randn(2, HQ, D, device="cuda").to(torch.bfloat16)
    free = sorted(set(range(kd.shape[0])) - set(np.concatenate(at).tolist()) - {0})
    for s in free:
        kc.view(torch.uint8)[s] = 0x7f
        vc.view(torch.uint8)[s] = 0x7f
        sc.view(torch.uint8)[s] = 255
    bad = idx.clone()
    bad[3], bad[100] = -4, 1 << 30
    at0 = [a.copy() for a in at]
    at0[0][3] = 0
    at0[1][30] = 0
    for variant in range(4):
        o = _decode(q, pool, ptr, bad, 4, 0, 64, 8, variant)
        _check_decode(o, q, pool, at0)
    kc.view(torch.uint8)[int(at[0][50]), 3] = 0x7f   # head 3 of one key of request 0
    sc.view(torch.uint8)[int(at[0][50]), 3, 0] = 255
    for variant in range(4):
        o = _decode(q, pool, ptr, idx, 4, 0, 64, 8, variant)
        assert o[0, 6:8].isnan().all()
        assert not o[0, :6].isnan().any() and not o[0, 8:].isnan().any() and not o[1].isnan().any()


# ---- chunk ------------------------------------------------------------------------------------

def _chunk_batch(specs, seed=0, page=None):
    lens = [p + e for p, e in specs]
    pool, ptr, idx, at = _batch(lens, seed=seed, page=page)
    qo = np.concatenate([[0], np.cumsum([e for _, e in specs])])
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(int(qo[-1]), HQ, D, generator=g).to(torch.bfloat16).cuda()
    return q, pool, _i32(qo.tolist()), ptr, idx, at, qo


def _chunk(q, pool, qo, ptr, idx, specs, workspace=True):
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.jit import load_ext
    me, mk = max(e for _, e in specs), max(p + e for p, e in specs)
    if workspace:
        return extend_attention_fwd(q, pool[0], pool[1], qo, ptr, idx, me, SCALE, max_kv_len=mk,
                                    kv_scales=pool[2])
    o = torch.full_like(q, float("nan"))
    load_ext().extend_attention_fwd(q, pool[0], pool[1], qo, ptr, idx, me, SCALE, o, mk, None,
                                    kv_scales=pool[2])
    return o


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
    """With and without the workspace, alone and in a batch, whole or window by window."""
    specs = [(300, 64), (0, 40), (1023, 33)]
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


@pytest.mark.parametrize("batch,lo,hi,pre", [(2, 900, 2100, 700), (17, 1, 400, 900),
                                             (63, 1, 50, 300), (64, 1, 40, 100), (65, 20, 40, 5),
                                             (200, 1, 30, 60), (256, 0, 9, 40), (257, 1, 9, 40),
                                             (300, 1, 3, 20)])
def test_chunk_placement_covers_every_tile(batch, lo, hi, pre):
    """Ragged batches whose grid is placed by key count (up to 256 requests) or plainly: every
    row is there, with the bits that its request alone gives (fanned out)."""
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
@pytest.mark.parametrize("specs", [[(100, 70)], [(5, 1200)] * 4], ids=["fanout", "grid"])
def test_chunk_nan_reaches_only_rows_that_see_it(specs, which):
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=8)
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    key, head = specs[0][0] + 37, 5
    pool[which].view(torch.uint8)[int(at[0][key]), head] = 0x7f
    pool[2].view(torch.uint8)[int(at[0][key]), head, which] = 255
    o = _chunk(q, pool, qo, ptr, idx, specs)
    hit = torch.zeros(o.shape, dtype=torch.bool, device="cuda")
    hit[37:int(qoh[1]), 2 * head:2 * head + 2] = True
    assert o[hit].isnan().all()
    assert torch.equal(o[~hit], clean[~hit])


@pytest.mark.parametrize("which", [0, 1], ids=["nan_k", "nan_v"])
@pytest.mark.parametrize("specs,key", [([(100, 70)], 169), ([(100, 70)], 128), ([(5, 1200)] * 4, 1204),
                                       ([(5, 1200)] * 4, 512)],
                         ids=["fanout_last", "fanout_tile", "grid_last", "grid_split"])
def test_chunk_nan_in_the_last_key_and_at_edges(specs, key, which):
    """The last key, which stands in for the keys past the sequence's end, and a tile's and a
    split's first."""
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=21)
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    pool[which].view(torch.uint8)[int(at[0][key]), 3] = 0x7f
    pool[2].view(torch.uint8)[int(at[0][key]), 3, which] = 255
    o = _chunk(q, pool, qo, ptr, idx, specs)
    hit = torch.zeros(o.shape, dtype=torch.bool, device="cuda")
    hit[max(0, key - specs[0][0]):int(qoh[1]), 6:8] = True
    assert o[hit].isnan().all()
    assert torch.equal(o[~hit], clean[~hit])


def _ramp(lens, seed, up):
    """A pool whose scores rise (or fall) by about 12 octaves of exp every 64 positions, and
    queries for it: every tile moves its rows' maxima (or none but the first does)."""
    g = torch.Generator().manual_seed(seed)
    _, ptr, idx, at = _batch(lens, seed=seed, page=16)
    size = int(idx.max()) + 17
    w = torch.randn(HKV, D, generator=g)
    x = torch.randn(2, size, HKV, D, generator=g)
    for a in at:
        pos = torch.arange(len(a), dtype=torch.float32)
        x[0, torch.from_numpy(a)] += (pos if up else -pos)[:, None, None] * w / 87.0
    pool, vals, bytes_ = [], [], []
    for s in (0, 1):
        codes, b = store_ref(x[s].to(torch.bfloat16).double().numpy())
        pool.append(torch.from_numpy(codes).cuda().view(FP8))
        bytes_.append(b)
        vals.append(load_ref(codes, b))
    scales = torch.from_numpy(np.stack(bytes_, -1)).cuda().view(E8M0)

    def queries(n):
        q = torch.randn(n, HQ, D, generator=g) * 0.3 + w.repeat_interleave(2, 0)
        return q.to(torch.bfloat16).cuda()
    return (pool[0], pool[1], scales, *vals), ptr, idx, at, queries


@pytest.mark.parametrize("up", [True, False], ids=["rising", "falling"])
@pytest.mark.parametrize("workspace", [True, False])
def test_chunk_scores_that_move_every_tile(up, workspace):
    specs = [(0, 130), (700, 50), (1000, 40)]
    pool, ptr, idx, at, queries = _ramp([p + e for p, e in specs], 5, up)
    qoh = np.concatenate([[0], np.cumsum([e for _, e in specs])])
    q = queries(int(qoh[-1]))
    o = _chunk(q, pool, _i32(qoh.tolist()), ptr, idx, specs, workspace)
    for i, (p, e) in enumerate(specs):
        a, b = int(qoh[i]), int(qoh[i + 1])
        _bounded(o[a:b], q[a:b], pool[3][at[i]], pool[4][at[i]], first=p, chunk=True)


@pytest.mark.parametrize("up", [True, False], ids=["rising", "falling"])
@pytest.mark.parametrize("variant", [2, 3])
def test_decode_scores_that_move_every_tile(up, variant):
    lens = [1, 70, 500, 1300]
    pool, ptr, idx, at, queries = _ramp(lens, 6, up)
    q = queries(len(lens))
    for args in ((1, 0, 0, 1), (1, 0, 256, 6)):
        _check_decode(_decode(q, pool, ptr, idx, *args, variant), q, pool, at)


def test_chunk_unwritten_slot_zero_and_tail_rows_untouched():
    """Slot 0 holding NaNs is behind every tile's end; rows past the last sequence stay."""
    specs = [(10, 7), (64, 30)]
    q, pool, qo, ptr, idx, at, qoh = _chunk_batch(specs, seed=12)
    used = set(np.concatenate(at).tolist())
    if 0 in used:  # give slot 0's row another place
        spare = next(s for s in range(pool[3].shape[0]) if s not in used)
        for t in pool[:3]:
            t.view(torch.uint8)[spare] = t.view(torch.uint8)[0]
        idx[idx == 0] = spare
    clean = _chunk(q, pool, qo, ptr, idx, specs)
    for t, val in zip(pool[:3], (0x7f, 0x7f, 255)):
        t.view(torch.uint8)[0] = val
    from sid.kernels.jit import load_ext
    qq = torch.cat([q, q[:3]])
    for ws in (True, False):
        assert torch.equal(_chunk(q, pool, qo, ptr, idx, specs, ws), clean)
    o = torch.full_like(qq, 7.0)
    load_ext().extend_attention_fwd(qq, pool[0], pool[1], qo, ptr, idx, 30, SCALE, o, 94, None,
                                    kv_scales=pool[2])
    assert torch.equal(o[:q.shape[0]], clean) and (o[q.shape[0]:] == 7.0).all()


# ---- together ---------------------------------------------------------------------------------

def test_pool_that_grows():
    """Prompts written and attended to, then read back, then single tokens appended and decoded,
    then a window over everything: each step against 64 bits of what the pool stands for."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.kv_fp8 import gather_cache_fp8, reshape_and_cache_fp8
    lens = [40, 3, 129]
    cap = 260
    perm = torch.randperm(3 * cap, generator=torch.Generator().manual_seed(5))
    slots = [perm[i * cap:(i + 1) * cap] for i in range(3)]
    kc, vc, sc = _empty(3 * cap)
    vals = [(np.zeros((0, HKV, D)), np.zeros((0, HKV, D))) for _ in lens]
    attn = DecodeAttention(3, HQ, HKV, D, 32, 256, 4096, "cuda")
    g = torch.Generator().manual_seed(6)

    def write(counts):
        at = torch.cat([slots[i][len(vals[i][0]):len(vals[i][0]) + c] for i, c in enumerate(counts)])
        k, v = (torch.randn(len(at), HKV, D, generator=g).to(torch.bfloat16) for _ in range(2))
        reshape_and_cache_fp8(k.cuda(), v.cuda(), kc, vc, sc, at.cuda())
        n = 0
        for i, c in enumerate(counts):
            new = [load_ref(*store_ref(x[n:n + c].double().numpy())) for x in (k, v)]
            vals[i] = tuple(np.concatenate([a, b]) for a, b in zip(vals[i], new))
            n += c

    def inputs():
        full = [len(v[0]) for v in vals]
        idx = torch.cat([slots[i][:n] for i, n in enumerate(full)])
        return full, _i32(np.concatenate([[0], np.cumsum(full)]).tolist()), idx.int().cuda()

    def chunk(counts):
        full, ptr, idx = inputs()
        q = torch.randn(sum(counts), HQ, D, generator=g).to(torch.bfloat16).cuda()
        qo = np.concatenate([[0], np.cumsum(counts)])
        specs = [(f - c, c) for f, c in zip(full, counts)]
        o = _chunk(q, (kc, vc, sc), _i32(qo.tolist()), ptr, idx, specs)
        for i, c in enumerate(counts):
            a, b = int(qo[i]), int(qo[i + 1])
            _bounded(o[a:b], q[a:b], *vals[i], first=full[i] - c, chunk=True)

    write(lens)
    chunk(lens)
    for i in range(3):
        k, v = gather_cache_fp8(kc, vc, sc, slots[i][:lens[i]].cuda())
        assert np.array_equal(k.double().cpu().numpy(), vals[i][0])
        assert np.array_equal(v.double().cpu().numpy(), vals[i][1])
    for _ in range(4):
        write([1, 1, 1])
        full, ptr, idx = inputs()
        q = torch.randn(3, HQ, D, generator=g).to(torch.bfloat16).cuda()
        o = attn.forward(q, kc, vc, ptr, idx, _i32(full), max(full), SCALE, False, kv_scales=sc,
                         **attn.step_plan(full, kv_fp8=True))
        for i in range(3):
            _bounded(o[i:i + 1], q[i:i + 1], *vals[i])
    write([70, 33, 64])
    chunk([70, 33, 64])


def test_graph_replays_on_another_stream():
    """store + decode + chunk + load captured once and replayed with other inputs, on a stream of
    its own, with eager work between the replays."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.kv_fp8 import gather_cache_fp8, reshape_and_cache_fp8
    lens = [300, 77]
    pool, ptr, idx, at = _batch(lens, seed=1)
    kc, vc, sc = pool[:3]
    attn = DecodeAttention(2, HQ, HKV, D, 32, 256, 4096, "cuda")
    plan = attn.step_plan(lens, kv_fp8=True)
    q = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device="cuda")
    qc = torch.zeros(8, HQ, D, dtype=torch.bfloat16, device="cuda")
    kn, vn = (torch.zeros(2, HKV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    new = torch.tensor([int(a[-1]) for a in at], device="cuda")
    seq, qo = _i32(lens), _i32([0, 4, 8])

    def run():
        reshape_and_cache_fp8(kn, vn, kc, vc, sc, new)
        o = attn.forward(q, kc, vc, ptr, idx, seq, max(lens), SCALE, False, kv_scales=sc, **plan)
        c = extend_attention_fwd(qc, kc, vc, qo, ptr, idx, 4, SCALE, max_kv_len=300, kv_scales=sc)
        return (o, c, *gather_cache_fp8(kc, vc, sc, new))

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    side = torch.cuda.Stream()
    for step in range(4):
        g = torch.Generator().manual_seed(step)
        for x in (q, qc, kn, vn):
            x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
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


def test_two_graphs_share_the_split_workspace():
    """Two captured steps of different batches over one pool and one DecodeAttention, replayed in
    turn with other inputs: each as its eager run."""
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.ops import qkv_post
    g = torch.Generator().manual_seed(31)
    attn = DecodeAttention(5, HQ, HKV, D, 32, 256, 4096, "cuda")
    pool, ptr, idx, at = _batch([900, 33, 400, 1, 2000], seed=4)
    kc, vc, sc = pool[:3]
    norm = (1 + 0.1 * torch.randn(2, D, generator=g)).to(torch.bfloat16).cuda()
    cos_sin = torch.randn(4096, D, generator=g).cuda()

    def step(pick):
        lens = [len(at[i]) for i in pick]
        b = len(pick)
        p = _i32(np.concatenate([[0], np.cumsum(lens)]).tolist())
        i = _i32(np.concatenate([at[i] for i in pick]).tolist())
        slots = torch.tensor([int(at[i][-1]) for i in pick], device="cuda")
        pos = torch.tensor([n - 1 for n in lens], device="cuda")
        proj = torch.zeros(b, (HQ + 2 * HKV) * D, dtype=torch.bfloat16, device="cuda")
        seq, qo, plan = _i32(lens), _i32(list(range(b + 1))), attn.step_plan(lens, kv_fp8=True)

        def run():
            q = qkv_post(proj, norm[0], norm[1], 1e-6, pos, cos_sin, slots, kc, vc, HQ, kv_scales=sc)
            o = attn.forward(q, kc, vc, p, i, seq, max(lens), SCALE, False, kv_scales=sc, **plan)
            c = extend_attention_fwd(q, kc, vc, qo, p, i, 1, SCALE, max_kv_len=max(lens),
                                     kv_scales=sc)
            return q, o, c
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        return proj, run, graph, out

    steps = [step([0, 3, 4]), step([4, 2, 1, 0, 3]), step([1])]
    for _ in range(3):
        for proj, run, graph, out in steps:
            proj.copy_(torch.randn(proj.shape, generator=g).to(torch.bfloat16))
            graph.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in out]
            for a, b in zip(got, run()):
                assert torch.equal(a, b)


# ---- refusals ---------------------------------------------------------------------------------

def test_refusals():
    from sid.kernels.decode_attention import DecodeAttention
    from sid.kernels.extend_attention import extend_attention_fwd
    from sid.kernels.kv_fp8 import gather_cache_fp8, reshape_and_cache_fp8
    kc, vc, sc = _empty(8)
    x = torch.zeros(2, HKV, D, dtype=torch.bfloat16, device="cuda")
    at = torch.arange(2, device="cuda")

    def refused(match, fn, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            fn(*a, **kw)

    store = reshape_and_cache_fp8
    refused("bf16", store, x.float(), x, kc, vc, sc, at)
    refused("k's shape", store, x, x[:1], kc, vc, sc, at)
    refused("float8_e4m3fn", store, x, x, x, x, sc, at)
    refused("e8m0", store, x, x, kc, vc, sc.view(torch.uint8), at)
    refused("kv_scales must be", store, x, x, kc, vc, sc[:4], at)
    refused("contiguous", store, x, x, kc, vc, sc[:, :, :1].expand(8, HKV, 2), at)
    refused("int64", store, x, x, kc, vc, sc, at.int())
    refused("T entries", store, x, x, kc, vc, sc, at[:1])
    refused("matching the cache", store, x[:, :4].contiguous(), x[:, :4].contiguous(), kc, vc, sc, at)
    y = torch.zeros(2, HKV, 64, dtype=torch.bfloat16, device="cuda")
    refused("must both be", store, y, y, kc, vc, sc, at)
    z = torch.zeros(2 * HKV * D + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, HKV, D)
    refused("16-byte", store, z, x, kc, vc, sc, at)
    refused("int64", gather_cache_fp8, kc, vc, sc, at.int())
    refused("must both be", gather_cache_fp8, kc, vc[:4], sc, at)

    attn = DecodeAttention(2, HQ, HKV, D, 32, 256, 4096, "cuda")
    q = torch.zeros(2, HQ, D, dtype=torch.bfloat16, device="cuda")
    ptr, idx, seq = _i32([0, 2, 4]), _i32([1, 2, 3, 4]), _i32([2, 2])
    # codes without their scales, and bf16 pools with some
    refused("bfloat16", attn.forward, q, kc, vc, ptr, idx, seq, 2, SCALE, False)
    refused("float8_e4m3fn", attn.forward, q, x, x, ptr, idx, seq, 2, SCALE, False, kv_scales=sc)
    refused("B\\+1", attn.forward, q, kc, vc, ptr[:2], idx, seq, 2, SCALE, False, kv_scales=sc)
    refused("int32", attn.forward, q, kc, vc, ptr.long(), idx, seq, 2, SCALE, False, kv_scales=sc)
    q4 = torch.zeros(2, 8, D, dtype=torch.bfloat16, device="cuda")
    refused("workspace|q heads", attn.forward, q4, kc, vc, ptr, idx, seq, 2, SCALE, False,
            kv_scales=sc)
    refused("bfloat16", extend_attention_fwd, q, kc, vc, _i32([0, 1, 2]), ptr, idx, 1, SCALE)
    refused("q heads", extend_attention_fwd, q4, kc, vc, _i32([0, 1, 2]), ptr, idx, 1, SCALE,
            kv_scales=sc)
    assert reshape_and_cache_fp8(x[:0], x[:0], kc, vc, sc, at[:0]) is None
    k0, v0 = gather_cache_fp8(kc, vc, sc, at[:0])
    assert k0.shape == (0, HKV, D) and v0.shape == (0, HKV, D)
