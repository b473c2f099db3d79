"""The 8-bit KV pool's attention where its inputs are unusual: queries and keys that are not numbers.
Where a kernel is shared with the bf16 pool, its form is run too."""

from __future__ import annotations

import pytest
import torch

from conftest import HQ, D, SCALE
from test_gpu_kv_fp8 import _batch, _decode

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
