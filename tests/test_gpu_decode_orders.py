"""Stage-1 orders of the decode attention with entries outside the grid, negative ones among them:
they are skipped, over every pool."""

from __future__ import annotations

import pytest
import torch

from conftest import HKV, D
from test_gpu_kv_fp8 import _decode, _i32, _say

pytestmark = pytest.mark.gpu

LENS = [70, 300, 40]
BAD = [-1, -(1 << 31), -(1 << 31) | 1 << 30, -(1 << 31) | 2 << 12 | 1, (1 << 30) - 1, 3 << 12, 1 << 12 | 4000]


def _pool_of(kind):
    n = sum(LENS)
    if kind == "bf16":
        g = torch.Generator().manual_seed(1)
        k, v = (torch.randn(n, HKV, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        return k, v, None
    if kind == "fp8":
        from test_gpu_kv_fp8 import _pool
    else:
        from test_gpu_kv_fp4_attention import _pool
    return _pool(n, seed=1)[:3]


@pytest.mark.parametrize("workers", [0, 1, 3])
@pytest.mark.parametrize("kind", ["bf16", "fp8", "fp4"])
def test_entries_outside_the_grid_are_skipped(kind, workers):
    _say("orders", kind, workers)
    pool = _pool_of(kind)
    idx = torch.randperm(sum(LENS), generator=torch.Generator().manual_seed(2)).int().cuda()
    ptr = _i32([0, 70, 370, 410])
    q = torch.randn(3, 16, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    for args in ((1, 0, 0, 1), (1, 0, 64, 5)):
        slots = args[3]
        if slots == 1 and workers:
            continue
        base = _decode(q, pool, ptr, idx, *args, 3)
        items = [b << 12 | y for y in range(slots) for b in range(3)]
        for bad in BAD:
            order = [bad if i >> 12 == 0 else i for i in items]
            if bad >= 0 or bad & 1 << 30:
                order.sort(key=lambda i: bool(i & 1 << 30))  # flagged entries come last
            o = _decode(q, pool, ptr, idx, *args, 3, order=_i32(order), workers=workers)
            assert torch.equal(o[1:], base[1:]), bad
            assert o[0].isnan().all(), bad  # what the workspace and the output held before
