"""Host-side rules of the KV pools and what is built over them (no GPU)."""

from __future__ import annotations

import types

import numpy as np
import pytest
import torch


def test_native_executor_goes_by_the_cache_itself(monkeypatch):
    """A KV cache made after another one was dropped may get the same id: the native executor's
    descriptor, which holds the pools' addresses, is made anew."""
    import sid.model.native
    from sid.model.qwen3 import Qwen3Model

    built = []

    class Recorder:
        def __init__(self, model, kv_cache, *_):
            built.append(kv_cache.tag)

        def forward(self, *a, **kw):
            return built[-1]

    class Cache:
        def __init__(self, tag):
            self.tag = tag

        def layer(self, i):
            return torch.zeros(4, 8, 128), None

    monkeypatch.setattr(sid.model.native, "NativeQwen3", Recorder)
    model = Qwen3Model.__new__(Qwen3Model)
    model._native, model.decode_chain = None, True
    fb = types.SimpleNamespace(sample_tiles=None)
    old = Cache("old")
    assert model._native_forward(fb, old, True) == "old"
    assert model._native_forward(fb, old, True) == "old" and built == ["old"]
    was, others = id(old), []
    del old
    for _ in range(10000):
        new = Cache("new")
        if id(new) == was:
            break
        others.append(new)
    assert id(new) == was, "no object took the dropped one's place"
    assert model._native_forward(fb, new, True) == "new"
    assert model._native_forward(fb, new, True) == "new" and built == ["old", "new"]
    model.decode_chain = False
    assert model._native_forward(fb, new, True) == "new" and built == ["old", "new", "new"]


def _host_only_attention(monkeypatch):
    from sid.kernels.decode_attention import DecodeAttention, workspace_slots
    da = DecodeAttention.__new__(DecodeAttention)
    da.num_kv_heads, da.max_kv_splits, da.invariant_split_size = 8, 32, 256
    da.device = torch.device("cpu")
    da.ws_splits = workspace_slots(16384, 32, 256)
    monkeypatch.setattr(DecodeAttention, "cu_count", lambda self: 256)
    return da


@pytest.mark.parametrize("kv_fp8", [False, True])
@pytest.mark.parametrize("lens", [[1], [1024], [300] * 5, [2000, 64, 7, 900] * 8, [2048] * 64,
                                  [700 + i for i in range(96)], [40] * 200], ids=lambda s: f"b{len(s)}")
def test_step_plan_is_the_plan_that_the_engine_runs(monkeypatch, lens, kv_fp8):
    from sid.engine.model_runner import ModelRunner
    da = _host_only_attention(monkeypatch)
    runner = ModelRunner.__new__(ModelRunner)
    runner.decode_attn, runner.graphs, runner.device = da, None, "cpu"
    runner.kv_cache = types.SimpleNamespace(kv_scales=[] if kv_fp8 else None)
    fb = types.SimpleNamespace(seq_lens_host=np.asarray(lens))
    geom = runner._pick_variant(fb, max(lens))
    ordered = runner._attach_order(fb, len(lens), False, max(lens), geom)
    plan = da.step_plan(lens, kv_fp8=kv_fp8)
    assert plan["geometry"] == geom == fb.decode_geometry and plan["variant"] == fb.decode_variant
    assert plan["workers"] == fb.decode_workers and geom[2] <= da.ws_splits
    assert (plan["wg_order"] is None) == (fb.decode_wg_order is None) == (ordered == 0)
    if ordered:
        assert torch.equal(plan["wg_order"], fb.decode_wg_order)
        want = torch.arange(len(lens))[:, None] << 12 | torch.arange(geom[2])
        assert torch.equal((plan["wg_order"] & ~(1 << 30)).sort()[0], want.reshape(-1).int().sort()[0])


def test_a_library_from_before_the_8bit_pool_is_refused(tmp_path):
    """A library of the same ABI version that lacks the entry points added since is named as such."""
    import subprocess

    from sid.kernels._native import ABI_REVISION, ABI_VERSION, NativeLib
    for rev, text in ((None, "revision 0"), (ABI_REVISION - 1, f"revision {ABI_REVISION - 1}")):
        src = tmp_path / f"old{rev}.c"
        src.write_text('const char* sid_last_error(void) { return ""; }\n'
                       f"int sid_abi_version(void) {{ return {ABI_VERSION}; }}\n"
                       + ("" if rev is None else f"int sid_abi_revision(void) {{ return {rev}; }}\n"))
        lib = tmp_path / f"libold{rev}.so"
        subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
        with pytest.raises(RuntimeError, match=text):
            NativeLib(lib)


def test_library_reports_its_revision():
    from sid.kernels._native import ABI_REVISION
    from sid.kernels.jit import load_ext
    assert load_ext().lib.sid_abi_revision() == ABI_REVISION == 1
