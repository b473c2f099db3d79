"""Host side of the 4-bit KV pool and of scaled rotary positions: the engine's plans, configurations."""

from __future__ import annotations

import json
import types

import numpy as np
import pytest
import torch

from test_kv_fp8_host import _host_only_attention


@pytest.mark.parametrize("lens", [[1], [1024], [300] * 5, [2000, 64, 7, 900] * 8, [2048] * 64,
                                  [700 + i for i in range(96)], [40] * 200, [5000] * 200],
                         ids=lambda s: f"b{len(s)}")
def test_step_plan_is_the_plan_that_the_engine_runs(monkeypatch, lens):
    from sid.engine.model_runner import ModelRunner
    da = _host_only_attention(monkeypatch)
    runner = ModelRunner.__new__(ModelRunner)
    runner.decode_attn, runner.graphs, runner.device = da, None, "cpu"
    runner.kv_cache = types.SimpleNamespace(kv_scales=[], dtype="fp4_e2m1")
    fb = types.SimpleNamespace(seq_lens_host=np.asarray(lens))
    geom = runner._pick_variant(fb, max(lens))
    ordered = runner._attach_order(fb, len(lens), False, max(lens), geom)
    plan = da.step_plan(lens, kv_fp4=True)
    assert plan["geometry"] == geom == fb.decode_geometry and plan["variant"] == fb.decode_variant == 3
    assert plan["workers"] == fb.decode_workers and geom[2] <= da.ws_splits
    assert (plan["wg_order"] is None) == (fb.decode_wg_order is None) == (ordered == 0)
    if ordered:
        assert torch.equal(plan["wg_order"], fb.decode_wg_order)
        want = torch.arange(len(lens))[:, None] << 12 | torch.arange(geom[2])
        assert torch.equal((plan["wg_order"] & ~(1 << 30)).sort()[0], want.reshape(-1).int().sort()[0])


def test_order_where_the_grid_does_not_start_at_once():
    """230 segments with tokens among 512 slots: ordered for a 4-bit pool, the grid's own otherwise."""
    from sid.kernels.decode_attention import placement, stage1_workers_fp4
    lens = [4096] + [1700] * 31
    four = placement(lens, 32, 1, 0, 256, 16, 3, 256, workers_of=stage1_workers_fp4, kv_fp4=True)
    assert four[0] is not None and four[0].size == 512 and four[1] == 0
    order, workers = placement([5000] * 64, 64, 1, 0, 256, 20, 3, 256, workers_of=stage1_workers_fp4,
                               kv_fp4=True)
    assert workers == 512 and order.size == 1280
    assert placement([100] * 4, 4, 1, 0, 32, 4, 3, 256, workers_of=stage1_workers_fp4,
                     kv_fp4=True) == (None, 0)


def test_config_names_the_pool():
    from sid.config import EngineConfig
    assert EngineConfig(kv_cache_dtype="fp4_e2m1").kv_cache_dtype == "fp4_e2m1"
    with pytest.raises(ValueError, match="fp4_e2m1"):
        EngineConfig(kv_cache_dtype="fp4")


def _write_config(tmp_path, scaling):
    hf = dict(model_type="qwen3", num_hidden_layers=2, hidden_size=1024, num_attention_heads=16,
              num_key_value_heads=8, head_dim=128, intermediate_size=2048, vocab_size=1000,
              rms_norm_eps=1e-6, rope_theta=1e6, max_position_embeddings=40960)
    if scaling is not None:
        hf["rope_scaling"] = scaling
    (tmp_path / "config.json").write_text(json.dumps(hf))


YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


@pytest.mark.parametrize("given", ["checkpoint", "dict"])
@pytest.mark.parametrize("scaling,want,positions", [
    (None, None, 40960), ({}, None, 40960), ({"rope_type": "default"}, None, 40960),
    ({"type": "linear", "factor": 2.0}, {"type": "linear", "factor": 2.0}, 81920),
    (YARN, YARN, 131072), (dict(YARN, factor=1.0), dict(YARN, factor=1.0), 40960),
], ids=str)
def test_scaled_positions_of_a_model(tmp_path, given, scaling, want, positions):
    from sid.model.loader import build_model_config
    _write_config(tmp_path, scaling)
    got, _ = build_model_config(str(tmp_path), rope_scaling="checkpoint" if given == "checkpoint"
                                else scaling)
    assert got.rope_scaling == want and got.max_position_embeddings == positions
    plain, _ = build_model_config(str(tmp_path))
    assert plain.rope_scaling is None and plain.max_position_embeddings == 40960
    random, _ = build_model_config("random:qwen3-0.6b", rope_scaling=scaling)
    assert random.rope_scaling == want and random.max_position_embeddings == positions


@pytest.mark.parametrize("scaling", [{"rope_type": "other", "factor": 2.0}, {"rope_type": "linear"},
                                     {"rope_type": "yarn", "factor": 4.0},
                                     {"type": "linear", "factor": 0.5}], ids=str)
def test_scaled_positions_that_are_refused(tmp_path, scaling):
    from sid.config import EngineConfig
    from sid.model.loader import build_model_config
    _write_config(tmp_path, scaling)
    for given in ("checkpoint", scaling):
        with pytest.raises(ValueError):
            build_model_config(str(tmp_path), rope_scaling=given)
    build_model_config(str(tmp_path))  # not asked for: not read
    with pytest.raises(ValueError, match="checkpoint"):
        EngineConfig(rope_scaling="yarn")


def test_executor_workspace_is_its_pools():
    """The 4-bit pool's attention splits the keys of a window that the bf16 pool's walks, or the
    other way round: the workspace differs by what each asks for."""
    import ctypes

    from sid.kernels.jit import load_ext
    from sid.model.native import Batch, Model, _bind
    ext = load_ext()
    _bind(ext.lib)
    m, b = Model(), Batch()
    m.num_layers, m.hidden, m.num_q_heads, m.num_kv_heads, m.head_dim = 1, 1024, 16, 8, 128
    m.intermediate, m.vocab, m.split_k_max_tokens = 2048, 1000, 64
    args = (ctypes.byref(m), ctypes.byref(b))
    for batch, e, keys in ((1, 32, 2048), (16, 32, 2048), (1, 512, 512), (4, 256, 2048), (1, 64, 100000)):
        b.num_tokens, b.batch, b.max_extend_len, b.max_kv_len = batch * e, batch, e, keys
        plain = ext.lib.sid_qwen3_extend_workspace_bytes(*args)
        four = ext.lib.sid_qwen3_extend_fp4_workspace_bytes(*args)
        own = [ext.extend_attention_workspace_bytes(batch, batch * e, 16, 8, e, keys, fp4=x)
               for x in (False, True)]
        assert abs((plain - own[0]) - (four - own[1])) <= 512  # (each piece starts on 256 bytes)


def test_executor_refuses_missing_scales():
    import ctypes

    from sid.kernels.jit import load_ext
    from sid.model.native import Batch, Model, _bind
    lib = load_ext().lib
    _bind(lib)
    m, b = Model(), Batch()
    m.num_layers = 1
    none = (ctypes.c_void_p * 1)(None)
    args = (ctypes.byref(m), ctypes.byref(b))
    assert lib.sid_qwen3_extend_forward_fp4(*args, None, None, 0, None, None, None) != 0
    assert lib.sid_qwen3_extend_forward_fp4(*args, none, None, 0, None, None, None) != 0
    assert b"layer 0 has no scales" in lib.sid_last_error()
