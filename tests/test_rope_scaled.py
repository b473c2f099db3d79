"""Rotary frequencies of the scaled layouts against their formulas, and refusals (no GPU)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from sid.kernels.rope import _turn_fractions, scaled_frequencies

YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)


def test_default_and_linear():
    f, g = scaled_frequencies(128, 1e6)
    want = torch.tensor([1e6 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64)
    assert g == 1.0 and torch.allclose(f, want, rtol=1e-15, atol=0)
    f2, g2 = scaled_frequencies(128, 1e6, dict(type="linear", factor=2.5))
    assert g2 == 1.0 and torch.allclose(f2 * 2.5, f, rtol=1e-15, atol=0)


def test_ntk_keeps_the_first_pair_and_divides_the_last():
    f, _ = scaled_frequencies(64, 1e4)
    s, g = scaled_frequencies(64, 1e4, dict(rope_type="ntk", factor=4.0))
    assert g == 1.0 and s[0] == 1.0
    assert math.isclose(float(s[-1]) * 4.0, float(f[-1]), rel_tol=1e-12)


def test_yarn_by_hand():
    """128 dims, base 1e6, 32768 positions: 32768 / (2 pi 32) = 163.0 and 32768 / (2 pi) = 5215.2,
    whose logarithms over ln(1e6) times 64 are 23.6 and 39.6: pairs up to 23 are kept, those from
    40 on divided by 4."""
    f, _ = scaled_frequencies(128, 1e6)
    s, g = scaled_frequencies(128, 1e6, YARN)
    assert math.isclose(g, 0.1 * math.log(4.0) + 1.0)
    assert torch.allclose(s[:24], f[:24], rtol=1e-15, atol=0)
    assert torch.allclose(s[40:], f[40:] / 4.0, rtol=1e-15, atol=0)
    r = (30 - 23) / (40 - 23)
    assert math.isclose(float(s[30]), float(f[30]) * (r / 4 + 1 - r), rel_tol=1e-14)
    assert scaled_frequencies(128, 1e6, dict(YARN, attention_factor=1.0))[1] == 1.0
    kept = scaled_frequencies(128, 1e6, dict(YARN, beta_fast=2.0))[0]
    assert torch.allclose(kept[:36], f[:36], rtol=1e-15, atol=0)


@pytest.mark.parametrize("scaling,text", [
    (dict(rope_type="other", factor=2.0), "unknown rope_type"), (dict(rope_type="linear"), "factor"),
    (dict(rope_type="ntk", factor=0.5), "factor"), (dict(rope_type="yarn", factor=2.0), "original"),
    (dict(rope_type="linear", factor=float("inf")), "factor"),
    (dict(YARN, beta_fast=1.0, beta_slow=2.0), "beta_fast"),
])
def test_bad_scalings(scaling, text):
    with pytest.raises(ValueError, match=text):
        scaled_frequencies(64, 1e4, scaling)


def test_bad_layouts():
    from sid.kernels.rope import RotaryEmbedding
    for n in (0, 3, 66):
        with pytest.raises(ValueError, match="rotary_dim"):
            RotaryEmbedding(64, 16, 1e4, "cpu", rotary_dim=n)
    with pytest.raises(ValueError, match="theta"):
        scaled_frequencies(64, 1.0)


def test_turn_fractions():
    """Fractions of a turn to 2^-65: pos times one, modulo 2^64, is the angle in turns."""
    f, _ = scaled_frequencies(128, 1e6, YARN)
    t = _turn_fractions(f, "cpu")
    assert t.dtype == torch.int64 and int(t.min()) > 0
    for i in (0, 13, 40, 63):
        got = (int(t[i]) * 131071) % (1 << 64) / 2.0 ** 64
        want = math.fmod(float(f[i]) * 131071 / (2 * math.pi), 1.0)
        assert abs(got - want) < 1e-11


def test_tables_of_the_whole_head():
    from sid.kernels.rope import RotaryEmbedding, rope_table
    plain = RotaryEmbedding(64, 50, 1e4, "cpu", scaling=dict(rope_type="default"))
    assert torch.equal(plain.cos_sin, rope_table(64, 50, 1e4, "cpu"))
    r = RotaryEmbedding(64, 50, 1e4, "cpu", scaling=dict(YARN, original_max_position_embeddings=16))
    f, g = scaled_frequencies(64, 1e4, dict(YARN, original_max_position_embeddings=16))
    angle = 49 * f
    want = torch.cat([angle.cos(), angle.sin()]) * g
    assert torch.allclose(r.cos_sin[49].double(), want, rtol=0, atol=2.0 ** -23)
    assert RotaryEmbedding(64, 50, 1e4, "cpu", interleaved=True).cos_sin is None
    assert RotaryEmbedding(64, 50, 1e4, "cpu", rotary_dim=32).cos_sin is None


def test_entry_point_refuses_bad_arguments():
    from sid.kernels.jit import load_ext
    lib = load_ext().lib

    def call(q=16, ldq=512, k=16, ldk=256, pos=16, rot=64, t=1, hq=4, hkv=2, d=128, qo=32, ldqo=512,
             ko=32, ldko=256):
        return lib.sid_rope_rotate(q, ldq, k, ldk, pos, 16, ctypes.c_float(1.0), rot, 0, t, hq, hkv,
                                   d, 100, qo, ldqo, ko, ldko, None)

    for bad, text in ((dict(t=-1), b"negative"), (dict(q=0), b"null"), (dict(ko=0), b"null"),
                      (dict(pos=0), b"null"), (dict(rot=63), b"rotary_dim"), (dict(rot=0), b"rotary_dim"),
                      (dict(rot=130), b"rotary_dim"), (dict(d=2048, ldq=1 << 20), b"head_dim"),
                      (dict(ldq=500), b"stride"), (dict(ldko=255), b"stride"),
                      (dict(qo=16, ldqo=1024), b"in place"), (dict(hq=-1), b"head counts"),
                      (dict(hq=0, hkv=0), b"head counts"), (dict(t=1 << 31), b"too many")):
        assert call(**bad) == 1 and text in lib.sid_last_error(), bad
    assert call(t=0) == 0


@pytest.mark.parametrize("scaling,text", [
    (dict(YARN, mscale=1.0, mscale_all_dim=1.0), "mscale, mscale_all_dim"),
    (dict(YARN, truncate=False), "truncate"), (dict(YARN, mrope_section=[16, 24, 24]), "mrope_section"),
    (dict(rope_type="linear", factor=2.0, beta_fast=32.0), "beta_fast"),
    (dict(rope_type="ntk", factor=2.0, attention_factor=1.0), "attention_factor"),
    (dict(rope_type="default", mrope_section=[16, 24, 24]), "mrope_section"),
    (dict(factor=4.0), "names no rope_type"), (dict(YARN, type="linear"), "rope_type"),
    (dict(YARN, rope_theta=5e5), "rope_theta"), (["yarn", 4.0], "dict"),
], ids=str)
def test_what_a_scaling_says_is_done_or_refused(scaling, text):
    """A key that would change positions or gain and is not read; a type that is not clear."""
    from sid.config import ModelConfig
    from sid.model.loader import scale_positions
    with pytest.raises(ValueError, match=text):
        scaled_frequencies(128, 1e6, scaling)
    with pytest.raises(ValueError, match=text):
        scale_positions(ModelConfig(model_path="random:"), scaling)


def test_keys_that_say_nothing_more_are_taken():
    f, g = scaled_frequencies(128, 1e6, YARN)
    for more in (dict(type="yarn"), dict(truncate=True), dict(mscale=None, truncate=None),
                 dict(rope_theta=1e6), dict(beta_fast=None, beta_slow=None, attention_factor=None)):
        f2, g2 = scaled_frequencies(128, 1e6, dict(YARN, **more))
        assert torch.equal(f, f2) and g == g2


@pytest.mark.parametrize("scaling,text", [
    (dict(rope_type="linear", factor=None), "factor"), (dict(rope_type="ntk", factor="much"), "factor"),
    (dict(YARN, factor=float("nan")), "factor"), (dict(YARN, factor=True), "factor"),
    (dict(YARN, attention_factor=float("nan")), "attention_factor"),
    (dict(YARN, attention_factor=float("inf")), "attention_factor"),
    (dict(YARN, attention_factor=0.0), "attention_factor"),
    (dict(YARN, beta_slow=0), "beta_slow"), (dict(YARN, beta_fast=0.0), "beta_fast"),
    (dict(YARN, beta_fast=float("inf")), "beta_fast"),
    (dict(YARN, original_max_position_embeddings=None), "original"),
    (dict(YARN, original_max_position_embeddings=float("inf")), "original"),
    (dict(YARN, original_max_position_embeddings=True), "original"),
    (dict(YARN, original_max_position_embeddings=-5), "original"),
], ids=str)
def test_values_that_are_no_numbers_are_refused(scaling, text):
    from sid.config import ModelConfig
    from sid.model.loader import scale_positions
    with pytest.raises(ValueError, match=text):
        scaled_frequencies(128, 1e6, scaling)
    with pytest.raises(ValueError, match=text):
        scale_positions(ModelConfig(model_path="random:"), scaling)


@pytest.mark.parametrize("kind", ["linear", "ntk"])
def test_trained_positions_that_are_null_are_the_models(kind):
    from sid.config import ModelConfig
    from sid.model.loader import scale_positions
    mcfg = ModelConfig(model_path="random:")
    trained = mcfg.max_position_embeddings
    scale_positions(mcfg, dict(rope_type=kind, factor=2.0, original_max_position_embeddings=None))
    assert mcfg.max_position_embeddings == 2 * trained
    for bad in (float("nan"), float("inf"), 0, "many"):
        with pytest.raises(ValueError, match="original"):
            scale_positions(mcfg, dict(rope_type=kind, factor=2.0, original_max_position_embeddings=bad))


def test_yarn_where_every_pair_is_on_one_side():
    """Trained positions of less than a turn of the fastest pair: all pairs are divided; of more than
    32 turns of the slowest one: none is."""
    few = dict(YARN, original_max_position_embeddings=2)
    f, _ = scaled_frequencies(128, 1e6)
    s, _ = scaled_frequencies(128, 1e6, few)
    assert torch.allclose(s, f / 4.0, rtol=1e-15, atol=0)
    f, _ = scaled_frequencies(4, 10.0)
    s, _ = scaled_frequencies(4, 10.0, dict(YARN, original_max_position_embeddings=1 << 20))
    assert torch.allclose(s, f, rtol=1e-15, atol=0)


@pytest.mark.parametrize("theta", [1.0, 0.5])
def test_a_table_of_any_base(theta):
    """Unscaled tables of a whole head in halves do not ask for a base above 1; what needs frequencies
    below half a turn does."""
    from sid.kernels.rope import RotaryEmbedding, rope_table
    rope = RotaryEmbedding(64, 50, theta, "cpu")
    assert torch.equal(rope.cos_sin, rope_table(64, 50, theta, "cpu"))
    x = torch.zeros(1, 1, 64)
    with pytest.raises(ValueError, match="theta"):
        rope.rotate(x, x, torch.zeros(1, dtype=torch.int64))
    for more in (dict(rotary_dim=32), dict(interleaved=True), dict(scaling=YARN)):
        with pytest.raises(ValueError, match="theta"):
            RotaryEmbedding(64, 50, theta, "cpu", **more)


def test_checkpoints_that_name_their_scaling_rope_parameters(tmp_path):
    import json

    from sid.model.loader import build_model_config
    hf = dict(model_type="qwen3", num_hidden_layers=2, hidden_size=1024, num_attention_heads=16,
              num_key_value_heads=8, head_dim=128, intermediate_size=2048, vocab_size=1000,
              rms_norm_eps=1e-6, rope_theta=1e6, max_position_embeddings=40960)

    def config(**more):
        (tmp_path / "config.json").write_text(json.dumps(dict(hf, **more)))
        return build_model_config(str(tmp_path), rope_scaling="checkpoint")[0]
    said = dict(YARN, rope_theta=1e6)
    mcfg = config(rope_parameters=said)
    assert mcfg.rope_scaling == said and mcfg.max_position_embeddings == 131072
    mcfg = config(rope_parameters=dict(rope_type="default", rope_theta=1e6), rope_scaling=None)
    assert mcfg.rope_scaling is None and mcfg.max_position_embeddings == 40960
    with pytest.raises(ValueError, match="rope_theta"):
        config(rope_parameters=dict(said, rope_theta=5e6))
