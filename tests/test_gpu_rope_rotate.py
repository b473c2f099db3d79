"""Rotary positions in every layout (RotaryEmbedding.rotate, and apply where there is no table)
against the formula in 64 bits.

Bound: an output is x cos -+ y sin in fp32, rounded once to bf16 (2^-8 of it). Sine and cosine are
off by at most 2^-22 of the gain (their sums' last terms 2.5e-8, the angle's 24 bits and five
roundings), the two products and their sum by 2^-23 more: 2^-21 gain (|x| + |y|)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)


def _want(x, pos, freq, gain, rotary, interleaved):
    x = x.double().cpu()
    angle = (pos.double().cpu()[:, None] * freq)[:, None]
    c, s = angle.cos() * gain, angle.sin() * gain
    r = x[..., :rotary]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else r.chunk(2, -1)
    z = (a * c - b * s, b * c + a * s)
    mag = a.abs() + b.abs()
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else \
        (lambda u, v: torch.cat([u, v], -1))
    return torch.cat([join(*z), x[..., rotary:]], -1), torch.cat([join(mag, mag), 0 * x[..., rotary:]], -1)


def _near(got, x, pos, freq, gain, rotary, interleaved):
    want, mag = _want(x, pos, freq, gain, rotary, interleaved)
    off = (got.double().cpu() - want).abs()
    bound = want.abs() * 2.0 ** -8 + mag * gain * 2.0 ** -21
    assert (off <= bound).all(), float((off - bound).max())
    assert torch.equal(got[..., rotary:], x[..., rotary:])


def _inputs(t, hq, hkv, d, seed=0, strided=True):
    g = torch.Generator().manual_seed(seed)
    proj = torch.randn(t, hq + 2 * hkv, d, generator=g).to(torch.bfloat16).cuda()
    q, k = proj[:, :hq], proj[:, hq:hq + hkv]
    return (q, k) if strided else (q.contiguous(), k.contiguous())


CASES = [
    # t, hq, hkv, d, rotary, interleaved, scaling
    (1, 16, 8, 128, 128, False, YARN), (1, 16, 8, 128, 128, True, None),
    (7, 16, 8, 128, 64, False, dict(rope_type="linear", factor=2.0)),
    (33, 16, 8, 128, 64, True, dict(rope_type="ntk", factor=4.0)),
    (5, 3, 1, 80, 40, False, None), (5, 3, 1, 80, 38, True, YARN), (4, 2, 2, 80, 2, False, YARN),
    (3, 1, 1, 2, 2, True, None), (9, 4, 4, 256, 250, False, YARN), (2, 2, 1, 1024, 1024, False, YARN),
    (1500, 16, 8, 128, 128, False, None), (1023, 2, 1, 64, 48, True, YARN),
    (2049, 4, 2, 64, 16, False, dict(rope_type="ntk", factor=1.5)), (1024, 1, 1, 1024, 1000, True, None),
]


@pytest.mark.parametrize("t,hq,hkv,d,rotary,interleaved,scaling", CASES)
def test_rotate_matches_formula(t, hq, hkv, d, rotary, interleaved, scaling):
    from sid.kernels.rope import RotaryEmbedding, scaled_frequencies
    print(t, hq, hkv, d, rotary, interleaved, scaling, flush=True)
    limit = 131072 if d * hq < 512 or t < 2000 else 40960
    rope = RotaryEmbedding(d, limit, 1e6, "cuda", rotary_dim=rotary, interleaved=interleaved,
                           scaling=scaling)
    freq, gain = scaled_frequencies(rotary, 1e6, scaling)
    q, k = _inputs(t, hq, hkv, d)
    keep = q.clone()
    g = torch.Generator().manual_seed(t)
    pos = torch.randint(0, limit, (t,), generator=g).cuda()
    pos[0] = limit - 1
    q2, k2 = rope.rotate(q, k, pos)
    assert q2.is_contiguous() and k2.is_contiguous() and torch.equal(q, keep)
    _near(q2, q, pos, freq, gain, rotary, interleaved)
    _near(k2, k, pos, freq, gain, rotary, interleaved)


def test_word_and_element_paths_agree():
    """The same heads at an address that is no multiple of 16 bytes: the same bits."""
    from sid.kernels.rope import RotaryEmbedding
    for interleaved in (False, True):
        rope = RotaryEmbedding(128, 40960, 1e6, "cuda", rotary_dim=96, interleaved=interleaved)
        q, k = _inputs(20, 4, 2, 128, strided=False)
        pos = torch.arange(20, device="cuda") * 1999
        want = rope.rotate(q, k, pos)
        room = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device="cuda")
        odd = room[1:].view_as(q).copy_(q)
        got = rope.rotate(odd, k, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("interleaved", [False, True])
def test_apply_without_a_table_is_rotate_in_place(interleaved):
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(128, 1000, 1e6, "cuda", rotary_dim=64, interleaved=interleaved)
    assert rope.cos_sin is None
    q, k = _inputs(70, 16, 8, 128, strided=False)
    pos = torch.arange(70, device="cuda") * 13
    want = rope.rotate(q, k, pos)
    rope.apply(q, k, pos)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_scaled_table_is_what_apply_and_the_fused_epilogue_read():
    """A whole head in halves, scaled: apply goes by the table, within a rounding of rotate."""
    from sid.kernels.rope import RotaryEmbedding, scaled_frequencies
    rope = RotaryEmbedding(128, 131072, 1e6, "cuda", scaling=YARN)
    q, k = _inputs(90, 16, 8, 128, strided=False)
    pos = torch.randint(0, 131072, (90,), generator=torch.Generator().manual_seed(1)).cuda()
    a, b = q.clone(), k.clone()
    rope.apply(a, b, pos)
    freq, gain = scaled_frequencies(128, 1e6, YARN)
    for got, x in ((a, q), (b, k)):
        _near(got, x, pos, freq, gain, 128, False)


def test_positions_outside_are_copied():
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(64, 100, 1e4, "cuda", rotary_dim=32, scaling=dict(YARN, factor=2.0))
    q, k = _inputs(5, 2, 1, 64)
    pos = torch.tensor([-1, 100, 3, 1 << 40, -(1 << 62)], device="cuda")
    q2, k2 = rope.rotate(q, k, pos)
    at = [0, 1, 3, 4]
    assert torch.equal(q2[at], q[at]) and torch.equal(k2[at], k[at])
    assert not torch.equal(q2[2], q[2])


def test_nothing_special_values_and_refusals():
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(64, 100, 1e4, "cuda", rotary_dim=32)
    q, k = _inputs(3, 2, 1, 64)
    pos = torch.arange(3, device="cuda")
    assert rope.rotate(q[:0], k[:0], pos[:0])[0].shape == (0, 2, 64)
    x = q.clone()
    x[1, 0, 3] = float("inf")
    x[2, 1, 40] = float("nan")
    y = rope.rotate(x, k, pos)[0]
    bad = ~torch.isfinite(y)
    assert bad[1, 0, [3, 19]].all() and bad[2, 1, 40] and int(bad.sum()) == 3
    for args, text in (((q, k[:2], pos), "matching q"), ((q, k, pos[:2]), "T entries"),
                       ((q, k, pos.int()), "positions must be"), ((q.float(), k, pos), "bf16"),
                       ((q.cpu(), k, pos), "GPU"), ((q[..., :32], k, pos), "q must be"),
                       ((q.transpose(1, 2).contiguous().transpose(1, 2), k, pos), "contiguous"),
                       ((q[:1].expand(3, -1, -1), k, pos), "stride")):
        with pytest.raises(RuntimeError, match=text):
            rope.rotate(*args)


def test_rotate_in_a_graph_and_on_another_stream():
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(128, 131072, 1e6, "cuda", interleaved=True, scaling=YARN)
    q, k = _inputs(64, 16, 8, 128)
    pos = torch.randint(0, 131072, (64,), device="cuda")
    want = rope.rotate(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rope.rotate(q, k, pos)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    static = torch.zeros_like(pos)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rope.rotate(q, k, static)
    for i in range(3):
        static.copy_(pos + i)
        graph.replay()
        torch.cuda.synchronize()
        eager = rope.rotate(q, k, pos + i)
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])


@pytest.mark.parametrize("rotary,interleaved", [(64, False), (64, True), (32, False), (6, True)])
def test_positions_outside_keep_every_bit(rotary, interleaved):
    """Infinities, NaNs and zeros of both signs too, out of place and in place, by words and by
    elements."""
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(64, 100, 1e4, "cuda", rotary_dim=rotary, interleaved=interleaved,
                           scaling=dict(YARN, factor=2.0))
    g = torch.Generator().manual_seed(rotary)
    bits = torch.randint(-(1 << 15), 1 << 15, (6, 3, 64), generator=g).to(torch.int16)
    for i, special in enumerate((0x7f80, -0x80, 0x7fc0, -0x3f, -0x8000, 0)):  # inf, -inf, NaNs, -0, 0
        bits[:, :, i::7] = special
    proj = bits.view(torch.bfloat16).cuda()
    q, k = proj[:, :2], proj[:, 2:]
    pos = torch.tensor([-1, 100, 3, 1 << 40, -(1 << 62), 99], device="cuda")
    out = [0, 1, 3, 4]
    for got, x in zip(rope.rotate(q, k, pos), (q, k)):
        assert torch.equal(got[out].view(torch.int16), x[out].contiguous().view(torch.int16))
    a, b = q.contiguous(), k.contiguous()
    rope.apply(a, b, pos)
    for got, x in ((a, q), (b, k)):
        assert torch.equal(got[out].view(torch.int16), x[out].contiguous().view(torch.int16))


@pytest.mark.parametrize("interleaved", [False, True])
def test_small_angles_keep_their_sines(interleaved):
    """Pairs (0, y): out is (-y sin, y cos), to the rounding of bf16 (2^-8) and a few of fp32's, the
    angle's, the sum's and the product's (2^-20), of each value itself."""
    from sid.kernels.rope import RotaryEmbedding, scaled_frequencies
    scaling = dict(rope_type="linear", factor=64.0)
    rope = RotaryEmbedding(128, 131072, 1e6, "cuda", interleaved=interleaved, scaling=scaling)
    freq, _ = scaled_frequencies(128, 1e6, scaling)
    q, k = _inputs(70, 4, 2, 128, strided=False)
    x, y = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 64), slice(64, None))
    q[..., x] = 0.0
    pos = torch.arange(70, device="cuda")
    got = rope.rotate(q, k, pos)[0].double().cpu()
    angle = (pos.double().cpu()[:, None] * freq)[:, None]
    v = q.double().cpu()[..., y]
    for part, want in ((x, -v * angle.sin()), (y, v * angle.cos())):
        over = (got[..., part] - want).abs() - want.abs() * (2.0 ** -8 + 2.0 ** -20)
        assert float(over.max()) <= 0.0


def test_no_tokens_of_q_are_none_of_k():
    from sid.kernels.rope import RotaryEmbedding
    rope = RotaryEmbedding(64, 100, 1e4, "cuda", rotary_dim=32)
    q, k = _inputs(3, 2, 1, 64)
    pos = torch.arange(3, device="cuda")
    for args in ((q[:0], k, pos[:0]), (q[:0], k, pos), (q[:0], k[:0], pos), (q[:0], k[:0].float(), pos[:0])):
        with pytest.raises(RuntimeError):
            rope.rotate(*args)
    none = rope.rotate(q[:0], k[:0], pos[:0])
    assert none[0].shape == (0, 2, 64) and none[1].shape == (0, 1, 64)
