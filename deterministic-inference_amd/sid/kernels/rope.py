"""Rotary position embedding: NeoX rotate-half (Qwen3) from a table, applied in place to Q and K, and
from the angles themselves for other layouts, parts of a head and contexts scaled beyond the
trained length.

Table layout follows sid/kernels/rope.py:40-48 of the reference: fp32 [max_pos, D] =
[cos(D/2) | sin(D/2)] with inv_freq = theta^(-i / (D/2)). The table is computed once in
float64 on the device and rounded to fp32.

Scaled frequencies (`scaling`, a model configuration's dict; n = rotary_dim, the angle of pair i at
position p is p f_i):

    rope_type "linear"   f_i = theta^(-2i/n) / factor
    rope_type "ntk"      f_i = (theta factor^(n/(n-2)))^(-2i/n): the last pair's angle is divided
                         by the factor, the first one's is kept
    rope_type "yarn"     f_i = theta^(-2i/n) (r_i / factor + 1 - r_i), r_i going linearly from 0 at
                         the pair that turns beta_fast (32) times within
                         original_max_position_embeddings (rounded down) to 1 at the one that turns
                         beta_slow (1) times (rounded up); cos and sin are multiplied with
                         attention_factor (0.1 ln(factor) + 1)
"""

from __future__ import annotations

import math
from fractions import Fraction

import torch

from sid.kernels.jit import load_ext

ROPE_TYPES = ("default", "linear", "ntk", "yarn")

# What a scaling dict may say, yarn's beside the others'.
_KEYS = ("rope_type", "type", "factor", "original_max_position_embeddings", "rope_theta")
_YARN_KEYS = ("beta_fast", "beta_slow", "attention_factor", "truncate")


def rope_type(scaling: dict | None) -> str:
    """One of ROPE_TYPES: a scaling dict's rope_type (or type). A key that is not read here would
    mean other positions than these, so it is refused unless it is None."""
    scaling = scaling or {}
    if not isinstance(scaling, dict):
        raise ValueError(f"rope scaling must be a dict, got {scaling!r}")
    said = {key: value for key, value in scaling.items() if value is not None}
    kind = said.get("rope_type", said.get("type", "default"))
    if kind not in ROPE_TYPES:
        raise ValueError(f"unknown rope_type {kind!r}: use one of {', '.join(ROPE_TYPES)}")
    if said.get("type", kind) != kind:
        raise ValueError(f"rope_type {kind!r} and type {said['type']!r} disagree")
    if said and "rope_type" not in said and "type" not in said:
        raise ValueError(f"rope scaling names no rope_type: {scaling!r}")
    other = [key for key in said if key not in _KEYS + (_YARN_KEYS if kind == "yarn" else ())]
    if said.get("truncate", True) is not True:
        other.append("truncate other than True")
    if other:
        raise ValueError(f"{kind} rope scaling does not take {', '.join(map(str, other))}")
    return kind


def scaling_number(scaling: dict, key: str, default: float | None = None, least: float = 0.0) -> float:
    """A scaling dict's number above 0, finite and at least `least`; None is the default."""
    value = default if scaling.get(key) is None else scaling[key]
    try:
        x = math.nan if isinstance(value, bool) else float(value)
    except (TypeError, ValueError, OverflowError):
        x = math.nan
    if not (0.0 < x < math.inf and x >= least):
        raise ValueError(f"rope scaling needs a finite {key} "
                         f"{f'of at least {least:g}' if least else 'above 0'}, got {value!r}")
    return x


def scaled_frequencies(rotary_dim: int, theta: float, scaling: dict | None = None) -> tuple:
    """(float64 [rotary_dim / 2] radians a position, the gain of cos and sin) of a scaling dict:
    rope_type (or type), factor, and for yarn original_max_position_embeddings, beta_fast,
    beta_slow, attention_factor; any other key that says something is refused (rope_type)."""
    kind, scaling = rope_type(scaling), dict(scaling or {})
    if not theta > 1.0:
        raise ValueError(f"rope theta must be above 1, got {theta}")
    if scaling.get("rope_theta") not in (None, theta):
        raise ValueError(f"rope scaling's rope_theta {scaling['rope_theta']!r} is not the model's {theta}")
    n = rotary_dim
    at = torch.arange(0, n, 2, dtype=torch.float64) / n
    if kind == "default":
        return theta ** -at, 1.0
    factor = scaling_number(scaling, "factor", least=1.0)
    if kind == "linear":
        return theta ** -at / factor, 1.0
    if kind == "ntk":
        return (theta * factor ** (n / max(n - 2, 1))) ** -at, 1.0
    trained = scaling_number(scaling, "original_max_position_embeddings")
    fast, slow = (scaling_number(scaling, key, x) for key, x in (("beta_fast", 32.0), ("beta_slow", 1.0)))
    if not fast > slow:
        raise ValueError(f"yarn scaling needs beta_fast > beta_slow, got {fast}, {slow}")

    def pair_of(turns: float) -> float:  # the pair that turns that often in the trained positions
        return n * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(theta))

    low, high = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), n - 1)
    ramp = (torch.arange(n // 2, dtype=torch.float64) - low) / (high - low or 0.001)
    ramp = ramp.clamp(0.0, 1.0)
    if high < low:  # no pair is between the two: all turn less than beta_slow times, or none less than beta_fast
        ramp.fill_(1.0 if high < 0 else 0.0)
    gain = scaling_number(scaling, "attention_factor", 0.1 * math.log(factor) + 1.0)
    return theta ** -at * (ramp / factor + (1.0 - ramp)), gain


# 2 pi to 50 digits, for frequencies as fractions of a turn.
_TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937511")


def _turn_fractions(freq: torch.Tensor, device) -> torch.Tensor:
    """int64 [n]: radians a position as 64-bit fractions of a turn (below half a turn)."""
    turns = [round(Fraction(f) / _TWO_PI * (1 << 64)) for f in freq.tolist()]
    return torch.tensor(turns, dtype=torch.int64, device=device)


def _table(freq: torch.Tensor, gain: float, max_positions: int, device) -> torch.Tensor:
    pos = torch.arange(max_positions, dtype=torch.float64, device=device)
    angle = torch.outer(pos, freq)
    table = torch.cat([angle.cos(), angle.sin()], dim=-1)
    return (table if gain == 1.0 else table * gain).to(torch.float32).contiguous()


def rope_table(head_dim: int, max_positions: int, theta: float, device) -> torch.Tensor:
    half = head_dim // 2
    inv_freq = 1.0 / (theta ** (torch.arange(0, half, dtype=torch.float64, device=device) / half))
    return _table(inv_freq, 1.0, max_positions, device)


class RotaryEmbedding:
    """rotary_dim (default: the whole head): only a head's first dims turn; interleaved: the pairs
    are neighbours (2i, 2i + 1), else halves (i, i + rotary_dim / 2); scaling: see
    scaled_frequencies. `cos_sin` is the table of the whole head in halves, which apply and the
    fused kernels (sid.kernels.ops) read; None for other layouts."""

    def __init__(self, head_dim: int, max_positions: int, theta: float, device: str,
                 rotary_dim: int | None = None, interleaved: bool = False,
                 scaling: dict | None = None):
        self.head_dim = head_dim
        self.max_positions = max_positions
        self.rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if not (0 < self.rotary_dim <= head_dim and self.rotary_dim % 2 == 0):
            raise ValueError(f"rotary_dim {rotary_dim} must be even and at most head_dim {head_dim}")
        self.interleaved = bool(interleaved)
        table = self.rotary_dim == head_dim and not self.interleaved
        plain = table and rope_type(scaling) == "default"
        self.gain, self.turns, self.cos_sin = 1.0, None, None
        if theta > 1.0 or not plain:  # (a plain table takes any base)
            freq, self.gain = scaled_frequencies(self.rotary_dim, theta, scaling)
            self.turns = _turn_fractions(freq, device)
        if plain:
            self.cos_sin = rope_table(head_dim, max_positions, theta, device)
        elif table:
            self.cos_sin = _table(freq.to(device), self.gain, max_positions, device)

    def apply(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> None:
        """In place. q: [T, HQ, D] bf16, k: [T, HKV, D] bf16, positions: int64 [T]. A position
        outside [0, max_positions) leaves its token as it is."""
        t, _, head_dim = q.shape
        assert head_dim == self.head_dim and q.is_contiguous() and k.is_contiguous()
        if t == 0:
            return
        if self.cos_sin is not None:
            load_ext().rope_apply(q, k, positions, self.cos_sin)
        else:
            load_ext().rope_rotate(q, k, positions, self.turns, self.gain, self.rotary_dim,
                                   self.interleaved, self.max_positions, q, k)

    def rotate(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> tuple:
        """(q, k) rotated, as new contiguous tensors: apply for tensors that are to be kept or that
        are columns of a projection (any token stride). Its sines and cosines are those of the
        exact angles to fp32's accuracy, apply's with a table that table's: the two can differ by
        the last bf16 rounding."""
        if self.turns is None:
            raise ValueError("rotate needs a rope theta above 1; apply takes any")
        if q.dim() != 3 or q.shape[2] != self.head_dim:
            raise RuntimeError(f"q must be [T, HQ, {self.head_dim}]")
        q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), \
            torch.empty_like(k, memory_format=torch.contiguous_format)
        load_ext().rope_rotate(q, k, positions, self.turns, self.gain, self.rotary_dim,
                               self.interleaved, self.max_positions, q_out, k_out)
        return q_out, k_out
