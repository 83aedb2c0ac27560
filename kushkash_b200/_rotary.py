"""Rotary position plans: the frequencies of Ops.rope(), as turns per position in 64-bit fixed point.

A pair's angle is position * frequency.  The kernel takes it modulo one turn in integers: turns[i] = frequency / (2 pi) *
2^64, and position * turns[i] modulo 2^64 is the fraction of a turn, for any position; so a plan has no table over
positions and no longest position.  Frequencies are worked out in 45 digits: turns[i] is the nearest integer (doubles would be
off by hundreds), so a position's angle is off by at most |position| 2^-65 turns.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from decimal import Context, Decimal, localcontext

import torch

_TWO_PI = Decimal("6.28318530717958647692528676655900576839433879875021")

# keys that every type allows without reading them (rope_theta is compared), and those that each reads
_COMMON_KEYS = {"rope_type", "type", "rope_theta", "original_max_position_embeddings", "finetuned"}
_KEYS = {"default": set(), "linear": {"factor"}, "ntk": {"factor"},
         "yarn": {"factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"},
         "llama3": {"factor", "low_freq_factor", "high_freq_factor"}}


def _yarn_factor(factor: float, scaling: dict) -> float:
    """The factor of the cosines and sines under yarn scaling."""
    def grow(m: float) -> float:
        return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0

    if "attention_factor" in scaling:
        return float(scaling["attention_factor"])
    mscale, all_dim = float(scaling.get("mscale", 0)), float(scaling.get("mscale_all_dim", 0))
    if mscale and all_dim:
        return grow(mscale) / grow(all_dim)
    if all_dim or mscale not in (0.0, 1.0):       # (1 alone is the default's own factor)
        raise ValueError("rotary: mscale and mscale_all_dim go together")
    return grow(1.0)


def _frequencies(r: int, theta: float, scaling: dict | None) -> tuple[list[Decimal], float]:
    """rotary_frequencies() in 45 digits."""
    theta = float(theta)
    if not 0 < theta < math.inf:
        raise ValueError(f"rotary: theta must be positive, got {theta}")
    with localcontext(Context(prec=45)):
        base = Decimal(theta)
        freq = [base ** (Decimal(-2 * i) / r) for i in range(r // 2)]
        return _scaled(freq, r, theta, scaling) if scaling else (freq, 1.0)


def _scaled(freq: list[Decimal], r: int, theta: float, scaling: dict) -> tuple[list[Decimal], float]:
    def number(key: str) -> Decimal:
        return Decimal(float(scaling[key]))

    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in _KEYS:
        raise ValueError(f"rotary: unknown scaling {kind!r} (linear, ntk, yarn, llama3 or default)")
    scaling = {key: value for key, value in scaling.items() if value is not None}
    unread = sorted(set(scaling) - _COMMON_KEYS - _KEYS[kind])
    if unread:
        raise ValueError(f"rotary: {kind} scaling does not know {', '.join(unread)}")
    if float(scaling.get("rope_theta", theta)) != theta:
        raise ValueError(f"rotary: rope_theta {scaling['rope_theta']} of the scaling is not theta {theta}")
    try:
        if kind == "default":
            return freq, 1.0
        factor = number("factor")
        if not 0 < factor < Decimal("inf"):
            raise ValueError(f"rotary: factor must be positive, got {factor}")
        if kind == "linear":
            return [f / factor for f in freq], 1.0
        if kind == "ntk":
            if r <= 2:
                raise ValueError("rotary: ntk scaling needs rotary_dim > 2")
            return [f * factor ** (Decimal(-2 * i) / (r - 2)) for i, f in enumerate(freq)], 1.0
        if kind == "yarn":
            if theta == 1:
                raise ValueError("rotary: yarn scaling needs theta != 1")
            context, turns = number("original_max_position_embeddings"), (scaling.get("beta_fast") or 32, scaling.get("beta_slow") or 1)
            if context <= 0 or min(turns) <= 0:
                raise ValueError(f"rotary: yarn scaling of {context} positions, beta {turns}")
            at = [r * (context / (Decimal(float(beta)) * _TWO_PI)).ln() / (2 * Decimal(theta).ln()) for beta in turns]
            if scaling.get("truncate", True):
                at = [Decimal(math.floor(at[0])), Decimal(math.ceil(at[1]))]
            lo, hi = max(at[0], Decimal(0)), min(at[1], Decimal(r - 1))
            keep = [1 - min(max((i - lo) / max(hi - lo, Decimal("1e-3")), Decimal(0)), Decimal(1)) for i in range(r // 2)]
            return [f / factor * (1 - w) + f * w for f, w in zip(freq, keep)], _yarn_factor(float(factor), scaling)
        context = number("original_max_position_embeddings")                  # llama3
        low, high = number("low_freq_factor"), number("high_freq_factor")
        if high <= low:
            raise ValueError("rotary: high_freq_factor must be above low_freq_factor")
        keep = [min(max((context * f / _TWO_PI - low) / (high - low), Decimal(0)), Decimal(1)) for f in freq]
        return [f / factor * (1 - w) + f * w for f, w in zip(freq, keep)], 1.0
    except KeyError as e:
        raise ValueError(f"rotary: {kind} scaling needs {e.args[0]}") from None


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None) -> tuple[list[float], float]:
    """(radians per position of pair i, factor of the cosines and sines).  Base frequencies theta^(-2i / rotary_dim);
    `scaling` stretches them for contexts longer than the trained one, in the keys model configurations use:
      rope_type "linear"   factor: every frequency divided by it
                "ntk"      factor: theta becomes theta * factor^(r / (r - 2)): the fastest pair unchanged, the slowest / factor
                "yarn"     factor, original_max_position_embeddings [, beta_fast 32, beta_slow 1, truncate True]: pairs that
                           turn more than beta_fast times over the original context kept, those below beta_slow divided
                           by factor, a ramp over the pair's index between (its ends whole indices unless truncate is
                           False); the factor of cosines and sines is attention_factor, or from mscale and mscale_all_dim
                           (0.1 mscale ln(factor) + 1) / (0.1 mscale_all_dim ln(factor) + 1), or 0.1 ln(factor) + 1
                "llama3"   factor, low_freq_factor, high_freq_factor, original_max_position_embeddings: the same with a ramp
                           over the number of turns
                "default"  none
    A key given as None counts as absent; rope_theta has to be theta; a key that the type does not read is refused."""
    freq, factor = _frequencies(rotary_dim, theta, scaling)
    return [float(f) for f in freq], factor


@dataclass(frozen=True)
class Rotary:
    """A plan made by Ops.rotary(): pass it to Ops.rope() of the same head_dim on the same device."""
    head_dim: int
    rotary_dim: int
    interleaved: bool
    factor: float                # of the cosines and sines
    turns: torch.Tensor          # [rotary_dim / 2] int64 (the bits of uint64): turns per position * 2^64


def make_rotary(device: torch.device, head_dim: int, rotary_dim: int | None, theta: float, interleaved: bool,
                scaling: dict | None) -> Rotary:
    r = head_dim if rotary_dim is None else int(rotary_dim)
    if r < 2 or r > head_dim or r % 2:
        raise ValueError(f"rotary: rotary_dim must be even and in [2, {head_dim}], got {rotary_dim}")
    freq, factor = _frequencies(r, float(theta), scaling)
    with localcontext(Context(prec=45)):
        bits = [int((f / _TWO_PI * 2 ** 64).to_integral_value()) % 2 ** 64 for f in freq]
    turns = torch.tensor([b - 2 ** 64 if b >= 2 ** 63 else b for b in bits], dtype=torch.int64, device=device)
    return Rotary(head_dim, r, bool(interleaved), factor, turns)
