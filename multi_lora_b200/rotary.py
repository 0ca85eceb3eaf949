"""Rotary positions: queries and keys turned by angles that grow with their position.

The reference leaves them to the model library. Here they are one launch over the packed rows of a step, or ride
on the cache append (:func:`multi_lora_b200.paged_kv.append_paged_kv`). Pair i of a row at position t is turned by
t * f_i radians and multiplied by a factor:

    (a, b) -> factor * (a cos - b sin, b cos + a sin)

:class:`RotaryPositions` keeps the frequencies as whole numbers of 2^-64 turns a position, so that angles of the
frequencies as they are held are exact modulo a turn at every position, however far; no table of cosines bounds the
length. A frequency up to one radian is held to 2^-55 turns a position, what a quotient of doubles leaves.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Mapping, Optional, Sequence

import torch

from multi_lora_b200 import _native


@dataclass
class RotaryPositions:
    """Frequencies of the rotated pairs: what a model keeps, one for all its layers."""

    turns: torch.Tensor        # int64 [pairs] on the device: turns a position, times 2^64, modulo 2^64
    interleaved: bool = False  # pairs are elements (2i, 2i + 1); otherwise (i, i + pairs)
    factor: float = 1.0        # of the rotated elements

    @classmethod
    def from_frequencies(cls, radians: Sequence[float], device: torch.device, *, interleaved: bool = False,
                         factor: float = 1.0) -> "RotaryPositions":
        """From radians a position of each pair, in Python's floats (a model's ``inv_freq.tolist()``)."""
        turns = []
        for f in radians:
            if not math.isfinite(f):
                raise ValueError(f"RotaryPositions: a frequency of {f}")
            whole = int(math.fmod(f / (2 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64
            turns.append(whole - 2 ** 64 if whole >= 2 ** 63 else whole)
        return cls(torch.tensor(turns, dtype=torch.int64, device=device), interleaved, float(factor))

    @classmethod
    def new(cls, rotary_dim: int, device: torch.device, *, base: float = 10000.0, interleaved: bool = False,
            scaling: Optional[Mapping[str, object]] = None,
            max_position_embeddings: Optional[int] = None) -> "RotaryPositions":
        """Pair i of ``rotary_dim // 2`` turns by base^(-2i / rotary_dim) radians a position, changed for long contexts by
        ``scaling``, a model configuration's ``rope_scaling`` of ``rope_type`` (or ``type``) "default", "linear",
        "llama3" or "yarn". ``max_position_embeddings``, the configuration's own, is the trained length where a
        "llama3" or "yarn" scaling has no ``original_max_position_embeddings``."""
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError(f"RotaryPositions: rotary_dim {rotary_dim}: an even number is wanted")
        freqs = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
        freqs, factor = _scaled(freqs, rotary_dim, base, dict(scaling or {}), max_position_embeddings)
        return cls.from_frequencies(freqs, device, interleaved=interleaved, factor=factor)


def _scaled(freqs: List[float], dim: int, base: float, scaling: dict, longest: Optional[int]):
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return freqs, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f"RotaryPositions: unknown rope_type {kind!r}")

    def wanted(name: str, otherwise=None) -> float:
        value = scaling.get(name)
        value = otherwise if value is None else value
        if value is None:
            raise ValueError(f"RotaryPositions: a scaling of rope_type {kind!r} without {name!r}")
        return float(value)

    factor = wanted("factor")
    if kind == "linear":
        return [f / factor for f in freqs], 1.0
    trained = wanted("original_max_position_embeddings", longest)
    if kind == "llama3":
        # by the turns that a pair makes over the trained length: many, left alone; few, slowed down; a blend between
        low, high = wanted("low_freq_factor"), wanted("high_freq_factor")
        keep = [(trained * f / (2 * math.pi) - low) / (high - low) for f in freqs]
        attention = 1.0
    else:
        fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

        def pair_of(turns: float) -> float:  # the pair, as a real number, that makes so many turns over the trained length
            return dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = pair_of(fast), pair_of(slow)
        if scaling.get("truncate", True):
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, dim - 1)
        last += 0.001 if first == last else 0.0
        keep = [1.0 - (i - first) / (last - first) for i in range(len(freqs))]

        def magnitude(weight: float) -> float:
            return 1.0 if factor <= 1.0 else 0.1 * weight * math.log(factor) + 1.0

        attention = scaling.get("attention_factor")
        if attention is None:
            m, every = scaling.get("mscale"), scaling.get("mscale_all_dim")
            attention = magnitude(float(m)) / magnitude(float(every)) if m and every else magnitude(1.0)
    keep = [min(1.0, max(0.0, k)) for k in keep]
    return [k * f + (1.0 - k) * f / factor for k, f in zip(keep, freqs)], float(attention)


def rotate(x: torch.Tensor, positions: torch.Tensor, rotary: RotaryPositions, *,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` [tokens, heads, head_dim] turned by ``positions`` (int32 [tokens]); elements behind the
    ``2 * len(rotary.turns)`` rotated ones are copied.

    Slices of a fused projection are read where they are. ``out`` may be ``x`` itself and does not overlap it
    otherwise. bfloat16, float16 or float32, rounded once; head_dim up to 512. It has no gradient.
    """
    if not x.is_cuda:
        raise RuntimeError("mlora: rotate needs CUDA tensors (no CPU path)")
    return _native.direct("rotate")(x, positions, rotary.turns, rotary.interleaved, rotary.factor, out)
