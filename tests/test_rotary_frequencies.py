"""How exactly frequencies are held, and configurations that lack something (no GPU needed)."""

from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from multi_lora_b200.rotary import RotaryPositions

CPU = torch.device("cpu")
PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923078164, 10 ** 70)


@pytest.mark.parametrize("base", [10000.0, 500000.0, 1e6, 1.5])
def test_frequencies_are_within_2_to_the_minus_55_turns(base):
    """2 pi as a double is off by 2^-54.5 of itself, the quotient by 2^-53, which is 2^-55 of a turn for the 0.16 turns of one
    radian, and less than one whole number is cut off."""
    freqs = [base ** (-i / 64) for i in range(64)]
    held = RotaryPositions.from_frequencies(freqs, CPU).turns.tolist()
    error = [abs(Fraction(t, 2 ** 64) - Fraction(f) / (2 * PI)) for t, f in zip(held, freqs)]
    assert max(error) <= Fraction(1, 2 ** 55) + Fraction(1, 2 ** 64)
    assert abs(PI - Fraction(math.pi)) < Fraction(1, 2 ** 52)


BANDS = {"low_freq_factor": 1.0, "high_freq_factor": 4.0}


@pytest.mark.parametrize("kind, extra", [("yarn", {}), ("llama3", BANDS)])
def test_the_model_s_own_maximum_stands_for_a_trained_length_that_is_missing(kind, extra):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    scaling = {"rope_type": kind, "factor": 8.0, **extra}
    config = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=64, max_position_embeddings=8192,
                         rope_parameters={"rope_theta": 10000.0, **scaling})
    want, factor = ROPE_INIT_FUNCTIONS[kind](config, CPU)
    got = RotaryPositions.new(64, CPU, scaling=scaling, max_position_embeddings=8192)
    assert [t / 2.0 ** 64 * 2 * math.pi for t in got.turns.tolist()] == pytest.approx(want.double().tolist(), rel=2.0 ** -20)
    assert got.factor == pytest.approx(factor, rel=1e-6)
    given = dict(scaling, original_max_position_embeddings=4096)  # comes first
    assert (RotaryPositions.new(64, CPU, scaling=given, max_position_embeddings=8192).turns.tolist()
            == RotaryPositions.new(64, CPU, scaling=given).turns.tolist() != got.turns.tolist())


@pytest.mark.parametrize("scaling, name", [
    ({"rope_type": "linear"}, "factor"), ({"rope_type": "yarn", "original_max_position_embeddings": 64}, "factor"),
    ({"rope_type": "yarn", "factor": 2.0}, "original_max_position_embeddings"),
    ({"type": "llama3", "factor": 2.0, **BANDS}, "original_max_position_embeddings"),
    ({"rope_type": "llama3", "factor": 2.0, "original_max_position_embeddings": 64, "low_freq_factor": 1.0}, "high_freq_factor"),
    ({"rope_type": "llama3", "factor": None, "original_max_position_embeddings": 64, **BANDS}, "'factor'"),
])
def test_what_a_scaling_lacks_is_named(scaling, name):
    with pytest.raises(ValueError, match=name):
        RotaryPositions.new(64, CPU, scaling=scaling)
