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
