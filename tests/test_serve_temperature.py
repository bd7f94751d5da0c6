"""CPU: temperatures whose reciprocal times log2(e) has no float are refused:
with an infinite scale even equal logits would differ by 0 * inf."""
import math

import pytest

import quantr
from test_serve_args import BAD_ARG, P

SMALLEST = 1.4426950408889634 / 3.4028234e38  # about 4.24e-39


@pytest.mark.parametrize("temperature", [SMALLEST * 0.999, 3e-39])
def test_too_small(temperature):
    assert math.isfinite(1.0 / temperature)
    assert quantr.lib().quantr_logprobs_dev(P, 100, 0, 2, 100, temperature, P, P, None, None, 0, None, None, None, 0,
                                            None) == BAD_ARG
