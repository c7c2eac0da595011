"""The yarn table against its definition where the trained context is short."""
import numpy as np
import pytest

import aigpu


@pytest.mark.parametrize("dims", [2, 64, 128])
@pytest.mark.parametrize("original,low,high", [(4.0, 1.0, 32.0), (6.0, 1.0, 2.0), (100.0, 20.0, 40.0), (1.0, 0.5, 1.0)])
def test_pairs_of_few_turns_are_all_divided(dims, original, low, high):
    """original below 2 pi low: no pair makes `low` turns over it, so every one is divided by the factor"""
    got, _ = aigpu.rotary_frequencies(dims, 1e4, "yarn", factor=8.0, original=original, low=low, high=high)
    f = 1e4 ** (-np.arange(dims // 2) * 2.0 / dims)
    assert (original * f / (2 * np.pi) <= low).all()
    assert (np.abs(got - f / 8.0) <= 2.0 ** -24 * f).all()


def test_pairs_of_many_turns_are_all_kept():
    """every pair makes more than `high` turns"""
    got, _ = aigpu.rotary_frequencies(64, 1.5, "yarn", factor=8.0, original=1e6, low=1.0, high=32.0)
    f = 1.5 ** (-np.arange(32) * 2.0 / 64)
    assert (np.abs(got - f) <= 2.0 ** -24 * f).all()
