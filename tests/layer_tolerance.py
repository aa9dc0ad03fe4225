"""Tolerances of the layer operators' GPU tests, counted in roundings.

``U`` is half a step of float32 and ``half(dtype)`` half a step of the result's type, both relative to the value.
A sum of n terms in float32 is off by at most n U times the sum of the terms' magnitudes; a kernel's longest chain
of additions is far below the constants used here only by the counts named at each use.
"""

import numpy as np
import torch

U = 2.0**-24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance of subnormals: what a rounding of a tiny value may be off by, absolutely."""

    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def assert_within(got, want, bound, what):
    """|got - want| <= bound, elementwise; bound is an array or a number."""

    got = f64(got)
    assert got.shape == want.shape, f"{what}: shape {got.shape}, expected {want.shape}"
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN at other places"
    over = np.abs(got - want) - bound
    worst = np.nanmax(over) if over.size else 0.0
    assert worst <= 0, f"{what}: {int((over > 0).sum())} values out of bounds, by up to {worst:.3g}"
