"""The scaled rotary table against 64 bits, within the bound of the polynomials that compute it."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from test_serving_operators_gpu import E, _lib, _stream, assert_within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,rotary,positions,theta,factor,high", [
    (0, 128, 5000, 1e4, 1.0, 4.0), (1, 34, 333, 1e4, 4.0, 4.0), (2, 128, 8192, 5e5, 8.0, 4.0), (3, 64, 131_072, 1e6, 4.0, 32.0),
    (3, 512, 129, 1e4, 40.0, 32.0), (0, 2, 3_000_000, 1e4, 1.0, 4.0)])
def test_table_within_its_polynomials_bound(cuda, kind, rotary, positions, theta, factor, high):
    """The angle is p times an fp64 frequency in quarter turns, relative error under 2^-50: p 2^-50 turns.
    Its remainder |u| <= 1/2 of a quarter turn is rounded to fp32 (at most 2^-26) and a polynomial evaluated:

                                                         sin                       cos
      rounding of u times the slope                      2^-26 pi/2 = 0.40 e       2^-26 pi/2 0.71 = 0.28 e
      the polynomials with their fp32 constants          3.0e-8     = 0.51 e       6.7e-9          = 0.12 e
      rounding of the result                             2^-25      = 0.50 e       2^-25           = 0.50 e
      of the last inner sum (below 2) times u, u^2       2^-24 / 2  = 0.50 e       2^-24 / 4       = 0.25 e
      of u^2 and the sums further in                     0.11 e                    0.17 e

    2.02 e and 1.32 e in all. The multiplier A is rounded once (e A), the product once (e A)."""
    import torch
    native = _lib()
    s = native.RopeScalingStruct(theta, rotary, kind, factor, 1.0, high, 8192, 0.0)
    f, multiplier = np.zeros(rotary // 2), ctypes.c_double()
    native.check(native.lib.ar_rope_frequencies(ctypes.byref(s), f.ctypes.data, ctypes.byref(multiplier)))
    cos, sin = (torch.empty(positions, rotary // 2, device=cuda) for _ in range(2))
    native.check(native.lib.ar_rope_table_scaled(ctypes.byref(s), positions, cos.data_ptr(), sin.data_ptr(), _stream()))
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=cuda), torch.from_numpy(f).to(cuda))
    a = multiplier.value
    bound = a * (2.05 * E + 2 * E + 2 * math.pi * positions * 2.0 ** -50)
    assert_within(cos, a * angle.cos(), bound, "cos")
    assert_within(sin, a * angle.sin(), bound, "sin")
