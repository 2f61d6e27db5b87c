"""What the paged write's norm rests on (runs without a GPU)."""

from __future__ import annotations

import numpy as np


def test_no_reciprocal_square_root_of_an_fp32_number_is_near_a_rounding_boundary():
    """The dense cache's kernel takes 1 / sqrt(t) in fp64 (a root and a division, each correctly rounded: 2^-52 in
    all), the paged write CUDA's fp64 rsqrt (1 ulp: 2^-52 at most); both round to fp32. They agree for every fp32
    t if no 1 / sqrt(t) comes within 2^-52 of the middle of two fp32 numbers. Powers of 4 scale t exactly and no result is
    subnormal, so t in [1, 4) is all of it; 2^-60 is what 64 bits leave in this check."""
    for base in (1.0, 2.0):
        t = (1 + np.arange(2**23) * 2.0**-23) * base
        y = 1 / np.sqrt(t.astype(np.longdouble)) * np.longdouble(2.0**24)  # in (2^23, 2^24]: fp32's step is 1
        away = np.abs(y - np.floor(y) - np.longdouble(0.5)) / y
        assert np.finfo(np.longdouble).nmant >= 63 and float(away.min()) > 2.0**-52 + 2.0**-60
