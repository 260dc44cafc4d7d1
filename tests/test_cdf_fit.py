"""The polynomial behind gelu's 8-bit kernels (csrc/act8.hip) against the normal distribution in 64 bits, without a GPU."""
import os
import re

import numpy as np
import pytest
import torch

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "transcodon_amd", "csrc", "act8.hip")


def _source():
    text = open(SOURCE).read()
    body = text[text.index("float normal_cdf("):]
    body = body[:body.index("\n}")]
    first = float(re.search(r"float q = ([-0-9.e]+)f;", body).group(1))
    rest = [float(c) for c in re.findall(r"q = fmaf\(q, t, ([-0-9.e]+)f\);", body)]
    slope = float(re.search(r"fmaf\(a, ([0-9.]+)f, 1\.0f\)", body).group(1))
    stated = float(re.search(r"least relative error \(([0-9.e-]+)\)", text).group(1))
    return [first, *rest], slope, stated


def test_relative_error_of_the_fit_is_the_stated_one():
    """Coefficients as the kernel holds them (f32), arithmetic in 64 bits; a in [0, 14]."""
    coefficients, slope, stated = _source()
    assert len(coefficients) == 8
    a = torch.linspace(0, 14, 400001, dtype=torch.float64)
    t = 1 / (1 + float(np.float32(slope)) * a)
    p = torch.zeros_like(a)
    for c in coefficients:
        p = p * t + float(np.float32(c))
    # exp(a^2 / 2) Phi(-a)
    want = 0.5 * torch.special.erfcx(a * 0.5 ** 0.5)
    worst = float((p * t / want - 1).abs().max())
    assert worst <= stated, (worst, stated)
    # and what the tolerance of the GPU tests leaves for it: 32 C in all, of which evaluation, reciprocal and exponential take 28
    assert worst <= 4 * 2.0 ** -24
    assert stated == pytest.approx(worst, rel=0.05)               # not a loose upper bound either
