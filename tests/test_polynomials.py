"""The kernels' polynomials as they stand in the sources, in 64 bits over the intervals on which they
are used: their errors are no larger than the comments beside them say."""

import re
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parent.parent / "flash_ulysses_b200" / "csrc"
ATTENTION, CACHE = ((CSRC / name).read_text() for name in ("fu_attention.cu", "fu_kvcache.cu"))


def coefficients(text, begin, end):
    """The float literals between two marks, in their order."""
    a = text.index(begin)
    return [float(x) for x in re.findall(r"-?\d+\.\d*(?:e-?\d+)?(?=f\b)",
                                         text[a:text.index(end, a)])]


def horner(x, high_to_low):
    y = np.zeros_like(x)
    for c in high_to_low:
        y = y * x + c
    return y


def tanh_errors(z, odd_low_to_high):
    """Largest relative and absolute error of z (c0 + c1 z^2 + ..) against tanh(z)."""
    got, want = z * horner(z * z, odd_low_to_high[::-1]), np.tanh(z)
    return np.abs(got / want - 1).max(), np.abs(got - want).max()


HALF, ONE = np.linspace(1e-6, 0.5, 400001), np.linspace(1e-6, 1.0, 400001)


def test_power_of_two():
    c = coefficients(ATTENTION, "f32x2 r = fma2(f,", "const float2 n = both(t)")
    assert len(c) == 4
    f = np.linspace(0, 1, 400001)
    off = np.abs(horner(f, c) / 2 ** f - 1).max()
    assert off <= 7.5e-5 <= 2.0 ** -8 / 50            # a fiftieth of a rounding to BF16


def test_short_tanh_of_attention():
    c = coefficients(ATTENTION, "const float cap_low[4]", "const bool cap_small")
    assert len(c) == 3
    relative, absolute = tanh_errors(HALF, [1.0] + c)
    assert relative <= 1.0e-6 and absolute <= 2e-7


def test_long_tanh_of_attention():
    c = coefficients(ATTENTION, "const auto degree_11", "return both(mul2(mul2")
    assert len(c) == 6 and c[-1] == 1.0
    relative, absolute = tanh_errors(ONE, c[::-1])
    assert relative <= 1.2e-6 <= 2.0 ** -19 and absolute <= 7.3e-7


def test_tanh_of_decode():
    c = coefficients(CACHE, "float near = fmaf(u,", "x = fabsf(x) <= LOG2E")
    assert len(c) == 3
    relative, absolute = tanh_errors(HALF, [1.0] + c[::-1])
    assert relative <= 1.0e-6 <= 2.0 ** -19 and absolute <= 2e-7
