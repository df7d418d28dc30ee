"""The rotation at far positions (boonta_b200.rotary) against phases in exact arithmetic.

Bound: a phase is off by |position| 2^-64 + 2^-32 of a turn and the rounding of a float32 angle within half a
turn (2^-25 of a half turn), a sine or cosine by 2^-23 more; with the norm's own (D + 32) 2^-24 as in
tests/test_gpu_rotary.py, which has room for the last three."""
import math
from fractions import Fraction

import numpy as np
import pytest

from _sequence import U, numpy64

pytestmark = pytest.mark.gpu

BITS = 400


def pi():
    """pi by Machin's formula, to BITS - 10 bits."""
    def arctan_of_inverse(x):
        s, t, n, sign = 0, (1 << BITS) // x, 1, 1
        while t:
            s, t, n, sign = s + sign * (t // n), t // (x * x), n + 2, -sign
        return s
    return Fraction(4 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239)), 1 << BITS)


def phases(pos, freq):
    """pos * freq less whole turns, in (-pi, pi], rounded once."""
    turn = 1 / (2 * pi())
    out = np.empty((len(pos), len(freq)))
    for i, p in enumerate(pos):
        for j, f in enumerate(freq):
            t = int(p) * Fraction(float(f)) * turn
            out[i, j] = 2 * math.pi * float(t - round(t))
    return out


def test_pi():
    assert float(pi()) == math.pi


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D", [8, 64, 80])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_far_positions(base, D, interleaved):
    import torch

    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    half = D // 2
    g = torch.Generator("cuda").manual_seed(D)
    pos = torch.tensor([0, 1, -1, 10 ** 6, -10 ** 6, 2 ** 31 - 1, 2 ** 31 + 12345, 10 ** 10, -10 ** 10, 2 ** 40,
                        2 ** 40 - 977, -2 ** 40 + 1], device="cuda")
    f = rotary_frequencies(D, base)
    f[1::3] *= -1
    f[2::3] *= 37.0
    f[0] = 1e-18  # next to none, of either sign
    f[half - 1] = -1e-18
    x = torch.randn(1, len(pos), 1, D, device="cuda", generator=g)
    y = qk_norm_rotary(x, x, None, None, pos, f, interleaved=interleaved)[0]
    ph = phases(pos.tolist(), f.tolist())
    n = numpy64(x)[0, :, 0]
    n = n / np.sqrt((n * n).mean(-1, keepdims=True) + 1e-6)
    a, b = (n[:, 0::2], n[:, 1::2]) if interleaved else (n[:, :half], n[:, half:])
    want = a * np.cos(ph) - b * np.sin(ph), b * np.cos(ph) + a * np.sin(ph)
    got = numpy64(y)[0, :, 0]
    got = (got[:, 0::2], got[:, 1::2]) if interleaved else (got[:, :half], got[:, half:])
    far = np.abs(pos.cpu().numpy()).astype(float)[:, None] * 2.0 ** -64 * 2 * math.pi
    for u, v in zip(got, want):
        over = np.abs(u - v) - ((D + 32) * U["f32"] + far) * (np.abs(a) + np.abs(b))
        assert (over <= 0).all(), (over.max(), np.unravel_index(over.argmax(), over.shape))
