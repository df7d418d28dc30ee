"""Bounds of the sequence-torso operators' GPU tests (imported by the test modules; not a test).

Every output is held to two bounds against the float64 oracle. `scale` is the oracle's sum of the
absolute values of the products that enter an element.

* Element by element, rigorous: a rounding to a type is off by at most u = eps / 2 of the value
  (bf16 2^-8, fp32 2^-24). An fp32 sum of n terms is off by at most n 2^-24 of the terms' absolute
  sum (here n counts features, steps and the decay factors' own roundings). A bf16 call may round
  one factor of each product (weighted scores, or the state, as a tensor-core operand) to bf16:
  2^-8 of the absolute sum, and its output once more. What is below fp32's smallest normal number,
  2^-126, may become zero.
* In the 2-norm, for the tests' random inputs: the roundings of different terms are independent, so
  their sum grows with the root of their number: n is replaced by 4 sqrt(n), four standard
  deviations of a sum of n roundings, and the absolute sum by the result's own norm.

Tensor-core sums are kept in fp32 but truncated rather than rounded at each of a chunk's 24 steps
(2^-22 of the running value at most, as the learner's GEMMs measure it): 24 x 2^-22 < 2^-17.
"""
import numpy as np

U = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def numpy64(t):
    return t.detach().double().cpu().numpy()


def check(name, got, want, scale, n, out, operands, tensor_cores=False):
    """got: tensor; want, scale: oracle arrays; n: terms of a sum; out: the output's type;
    operands: the call's type (bf16: one factor of each product may have been rounded)."""
    got = numpy64(got)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert np.isfinite(got).all(), name
    factor = U["bf16"] if operands == "bf16" and out == "bf16" else 0.0
    chain = 2.0 ** -17 if tensor_cores else 0.0
    each = n * U["f32"] + chain + factor
    worst = np.abs(got - want) - (U[out] * np.abs(want) + (1 + U[out]) * each * scale + 2.0 ** -126)
    assert (worst <= 0).all(), (name, float(worst.max()), np.unravel_index(worst.argmax(), worst.shape))
    norm = np.linalg.norm(want)
    both = 4 * np.sqrt(n) * U["f32"] + chain + 2 * factor + U[out]
    # an element's own smallness does not shrink the roundings of the terms that cancel in it
    floor = 1e-3 * both * np.linalg.norm(scale)
    assert np.linalg.norm(got - want) <= both * norm + floor, (name, np.linalg.norm(got - want) / max(norm, 1e-300), both)
