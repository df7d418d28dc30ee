"""The float64 oracle of the sequence-torso operators (oracle/sequence.py): its gradients against
central differences, and its recurrence against the closed form (CPU)."""
import numpy as np
import pytest

from oracle import sequence as seq

# central differences of a function that is smooth over the step: truncation ~ h^2, rounding
# ~ 2^-53 / h times the value; h = 1e-5 leaves about 1e-9 of values of order 10
H, TOL = 1e-5, 1e-6


def differences(f, x, dy):
    """d sum(f(x) * dy) / dx for every element of x."""
    g = np.empty(x.shape)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += H
        down[i] -= H
        g[i] = sum(((a - b) * d).sum() for a, b, d in zip(f(up), f(down), dy)) / (2 * H)
    return g


def problem(seed, resets):
    r = np.random.default_rng(seed)
    B, T, N, dk, dv = 2, 4, 2, 3, 2
    x = [r.standard_normal(s) for s in ((B, T, N, dk), (B, T, N, dk), (B, T, N, dv), (B, N, dk, dv))]
    reset = None if not resets else r.random((B, T)) < 0.4
    dy = r.standard_normal((B, T, N, dv)), r.standard_normal((B, N, dk, dv))
    return x, np.log([0.9, 0.5]), reset, dy


@pytest.mark.parametrize("resets", [False, True])
def test_linear_attention_gradients_are_its_differences(resets):
    x, ld, reset, dy = problem(3, resets)
    q, k, v, s = x
    got = seq.linear_attention_backward(q, k, v, ld, s, reset, 0.7, *dy)
    for i in range(4):
        f = lambda z, i=i: seq.linear_attention(*[z if j == i else x[j] for j in range(3)], ld,
                                                z if i == 3 else s, reset, 0.7)
        np.testing.assert_allclose(got[i], differences(f, x[i], dy), atol=TOL)


def test_linear_attention_is_the_sum_over_pairs_within_a_segment():
    (q, k, v, s), ld, reset, _ = problem(5, True)
    out, final = seq.linear_attention(q, k, v, ld, s, reset, 0.7)
    B, T, N, _ = q.shape
    seg = np.cumsum(reset, 1)
    for b in range(B):
        for n in range(N):
            for t in range(T):
                o = sum(np.exp((t - j) * ld[n]) * (q[b, t, n] @ k[b, j, n]) * v[b, j, n]
                        for j in range(t + 1) if seg[b, j] == seg[b, t])
                if seg[b, t] == 0:
                    o = o + np.exp((t + 1) * ld[n]) * q[b, t, n] @ s[b, n]
                np.testing.assert_allclose(out[b, t, n], 0.7 * o, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rotary_gradients_are_its_differences(interleaved):
    r = np.random.default_rng(7)
    x, w = r.standard_normal((2, 3, 2, 6)), 1 + 0.3 * r.standard_normal(6)
    pos, f = r.integers(0, 50, (2, 3)), np.array([1.0, 0.1])
    dy = r.standard_normal(x.shape)
    dx, dw = seq.norm_rotary_backward(x, w, pos, f, 1e-3, interleaved, dy)
    np.testing.assert_allclose(
        dx, differences(lambda z: (seq.norm_rotary(z, w, pos, f, 1e-3, interleaved),), x, (dy,)), atol=TOL)
    np.testing.assert_allclose(
        dw, differences(lambda z: (seq.norm_rotary(x, z, pos, f, 1e-3, interleaved),), w, (dy,)), atol=TOL)


@pytest.mark.parametrize("act", ["silu", "tanh", "relu", "none"])
def test_glu_gradients_are_its_differences(act):
    r = np.random.default_rng(11)
    x = [r.standard_normal(s) for s in ((4, 3), (3, 5), (3, 5))]
    dh = r.standard_normal((4, 5))
    got = seq.glu_backward(*x, act, dh)
    for i in range(3):
        f = lambda z, i=i: (seq.glu(*[z if j == i else x[j] for j in range(3)], act),)
        np.testing.assert_allclose(got[i], differences(f, x[i], (dh,)), atol=TOL)
