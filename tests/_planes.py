"""Problems whose results show whether every one of an operand's 24 bits counts (imported by test modules; not
a test), with their bounds.

The gated layer takes a float32 operand as three bf16 planes. Its problems have operands z = 1 + i 2^-14 +-
31 2^-22 (32 <= i < 64): the planes are 1, i 2^-14 and +-31 2^-22. Along the sum, pairs of neighbours have the
same i, opposite last planes and meet factors +1 and -1, so the first two planes cancel and the result, 31 2^-22
for each term, is the third plane's alone: with two planes it is 0. Bound: products of size one at most; an
accumulator step is off by 2^-22 of the largest value in it at most, and a 64-deep block takes 6 x 4 steps, so
24 2^-22 for each 64 terms, 24 / (64 x 31) of the result, and fp32 sums of blocks far below it.

The attention's states take bf16 factors b and weighted values w c as three planes cut at 8 bits each. With random
signs the result's size is that of sqrt(T) terms. Bound of the error's 2-norm, relative to the result's: 8 steps of the
first plane's products, 2^-22 of the running value each, 2^-7 of that for the two other planes' steps, and the two
roundings of each term (of the weight, of its product with c: 2^-24 at most, independent, so relative to the result as
to the term; four standard deviations are below 8 2^-24). Two planes lose 2^-17 of every term on average, all
towards zero, four times the bound.
"""
import numpy as np

BLOCK = 24 * 2.0 ** -22
STATE_BOUND = 8 * 2.0 ** -22 * (1 + 2.0 ** -7) + 8 * 2.0 ** -24

GLU_CASES = [(what, which) for what in ("x", "w", "grad of dx", "w of dx", "x of dw", "grad of dw")
             for which in ("up", "gate")]


def rounded_planes(x, n):
    """x (float64 values of float32) as the sum of n bf16 planes, each rounded to nearest."""
    left, total = x.astype(np.float64), np.zeros_like(x, dtype=np.float64)
    for _ in range(n):
        plane = bf16(left)
        total += plane
        left = left - plane
    return total


def cut_planes(x, n):
    """x as the sum of n bf16 planes, each the leading 8 bits of what is left."""
    left, total = x.astype(np.float32), np.zeros_like(x, dtype=np.float64)
    for _ in range(n):
        plane = (left.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        total += plane
        left = left - plane
    return total


def bf16(x):
    """Rounded to nearest even at 8 bits (normal values)."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 256), e - 8)


def signs(n):
    return np.where(np.arange(n) % 2, -1.0, 1.0)


def last_bits(rng, lead, length):
    """z [lead, length]: pairs along the length with one i and opposite last planes, the first one's sign per row."""
    i = np.repeat(rng.integers(32, 64, (lead, length // 2)), 2, axis=1)
    sigma = rng.choice([-1.0, 1.0], (lead, 1))
    return 1 + i * 2.0 ** -14 + sigma * signs(length) * 31 * 2.0 ** -22, sigma


def glu_problem(what, which, length, seed=0):
    """(x, w_gate, w_up, dh) in float64 (float32 values), activation "none", and what to look at: the index of the
    result among (h, dx, dw_gate, dw_up), a slice of it, its exact value and its bound."""
    rng = np.random.default_rng(seed)
    A, B = 70, 40  # the two axes that are not summed over
    tau = rng.choice([-1.0, 1.0], (1, B))
    z, sigma = last_bits(rng, A, length)
    value = sigma * tau * 31 * 2.0 ** -22 * length
    plain = signs(length)[:, None] * tau  # [length, B]
    bound = BLOCK * -(-length // 64)
    one = {"up": 0, "gate": 1}[which]  # the projection that is 1 everywhere: a last feature of 1s, alone
    if what in ("x", "w"):  # h[m, n] = sum over features
        x = z if what == "x" else plain.T
        w = plain if what == "x" else z.T
        x = np.concatenate([x, np.ones((len(x), 1))], 1)
        w = np.concatenate([w, np.zeros((1, w.shape[1]))])
        ones = np.zeros_like(w)
        ones[-1] = 1
        weights = (ones, w) if one == 0 else (w, ones)
        value = value if what == "x" else value.T
        return (x, *weights, np.ones((len(x), w.shape[1]))), (0, np.s_[:], value, bound)
    if what in ("grad of dx", "w of dx"):  # dx[m, k] = sum over outputs n of dU[m, n] w[k, n]
        dh = z if what == "grad of dx" else plain.T
        w = plain.T if what == "grad of dx" else z
        value = value if what == "grad of dx" else value.T
        x = np.concatenate([rng.choice([-1.0, 1.0], (len(dh), len(w))), np.ones((len(dh), 1))], 1)
        w = np.concatenate([w, np.zeros((1, length))])
        ones = np.zeros_like(w)
        ones[-1] = 1
        weights = (ones, w) if one == 0 else (w, ones)
        return (x, *weights, dh), (1, np.s_[:, :-1], value, bound)
    # dw[k, n] = sum over rows m of x[m, k] dU[m, n]
    x, dh = (z.T, plain) if what == "x of dw" else (plain, z.T)
    value = value if what == "x of dw" else value.T
    x = np.concatenate([x, np.ones((length, 1))], 1)
    w = np.zeros((x.shape[1], dh.shape[1]))
    ones = w.copy()
    ones[-1] = 1
    weights = (ones, w) if one == 0 else (w, ones)
    return (x, *weights, dh), (3 if one == 0 else 2, np.s_[:-1], value, bound)


def glu_of_planes(a, n):
    """(h, dx, dw_gate, dw_up) in float64 with every operand of a product in n planes."""
    x, wg, wu, dh = a
    p = lambda t: rounded_planes(t, n)
    g, u = p(x) @ p(wg), p(x) @ p(wu)
    dg, du = dh * u, dh * g
    return g * u, p(dg) @ p(wg).T + p(du) @ p(wu).T, p(x).T @ p(dg), p(x).T @ p(du)


def state_problem(T, dk, dv, decays, seed=0):
    """(k [T, H, dk] of +-1, v [T, H, dv] in bf16) as float64."""
    rng = np.random.default_rng(seed)
    H = len(decays)
    return rng.choice([-1.0, 1.0], (T, H, dk)), bf16(rng.standard_normal((T, H, dv)))


def weights(T, decays, scale=1.0):
    """[T, H]: what a step's product counts in the state after the last one."""
    return scale * np.exp((T - 1 - np.arange(T))[:, None] * np.asarray(decays, dtype=np.float64))


def state(k, wv):
    return np.einsum("thx,thy->hxy", k, wv)


def state_off(got, want):
    """The error's 2-norm relative to the result's, the largest of the heads."""
    return max(np.linalg.norm(g - w) / np.linalg.norm(w) for g, w in zip(got, want))
