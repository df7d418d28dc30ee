"""The gated feed-forward layer (boonta_b200.glu) against the float64 oracle: sizes off every tile,
single rows, both types, every activation, strided inputs, gradients, streams and graphs.

Bounds. With u the type's rounding, P = |x| |W| the absolute sums of the projections and e = (K + 64)
2^-24 + 2^-18 their relative error (sums of K terms in fp32, which the tensor cores truncate every
few hundred terms; the activations' 2^-20 with them), the gate's slope at most 1.1 and the
activations' second derivative at most 1 (relu: none, away from its border):
  h        u |h| + e (1.1 Pg |U| + (|act| + 1.1 e Pg) Pu)
  dG, dU   rounded once to the type: u |dG| + e-terms as above, then summed in fp32.
relu's border: a gate within its error of 0 may fall on either side, so rows near it are left out by
construction: the test's gates are multiples of 2^-6 in exact arithmetic.
"""
import numpy as np
import pytest

from _sequence import U, numpy64
from oracle import sequence as seq

pytestmark = pytest.mark.gpu

ACTS = ("silu", "tanh", "relu", "none")


def inputs(seed, M, K, N, dtype, act):
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x, wg, wu, dh = r(M, K), r(K, N) * K ** -0.5, r(K, N) * K ** -0.5, r(M, N)
    if act == "relu":  # sums of products of multiples of 1/8: exact in fp32 and any order
        x, wg = (x * 4).round().clamp(-8, 8) / 8, (wg * 8).round().clamp(-8, 8) / 8
    return [t.to(dt) for t in (x, wg, wu, dh)]


def compare(got, a, dtype, act):
    x, wg, wu, dh = (numpy64(t) for t in a)
    M, K = x.shape
    N = wg.shape[1]
    u, f = U[dtype], U["f32"]
    e = (K + 64) * f + 2.0 ** -18
    pg, pu = np.abs(x) @ np.abs(wg), np.abs(x) @ np.abs(wu)
    eg = 0.0 if act == "relu" else e
    A, slope = seq._act(act, x @ wg)
    Uv = np.abs(x @ wu)
    eA = 1.1 * eg * pg + 2.0 ** -20 * np.abs(A)
    h = seq.glu(x, wg, wu, act)

    def near(name, g, want, bound):
        g = numpy64(g)
        assert g.shape == want.shape
        over = np.abs(g - want) - bound
        assert (over <= 0).all(), (name, float(over.max()), np.unravel_index(over.argmax(), over.shape))

    near("h", got[0], h, u * np.abs(h) + (1 + u) * (eA * Uv + (np.abs(A) + eA) * e * pu))
    if len(got) == 1:
        return
    dx, dwg, dwu, dg, du = seq.glu_backward(x, wg, wu, act, dh)
    # errors of the rounded dG and dU, element by element
    eslope = (eg * pg if act in ("silu", "tanh") else 0.0) + 2.0 ** -20
    bg = u * np.abs(dg) + (1 + u) * np.abs(dh) * (eslope * Uv + (np.abs(slope) + eslope) * e * pu)
    bu = u * np.abs(du) + (1 + u) * np.abs(dh) * eA
    for name, g, want, err, size, n in (
            ("dx", got[1], dx, bg @ np.abs(wg).T + bu @ np.abs(wu).T,
             np.abs(dg) @ np.abs(wg).T + np.abs(du) @ np.abs(wu).T, 2 * N),
            ("dwg", got[2], dwg, np.abs(x).T @ bg, np.abs(x).T @ np.abs(dg), M),
            ("dwu", got[3], dwu, np.abs(x).T @ bu, np.abs(x).T @ np.abs(du), M)):
        near(name, g, want, u * np.abs(want) + (1 + u) * (err + ((n + 64) * f + 2.0 ** -18) * size))
        # 2-norm: independent roundings of dG, dU (u) and of the result (u), e for the rest
        bound = (2 * u + 4 * np.sqrt(max(n, K) + 64) * f + 2.0 ** -16) * np.linalg.norm(want) + \
            1e-3 * u * np.linalg.norm(size)
        assert np.linalg.norm(numpy64(g) - want) <= bound, (name, np.linalg.norm(numpy64(g) - want) / np.linalg.norm(want))


def run(a, act, grads=True):
    import torch

    from boonta_b200.glu import gated_linear_unit

    x, wg, wu, dh = a
    if not grads:
        return [gated_linear_unit(x, wg, wu, act)]
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = gated_linear_unit(*leaves, act)
    return [h, *torch.autograd.grad(h, leaves, dh)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (3, 5, 7), (1, 512, 1408), (16, 512, 1408), (8, 64, 64), (17, 72, 200),
                                   (33, 200, 136), (128, 64, 128), (129, 65, 129), (300, 328, 520), (127, 1024, 96),
                                   (640, 256, 1000), (2500, 40, 24)])
def test_sizes(M, K, N, dtype):
    a = inputs(M + N, M, K, N, dtype, "silu")
    compare(run(a, "silu"), a, dtype, "silu")
    compare(run(a, "silu", grads=False), a, dtype, "silu")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [5, 200])
def test_activations(M, act, dtype):
    a = inputs(M, M, 96, 144, dtype, act)
    compare(run(a, act), a, dtype, act)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_long_sum_over_rows(dtype):
    """The weight gradients of many rows, all of one sign (their error grows with the chain)."""
    a = [t.abs() for t in inputs(3, 20000, 64, 72, dtype, "none")]
    compare(run(a, "none"), a, dtype, "none")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_inputs_and_leading_axes(dtype):
    import torch

    from boonta_b200.glu import gated_linear_unit

    x, wg, wu, dh = inputs(5, 60, 64, 96, dtype, "silu")
    wide = torch.zeros(60, 2, 64, dtype=x.dtype, device="cuda")
    wide[:, 1] = x
    want = gated_linear_unit(x, wg, wu)
    assert torch.equal(gated_linear_unit(wide[:, 1], wg.t().contiguous().t(), wu), want)
    both = torch.cat([wg, wu], 1)
    assert torch.equal(gated_linear_unit(x, both[:, :96], both[:, 96:]), want)
    assert torch.equal(gated_linear_unit(x.view(3, 4, 5, 64), wg, wu), want.view(3, 4, 5, 96))
    off = torch.zeros(60 * 64 + 1, dtype=x.dtype, device="cuda")[1:].view(60, 64).copy_(x)
    assert torch.equal(gated_linear_unit(off, wg, wu), want)
    # an expanded gradient, and only one of the gradients wanted
    w = wg.clone().requires_grad_()
    g = torch.autograd.grad(gated_linear_unit(x, w, wu).sum(), w)[0]
    full = torch.autograd.grad(gated_linear_unit(x, w, wu), w, torch.ones_like(dh))[0]
    assert torch.equal(g, full)
    xs = x.clone().requires_grad_()
    assert torch.autograd.grad(gated_linear_unit(xs, wg, wu).sum(), xs)[0].shape == x.shape


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows(dtype):
    import torch

    a = inputs(1, 0, 16, 24, dtype, "silu")
    got = run(a, "silu")
    assert got[0].shape == (0, 24) and got[1].shape == (0, 16)
    assert not got[2].any() and not got[3].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M", [4, 700])
def test_another_stream_and_a_captured_pass_give_the_same_bits(M, dtype):
    import torch

    a = inputs(7, M, 128, 320, dtype, "silu")
    want = [t.detach().clone() for t in run(a, "silu")]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(a, "silu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(a, "silu")
    for t, s in zip(a, inputs(8, M, 128, 320, dtype, "silu")):
        t.copy_(s)
    graph.replay()
    torch.cuda.synchronize()
    compare([t.detach() for t in got], a, dtype, "silu")
