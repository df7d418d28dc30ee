"""The gated layer (boonta_b200.glu) at the ends of its types' ranges: a gate that is not a number, float32 values
next to the largest, infinities."""
import math

import pytest

pytestmark = pytest.mark.gpu

ACTS = ("silu", "tanh", "relu", "none")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_nan_shows_in_what_it_enters_and_nowhere_else(which, act, dtype):
    """NaN in one element of x, w_gate or w_up: its row (column) of the output is NaN, the rest as it was."""
    import torch

    from boonta_b200.glu import gated_linear_unit

    g = torch.Generator("cuda").manual_seed(1)
    a = [torch.randn(*s, device="cuda", generator=g).to(getattr(torch, dtype)) for s in ((70, 96), (96, 136), (96, 136))]
    clean = gated_linear_unit(*a, act)
    a[which] = a[which].clone()
    a[which][5, 3] = math.nan
    got = gated_linear_unit(*a, act)
    hit = torch.zeros_like(got, dtype=torch.bool)
    if which:
        hit[:, 3] = True
    else:
        hit[5] = True
    assert got[hit].isnan().all()
    assert torch.equal(got[~hit], clean[~hit])


# 2^-20 of the absolute sum: float32 operands keep 24 bits, and a sum of this few terms is off by less than 16
# truncations of 2^-24 (an output here has one large term, the others are below 2^-100 of it)
@pytest.mark.parametrize("where", [0, 1, 2, 3])  # x, w_gate, w_up, dh
def test_float32_values_next_to_the_largest(where):
    import torch

    from boonta_b200.glu import gated_linear_unit

    big = torch.finfo(torch.float32).max
    M, K, N = 40, 24, 48
    g = torch.Generator("cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).sign()
    x, wg, wu, dh = r(M, K), r(K, N) * 2.0 ** -60, r(K, N) * 2.0 ** -60, r(M, N)
    if where == 0:
        x[:, 7] = big * r(M)
    elif where < 3:
        x = x * 2.0 ** -60
        (wg, wu)[where - 1][7] = big * r(N)
        (wu, wg)[where - 1].mul_(2.0 ** 60)
    else:
        dh = big * dh
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    h = gated_linear_unit(*leaves, "none")
    got = [h, *torch.autograd.grad(h, leaves, dh)]
    X, G, U, D = (t.detach().double() for t in (x, wg, wu, dh))
    dg, du = D * (X @ U), D * (X @ G)
    A = lambda t: t.abs()
    want = [(X @ G) * (X @ U), dg @ G.T + du @ U.T, X.T @ dg, X.T @ du]
    size = [(A(X) @ A(G)) * (A(X) @ A(U)), A(D) * (A(X) @ A(U)) @ A(G).T + A(D) * (A(X) @ A(G)) @ A(U).T,
            A(X).T @ (A(D) * (A(X) @ A(U))), A(X).T @ (A(D) * (A(X) @ A(G)))]
    for n, a, b, s in zip(("h", "dx", "dwg", "dwu"), got, want, size):
        fits = s < big  # what leaves the range of float32 may be infinite
        assert fits.any() or n != ("dx", "h", "h", "h")[where], n  # (x = 2^128: h is 2^136)
        over = (a.double() - b).abs() - (2.0 ** -20 * s + 2.0 ** -126)
        assert (over[fits] <= 0).all(), (n, over[fits].max().item())


def test_gradients_next_to_the_largest():
    """dU is as large as dh (a gate of 1), and its product with small weights is not."""
    import torch

    from boonta_b200.glu import gated_linear_unit

    big = torch.finfo(torch.float32).max
    M, K, N = 40, 24, 48
    g = torch.Generator("cuda").manual_seed(4)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).sign()
    x, wu, dh = r(M, K), r(K, N) * 2.0 ** -60, r(M, N) * big
    wg = torch.zeros(K, N, device="cuda")
    wg[0] = 1
    x.requires_grad_()
    dx = torch.autograd.grad(gated_linear_unit(x, wg, wu, "none"), x, dh)[0].double()
    X, G, U, D = (t.detach().double() for t in (x, wg, wu, dh))
    dg, du = D * (X @ U), D * (X @ G)
    want, size = dg @ G.T + du @ U.T, dg.abs() @ G.abs().T + du.abs() @ U.abs().T
    assert (size < big).all()
    assert ((dx - want).abs() <= 2.0 ** -20 * size).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_an_infinity_is_not_lost(bad, dtype):
    import torch

    from boonta_b200.glu import gated_linear_unit

    x = torch.ones(20, 40, device="cuda", dtype=getattr(torch, dtype))
    w = torch.ones(40, 24, device="cuda", dtype=getattr(torch, dtype))
    clean = gated_linear_unit(x, w, w, "none")
    x[4, 9] = bad
    got = gated_linear_unit(x, w, w, "none")
    assert not got[4].isfinite().any()
    keep = torch.arange(20, device="cuda") != 4
    assert torch.equal(got[keep], clean[keep])
