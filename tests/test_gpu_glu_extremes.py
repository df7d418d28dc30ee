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
