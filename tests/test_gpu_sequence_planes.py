"""Every one of an operand's 24 bits counts in the tensor-core kernels (the problems and bounds: tests/_planes.py;
that they tell two planes from three: tests/test_sequence_planes.py)."""
import numpy as np
import pytest

import _planes as pl
from _sequence import numpy64
from test_sequence_planes import DECAYS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [2, 64, 130, 500, 2000])
@pytest.mark.parametrize("what,which", pl.GLU_CASES)
def test_the_gated_layers_operands_keep_their_bits(what, which, length):
    import torch

    from boonta_b200.glu import gated_linear_unit

    a, (i, part, value, bound) = pl.glu_problem(what, which, length)
    x, wg, wu, dh = (torch.tensor(t, dtype=torch.float32, device="cuda") for t in a)
    leaves = [t.requires_grad_() for t in (x, wg, wu)]
    h = gated_linear_unit(*leaves, "none")
    got = [h, *torch.autograd.grad(h, leaves, dh)][i]
    off = np.abs(numpy64(got)[part] - value).max()
    assert off <= bound, (off / bound, off / np.abs(value).max())


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 128), (128, 64)])
@pytest.mark.parametrize("T", [20, 64, 127, 128])
def test_the_attentions_states_keep_their_bits(T, dk, dv):
    import torch

    from boonta_b200.linear_attention import linear_attention

    k, v = pl.state_problem(T, dk, dv, DECAYS)
    scale = float(np.float32(1 / 3))
    ld = torch.tensor(DECAYS, device="cuda")
    to = lambda t: torch.tensor(t[None], dtype=torch.bfloat16, device="cuda")
    final = linear_attention(to(k), to(k), to(v), ld)[1]
    off = pl.state_off(numpy64(final)[0], pl.state(k, pl.weights(T, DECAYS)[..., None] * v))
    assert off <= pl.STATE_BOUND, off / pl.STATE_BOUND
    # the initial state's gradient: sum of scale e^{(t + 1) g} q_t dout_t^T, the steps taken the other way
    s = torch.zeros(1, len(DECAYS), dk, dv, device="cuda", requires_grad=True)
    out = linear_attention(to(k), to(k), to(v), ld, s, scale=scale)[0]
    got = torch.autograd.grad(out, s, to(v))[0]
    w = pl.weights(T, DECAYS, scale)[::-1] * np.exp(DECAYS.astype(np.float64))
    off = pl.state_off(numpy64(got)[0], pl.state(k, w[..., None] * v))
    assert off <= pl.STATE_BOUND, off / pl.STATE_BOUND
