"""What a reset hides stays hidden whatever it holds (boonta_b200.linear_attention): NaN and infinities in one
episode of an unroll leave the outputs, gradients and states of every other episode as they are, bit for bit,
on the tensor cores (bfloat16 heads of a multiple of 8 features) as on the CUDA cores."""
import math

import pytest

from test_gpu_linear_attention import NAMES, inputs, run

pytestmark = pytest.mark.gpu

# T 1111 with two sequences is split along the steps
CASES = [(2, 300, 2, 64, 64), (2, 300, 2, 128, 128), (3, 130, 3, 48, 72), (1, 1111, 2, 64, 128), (2, 100, 2, 20, 12)]


def problem(B, T, H, dk, dv, dtype, decay):
    import torch

    a = list(inputs(T + dk, B, T, H, dk, dv, dtype, resets="none"))
    a[3] = torch.full((H,), decay, device="cuda")
    a[5] = torch.zeros(B, T, dtype=torch.bool, device="cuda")
    # episodes that begin inside a chunk, one step after another, and at a chunk's edge
    for t in (40, 75, 76, 99, 128, 250, 600, 1000):
        if t < T:
            a[5][:, t] = True
    return a


def episodes(reset):
    return reset.int().cumsum(1)


@pytest.mark.parametrize("decay", [-0.02, -0.9])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", [0, 1, 2, 6])  # q, k, v, the outputs' gradient
@pytest.mark.parametrize("B,T,H,dk,dv", CASES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_episode_does_not_reach_another(dtype, B, T, H, dk, dv, where, bad, decay):
    import torch

    a = problem(B, T, H, dk, dv, dtype, decay)
    clean = run(a)
    ep = episodes(a[5])
    last = int(ep.max())
    for t in (7, 39, 80, 127, 249):
        if t >= T - 1:
            continue
        b = list(a)
        b[where] = a[where].clone()
        b[where][0, t, 0, 3] = bad
        got = run(b)
        others = (ep != ep[0, t])
        others[1:] = True
        for i, (g, c) in enumerate(zip(got, clean)):
            if i in (1, 5):  # the final state: of the last episode; its gradient: of the first
                if int(ep[0, t]) != (last if i == 1 else 0):
                    assert torch.equal(g, c), (NAMES[i], t)
            else:
                assert torch.equal(g[others], c[others]), (NAMES[i], t)
                assert torch.equal(g[:, :, 1:], c[:, :, 1:]), (NAMES[i], t)
        # and it is not lost either: the step itself shows it
        shown = {0: 0, 1: 0, 2: 0, 6: 2}[where]
        assert not got[shown][0, t, 0].isfinite().all(), t


@pytest.mark.parametrize("decay", [-0.02, -0.9])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_column_that_is_not_finite_reaches_later_steps_of_its_episode_only(dtype, decay):
    """In a chunk with a cut a value of v shows in its own column, from its own step to its episode's end."""
    import torch

    a = problem(2, 128, 2, 64, 64, dtype, decay)
    clean = run(a, grads=False)
    b = list(a)
    b[2] = a[2].clone()
    b[2][1, 20, 1, 5] = math.nan
    b[2][1, 110, 0, 63] = math.inf
    got = run(b, grads=False)
    hit = torch.zeros_like(clean[0], dtype=torch.bool)
    hit[1, 20:40, 1, 5] = True
    hit[1, 110:, 0, 63] = True
    assert not got[0][hit].isfinite().any()
    assert torch.equal(got[0][~hit], clean[0][~hit])
    state = torch.zeros_like(clean[1], dtype=torch.bool)
    state[1, 0, :, 63] = True
    assert not got[1][state].isfinite().any()
    assert torch.equal(got[1][~state], clean[1][~state])


@pytest.mark.parametrize("B,T,H,dk,dv", CASES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_given_states_end_with_their_episode(dtype, B, T, H, dk, dv):
    import torch

    a = problem(B, T, H, dk, dv, dtype, -0.02)
    clean = run(a)
    ep = episodes(a[5])
    b = list(a)
    b[4] = torch.full_like(a[4], math.nan)
    b[7] = torch.full_like(a[7], math.inf)
    got = run(b)
    inner = (ep != 0) & (ep != ep[:, -1:])
    for i in (0, 2, 3, 4):
        assert torch.equal(got[i][inner], clean[i][inner]), NAMES[i]
    assert torch.equal(got[0][ep != 0], clean[0][ep != 0]) and torch.equal(got[1], clean[1])
    assert torch.equal(got[5], clean[5])
