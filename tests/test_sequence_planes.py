"""The problems of tests/_planes.py tell two planes from three (CPU: the planes are formed here)."""
import numpy as np
import pytest

import _planes as pl


@pytest.mark.parametrize("length", [2, 64, 130, 500])
@pytest.mark.parametrize("what,which", pl.GLU_CASES)
def test_two_planes_of_the_gated_layer_are_noticed(what, which, length):
    a, (i, part, value, bound) = pl.glu_problem(what, which, length)
    for t in a:
        assert np.array_equal(t, t.astype(np.float32))
    assert np.abs(pl.glu_of_planes(a, 3)[i][part] - value).max() == 0
    assert np.abs(pl.glu_of_planes(a, 2)[i][part] - value).min() > 2 * bound or length == 2


DECAYS = np.float32([-0.003, -0.02, -0.1, -0.2299, -0.3, -2.0])


@pytest.mark.parametrize("T", [20, 64, 127, 128])
@pytest.mark.parametrize("scale", [1.0, float(np.float32(1 / 3))])
def test_two_planes_of_the_attentions_states_are_noticed(scale, T):
    k, v = pl.state_problem(T, 64, 128, DECAYS)
    w = pl.weights(T, DECAYS, scale)
    want = pl.state(k, w[..., None] * v)
    wv = w.astype(np.float32)[..., None] * v.astype(np.float32)
    three, two = (pl.state(k, pl.cut_planes(wv, n)) for n in (3, 2))
    for h in range(len(DECAYS)):
        assert pl.state_off(three[h:h + 1], want[h:h + 1]) <= pl.STATE_BOUND / 8
        # (a head that forgets at once ends in its last term, whose weight 1 takes one plane)
        assert pl.state_off(two[h:h + 1], want[h:h + 1]) > 1.5 * pl.STATE_BOUND or DECAYS[h] < -1, h
