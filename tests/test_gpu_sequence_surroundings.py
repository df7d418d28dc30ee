"""What lies around the outputs of linear attention's C entries stays as it was: gradients and outputs
written into views of wider buffers, rows that end off a 16-byte boundary among them, with step counts
that leave the backward walk's earliest chunk before step 0. The bounds of the values are those of
tests/_sequence.py."""
import pytest

from _sequence import check
from test_gpu_linear_attention import NAMES, inputs, oracle, terms

pytestmark = pytest.mark.gpu

GAP = 3.0


def room(t, stride):
    """A buffer of GAP everywhere with a view of t's shape in it: rows `stride` elements apart, two more
    heads, and steps before and behind."""
    import torch

    B, T, H, d = t.shape
    wide = torch.full((B, T + 7, H + 2, stride), GAP, device="cuda", dtype=t.dtype)
    return wide, wide[:, 3:3 + T, 1:1 + H, :d]


@pytest.mark.parametrize("resets", ["none", "some"])
@pytest.mark.parametrize("T", [1, 100, 130, 256, 700])
@pytest.mark.parametrize("dk,dv,stride", [(60, 60, 64), (64, 60, 64), (60, 64, 64), (3, 13, 16), (100, 67, 104),
                                          (64, 64, 64), (128, 128, 128), (64, 64, 72)])
def test_the_gradients_leave_their_surroundings(dk, dv, stride, T, resets):
    import torch

    from boonta_b200 import _lib
    from boonta_b200.linear_attention import _heads, _shape, _workspace

    q, k, v, ld, s, m, dout, dfinal = inputs(T + dk, 2, T, 3, dk, dv, "bf16", resets=resets)
    want, scale = oracle(q, k, v, ld, s, m, dout, dfinal)

    def strided(t):
        wide, view = room(t, stride)
        view.copy_(t)
        return view

    q, k, v, dout = (strided(t) for t in (q, k, v, dout))
    rooms = [room(t, stride) for t in (v, q, k, v)]  # out, dq, dk, dv
    states = [torch.full((8, dk, dv), GAP, device="cuda") for _ in range(2)]
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    shape = _shape(q, v, ld, m, dk ** -0.5)
    for back in (0, 1):
        ws, n = _workspace(shape, back, q.device)
        p = None if ws is None else ws.data_ptr()
        if back:
            _lib.check(lib.bt_linear_attention_backward(
                shape, _heads(q), _heads(k), _heads(v), s.data_ptr(), _heads(dout), dfinal.data_ptr(),
                *[_heads(r[1]) for r in rooms[1:]], states[1][1:7].data_ptr(), p, n, stream))
        else:
            _lib.check(lib.bt_linear_attention(
                shape, _heads(q), _heads(k), _heads(v), s.data_ptr(), _heads(rooms[0][1]),
                states[0][1:7].data_ptr(), p, n, stream))
    got = [rooms[0][1], states[0][1:7].view(2, 3, dk, dv), *[r[1] for r in rooms[1:]],
           states[1][1:7].view(2, 3, dk, dv)]
    for i, (g, w, sc) in enumerate(zip(got, want, scale)):
        check(NAMES[i], g, w, sc, terms(T, dk, dv), "f32" if i in (1, 5) else "bf16", "bf16", tensor_cores=True)
    for i, (wide, view) in enumerate(rooms):
        view.fill_(GAP)
        assert (wide == GAP).all(), ("out", "dq", "dk", "dv")[i]
    for st in states:
        assert (st[0] == GAP).all() and (st[7] == GAP).all()
