"""What the sequence-torso operators refuse, on the host and before any CUDA call (CPU)."""
import ctypes as C

import pytest
import torch

from boonta_b200 import _lib
from boonta_b200.glu import gated_linear_unit
from boonta_b200.linear_attention import linear_attention, linear_attention_step
from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies


def attention_args(**change):
    a = dict(q=torch.zeros(2, 5, 3, 8), k=torch.zeros(2, 5, 3, 8), v=torch.zeros(2, 5, 3, 4),
             log_decay=torch.zeros(3), state=torch.zeros(2, 3, 8, 4),
             reset=torch.zeros(2, 5, dtype=torch.bool))
    return a | change


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "CUDA"),
    ({"k": torch.zeros(2, 5, 3, 9)}, ValueError, "features"),
    ({"k": torch.zeros(2, 5, 1, 8)}, ValueError, "alike"),
    ({"v": torch.zeros(2, 4, 3, 4)}, ValueError, "alike"),
    ({"v": torch.zeros(2, 5, 3, 4, dtype=torch.bfloat16)}, TypeError, "bfloat16"),
    ({"q": torch.zeros(2, 5, 3, 8).half(), "k": torch.zeros(2, 5, 3, 8).half(),
      "v": torch.zeros(2, 5, 3, 4).half()}, TypeError, "float16"),
    ({"v": torch.zeros(2, 5, 3, 129)}, ValueError, "129"),
    ({"log_decay": torch.zeros(2)}, ValueError, "log_decay"),
    ({"log_decay": torch.zeros(3, requires_grad=True)}, ValueError, "no gradient"),
    ({"log_decay": torch.zeros(3, dtype=torch.float64)}, ValueError, "log_decay"),
    ({"state": torch.zeros(2, 3, 4, 8)}, ValueError, "state"),
    ({"state": torch.zeros(2, 3, 8, 4, dtype=torch.bfloat16)}, ValueError, "state"),
    ({"reset": torch.zeros(2, 5)}, ValueError, "reset"),
    ({"reset": torch.zeros(2, 6, dtype=torch.bool)}, ValueError, "reset"),
])
def test_linear_attention_refuses(change, error, match):
    a = attention_args(**change)
    with pytest.raises(error, match=match):
        linear_attention(a["q"], a["k"], a["v"], a["log_decay"], a["state"], a["reset"])


def test_linear_attention_step_refuses():
    q, v, ld, s = torch.zeros(2, 3, 8), torch.zeros(2, 3, 4), torch.zeros(3), torch.zeros(2, 3, 8, 4)
    with pytest.raises(ValueError, match="CUDA"):
        linear_attention_step(q, q, v, ld, s)
    with pytest.raises(ValueError, match="heads"):
        linear_attention_step(q[None], q[None], v[None], ld, s)


def rotary_args(**change):
    a = dict(q=torch.zeros(2, 5, 3, 8), k=torch.zeros(2, 5, 1, 8), wq=torch.ones(8), wk=torch.ones(8),
             pos=torch.zeros(2, 5, dtype=torch.int64), f=torch.ones(4, dtype=torch.float64))
    return list((a | change).values())


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "CUDA"),
    ({"k": torch.zeros(2, 4, 1, 8)}, ValueError, "alike"),
    ({"k": torch.zeros(2, 5, 1, 8, dtype=torch.bfloat16)}, TypeError, "bfloat16"),
    ({"q": torch.zeros(2, 5, 3, 257), "k": torch.zeros(2, 5, 1, 257)}, ValueError, "257"),
    ({"wq": torch.ones(7)}, ValueError, "weights"),
    ({"wk": torch.ones(8, dtype=torch.bfloat16)}, ValueError, "weights"),
    ({"f": torch.ones(5, dtype=torch.float64)}, ValueError, "frequencies"),
    ({"f": torch.ones(4)}, ValueError, "frequencies"),
    ({"pos": torch.zeros(2, 5, dtype=torch.int32)}, ValueError, "positions"),
    ({"pos": torch.zeros(2, dtype=torch.int64)}, ValueError, "positions"),
])
def test_qk_norm_rotary_refuses(change, error, match):
    with pytest.raises(error, match=match):
        qk_norm_rotary(*rotary_args(**change))


def test_rotary_frequencies():
    f = rotary_frequencies(8, 100.0, device="cpu")
    assert f.dtype == torch.float64
    torch.testing.assert_close(f, 100.0 ** (-torch.tensor([0.0, 2, 4, 6], dtype=torch.float64) / 8))
    assert rotary_frequencies(0, device="cpu").shape == (0,)
    with pytest.raises(ValueError, match="even"):
        rotary_frequencies(7, device="cpu")


def test_gated_linear_unit_refuses():
    x, w = torch.zeros(4, 8), torch.zeros(8, 6)
    with pytest.raises(ValueError, match="CUDA"):
        gated_linear_unit(x, w, w)
    with pytest.raises(ValueError, match="activation"):
        gated_linear_unit(x, w, w, "gelu")
    with pytest.raises(ValueError, match="expected"):
        gated_linear_unit(x, w, torch.zeros(8, 5))
    with pytest.raises(ValueError, match="expected"):
        gated_linear_unit(torch.zeros(4, 7), w, w)
    with pytest.raises(TypeError, match="float16"):
        gated_linear_unit(x.half(), w.half(), w.half())
    with pytest.raises(TypeError, match="bfloat16"):
        gated_linear_unit(x, w.bfloat16(), w.bfloat16())
    with pytest.raises(ValueError, match="without"):
        gated_linear_unit(x, torch.zeros(8, 0), torch.zeros(8, 0))


def test_the_c_entries_refuse_before_any_cuda_call():
    lib, h = _lib.lib(), _lib.Heads()
    shape = _lib.LinearAttentionShape(2, 5, 3, 129, 4, 0, 1.0, 256, None, 0, 0)
    assert lib.bt_linear_attention_workspace(C.byref(shape), 0) == -1
    assert b"129" in lib.bt_last_error()
    shape.key_dim = 8
    assert lib.bt_linear_attention(C.byref(shape), h, h, h, None, h, None, None, 0, None) == _lib.BT_ERR_INVALID
    assert b"null" in lib.bt_last_error()
    shape.dtype = 5
    assert lib.bt_linear_attention_workspace(C.byref(shape), 1) == -1
    shape.dtype = 0
    one = _lib.Heads(256, 0, 0, 0)
    assert lib.bt_linear_attention_step(C.byref(shape), one, one, one, 256, 256, 256, None) == _lib.BT_ERR_INVALID
    assert b"steps" in lib.bt_last_error()
    # a long sequence is split, and the splits need their workspace
    shape = _lib.LinearAttentionShape(1, 4096, 1, 64, 64, 0, 1.0, 256, None, 0, 0)
    assert lib.bt_linear_attention_workspace(C.byref(shape), 0) > 0
    assert lib.bt_linear_attention(C.byref(shape), one, one, one, None, one, 256, None, 0, None) == _lib.BT_ERR_INVALID
    assert b"workspace" in lib.bt_last_error()
    rot = _lib.QkNormRotaryShape(2, 5, 3, 1, 8, 5, 0, 0, 0, 1e-6, 256, 0, 0, 256)
    assert lib.bt_qk_norm_rotary(C.byref(rot), one, one, None, None, one, one, None) == _lib.BT_ERR_INVALID
    assert b"frequencies" in lib.bt_last_error()
    rot.half = 4
    assert lib.bt_qk_norm_rotary(C.byref(rot), h, one, None, None, one, one, None) == _lib.BT_ERR_INVALID
    assert lib.bt_qk_norm_rotary_backward(C.byref(rot), one, one, None, None, one, one, one, one, None,
                                          None, None, 0, None) == _lib.BT_ERR_INVALID
    assert b"workspace" in lib.bt_last_error()
    glu = _lib.GluShape(4, 8, 6, 0, 9)
    assert lib.bt_glu(C.byref(glu), 256, 256, 256, 256, None, 0, None) == _lib.BT_ERR_INVALID
    assert b"activation" in lib.bt_last_error()
    glu.activation = 1
    assert lib.bt_glu(C.byref(glu), None, 256, 256, 256, None, 0, None) == _lib.BT_ERR_INVALID
    assert lib.bt_glu_backward(C.byref(glu), 256, 256, 256, 256, None, 256, None, 256, 1 << 30, None) == _lib.BT_ERR_INVALID
    assert b"dw_" in lib.bt_last_error()
    assert lib.bt_glu_backward(C.byref(glu), 256, 256, 256, 256, 256, 256, 256, None, 0, None) == _lib.BT_ERR_INVALID
    assert b"workspace" in lib.bt_last_error()


@pytest.mark.parametrize("which", ["q", "k", "v", "log_decay", "state"])
def test_linear_attention_refuses_forward_mode_tangents(which):
    """A dual tensor does not require a gradient: its tangent would be dropped without a word."""
    import torch.autograd.forward_ad as fw

    a = attention_args(reset=None)
    one = {n: a[n][:, 0] for n in ("q", "k", "v")} | {"log_decay": a["log_decay"], "state": a["state"]}
    with fw.dual_level():
        a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
        one[which] = fw.make_dual(one[which], torch.ones_like(one[which]))
        for context in (torch.enable_grad, torch.no_grad):
            with context(), pytest.raises(NotImplementedError, match="linear_attention: .*forward"):
                linear_attention(**a)
            with context(), pytest.raises(NotImplementedError, match="linear_attention_step: .*forward"):
                linear_attention_step(**one)
    with fw.dual_level():  # no tangent, no refusal
        with pytest.raises(ValueError, match="CUDA"):
            linear_attention(**attention_args())


@pytest.mark.parametrize("which", range(4))
def test_qk_norm_rotary_refuses_forward_mode_tangents(which):
    import torch.autograd.forward_ad as fw

    a = rotary_args()
    with fw.dual_level():
        a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(NotImplementedError, match="qk_norm_rotary: .*forward"):
            qk_norm_rotary(*a)
        a = rotary_args()
        a[5] = fw.make_dual(a[5], torch.ones_like(a[5]))
        with pytest.raises(NotImplementedError, match="forward"):
            qk_norm_rotary(*a)


@pytest.mark.parametrize("which", range(3))
def test_gated_linear_unit_refuses_forward_mode_tangents(which):
    import torch.autograd.forward_ad as fw

    a = [torch.zeros(4, 8), torch.zeros(8, 6), torch.zeros(8, 6)]
    with fw.dual_level():
        a[which] = fw.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises(NotImplementedError, match="gated_linear_unit: .*forward"):
            gated_linear_unit(*a)


def meta(*shape, dtype=torch.float32):
    """A tensor of any size without memory."""
    return torch.empty(shape, dtype=dtype, device="meta")


FAR = 2 ** 32 + 3  # the C entries' sizes are 32-bit: this one would arrive as 3


@pytest.mark.parametrize("shape", [(FAR, 2, 1, 1), (1, FAR, 1, 1), (1, 2, FAR, 1), (2 ** 31, 1, 1, 1)])
def test_sizes_beyond_32_bits_are_refused(shape):
    x = meta(*shape)
    with pytest.raises(ValueError, match="linear_attention: .*sizes"):
        linear_attention(x, x, x, meta(shape[2]))
    one = meta(shape[0], shape[2], 1)
    if shape[1] < 3:
        with pytest.raises(ValueError, match="linear_attention_step: .*sizes"):
            linear_attention_step(one, one, one, meta(shape[2]), meta(shape[0], shape[2], 1, 1))
    with pytest.raises(ValueError, match="qk_norm_rotary: .*sizes"):
        qk_norm_rotary(x, meta(*shape[:2], 1, 1), None, None, meta(*shape[:2], dtype=torch.int64),
                       meta(0, dtype=torch.float64))
    with pytest.raises(ValueError, match="qk_norm_rotary: .*sizes"):
        qk_norm_rotary(meta(*shape[:2], 1, 1), x, None, None, meta(*shape[:2], dtype=torch.int64),
                       meta(0, dtype=torch.float64))


@pytest.mark.parametrize("x,w", [((FAR, 1), (1, 4)), ((2 ** 16, 2 ** 16 + 1, 4), (4, 4)), ((2, FAR), (FAR, 1)),
                                 ((2, 1), (1, FAR))])
def test_a_gated_layer_beyond_32_bits_is_refused(x, w):
    with pytest.raises(ValueError, match="gated_linear_unit: .*sizes"):
        gated_linear_unit(meta(*x), meta(*w), meta(*w))


def test_steps_next_to_2_31_are_refused_where_a_chunks_end_would_pass_it():
    lib = _lib.lib()
    shape = _lib.LinearAttentionShape(1, 2 ** 31 - 1, 1, 1, 1, 0, 1.0, 256, None, 0, 0)
    assert lib.bt_linear_attention_workspace(C.byref(shape), 0) == -1
    assert b"steps" in lib.bt_last_error()
    shape.steps = 2 ** 30
    assert lib.bt_linear_attention_workspace(C.byref(shape), 0) >= 0


def test_frequencies_that_want_a_gradient_are_refused():
    """They are constants, as log_decay is: a gradient would be missing without a word."""
    a = rotary_args()
    a[5] = a[5].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        qk_norm_rotary(*a)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        qk_norm_rotary(*a)
