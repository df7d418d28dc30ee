"""Derivatives of the sequence-torso operators that must not go wrong in silence: a state that acting overwrites
after an unroll has saved it, forward-mode tangents."""
import pytest

pytestmark = pytest.mark.gpu


def problem(dtype="float32"):
    import torch

    g = torch.Generator("cuda").manual_seed(2)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    dt = getattr(torch, dtype)
    return [r(2, 9, 3, 16).to(dt) for _ in range(3)] + [-torch.rand(3, device="cuda", generator=g), r(2, 3, 16, 16)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_step_in_place_on_a_saved_state_is_noticed(dtype):
    import torch

    from boonta_b200.linear_attention import linear_attention, linear_attention_step

    q, k, v, ld, s = problem(dtype)
    x = q.clone().requires_grad_()
    out, _ = linear_attention(x, k, v, ld, s)
    linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, new_state=s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # into another tensor, or after the backward, nothing is lost
    room = torch.empty_like(s)
    out, _ = linear_attention(x, k, v, ld, s)
    before = room._version
    linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, new_state=room)
    assert room._version > before
    out.sum().backward()
    linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, new_state=s)


def test_a_step_in_place_in_inference_mode():
    import torch

    from boonta_b200.linear_attention import linear_attention_step

    q, k, v, ld, s = problem()
    want = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s)[1]
    with torch.inference_mode():
        room = s.clone()
        assert torch.equal(linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, room, new_state=room)[1], want)
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, new_state=s)
    assert torch.equal(s, want)


def test_a_tangent_of_the_outputs_gradient_is_refused():
    """Forward mode over the backward pass: the gradients of the outputs carry the tangent."""
    import torch
    import torch.autograd.forward_ad as fw

    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention
    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    q, k, v, ld, s = problem()
    x = q.clone().requires_grad_()
    rows = q.reshape(-1, 16).clone().requires_grad_()
    w = torch.randn(16, 16, device="cuda")
    pos = torch.arange(9, device="cuda")
    for leaf, y in ((x, linear_attention(x, k, v, ld, s)[0]), (x, linear_attention(x, k, v, ld, s)[1]),
                    (x, qk_norm_rotary(x, k, None, None, pos, rotary_frequencies(16))[0]),
                    (rows, gated_linear_unit(rows, w, w))):
        with fw.dual_level():
            d = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, d, retain_graph=True)
        assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].isfinite().all()
