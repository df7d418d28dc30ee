"""The sequence-torso operators where an element's offset passes 2^31: the same bits as on a copy
without gaps (a few GB on the device)."""
import pytest

pytestmark = pytest.mark.gpu

FAR = 2 ** 31 + 64


def far_views(dtype, T=150, H=2, D=64):
    """q, k, v whose second batch row lies FAR elements behind the first, and copies of them."""
    import torch

    g = torch.Generator("cuda").manual_seed(3)
    room = torch.empty(FAR + 3 * T * H * D, dtype=dtype, device="cuda")
    views = [room.as_strided((2, T, H, D), (FAR, 3 * H * D, D, 1), i * H * D) for i in range(3)]
    for v in views:
        v.copy_(torch.randn(2, T, H, D, device="cuda", generator=g))
    return views, [v.contiguous() for v in views]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_attention_and_norms_over_far_rows(dtype):
    import torch

    from boonta_b200.linear_attention import linear_attention, linear_attention_step
    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    far, near = far_views(getattr(torch, dtype))
    ld = torch.tensor([-0.05, -0.5], device="cuda")
    f, pos = rotary_frequencies(64), torch.arange(150, device="cuda")
    s = torch.randn(2, 2, 64, 64, device="cuda")

    def passes(q, k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out, last = linear_attention(*leaves, ld, s)
        grads = torch.autograd.grad((out, last), leaves, (near[0], s))
        step = linear_attention_step(q[:, 7], k[:, 7], v[:, 7], ld, s)
        return [out, last, *grads, *step, *qk_norm_rotary(q, k, None, None, pos, f)]

    for a, b in zip(passes(*far), passes(*near)):
        assert torch.equal(a, b)


def test_gated_layer_of_many_rows():
    import torch

    from boonta_b200.glu import gated_linear_unit

    M, K, N = 4_150_001, 520, 16  # M K is above 2^31
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, K, device="cuda")
    w = torch.randn(K, N, device="cuda").bfloat16()
    h = gated_linear_unit(x, w, w)
    assert torch.equal(h[-300:], gated_linear_unit(x[-300:].clone(), w, w))
    assert not h[:-300].any()
