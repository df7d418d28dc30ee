"""The sequence-torso operators used together, as one residual block of a recurrent policy: the
projections' heads normed and rotated, linear attention over the unroll, the gated layer; its
gradients against the float64 definition through torch's autograd, and acting step by step."""
import pytest

pytestmark = pytest.mark.gpu

D, H, F = 64, 4, 96


def weights(dtype, seed=0):
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: (torch.randn(*s, device="cuda", generator=g) * s[0] ** -0.5).to(dtype)
    return {"qkv": r(D, 3 * D), "wq": torch.ones(D // H, device="cuda", dtype=dtype),
            "wk": torch.ones(D // H, device="cuda", dtype=dtype), "gate": r(D, F), "up": r(D, F), "down": r(F, D)}


def block(p, x, ld, state, reset, pos, freq):
    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention
    from boonta_b200.rotary import qk_norm_rotary

    q, k, v = (t.unflatten(-1, (H, D // H)) for t in (x @ p["qkv"]).split(D, -1))
    q, k = qk_norm_rotary(q, k, p["wq"], p["wk"], pos, freq)
    o, state = linear_attention(q, k, v, ld, state, reset)
    x = x + o.flatten(-2)
    return x + gated_linear_unit(x, p["gate"], p["up"]) @ p["down"], state


def plain(p, x, ld, state, reset, pos, freq):
    """The same in float64 torch operations, step by step."""
    import torch

    q, k, v = (t.unflatten(-1, (H, D // H)) for t in (x @ p["qkv"]).split(D, -1))
    ang = pos[..., None].double() * freq
    turn = torch.polar(torch.ones_like(ang), ang)[:, :, None]

    def norm(y, w):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = y.chunk(2, -1)
        z = torch.complex(a, b) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k = norm(q, p["wq"]), norm(k, p["wk"])
    outs = []
    for t in range(x.shape[1]):
        keep = (~reset[:, t])[:, None, None, None] * torch.exp(ld)[:, None, None]
        state = keep * state + k[:, t, :, :, None] * v[:, t, :, None, :]
        outs.append((q[:, t, :, None] @ state)[:, :, 0] * (D // H) ** -0.5)
    x = x + torch.stack(outs, 1).flatten(-2)
    return x + (torch.nn.functional.silu(x @ p["gate"]) * (x @ p["up"])) @ p["down"], state


def problem(dtype, B=3, T=90):
    import torch

    from boonta_b200.rotary import rotary_frequencies

    g = torch.Generator("cuda").manual_seed(5)
    reset = torch.rand(B, T, device="cuda", generator=g) < 0.05
    t = torch.arange(T, device="cuda")
    start = torch.where(reset, t, 0).cummax(1).values
    return (torch.randn(B, T, D, device="cuda", generator=g).to(dtype),
            torch.log1p(-torch.exp2(-torch.linspace(2, 6, H, device="cuda"))),
            torch.randn(B, H, D // H, D // H, device="cuda", generator=g), reset, t - start,
            rotary_frequencies(D // H))


# float32: the block's 5 products of at most 192 terms in a row, each within 200 2^-24 of its terms'
# absolute sum (about 10 times the result): 1e-4 of the result's norm; bf16: about 12 roundings of
# 2^-8 that add as independent errors, and the products' operands: 12 x 2^-8 at most
@pytest.mark.parametrize("dtype,bound", [("float32", 1e-4), ("bfloat16", 12 * 2.0 ** -8)])
def test_a_block_and_its_gradients(dtype, bound):
    import torch

    dt = getattr(torch, dtype)
    x, ld, s, reset, pos, freq = problem(dt)
    p = weights(dt)
    leaves = {n: w.clone().requires_grad_() for n, w in p.items()}
    xs, ss = x.clone().requires_grad_(), s.clone().requires_grad_()
    y, last = block(leaves, xs, ld, ss, reset, pos, freq)
    want_leaves = {n: w.double().requires_grad_() for n, w in p.items()}
    wx, ws = x.double().requires_grad_(), s.double().requires_grad_()
    wy, wlast = plain(want_leaves, wx, ld.double(), ws, reset, pos, freq)
    dy, dl = torch.randn_like(y), torch.randn_like(last)
    got = torch.autograd.grad((y, last), [xs, ss, *leaves.values()], (dy, dl))
    want = torch.autograd.grad((wy, wlast), [wx, ws, *want_leaves.values()], (dy.double(), dl.double()))
    for n, a, b in zip(["y", "last", "x", "state", *p], (y, last, *got), (wy, wlast, *want)):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= bound, (n, off)


def test_acting_follows_the_unroll():
    import torch

    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention_step
    from boonta_b200.rotary import qk_norm_rotary

    x, ld, s, reset, pos, freq = problem(torch.float32)
    p = weights(torch.float32)
    want, last = block(p, x, ld, s, reset, pos, freq)
    for t in range(x.shape[1]):
        q, k, v = (z.unflatten(-1, (H, D // H)) for z in (x[:, t:t + 1] @ p["qkv"]).split(D, -1))
        q, k = qk_norm_rotary(q, k, p["wq"], p["wk"], pos[:, t:t + 1], freq)
        o, s = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, reset[:, t])
        y = x[:, t] + o.flatten(-2)
        y = y + gated_linear_unit(y, p["gate"], p["up"]) @ p["down"]
        # two float32 evaluations of the same sums (values of order one to ten)
        torch.testing.assert_close(y, want[:, t], rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(s, last, rtol=1e-4, atol=1e-4)
