"""Linear attention with a decay per head (boonta_b200.linear_attention) against the float64 oracle:
lengths from none to several splits, feature counts off every tile, strided and misaligned inputs,
resets, missing and given states, gradients, the single-step form, streams and graphs. The bounds
are derived in tests/_sequence.py."""
import math

import numpy as np
import pytest

from oracle import sequence as seq
from _sequence import check, numpy64

pytestmark = pytest.mark.gpu

RESETS = ("none", "some", "all", "first", "last")


def terms(T, dk, dv):
    return 2 * T + 2 * max(dk, dv) + 64


def inputs(seed, B, T, H, dk, dv, dtype, resets="some", state=True, layout="plain"):
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    r = lambda *s, d=dt: torch.randn(*s, device="cuda", generator=g).to(d)
    if layout == "plain":
        q, k, v = r(B, T, H, dk), r(B, T, H, dk), r(B, T, H, dv)
    elif layout == "fused":  # slices of one projection's output, off any alignment where dk is odd
        q, k, v = r(B, T, H, 2 * dk + dv).split([dk, dk, dv], -1)
    elif layout == "heads_first":
        q, k, v = (r(B, H, T, d).transpose(1, 2) for d in (dk, dk, dv))
    elif layout == "shifted":  # one element off a 16-byte boundary
        q, k, v = (r(B * T * H * d + 1)[1:].view(B, T, H, d) for d in (dk, dk, dv))
    elif layout == "expanded":  # one key head for all query heads
        q, v = r(B, T, H, dk), r(B, T, H, dv)
        k = r(B, T, 1, dk).expand(B, T, H, dk)
    ld = torch.log1p(-torch.exp2(-torch.linspace(1, 9, H, device="cuda")))
    s = r(B, H, dk, dv, d=torch.float32) if state else None
    m = {"none": None, "some": torch.rand(B, T, device="cuda", generator=g) < 0.05,
         "all": torch.ones(B, T, dtype=torch.bool, device="cuda"),
         "first": torch.arange(T, device="cuda").expand(B, T) == 0,
         "last": torch.arange(T, device="cuda").expand(B, T) == T - 1}[resets]
    return q, k, v, ld, s, m, r(B, T, H, dv), r(B, H, dk, dv, d=torch.float32)


def oracle(q, k, v, ld, s, m, dout=None, dfinal=None, scale=None):
    n = [numpy64(t) for t in (q, k, v, ld)]
    st = np.zeros((q.shape[0], q.shape[2], q.shape[3], v.shape[3])) if s is None else numpy64(s)
    mask = None if m is None else m.cpu().numpy()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want = seq.linear_attention(*n, st, mask, scale)
    g = ()
    if dout is not None:
        g = numpy64(dout), numpy64(dfinal)
        want += seq.linear_attention_backward(*n, st, mask, scale, *g)
    return want, seq.linear_attention_scale(*n, st, mask, scale, *g)


NAMES = ("out", "final", "dq", "dk", "dv", "dstate")


def compare(got, want, scale, T, dk, dv, dtype):
    for i, (g, w, s) in enumerate(zip(got, want, scale)):
        if w.size:
            check(NAMES[i], g, w, s, terms(T, dk, dv), "f32" if i in (1, 5) else dtype, dtype,
                  tensor_cores=dtype == "bf16")


def run(a, grads=True, **kw):
    import torch

    from boonta_b200.linear_attention import linear_attention

    q, k, v, ld, s, m, dout, dfinal = a
    leaves = [t.detach().requires_grad_() for t in (q, k, v) + (() if s is None else (s,))]
    out, final = linear_attention(*leaves[:3], ld, leaves[3] if s is not None else None, m, **kw)
    if not grads:
        return [out, final]
    return [out, final, *torch.autograd.grad((out, final), leaves, (dout, dfinal))]


def one(seed, B, T, H, dk, dv, dtype, **kw):
    a = inputs(seed, B, T, H, dk, dv, dtype, **kw)
    want, scale = oracle(*a)
    got = run(a)
    assert got[0].dtype == got[2].dtype == a[0].dtype
    compare(got, want, scale, T, dk, dv, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(T, dtype):
    one(T, 2, T, 3, 64, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("resets", RESETS)
@pytest.mark.parametrize("T", [1, 150])
def test_resets(T, resets, dtype):
    one(7 + T, 3, T, 2, 32, 64, dtype, resets=resets)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dk,dv", [(1, 1), (3, 5), (8, 16), (16, 8), (40, 72), (64, 128), (128, 64),
                                   (96, 33), (65, 64), (128, 128)])
def test_feature_counts(dk, dv, dtype):
    one(dk + dv, 2, 140, 2, dk, dv, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "shifted", "expanded"])
@pytest.mark.parametrize("d", [64, 24, 7])
def test_strides(d, layout, dtype):
    one(d, 2, 70, 3, d, d, dtype, layout=layout)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("resets", ["none", "some"])
def test_long_sequences_are_split(resets, dtype):
    one(17, 1, 1111, 2, 64, 64, dtype, resets=resets)
    one(18, 1, 900, 1, 16, 128, dtype, resets=resets)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_without_a_state_and_with_a_given_scale(dtype):
    a = inputs(5, 2, 100, 2, 64, 64, dtype, state=False)
    want, scale = oracle(*a, scale=0.5)
    compare(run(a, scale=0.5), want[:5], scale[:5], 100, 64, 64, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_steps_hand_the_state_on(dtype):
    import torch

    a = inputs(5, 2, 0, 2, 16, 8, dtype, resets="none")
    got = run(a)
    assert got[0].shape == (2, 0, 2, 8)
    assert torch.equal(got[1], a[4]) and torch.equal(got[5], a[7])
    a = inputs(5, 0, 4, 2, 16, 8, dtype, resets="none")
    assert run(a)[0].shape == (0, 4, 2, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_gradient_of_the_two(dtype):
    """Only the output's, or only the final state's gradient: the other counts as zero."""
    import torch

    from boonta_b200.linear_attention import linear_attention

    a = inputs(23, 2, 90, 2, 32, 32, dtype)
    q, k, v, ld, s, m, dout, dfinal = a
    for which in (0, 1):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, s)]
        y = linear_attention(*leaves[:3], ld, leaves[3], m)[which]
        got = torch.autograd.grad(y, leaves, (dout, dfinal)[which])
        g = [dout, dfinal]
        g[1 - which] = torch.zeros_like(g[1 - which])
        want, scale = oracle(q, k, v, ld, s, m, *g)
        for i in range(4):
            check(NAMES[2 + i], got[i], want[2 + i], scale[2 + i], terms(90, 32, 32),
                  "f32" if i == 3 else dtype, dtype, tensor_cores=dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_extreme_decays(dtype):
    """A head that forgets at once (log decay -inf), one that nearly does, one that never does."""
    import torch

    a = list(inputs(29, 2, 200, 4, 64, 64, dtype))
    a[3] = torch.tensor([-math.inf, -30.0, 0.0, -1e-6], device="cuda")
    clamped = list(a)
    clamped[3] = a[3].clamp(min=-700)
    want, scale = oracle(*clamped)
    compare(run(a), want, scale, 200, 64, 64, dtype)


@pytest.mark.parametrize("resets", ["none", "some"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decays_on_both_sides_of_the_two_forms_of_the_scores(dtype, resets):
    """Heads just above and just below the decay where the weights change their place; a negative scale."""
    import torch

    a = list(inputs(47, 2, 333, 5, 64, 128, dtype, resets=resets))
    a[3] = torch.tensor([-0.2299, -0.2301, -0.1, -0.6, -5.0], device="cuda")
    want, scale = oracle(*a, scale=-0.3)
    compare(run(a, scale=-0.3), want, scale, 333, 64, 128, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_nan_stays_in_its_sequence(dtype):
    import torch

    a = list(inputs(31, 2, 100, 2, 64, 64, dtype, resets="none"))
    clean = run(a)
    a[2] = a[2].clone()
    a[2][1, 50, 1] = math.nan
    a[6] = a[6].clone()
    a[6][1, 20, 1] = math.inf
    got = run(a)
    for i, (g, c) in enumerate(zip(got, clean)):
        heads = 1 if i in (1, 5) else 2
        keep = torch.ones(g.shape[:1] + g.shape[heads:heads + 1], dtype=torch.bool)
        keep[1, 1] = False
        pick = lambda x: (x if heads == 1 else x.transpose(1, 2))[keep.to(x.device)]
        assert torch.equal(pick(g), pick(c)), NAMES[i]
        assert not torch.isfinite((g if heads == 1 else g.transpose(1, 2))[1, 1]).all(), NAMES[i]


def test_what_a_reset_hides_has_no_part():
    """float32: values of any kind before a reset leave what comes after it alone."""
    import torch

    a = list(inputs(37, 2, 100, 2, 16, 16, "f32", resets="none"))
    a[5] = torch.zeros(2, 100, dtype=torch.bool, device="cuda")
    a[5][:, 40] = True
    clean = run(a, grads=False)
    a[1], a[2], a[4] = a[1].clone(), a[2].clone(), a[4].clone()
    a[1][:, 7], a[2][:, 39], a[4][0] = math.nan, math.inf, math.nan
    got = run(a, grads=False)
    assert torch.equal(got[0][:, 40:], clean[0][:, 40:]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,H,dk,dv", [(1, 1, 1, 1), (3, 2, 64, 64), (5, 3, 48, 40), (2, 2, 128, 128),
                                       (2, 2, 33, 7), (300, 4, 16, 64)])
def test_steps(B, H, dk, dv, dtype):
    import torch

    from boonta_b200.linear_attention import linear_attention_step

    a = inputs(B + dk, B, 1, H, dk, dv, dtype, resets="some")
    q, k, v, ld, s, m = a[:6]
    m[0] = True
    want, scale = oracle(q, k, v, ld, s, m)
    keep = s.clone()
    out, new = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, m[:, 0])
    assert torch.equal(s, keep) and out.dtype == v.dtype
    check("out", out[:, None], want[0], scale[0], terms(1, dk, dv), dtype, "f32")
    check("state", new, want[1], scale[1], terms(1, dk, dv), "f32", "f32")
    again, same = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, m[:, 0], new_state=s)
    assert same is s and torch.equal(s, new) and torch.equal(again, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_nan_decay_is_not_hidden(dtype):
    import torch

    a = list(inputs(33, 1, 140, 2, 64, 64, dtype, resets="none"))
    a[3] = torch.tensor([math.nan, -0.1], device="cuda")
    out, final = run(a, grads=False)
    assert out[:, :, 0].isnan().all() and final[:, 0].isnan().all()
    assert out[:, :, 1].isfinite().all() and final[:, 1].isfinite().all()


def test_steps_follow_the_unroll():
    """Acting step by step gives what the unroll gives, and the state between."""
    import torch

    from boonta_b200.linear_attention import linear_attention, linear_attention_step

    q, k, v, ld, s, m, _, _ = inputs(41, 3, 40, 2, 64, 64, "f32")
    # each side is within n 2^-24 of the terms' absolute sum of the exact values (tests/_sequence.py)
    scale, last = oracle(q, k, v, ld, s, m)[1]
    far = 2 * terms(40, 64, 64) * 2.0 ** -24
    out, final = linear_attention(q, k, v, ld, s, m)
    for t in range(40):
        o, s = linear_attention_step(q[:, t], k[:, t], v[:, t], ld, s, m[:, t])
        assert (np.abs(numpy64(o) - numpy64(out[:, t])) <= far * scale[:, t]).all()
    assert (np.abs(numpy64(s) - numpy64(final)) <= far * last).all()
    torch.testing.assert_close(s, final, rtol=1e-4, atol=1e-4)


def test_refusals_on_the_gpu():
    import torch

    from boonta_b200.linear_attention import linear_attention, linear_attention_step

    q, k, v, ld, s, m, _, _ = inputs(1, 2, 1, 2, 8, 8, "f32")
    with pytest.raises(ValueError, match="device"):
        linear_attention(q, k, v.cpu(), ld, s, m)
    step = [t[:, 0] for t in (q, k, v)]
    with pytest.raises(ValueError, match="no gradient"):
        linear_attention_step(step[0].clone().requires_grad_(), *step[1:], ld, s)
    with pytest.raises(ValueError, match="new_state"):
        linear_attention_step(*step, ld, s, new_state=torch.empty(2, 2, 8, 9, device="cuda"))
    room = torch.zeros(3, 2, 8, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        linear_attention_step(*step, ld, room[:2], new_state=room[1:])
    with pytest.raises(ValueError, match="overlaps"):
        linear_attention_step(*step, ld, room[0].transpose(2, 1).expand(2, 2, 8, 8), new_state=room[:2])
    with pytest.raises(ValueError, match="a state"):
        linear_attention_step(*step, ld, None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_another_stream_and_a_captured_pass_give_the_same_bits(dtype):
    import torch

    a = inputs(43, 2, 700, 2, 64, 64, dtype)
    want = [t.clone() for t in run(a)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(a)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(a)
    other = inputs(44, 2, 700, 2, 64, 64, dtype)
    second = [t.clone() for t in run(other)]
    for src, dst in zip(other, a):
        if dst is not None:
            dst.copy_(src)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, second))
