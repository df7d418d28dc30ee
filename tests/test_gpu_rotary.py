"""Query/key norms with the position rotation (boonta_b200.rotary) against the float64 oracle:
feature counts off every vector, partial rotations, both pairings, strided inputs, far positions,
missing weights, gradients, streams and graphs.

Bounds. A row's mean square is a sum of D terms in fp32, so its root's reciprocal is off by at most
(D + 4) 2^-25 relative; the products add 4 roundings, and an angle below 1e6 turns, reduced in 64
bits, is off by at most 2^-30 there and 2^-23 in fp32 sine and cosine (4 pi 2^-24 and two units of
the functions): each output is within e = (D + 32) 2^-24 of the sum of the absolute values of its
two products (1 + |xh| mean(|u xh|) for dx), plus its own rounding u. A weight gradient sums
`rows` such terms in fp32 and float64: (e + rows-per-thread 2^-24) of their absolute sum.
"""
import numpy as np
import pytest

from _sequence import U, numpy64
from oracle import sequence as seq

pytestmark = pytest.mark.gpu


def inputs(seed, B, T, hq, hk, D, dtype, wdtype=None, layout="plain", far=1000):
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    dts = {"f32": torch.float32, "bf16": torch.bfloat16}
    dt, wt = dts[dtype], dts[wdtype or dtype]
    r = lambda *s, d=dt: torch.randn(*s, device="cuda", generator=g).to(d)
    if layout == "plain":
        q, k = r(B, T, hq, D), r(B, T, hk, D)
    elif layout == "fused":
        q, k, _ = r(B, T, (hq + 2 * hk) * D).split([hq * D, hk * D, hk * D], -1)
        q, k = q.unflatten(-1, (hq, D)), k.unflatten(-1, (hk, D))
    elif layout == "shifted":
        q, k = (r(B * T * h * D + 1)[1:].view(B, T, h, D) for h in (hq, hk))
    elif layout == "heads_first":
        q, k = r(B, hq, T, D).transpose(1, 2), r(B, hk, T, D).transpose(1, 2)
    wq, wk = 1 + 0.3 * r(D, d=wt), 1 + 0.3 * r(D, d=wt)
    pos = torch.randint(0, far, (B, T), device="cuda", generator=g)
    return q, k, wq, wk, pos, r(B, T, hq, D), r(B, T, hk, D)


def check(name, got, want, scale, e, u):
    got = numpy64(got)
    assert got.shape == want.shape
    over = np.abs(got - want) - (u * np.abs(want) + e * scale)
    assert (over <= 0).all(), (name, float(over.max()))


def compare(a, dtype, wdtype, half, interleaved, eps=1e-6, base=10000.0):
    import torch

    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    q, k, wq, wk, pos, gq, gk = a
    D = q.shape[-1]
    f = rotary_frequencies(2 * half, base)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    y = qk_norm_rotary(*leaves, pos, f, eps=eps, interleaved=interleaved)
    grads = torch.autograd.grad(y, leaves, (gq, gk))
    e = (D + 32) * U["f32"]
    p, ff = pos.cpu().numpy(), f.cpu().numpy()
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        x, w, g = numpy64(x), numpy64(w), numpy64(g)
        want = seq.norm_rotary(x, w, p, ff, eps, interleaved)
        r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        spread = np.abs(x) * r * np.abs(w)
        pair = seq._turn(spread, np.zeros(p.shape + (half,)), interleaved)
        both = pair + partner(spread, half, interleaved)
        check("y", y[i], want, both, e, U[dtype])
        dx, dw = seq.norm_rotary_backward(x, w, p, ff, eps, interleaved, g)
        turned = np.abs(g) + partner(np.abs(g), half, interleaved)
        xh = np.abs(x) * r
        check("dx", grads[i], dx, r * (turned * np.abs(w) + xh * (turned * np.abs(w) * xh).mean(-1, keepdims=True)),
              2 * e, U[dtype])
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        check("dw", grads[2 + i], dw, (turned * xh).sum((0, 1, 2)), e + min(rows, 4096) * U["f32"], U[wdtype or dtype])


def partner(x, half, interleaved):
    y = np.zeros_like(x)
    if interleaved:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = x[..., 1:2 * half:2], x[..., 0:2 * half:2]
    else:
        y[..., :half], y[..., half:2 * half] = x[..., half:2 * half], x[..., :half]
    return y


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,half", [(64, 32), (128, 64), (256, 128), (80, 20), (80, 40), (96, 5), (2, 1),
                                    (1, 0), (33, 16), (7, 2), (130, 65), (200, 0), (8, 4)])
def test_feature_counts(D, half, interleaved, dtype):
    compare(inputs(D, 2, 9, 3, 2, D, dtype), dtype, None, half, interleaved)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,hq,hk", [(1, 1, 1, 1), (1, 1, 40, 1), (3, 1, 8, 8), (2, 700, 4, 1), (1, 2500, 16, 4),
                                       (700, 1, 2, 2)])
def test_shapes(B, T, hq, hk, dtype):
    compare(inputs(T, B, T, hq, hk, 64, dtype), dtype, None, 32, False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["fused", "shifted", "heads_first"])
@pytest.mark.parametrize("D", [64, 80, 10])
def test_strides(D, layout, dtype):
    compare(inputs(D, 2, 17, 4, 2, D, dtype, layout=layout), dtype, None, D // 2, False)


@pytest.mark.parametrize("dtype,wdtype", [("f32", "bf16"), ("bf16", "f32")])
def test_weights_of_the_other_type(dtype, wdtype):
    compare(inputs(3, 2, 33, 4, 2, 64, dtype, wdtype), dtype, wdtype, 32, True)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_keep_their_phase(interleaved):
    compare(inputs(5, 2, 50, 2, 2, 64, "f32", far=1_000_000), "f32", None, 32, interleaved)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_positions_before_zero(dtype):
    a = list(inputs(6, 2, 40, 2, 1, 64, dtype))
    a[4] = a[4] - 500
    compare(a, dtype, None, 32, False)


def test_missing_weights_count_as_ones_and_positions_may_be_shared():
    import torch

    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    q, k, _, wk, pos, _, _ = inputs(9, 3, 11, 2, 2, 64, "f32")
    f, one = rotary_frequencies(64), torch.ones(64, device="cuda")
    for a, b in zip(qk_norm_rotary(q, k, None, None, pos[0], f),
                    qk_norm_rotary(q, k, one, one, pos[0].expand(3, -1).contiguous(), f)):
        assert torch.equal(a, b)
    for a, b in zip(qk_norm_rotary(q, k, None, wk, pos, f), qk_norm_rotary(q, k, one, wk, pos, f)):
        assert torch.equal(a, b)
    x = q.clone().requires_grad_()
    y = qk_norm_rotary(x, k, None, wk, pos, f)[0]
    assert torch.autograd.grad(y.sum(), x)[0].isfinite().all()


def test_empty_calls():
    import torch

    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    f, w = rotary_frequencies(8), torch.ones(8, device="cuda", requires_grad=True)
    for B, T, hq, hk in ((0, 3, 2, 1), (2, 0, 2, 1), (2, 3, 0, 1), (2, 3, 2, 0)):
        q, k = torch.ones(B, T, hq, 8, device="cuda"), torch.ones(B, T, hk, 8, device="cuda")
        pos = torch.zeros(B, T, dtype=torch.int64, device="cuda")
        y = qk_norm_rotary(q, k, w, w, pos, f)
        assert y[0].shape == q.shape and y[1].shape == k.shape
        g = torch.autograd.grad(y, w, [torch.ones_like(t) for t in y])[0]
        # rows of ones: the norm is 1 / sqrt(1 + eps), the position 0 turns nothing
        want = B * T * (hq + hk) / np.sqrt(1 + 1e-6)
        torch.testing.assert_close(g, torch.full_like(g, want), rtol=1e-5, atol=0)


def test_the_passes_repeat_to_the_bit_on_another_stream_and_in_a_graph():
    import torch

    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    a = inputs(11, 4, 500, 4, 2, 64, "bf16")
    f = rotary_frequencies(64)

    def run():
        q, k, wq, wk, pos, gq, gk = a
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = qk_norm_rotary(*leaves, pos, f)
        return [*y, *torch.autograd.grad(y, leaves, (gq, gk))]

    want = [t.detach().clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
