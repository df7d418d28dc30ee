"""The stateless operators' report of waits that gave up, and calls that overlap: two streams, two
graphs of one capture pool, the same tensor in several places."""
import pytest

pytestmark = pytest.mark.gpu


def attention(seed, dtype="bfloat16", T=300):
    import torch

    g = torch.Generator("cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    return ([r(2, T, 3, 64).to(dt) for _ in range(3)] +
            [-torch.rand(3, device="cuda", generator=g), r(2, 3, 64, 64)])


def test_after_normal_calls_nothing_is_reported():
    import torch

    import boonta_b200
    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention

    linear_attention(*attention(1))
    x = torch.randn(200, 64, device="cuda")
    gated_linear_unit(x, x[:64], x[:64])
    boonta_b200.check_operators()
    boonta_b200.check_operators("cuda:0")


def test_two_streams_at_once_give_what_one_gives():
    import torch

    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention

    args = [attention(i, T=2000) for i in range(2)]
    xs = [torch.randn(700, 64, device="cuda").bfloat16() for _ in range(2)]
    w = torch.randn(64, 320, device="cuda").bfloat16()
    want = [(*linear_attention(*a), gated_linear_unit(x, w, w)) for a, x in zip(args, xs)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = (*linear_attention(*args[i]), gated_linear_unit(xs[i], w, w))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_captured_graphs_share_a_pool_and_replay_in_turn():
    import torch

    from boonta_b200.linear_attention import linear_attention

    args = [attention(i, T=2000) for i in range(2)]  # long enough for splits, so for workspaces
    want = [[t.clone() for t in linear_attention(*a)] for a in args]
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(linear_attention(*a))
        graphs.append(g)
    for _ in range(2):
        for i in (0, 1):
            graphs[i].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(outs[i], want[i]))


def test_one_tensor_in_several_places():
    import torch

    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention
    from boonta_b200.rotary import qk_norm_rotary, rotary_frequencies

    x = torch.randn(2, 100, 2, 32, device="cuda", requires_grad=True)
    ld = torch.tensor([-0.1, -0.2], device="cuda")
    g = torch.autograd.grad(linear_attention(x, x, x, ld)[0].sum(), x)[0]
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    want = torch.autograd.grad(linear_attention(*parts, ld)[0].sum(), parts)
    torch.testing.assert_close(g, want[0] + want[1] + want[2], rtol=1e-6, atol=1e-6)
    pos = torch.arange(100, device="cuda")
    f = rotary_frequencies(32)
    y = qk_norm_rotary(x, x, None, None, pos, f)
    assert torch.equal(y[0], y[1])
    w = torch.randn(32, 32, device="cuda", requires_grad=True)
    rows = x.detach().reshape(-1, 32)
    got = torch.autograd.grad(gated_linear_unit(rows, w, w).sum(), w)[0]
    a, b = w.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    ga, gb = torch.autograd.grad(gated_linear_unit(rows, a, b).sum(), (a, b))
    torch.testing.assert_close(got, ga + gb, rtol=1e-6, atol=1e-6)


def test_rows_behind_the_outputs_are_left_as_they_were():
    """Through the C entry, into views of larger buffers: what lies around the outputs stays."""
    import torch

    from boonta_b200 import _lib
    from boonta_b200.linear_attention import _heads, _shape, linear_attention

    for reverse_tail in (100, 130, 256):
        q, k, v, ld, s = attention(9, T=reverse_tail)
        want, final = linear_attention(q, k, v, ld, s)
        wide = torch.full((2, reverse_tail + 7, 5, 64), 3.0, device="cuda", dtype=q.dtype)
        out = wide[:, 3:3 + reverse_tail, 1:4]
        states = torch.full((8, 64, 64), 5.0, device="cuda")
        ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
        shape = _shape(q, v, ld, None, 0.125)
        _lib.check(_lib.lib().bt_linear_attention(
            shape, _heads(q), _heads(k), _heads(v), s.data_ptr(), _heads(out), states[1:7].data_ptr(),
            ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, want) and torch.equal(states[1:7], final.view(6, 64, 64))
        out.fill_(3.0)
        assert (wide == 3.0).all() and (states[0] == 5).all() and (states[7] == 5).all()


def test_a_fresh_host_thread_may_call_first():
    """A thread whose first CUDA call is an operator (its memory comes from torch's cache)."""
    import threading

    import torch

    from boonta_b200.glu import gated_linear_unit
    from boonta_b200.linear_attention import linear_attention

    a = attention(4)
    x, w = torch.randn(200, 64, device="cuda").bfloat16(), torch.randn(64, 64, device="cuda").bfloat16()
    calls = (lambda: gated_linear_unit(x, w, w), lambda: linear_attention(*a)[0])
    want = [f() for f in calls]
    for f in calls:  # the cache now holds blocks of every size that the threads will ask for
        del_me = [f() for _ in range(4)]
    del del_me
    got = [None, None]

    def go(i):
        try:
            got[i] = calls[i]()
        except Exception as e:  # noqa: BLE001
            got[i] = e

    for i in (0, 1):
        t = threading.Thread(target=go, args=(i,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    for g, b in zip(got, want):
        assert torch.is_tensor(g), g
        assert torch.equal(g, b)
