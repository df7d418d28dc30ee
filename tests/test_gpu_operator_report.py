"""The report of the stateless operators' waits: a wait that runs out (one thread, 20 ms, on a barrier that nothing
arrives at) is reported once, and calls go on afterwards. The first call of a process inside a graph's capture."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from boonta_b200 import _lib

pytestmark = pytest.mark.gpu


def test_a_wait_that_gave_up_is_reported_once():
    import torch

    import boonta_b200
    from boonta_b200.linear_attention import linear_attention

    boonta_b200.check_operators()
    s = torch.cuda.current_stream().cuda_stream
    _lib.check(_lib.lib().bt_selftest_operator_wait(20_000, s))
    with pytest.raises(_lib.BoontaError, match="gave up") as e:
        boonta_b200.check_operators()
    assert e.value.code == _lib.BT_ERR_TIMEOUT
    boonta_b200.check_operators()
    x = torch.randn(2, 200, 2, 64, device="cuda").bfloat16()
    out, _ = linear_attention(x, x, x, torch.tensor([-0.1, -0.2], device="cuda"))
    boonta_b200.check_operators()
    assert out.isfinite().all()


def test_the_report_comes_from_any_stream():
    import torch

    import boonta_b200

    side = torch.cuda.Stream()
    _lib.check(_lib.lib().bt_selftest_operator_wait(20_000, side.cuda_stream))
    side.synchronize()
    with pytest.raises(_lib.BoontaError, match="gave up"):
        boonta_b200.check_operators("cuda")
    boonta_b200.check_operators("cuda:0")


@pytest.mark.parametrize("limit", [0, -5, 2_000_001])
def test_limits_outside_the_bound_are_refused(limit):
    assert _lib.lib().bt_selftest_operator_wait(limit, None) == _lib.BT_ERR_INVALID
    assert b"limit" in _lib.lib().bt_last_error()


FIRST = """
import torch
from boonta_b200.{module} import *
torch.manual_seed(0)
r = lambda *s: torch.randn(*s, device="cuda").to(torch.{dtype})
{inputs}
def once():
    leaves = [t.detach().requires_grad_() for t in a]
    y = {call}
    y = y if isinstance(y, tuple) else (y,)
    return [*y, *torch.autograd.grad(y, leaves, [torch.ones_like(t) for t in y])]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = once()
graph.replay()
torch.cuda.synchronize()
want = once()
assert all(torch.equal(x, y) for x, y in zip(got, want))
print("same")
"""

CALLS = {
    "linear_attention": ("a = [r(2, 700, 2, 64) for _ in range(3)]; ld = torch.tensor([-0.1, -0.3], device='cuda')",
                         "linear_attention(*leaves, ld)"),
    "rotary": ("a = [r(2, 50, 4, 64), r(2, 50, 2, 64), r(64), r(64)]; p = torch.arange(50, device='cuda'); "
               "f = rotary_frequencies(64)", "qk_norm_rotary(*leaves, p, f)"),
    "glu": ("a = [r(700, 64), r(64, 320), r(64, 320)]", "gated_linear_unit(*leaves)"),
}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("module", sorted(CALLS))
def test_the_first_call_of_a_process_may_be_captured(module, dtype):
    inputs, call = CALLS[module]
    code = FIRST.format(module=module, dtype=dtype, inputs=inputs, call=call)
    root = Path(__file__).resolve().parents[1]
    p = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300,
                       env=os.environ | {"PYTHONPATH": str(root)})
    assert p.returncode == 0 and "same" in p.stdout, p.stderr[-2000:]


def test_the_first_step_of_a_process_may_be_captured():
    code = """
import torch
from boonta_b200.linear_attention import linear_attention_step
q = torch.randn(3, 2, 64, device="cuda")
s, ld = torch.randn(3, 2, 64, 64, device="cuda"), torch.tensor([-0.1, -0.3], device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = linear_attention_step(q, q, q, ld, s)
graph.replay()
torch.cuda.synchronize()
want = linear_attention_step(q, q, q, ld, s)
assert all(torch.equal(x, y) for x, y in zip(got, want))
print("same")
"""
    root = Path(__file__).resolve().parents[1]
    p = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300,
                       env=os.environ | {"PYTHONPATH": str(root)})
    assert p.returncode == 0 and "same" in p.stdout, p.stderr[-2000:]
