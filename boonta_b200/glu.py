"""The gated feed-forward layer h = act(x w_gate) * (x w_up), both projections, the activation and
the product in one kernel; differentiable through the native backward, which forms the projections
again tile by tile instead of keeping them.

The weights are kernels as the framework's Dense layers have them ([in features, out features]), the
activations its own ("silu", "relu", "tanh", "none").
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .linear_attention import _DTYPES, _device, _fits, _ptr, _refuse_tangents, _wants_grad


def _check(x, w_gate, w_up, activation):
    if activation not in _lib.ACT:
        raise ValueError(f"gated_linear_unit: unknown activation {activation!r}, have "
                         f"{sorted(_lib.ACT)}")
    if x.ndim < 1 or w_gate.ndim != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[0]:
        raise ValueError(f"gated_linear_unit: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, "
                         f"w_up {tuple(w_up.shape)}: [..., in], [in, out], [in, out] expected")
    if x.dtype not in _DTYPES or w_gate.dtype != x.dtype or w_up.dtype != x.dtype:
        raise TypeError(f"gated_linear_unit: x {x.dtype}, w_gate {w_gate.dtype}, w_up {w_up.dtype}: "
                        "float32 or bfloat16 expected, the same for all three")
    if min(w_gate.shape) < 1:
        raise ValueError(f"gated_linear_unit: weights {tuple(w_gate.shape)} without features")
    _fits("gated_linear_unit", math.prod(x.shape[:-1]), *w_gate.shape)
    _refuse_tangents("gated_linear_unit", x, w_gate, w_up)
    _device("gated_linear_unit", x, w_gate, w_up)


def _aligned(t):
    """t without gaps, from a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _shape(x, w, activation):
    return _lib.GluShape(x.shape[0], w.shape[0], w.shape[1], _DTYPES[x.dtype], _lib.ACT[activation])


def _workspace(shape, backward, device):
    n = _lib.lib().bt_glu_workspace(shape, backward)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None), n


def _forward(x, w_gate, w_up, activation):
    """The output, and the tensors that the call read."""
    x, w_gate, w_up = _aligned(x), _aligned(w_gate), _aligned(w_up)
    out = torch.empty((x.shape[0], w_gate.shape[1]), dtype=x.dtype, device=x.device)
    with _lib.on_device(x.get_device()) as stream:
        shape = _shape(x, w_gate, activation)
        ws, n = _workspace(shape, 0, x.device)
        _lib.check(_lib.lib().bt_glu(shape, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(),
                                     out.data_ptr(), _ptr(ws), n, stream))
    return out, (x, w_gate, w_up)


class _Glu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        out, read = _forward(x, w_gate, w_up, activation)
        ctx.save_for_backward(*read)
        ctx.activation = activation
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        x, w_gate, w_up = ctx.saved_tensors
        _refuse_tangents("gated_linear_unit", dout)
        dout = _aligned(dout.to(x.dtype))
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        weights = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dwg = torch.empty_like(w_gate) if weights else None
        dwu = torch.empty_like(w_up) if weights else None
        with _lib.on_device(x.get_device()) as stream:
            shape = _shape(x, w_gate, ctx.activation)
            ws, n = _workspace(shape, 1, x.device)
            _lib.check(_lib.lib().bt_glu_backward(
                shape, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), dout.data_ptr(), _ptr(dx),
                _ptr(dwg), _ptr(dwu), _ptr(ws), n, stream))
        return dx, dwg, dwu, None


def gated_linear_unit(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                      activation: str = "silu") -> torch.Tensor:
    """act(x @ w_gate) * (x @ w_up): x [..., in], weights [in, out], all float32 or all bfloat16;
    sums in float32, the result [..., out] in x's dtype. A float32 value that is not finite makes the
    sums it enters NaN; one below 2^-109 keeps fewer than 24 bits."""
    _check(x, w_gate, w_up, activation)
    rows = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    if _wants_grad(x, w_gate, w_up):
        out = _Glu.apply(rows, w_gate, w_up, activation)
    else:
        out = _forward(rows, w_gate, w_up, activation)[0]
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], w_gate.shape[1])
