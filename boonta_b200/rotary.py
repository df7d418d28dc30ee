"""Norms of the queries and keys of every head with the position rotation in the same pass.

`qk_norm_rotary(q, k, q_weight, k_weight, positions, frequencies)` divides every row of q and k
(one head of one step) by its root mean square, multiplies it by the weight, and turns its pairs of
features by position * frequency; what attention over an unroll (`boonta_b200.linear_attention`)
takes as its queries and keys. Differentiable in q, k and the weights through the native backward.
"""
from __future__ import annotations

import torch

from . import _lib
from .linear_attention import _DTYPES, _device, _fits, _heads, _ptr, _refuse_tangents, _rows, _wants_grad


def rotary_frequencies(dim: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """base^(-2 i / dim) for i < dim / 2, in float64: the frequencies of `dim` rotated features."""
    if dim < 0 or dim % 2:
        raise ValueError(f"rotary_frequencies: {dim} features, an even number expected")
    i = torch.arange(0, dim, 2, dtype=torch.float64, device=device)
    return base ** (-i / max(dim, 1))


def _check(q, k, q_weight, k_weight, positions, frequencies):
    if q.ndim != 4 or k.ndim != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
        raise ValueError(f"qk_norm_rotary: q {tuple(q.shape)}, k {tuple(k.shape)}: [batch, steps, "
                         "heads, features] expected, alike in all but their heads")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise TypeError(f"qk_norm_rotary: q {q.dtype}, k {k.dtype}: float32 or bfloat16 expected, "
                        "the same for both")
    dim = q.shape[3]
    if not 1 <= dim <= 256:
        raise ValueError(f"qk_norm_rotary: heads of {dim} features: 1 to 256 are supported")
    _fits("qk_norm_rotary", *q.shape, k.shape[2])
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (dim,) or w.dtype not in _DTYPES or w.dtype != weights[0].dtype:
            raise ValueError(f"qk_norm_rotary: weights of ({dim},) in float32 or bfloat16 expected, "
                             f"alike: got {tuple(w.shape)} {w.dtype}")
    if frequencies.ndim != 1 or frequencies.dtype != torch.float64 or 2 * frequencies.shape[0] > dim:
        raise ValueError(f"qk_norm_rotary: frequencies {tuple(frequencies.shape)} "
                         f"{frequencies.dtype}: at most {dim // 2} in float64 expected")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError("qk_norm_rotary: frequencies are constants and have no gradient; detach them")
    if positions.dtype != torch.int64 or (positions.shape != q.shape[:2] and positions.shape != q.shape[1:2]):
        raise ValueError(f"qk_norm_rotary: positions {tuple(positions.shape)} {positions.dtype}: "
                         f"{tuple(q.shape[:2])} or {tuple(q.shape[1:2])} int64 expected")
    _refuse_tangents("qk_norm_rotary", q, k, q_weight, k_weight, frequencies)
    _device("qk_norm_rotary", q, k, q_weight, k_weight, positions, frequencies)


def _forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
    """The outputs, and the tensors that the call read."""
    q, k = _rows(q), _rows(k)
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    frequencies = frequencies.contiguous()
    if positions.ndim == 1:
        positions = positions.expand(q.shape[0], -1)
    yq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    yk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    with _lib.on_device(q.get_device()) as stream:
        _lib.check(_lib.lib().bt_qk_norm_rotary(
            _shape(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved), _heads(q),
            _heads(k), _ptr(q_weight), _ptr(k_weight), _heads(yq), _heads(yk), stream))
    return yq, yk, (q, k, q_weight, k_weight, positions, frequencies)


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
        ctx.eps, ctx.interleaved = eps, interleaved
        yq, yk, read = _forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved)
        ctx.save_for_backward(*read)
        return yq, yk

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        _refuse_tangents("qk_norm_rotary", gq, gk)
        gq, gk = _rows(gq.to(q.dtype)), _rows(gk.to(q.dtype))
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        dwq = torch.empty_like(q_weight) if ctx.needs_input_grad[2] else None
        dwk = torch.empty_like(k_weight) if ctx.needs_input_grad[3] else None
        with _lib.on_device(q.get_device()) as stream:
            shape = _shape(q, k, q_weight, k_weight, positions, frequencies, ctx.eps, ctx.interleaved)
            n = _lib.lib().bt_qk_norm_rotary_workspace(shape)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n > 0 else None
            _lib.check(_lib.lib().bt_qk_norm_rotary_backward(
                shape, _heads(q), _heads(k), _ptr(q_weight), _ptr(k_weight), _heads(gq), _heads(gk),
                _heads(dq), _heads(dk), _ptr(dwq), _ptr(dwk), _ptr(ws), n, stream))
        return dq, dk, dwq, dwk, None, None, None, None


def _shape(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
    w = q_weight if q_weight is not None else k_weight
    return _lib.QkNormRotaryShape(
        q.shape[0], q.shape[1], q.shape[2], k.shape[2], q.shape[3], frequencies.shape[0],
        _DTYPES[q.dtype], 0 if w is None else _DTYPES[w.dtype], int(interleaved), eps,
        positions.data_ptr(), positions.stride(0), positions.stride(1), frequencies.data_ptr())


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None,
                   k_weight: torch.Tensor | None, positions: torch.Tensor,
                   frequencies: torch.Tensor, *, eps: float = 1e-6, interleaved: bool = False
                   ) -> tuple[torch.Tensor, torch.Tensor]:
    """q [batch, steps, query heads, features] and k [batch, steps, key heads, features] normed and
    turned. float32 or bfloat16, any strides with contiguous features, 1 to 256 features; weights
    [features] (None: ones); positions [batch, steps] or [steps] int64; frequencies [r] float64
    (`rotary_frequencies`; constants, without a gradient): the first 2 r features are turned, feature
    i with feature i + r, or 2 i with 2 i + 1 where `interleaved`, the others only normed."""
    _check(q, k, q_weight, k_weight, positions, frequencies)
    if not _wants_grad(q, k, q_weight, k_weight):
        return _forward(q, k, q_weight, k_weight, positions, frequencies, float(eps),
                        bool(interleaved))[:2]
    return _QkNormRotary.apply(q, k, q_weight, k_weight, positions, frequencies, float(eps),
                               bool(interleaved))
