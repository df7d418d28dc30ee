"""Linear attention with a decay per head: the matrix-valued recurrence of a sequence torso.

`linear_attention(q, k, v, log_decay, state, reset)` runs

    S_t = [not reset_t] exp(log_decay_h) S_{t-1} + k_t v_t^T,      out_t = scale * S_t^T q_t

over the steps of every (batch row, head), differentiable through the native backward kernels;
`linear_attention_step` is one step of it for acting. They stand beside `boonta_b200.scan`, whose
state is a vector: q, k are [batch, steps, heads, key features], v and out [batch, steps, heads,
value features], float32 or bfloat16 with any strides as long as features are contiguous; states
are float32 [batch, heads, key features, value features]. `reset` [batch, steps] (bool) clears the
state before a step, as the recurrent networks' `reset_carry` does at an episode's start, so an
unroll may hold several episodes.

`log_decay` [heads] (float32, at most 0) is a constant of the model: it has no gradient. A value
that is not finite may reach other steps of its own (batch row, head) sequence, never another's.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _heads(t: torch.Tensor) -> _lib.Heads:
    s = t.stride()
    return _lib.Heads(t.data_ptr(), s[0], s[1] if t.ndim == 4 else 0, s[-2])


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _on(device):
    """The device's context where it is not the current one."""
    return torch.cuda.device(device)


def _check(name, q, k, v, log_decay, state, reset):
    lead = "[batch, steps, heads" if name == "linear_attention" else "[batch, heads"
    ndim = 4 if name == "linear_attention" else 3
    if q.ndim != ndim or k.shape != q.shape or v.shape[:-1] != q.shape[:-1] or v.ndim != ndim:
        raise ValueError(f"{name}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: "
                         f"{lead}, features] expected, alike in all but v's features")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{name}: q {q.dtype}, k {k.dtype}, v {v.dtype}: float32 or bfloat16 "
                        "expected, the same for all three")
    if not (1 <= q.shape[-1] <= 128 and 1 <= v.shape[-1] <= 128):
        raise ValueError(f"{name}: heads of {q.shape[-1]} and {v.shape[-1]} features: 1 to 128 "
                         "are supported")
    batch, heads = q.shape[0], q.shape[-2]
    if log_decay.shape != (heads,) or log_decay.dtype != torch.float32:
        raise ValueError(f"{name}: log_decay {tuple(log_decay.shape)} {log_decay.dtype}: "
                         f"({heads},) float32 expected")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: log_decay is a constant and has no gradient; detach it")
    want = (batch, heads, q.shape[-1], v.shape[-1])
    if state is not None and (tuple(state.shape) != want or state.dtype != torch.float32):
        raise ValueError(f"{name}: state {tuple(state.shape)} {state.dtype}: {want} float32 expected")
    if reset is not None and (reset.shape != q.shape[:ndim - 2] or reset.dtype != torch.bool):
        raise ValueError(f"{name}: reset {tuple(reset.shape)} {reset.dtype}: "
                         f"{tuple(q.shape[:ndim - 2])} bool expected")
    for t in (q, k, v, log_decay, state, reset):
        if t is not None and (not t.is_cuda or t.device != q.device):
            raise ValueError(f"{name}: CUDA tensors on one device expected")


def _shape(q, v, log_decay, reset, scale) -> _lib.LinearAttentionShape:
    steps = q.shape[1] if q.ndim == 4 else 1
    rs = (0, 0) if reset is None else (reset.stride(0), reset.stride(1) if reset.ndim == 2 else 0)
    return _lib.LinearAttentionShape(
        q.shape[0], steps, q.shape[-2], q.shape[-1], v.shape[-1], _DTYPES[q.dtype], scale,
        log_decay.data_ptr(), None if reset is None else reset.data_ptr(), *rs)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(shape, backward, device):
    n = _lib.lib().bt_linear_attention_workspace(C.byref(shape), backward)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None), n


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, reset, scale):
        q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
        state = None if state is None else state.contiguous()
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        final = torch.empty(q.shape[0], q.shape[2], q.shape[3], v.shape[3], dtype=torch.float32,
                            device=q.device)
        with _on(q.device):
            shape = _shape(q, v, log_decay, reset, scale)
            ws, n = _workspace(shape, 0, q.device)
            _lib.check(_lib.lib().bt_linear_attention(
                C.byref(shape), _heads(q), _heads(k), _heads(v), _ptr(state), _heads(out),
                final.data_ptr(), _ptr(ws), n, torch.cuda.current_stream().cuda_stream))
        ctx.save_for_backward(q, k, v, log_decay, state, reset)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, state, reset = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 7
        dout = torch.zeros_like(v) if dout is None else _rows(dout.to(v.dtype))
        dfinal = None if dfinal is None else dfinal.contiguous()
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dstate = torch.empty(q.shape[0], q.shape[2], q.shape[3], v.shape[3], dtype=torch.float32,
                             device=q.device)
        with _on(q.device):
            shape = _shape(q, v, log_decay, reset, ctx.scale)
            ws, n = _workspace(shape, 1, q.device)
            _lib.check(_lib.lib().bt_linear_attention_backward(
                C.byref(shape), _heads(q), _heads(k), _heads(v), _ptr(state), _heads(dout),
                _ptr(dfinal), _heads(dq), _heads(dk), _heads(dv), dstate.data_ptr(), _ptr(ws), n,
                torch.cuda.current_stream().cuda_stream))
        return dq, dk, dv, None, (dstate if ctx.needs_input_grad[4] else None), None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     state: torch.Tensor | None = None, reset: torch.Tensor | None = None, *,
                     scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, final state) of the steps, from `state` (None: zeros). `scale` is 1 / sqrt(key
    features) unless given."""
    _check("linear_attention", q, k, v, log_decay, state, reset)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    return _LinearAttention.apply(q, k, v, log_decay, state, reset, scale)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          log_decay: torch.Tensor, state: torch.Tensor,
                          reset: torch.Tensor | None = None, *, scale: float | None = None,
                          new_state: torch.Tensor | None = None
                          ) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, new state) of one acting step: q, k [batch, heads, key features], v [batch, heads,
    value features], reset [batch]. `new_state` takes the updated state (it may be `state` itself);
    a new tensor unless given. It has no gradient: train through `linear_attention`."""
    _check("linear_attention_step", q, k, v, log_decay, state, reset)
    if state is None:
        raise ValueError("linear_attention_step: a state is expected")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or state.requires_grad):
        raise ValueError("linear_attention_step has no gradient: use linear_attention, or detach")
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    if new_state is None:
        new_state = torch.empty(state.shape, dtype=torch.float32, device=q.device)
    elif (new_state.shape != state.shape or new_state.dtype != torch.float32
          or new_state.device != q.device or not new_state.is_contiguous()):
        raise ValueError(f"linear_attention_step: new_state {tuple(new_state.shape)} "
                         f"{new_state.dtype}: a contiguous {tuple(state.shape)} float32 tensor expected")
    elif new_state.data_ptr() != state.data_ptr() and _overlap(new_state, state):
        raise ValueError("linear_attention_step: new_state overlaps state in part")
    state = state.contiguous()
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    with _on(q.device):
        shape = _shape(q, v, log_decay, reset, scale)
        _lib.check(_lib.lib().bt_linear_attention_step(
            C.byref(shape), _heads(q), _heads(k), _heads(v), state.data_ptr(), out.data_ptr(),
            new_state.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return out, new_state


def _span(t):
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a, b):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1
