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
that is not finite may reach other steps of its own episode (the steps of a (batch row, head) from
one reset to the next), never another's.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _heads(t: torch.Tensor) -> _lib.Heads:
    s = t.stride()
    return _lib.Heads(t.data_ptr(), s[0], s[1] if t.ndim == 4 else 0, s[-2])


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tiles(t: torch.Tensor) -> torch.Tensor:
    """_rows(t), and for bfloat16 a copy without gaps where the rows of `t` do not start on the
    16-byte boundaries that the tensor-core kernels read from but the copy's would (a shared head
    expanded over the others, a slice off the boundary)."""
    t = _rows(t)
    if t.dtype != torch.bfloat16 or t.shape[-1] % 8:
        return t
    fits = t.data_ptr() % 16 == 0 and all(
        n <= 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:-1], t.stride()))
    return t if fits else t.clone(memory_format=torch.contiguous_format)


def _device(name, first, *others) -> int:
    """The CUDA device of all the tensors (those that are not None)."""
    index = first.get_device()
    if index < 0:
        raise ValueError(f"{name}: CUDA tensors on one device expected")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name}: CUDA tensors on one device expected")
    return index


def _refuse_tangents(name, *tensors) -> None:
    """Forward-mode derivatives would be dropped: a dual tensor does not require a gradient."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name}: no forward-mode derivative; reverse mode is supported")


def _fits(name, *sizes) -> None:
    """The C entries take sizes as 32-bit integers, and ctypes would cut longer ones short."""
    if max(sizes, default=0) > 0x7fffffff:
        raise ValueError(f"{name}: sizes {sizes}: at most 2^31 - 1 is supported")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _check(name, ndim, q, k, v, log_decay, state, reset) -> int:
    """The device's index."""
    shape, vshape = q.shape, v.shape
    if len(shape) != ndim or k.shape != shape or len(vshape) != ndim or vshape[:-1] != shape[:-1]:
        lead = "[batch, steps, heads" if ndim == 4 else "[batch, heads"
        raise ValueError(f"{name}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: "
                         f"{lead}, features] expected, alike in all but v's features")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{name}: q {q.dtype}, k {k.dtype}, v {v.dtype}: float32 or bfloat16 "
                        "expected, the same for all three")
    if not (1 <= shape[-1] <= 128 and 1 <= vshape[-1] <= 128):
        raise ValueError(f"{name}: heads of {shape[-1]} and {vshape[-1]} features: 1 to 128 "
                         "are supported")
    _fits(name, *shape)
    if log_decay.shape != shape[-2:-1] or log_decay.dtype != torch.float32:
        raise ValueError(f"{name}: log_decay {tuple(log_decay.shape)} {log_decay.dtype}: "
                         f"({shape[-2]},) float32 expected")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: log_decay is a constant and has no gradient; detach it")
    _refuse_tangents(name, q, k, v, log_decay, state)
    if state is not None:
        want = (shape[0], shape[-2], shape[-1], vshape[-1])
        if state.shape != want or state.dtype != torch.float32:
            raise ValueError(f"{name}: state {tuple(state.shape)} {state.dtype}: {want} float32 expected")
    if reset is not None and (reset.shape != shape[:ndim - 2] or reset.dtype != torch.bool):
        raise ValueError(f"{name}: reset {tuple(reset.shape)} {reset.dtype}: "
                         f"{tuple(shape[:ndim - 2])} bool expected")
    return _device(name, q, k, v, log_decay, state, reset)


def _shape(q, v, log_decay, reset, scale) -> _lib.LinearAttentionShape:
    steps = q.shape[1] if q.ndim == 4 else 1
    rs = (0, 0) if reset is None else (reset.stride(0), reset.stride(1) if reset.ndim == 2 else 0)
    return _lib.LinearAttentionShape(
        q.shape[0], steps, q.shape[-2], q.shape[-1], v.shape[-1], _DTYPES[q.dtype], scale,
        log_decay.data_ptr(), None if reset is None else reset.data_ptr(), *rs)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(shape, backward, device):
    n = _lib.lib().bt_linear_attention_workspace(shape, backward)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None), n


def _forward(q, k, v, log_decay, state, reset, scale):
    """(out, final state) and the tensors that the call read."""
    q, k, v, log_decay = _tiles(q), _tiles(k), _tiles(v), log_decay.contiguous()
    state = None if state is None else state.contiguous()
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    final = torch.empty((q.shape[0], q.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32,
                        device=q.device)
    with _lib.on_device(q.get_device()) as stream:
        shape = _shape(q, v, log_decay, reset, scale)
        ws, n = _workspace(shape, 0, q.device)
        _lib.check(_lib.lib().bt_linear_attention(
            shape, _heads(q), _heads(k), _heads(v), _ptr(state), _heads(out), final.data_ptr(),
            _ptr(ws), n, stream))
    return out, final, (q, k, v, log_decay, state, reset)


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, reset, scale):
        out, final, read = _forward(q, k, v, log_decay, state, reset, scale)
        ctx.save_for_backward(*read)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, state, reset = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 7
        _refuse_tangents("linear_attention", dout, dfinal)
        dout = torch.zeros_like(v) if dout is None else _tiles(dout.to(v.dtype))
        dfinal = None if dfinal is None else dfinal.contiguous()
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        dstate = torch.empty((q.shape[0], q.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32,
                             device=q.device)
        with _lib.on_device(q.get_device()) as stream:
            shape = _shape(q, v, log_decay, reset, ctx.scale)
            ws, n = _workspace(shape, 1, q.device)
            _lib.check(_lib.lib().bt_linear_attention_backward(
                shape, _heads(q), _heads(k), _heads(v), _ptr(state), _heads(dout), _ptr(dfinal),
                _heads(dq), _heads(dk), _heads(dv), dstate.data_ptr(), _ptr(ws), n, stream))
        return dq, dk, dv, None, (dstate if ctx.needs_input_grad[4] else None), None, None


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                     state: torch.Tensor | None = None, reset: torch.Tensor | None = None, *,
                     scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, final state) of the steps, from `state` (None: zeros). `scale` is 1 / sqrt(key
    features) unless given."""
    _check("linear_attention", 4, q, k, v, log_decay, state, reset)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not _wants_grad(q, k, v, state):
        return _forward(q, k, v, log_decay, state, reset, scale)[:2]
    return _LinearAttention.apply(q, k, v, log_decay, state, reset, scale)


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                          log_decay: torch.Tensor, state: torch.Tensor,
                          reset: torch.Tensor | None = None, *, scale: float | None = None,
                          new_state: torch.Tensor | None = None
                          ) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, new state) of one acting step: q, k [batch, heads, key features], v [batch, heads,
    value features], reset [batch]. `new_state` takes the updated state (it may be `state` itself,
    overwritten as by torch's own in-place operations, and may overlap nothing else that the call
    reads); a new tensor unless given. It has no gradient: train through `linear_attention`."""
    device = _check("linear_attention_step", 3, q, k, v, log_decay, state, reset)
    if state is None:
        raise ValueError("linear_attention_step: a state is expected")
    _refuse_tangents("linear_attention_step", new_state)
    if _wants_grad(q, k, v, state, new_state):
        raise ValueError("linear_attention_step has no gradient: use linear_attention, or detach")
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    if new_state is None:
        new_state = torch.empty(state.shape, dtype=torch.float32, device=q.device)
    elif (new_state.shape != state.shape or new_state.dtype != torch.float32
          or new_state.get_device() != device or not new_state.is_contiguous()):
        raise ValueError(f"linear_attention_step: new_state {tuple(new_state.shape)} "
                         f"{new_state.dtype}: a contiguous {tuple(state.shape)} float32 tensor expected")
    elif _overlap(new_state, state) and not (new_state.data_ptr() == state.data_ptr()
                                             and state.is_contiguous()):
        raise ValueError("linear_attention_step: new_state overlaps state in part")
    state = state.contiguous()
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    with _lib.on_device(device) as stream:
        _lib.check(_lib.lib().bt_linear_attention_step(
            _shape(q, v, log_decay, reset, scale), _heads(q), _heads(k), _heads(v),
            state.data_ptr(), out.data_ptr(), new_state.data_ptr(), stream))
    if not new_state.is_inference():
        # autograd does not see the kernel's write: a graph that has saved the tensor must notice it
        torch.autograd.graph.increment_version(new_state)
    return out, new_state


def _span(t):
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else -1
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a, b):
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1
