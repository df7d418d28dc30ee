"""The sequence-torso operators in float64 (test infrastructure only): linear attention with a
decay per head, step by step; the norms of queries and keys with the position rotation; the gated
feed-forward layer; and their gradients, written from the same definitions. The `_scale` functions
give the sums of absolute values that bound an implementation's rounding errors.
"""
from __future__ import annotations

import numpy as np


def _f64(*xs):
    return [np.asarray(x, np.float64) for x in xs]


def _keep(reset, batch, steps):
    return np.ones((batch, steps)) if reset is None else 1.0 - np.asarray(reset, np.float64)


def _decay(log_decay):
    with np.errstate(over="ignore"):
        return np.exp(np.asarray(log_decay, np.float64))


def linear_attention(q, k, v, log_decay, state, reset, scale):
    """q, k [B, T, H, Dk], v [B, T, H, Dv], state [B, H, Dk, Dv] -> (out, final state)."""
    q, k, v, s = _f64(q, k, v, state)
    keep, lam = _keep(reset, *q.shape[:2]), _decay(log_decay)
    out = np.empty(v.shape)
    for t in range(q.shape[1]):
        f = keep[:, t, None, None, None] * lam[None, :, None, None]
        s = np.where(keep[:, t, None, None, None] > 0, f * s, 0.0)
        s = s + k[:, t, :, :, None] * v[:, t, :, None, :]
        out[:, t] = scale * np.einsum("bhi,bhij->bhj", q[:, t], s)
    return out, s


def linear_attention_backward(q, k, v, log_decay, state, reset, scale, dout, dfinal):
    """(dq, dk, dv, dstate)."""
    q, k, v, s, dout, r = _f64(q, k, v, state, dout, dfinal)
    keep, lam = _keep(reset, *q.shape[:2]), _decay(log_decay)
    T = q.shape[1]
    dq, dk, dv = np.empty(q.shape), np.empty(k.shape), np.empty(v.shape)
    factor = keep[:, :, None] * lam  # [B, T, H]
    for t in range(T):
        s = factor[:, t, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = scale * np.einsum("bhij,bhj->bhi", s, dout[:, t])
    for t in range(T - 1, -1, -1):
        r = r + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
        dv[:, t] = np.einsum("bhij,bhi->bhj", r, k[:, t])
        dk[:, t] = np.einsum("bhij,bhj->bhi", r, v[:, t])
        r = factor[:, t, :, None, None] * r
    return dq, dk, dv, r


def linear_attention_scale(q, k, v, log_decay, state, reset, scale, dout=None, dfinal=None):
    """The same sums over absolute values: of every product that enters an output."""
    a = [np.abs(np.asarray(x, np.float64)) for x in (q, k, v)]
    s = np.abs(np.asarray(state, np.float64))
    fwd = linear_attention(*a, log_decay, s, reset, abs(scale))
    if dout is None:
        return fwd
    return fwd + linear_attention_backward(*a, log_decay, s, reset, abs(scale), np.abs(dout),
                                           np.abs(dfinal))


def _turn(x, angle, interleaved):
    half = angle.shape[-1]
    c, s = np.cos(angle)[:, :, None], np.sin(angle)[:, :, None]
    y = x.copy()
    a = np.s_[..., 0:2 * half:2] if interleaved else np.s_[..., :half]
    b = np.s_[..., 1:2 * half:2] if interleaved else np.s_[..., half:2 * half]
    y[a] = x[a] * c - x[b] * s
    y[b] = x[b] * c + x[a] * s
    return y


def norm_rotary(x, weight, positions, frequencies, eps, interleaved):
    """x [B, T, H, D] -> y."""
    x, w, f = _f64(x, weight, frequencies)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return _turn(x * r * w, np.asarray(positions, np.float64)[..., None] * f, interleaved)


def norm_rotary_backward(x, weight, positions, frequencies, eps, interleaved, dy):
    """(dx, dweight)."""
    x, w, f, dy = _f64(x, weight, frequencies, dy)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    g = _turn(dy, -np.asarray(positions, np.float64)[..., None] * f, interleaved)
    xh = x * r
    u = g * w
    return r * (u - xh * (u * xh).mean(-1, keepdims=True)), (g * xh).sum((0, 1, 2))


def _act(name, z):
    if name == "silu":
        sig = 1.0 / (1.0 + np.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    if name == "tanh":
        return np.tanh(z), 1.0 - np.tanh(z) ** 2
    if name == "relu":
        return np.maximum(z, 0.0), (z > 0).astype(np.float64)
    return z, np.ones_like(z)


def glu(x, w_gate, w_up, activation):
    x, wg, wu = _f64(x, w_gate, w_up)
    return _act(activation, x @ wg)[0] * (x @ wu)


def glu_backward(x, w_gate, w_up, activation, dh):
    """(dx, dw_gate, dw_up, dG, dU)."""
    x, wg, wu, dh = _f64(x, w_gate, w_up, dh)
    u = x @ wu
    a, slope = _act(activation, x @ wg)
    dg, du = dh * u * slope, dh * a
    return dg @ wg.T + du @ wu.T, x.T @ dg, x.T @ du, dg, du
