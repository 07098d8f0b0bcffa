"""Rows quantized to int8 and their products with int8 weights, in NumPy: codes in fp32 steps as they are defined, sums
of codes as whole numbers, the rest in float64."""

from __future__ import annotations

import numpy as np

from oracle import moe

F32 = np.float32
TINY = F32(2.0 ** -100)


def half_entries(x):
    """(..., 8) float32 -> (..., c, b, re / im) float32: X / 2, each entry one rounded sum of two halves."""
    s, v1, v2, v3, b12, b13, b23, t = np.moveaxis(np.asarray(x, F32) * F32(0.5), -1, 0)
    e = [s + v3, t + b12, v1 - b13, b23 - v2, v1 + b13, b23 + v2, s - v3, t - b12]  # M00, M01, M10, M11
    return np.stack(e, -1).reshape(*s.shape, 2, 2, 2)


def quantize(x):
    """(rows, d, 8) -> codes (rows, d, c, b, re / im) int64 and scales (rows,) float32."""
    e = half_entries(x)
    a = np.abs(e).max((1, 2, 3, 4))
    finite = np.isfinite(a)
    top = np.maximum(np.where(finite, a, 0), TINY).astype(F32)
    inv = F32(127.0) / top
    q = np.rint(np.where(finite[:, None, None, None, None], e, 0) * inv[:, None, None, None, None]).astype(np.int64)
    return q, np.where(finite, top / F32(127.0), F32(np.nan)).astype(F32)


def codes_layout(q):
    """The codes in the layout of ``Int8Rows.codes``."""
    rows, d = q.shape[:2]
    steps = (d + 31) // 32
    out = np.zeros((rows, 2, steps, 2, 4, 16), np.int8)
    for i in range(d):
        for c in range(2):
            out[:, :, i // 32, :, i % 32 // 8, 2 * (i % 8) + c] = q[:, i, c]
    return out


def quantized_weights(w):
    """(E, d_out, d_in, 8) -> codes (E, d_out, d_in, a, c, re / im) int64 and scales (E, d_out) float32."""
    q, s = moe.quantize_int8_pauli(w)
    return q.reshape(*q.shape[:-1], 2, 2, 2).astype(np.int64), s


def product(q, scale, wq, ws, bias):
    """Before the activation, float64: (rows, d_out, 8), and the sum of the magnitudes of what is added in fp32."""
    x = q[..., 0] + 1j * q[..., 1]  # (rows, i, c, b)
    w = wq[..., 0] + 1j * wq[..., 1]  # (j, i, a, c)
    y = np.einsum("jiac,ricb->rjab", w, x) if len(x) else np.zeros((0, len(w), 2, 2), complex)
    y = y * ws.astype(np.float64)[None, :, None, None] * scale.astype(np.float64)[:, None, None, None]
    (a00, a01), (a10, a11) = [[y[:, :, a, b] for b in range(2)] for a in range(2)]

    def blades(f, p, m):
        return np.stack([p(f(a00).real, f(a11).real), p(f(a10).real, f(a01).real), m(f(a10).imag, f(a01).imag),
                         m(f(a00).real, f(a11).real), m(f(a00).imag, f(a11).imag), m(f(a10).real, f(a01).real),
                         p(f(a10).imag, f(a01).imag), p(f(a00).imag, f(a11).imag)], -1)

    out = blades(lambda v: v, np.add, np.subtract)
    size = blades(lambda v: np.abs(v.real) + 1j * np.abs(v.imag), np.add, np.add)
    if bias is not None:
        out, size = out + bias.astype(np.float64), size + np.abs(bias)
    return out, size


def grouped(q, scale, bounds, wq, ws, bias, gather=None):
    """Every expert's product of its rows [bounds[e], bounds[e + 1])."""
    parts = []
    for e in range(len(bounds) - 1):
        r = np.arange(bounds[e], bounds[e + 1])
        r = r if gather is None else gather[r]
        parts.append(product(q[r], scale[r], wq[e], ws[e], None if bias is None else bias[e]))
    return np.concatenate([p[0] for p in parts]), np.concatenate([p[1] for p in parts])


def activate(y, act):
    """The grade-wise activation in float64, and how much of an error of 1 in every value reaches each output."""
    if act == "none":
        return y, np.ones_like(y)
    out, gain = y.copy(), np.full_like(y, 4.0)
    if act == "relu":
        out[..., 0] = np.maximum(y[..., 0], 0)
        return out, np.ones_like(y)

    def f(v):
        if act == "sigmoid":
            return 1 / (1 + np.exp(-v))
        return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))

    out[..., 0], out[..., 7] = f(y[..., 0]), np.tanh(y[..., 7])
    for lo in (1, 4):
        g = y[..., lo:lo + 3]
        n = np.sqrt((g * g).sum(-1, keepdims=True) + 1e-12)
        out[..., lo:lo + 3] = g / n * f(n)
        if act == "sigmoid":  # the direction turns as fast as 1 / n
            gain[..., lo:lo + 3] = 4.0 + 2.0 / n
    return out, gain
