"""GPU: the activations' gradients at hidden values far from working sizes, which bf16 rows hold all the same.

With the unit weight the product hands dy on exactly (small whole numbers), so an output is the slope at h times dy,
rounded once to bf16: off by 2^-8 of its value.  The slope itself is some 16 fp32 operations, hardware reciprocals,
roots and exponentials of 1 or 2 steps among them: below 2^-19 of the sum of its terms -- s and m s' z' for gelu, whose
difference is small around its minimum; (slope + f / m) |g| for the grades with a length.  On top, a slope s' = e / (1 + e)^2
holds e = 2^-z2 of an exponent z2 that has two roundings, 2^-24 z2 each: 2^-23 ln 2 z2 < 2^-23 z2 of e.  e below fp32's
normal numbers is zero, so z2 < 126 wherever s' counts: 2^-16 of s' at most (30 in grade 3: z2 = 87, 2^-17.1 allowed,
2^-18.2 seen; with 2^-19 alone no fp32 exponent would pass).
"""

import numpy as np
import pytest
import torch

from _gpu_helpers import say

pytestmark = pytest.mark.gpu

SIZES = [0.0, 1e-3, 1.0, 30.0, 99.0, 101.0, 1e3, 1e5, 3e9, 9e11, 2e12, 1.3e13, 1e17, 1.7e19, 2e19, 1e25, 1e31, 1e37]


def _slopes(h, g, act):
    """The activation's gradient in float64, the size of its terms, and that of those with s'."""
    def f(m):  # value and slope of gelu or the sigmoid at m, and the slope's part with s'
        if act == "gelu":
            c = np.sqrt(2 / np.pi)
            t = np.tanh(c * (m + 0.044715 * m ** 3))
            s = 1 - t * t
            part = np.where(s == 0, 0, 0.5 * m * s * c * (1 + 3 * 0.044715 * m * m))
            return 0.5 * m * (1 + t), 0.5 * (1 + t) + part, part
        e = np.exp(-np.abs(m))
        return np.where(m >= 0, 1, e) / (1 + e), e / (1 + e) ** 2, e / (1 + e) ** 2

    out, size, part = np.empty_like(h), np.empty_like(h), np.empty_like(h)
    _, s, p = f(h[..., 0])
    out[..., 0], part[..., 0] = s * g[..., 0], np.abs(p * g[..., 0])
    size[..., 0] = (np.abs(s - p) + np.abs(p)) * np.abs(g[..., 0])
    out[..., 7] = g[..., 7] / np.cosh(np.minimum(np.abs(h[..., 7]), 300)) ** 2
    size[..., 7] = part[..., 7] = np.abs(out[..., 7])
    for lo in (1, 4):
        c, q = h[..., lo:lo + 3], g[..., lo:lo + 3]
        m = np.sqrt((c * c).sum(-1, keepdims=True) + 1e-12)
        v, s, p = f(m)
        u = c / m
        out[..., lo:lo + 3] = v / m * q + (s - v / m) * (u * q).sum(-1, keepdims=True) * u
        size[..., lo:lo + 3] = (np.abs(s) + v / m) * np.abs(q).max(-1, keepdims=True)
        part[..., lo:lo + 3] = np.abs(p) * np.abs(q).max(-1, keepdims=True)
    return out, size, part


@pytest.mark.parametrize("act", ["gelu", "sigmoid"])
@pytest.mark.parametrize("layout", ["pauli", "blade"])
def test_slopes_of_very_large_hidden_values(act, layout):
    from yggdrasil_amd import ops

    g = np.random.default_rng(31)
    d, reps = 34, 4
    P = len(SIZES) * reps
    h = np.repeat(SIZES, reps)[:, None, None] * np.where(g.random((P, d, 8)) < 0.5, -1, 1) * g.uniform(0.6, 1.0, (P, d, 8))
    h = torch.from_numpy(h.astype(np.float32)).bfloat16()
    dy = g.integers(-8, 9, (P, d, 8)).astype(np.float32)
    w = torch.zeros(1, d, d, 8)
    w[0, torch.arange(d), torch.arange(d), 0] = 1.0
    say(f"slopes of very large hidden values, {act}, {layout} rows")
    adj = ops.prepare_adjoint_weights(w.cuda(), "pauli")
    dyp = ops.pauli_rows_from_blade(torch.from_numpy(dy).bfloat16().cuda())
    offsets = torch.tensor([0, P], dtype=torch.int32, device="cuda")
    kw = dict(out_dtype=torch.float32) if layout == "blade" else {}
    got = ops.pauli_grouped_input_grad(dyp, adj, offsets, h.cuda(), act, y_layout=layout, **kw).cpu().double().numpy()
    want, size, part = _slopes(h.double().numpy(), dy.astype(np.float64), act)
    rounding = 0.0
    if layout == "pauli":  # the matrices' entries: each the sum of two blades, rounded to bf16
        def mat(v):
            s, a, b, c, ab, ac, bc, t = np.moveaxis(v, -1, 0)
            return np.stack([np.stack([s + c, t + ab, a + ac, bc + b], -1), np.stack([a - ac, bc - b, s - c, t - ab], -1)], 1)

        most = lambda v: 2 * v.max(-1)[:, None, :, None]
        want, size, part, rounding = mat(want), most(size), most(part), 2.0 ** -8
    assert np.isfinite(got).all()
    # (outputs below fp32's normal numbers may be flushed)
    assert (np.abs(got - want) <= rounding * np.abs(want) + 2.0 ** -19 * size + 2.0 ** -16 * part + 1e-37).all()
