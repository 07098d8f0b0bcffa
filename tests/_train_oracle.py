"""The training operators in float64 (numpy), with bounds on what 32-bit and bf16 arithmetic may add.

Plain loops and matrix products over blades, written from the definitions; no GPU needed.  Every
operator returns its result and, next to it, the same sum over absolute values, which the tests
multiply by the roundings that the kernels are allowed.
"""

from __future__ import annotations

import numpy as np

MASKS = (0, 1, 2, 4, 3, 5, 6, 7)  # generators of each blade: 1, e1, e2, e3, e12, e13, e23, e123
GRADE = np.array([0, 1, 1, 1, 2, 2, 2, 3])
REVERSE = np.where(GRADE >= 2, -1.0, 1.0)


def _sign(a, b):
    return -1.0 if sum(bin(a >> (s + 1)).count("1") for s in range(3) if b >> s & 1) % 2 else 1.0


# TABLE[p, q, r]: blade p times blade q is that times blade r
TABLE = np.array([[[_sign(a, b) if c == a ^ b else 0.0 for c in MASKS] for b in MASKS] for a in MASKS])

# the eight reals (re, im) of M00, M01, M10, M11 of each blade's matrix: rows blades, columns entries
TO_PAULI = np.zeros((8, 8))
for _e, (_plus, _minus, _other) in enumerate([(0, None, 3), (7, None, 4), (1, 5, None), (6, 2, None),
                                               (1, None, 5), (6, None, 2), (0, 3, None), (7, 4, None)]):
    TO_PAULI[_plus, _e] = 1.0
    if _other is not None:
        TO_PAULI[_other, _e] = 1.0
    if _minus is not None:
        TO_PAULI[_minus, _e] = -1.0
FROM_PAULI = np.linalg.inv(TO_PAULI)


def half_rows(x):
    """(rows, d, 8) -> (rows, 2, d, 4): column b of every matrix, (re, im) of its entries 0 and 1."""
    m = (np.asarray(x, np.float64) @ TO_PAULI).reshape(*x.shape[:2], 2, 2, 2)  # [a][b][re / im]
    return np.transpose(m, (0, 3, 1, 2, 4)).reshape(x.shape[0], 2, x.shape[1], 4)


def blade_rows(h):
    """The inverse of half_rows."""
    m = np.asarray(h, np.float64).reshape(h.shape[0], 2, h.shape[2], 2, 2)  # [r][b][i][a][re / im]
    return np.transpose(m, (0, 2, 3, 1, 4)).reshape(h.shape[0], h.shape[2], 8) @ FROM_PAULI


def weight_grad(dy, a, offsets):
    """dW[e, j, i] = sum over the expert's rows of dy_j ~a_i, db = sum dy_j; half-rows in, and the sums' magnitudes
    (of the products of matrix entries that make them up)."""
    u, v = blade_rows(dy), blade_rows(a) * REVERSE
    mu, mv = np.abs(np.asarray(dy, np.float64)), np.abs(np.asarray(a, np.float64))
    E = len(offsets) - 1
    dW = np.zeros((E, u.shape[1], v.shape[1], 8))
    db = np.zeros((E, u.shape[1], 8))
    mW, mb = np.zeros_like(dW), np.zeros_like(db)
    for e in range(E):
        s = slice(offsets[e], offsets[e + 1])
        dW[e] = np.einsum("rjp,riq,pqs->jis", u[s], v[s], TABLE, optimize=True)
        db[e] = u[s].sum(0)
        # any blade is half of a sum of two entries, an entry a sum over b and (re, im) of products
        mW[e] = np.einsum("rbjx,rbiy->ji", mu[s], mv[s], optimize=True)[..., None]
        mb[e] = mu[s].sum((0, 1, 3))[:, None]
    return dW, db, mW, mb


def linear_grad(dy, W, offsets):
    """sum_j ~W_e[j, i] dy_j of every expert's rows (half-rows in, blades out) and its magnitude, as above."""
    u = blade_rows(dy)
    mu = np.abs(np.asarray(dy, np.float64))
    W = np.asarray(W, np.float64)
    P, d_in = u.shape[0], W.shape[2]
    g, mg = np.zeros((P, d_in, 8)), np.zeros((P, d_in, 8))
    for e in range(len(offsets) - 1):
        s = slice(offsets[e], offsets[e + 1])
        g[s] = np.einsum("jip,rjq,pqs->ris", W[e] * REVERSE, u[s], TABLE, optimize=True)
        mw = np.abs(W[e] @ TO_PAULI).sum(-1)  # (j, i)
        mg[s] = np.einsum("ji,rbjx->ri", mw, mu[s], optimize=True)[..., None]
    return g, mg


def _gelu(v):
    k = np.sqrt(2.0 / np.pi)
    t = np.tanh(k * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)


def _sigmoid(v):
    s = 1.0 / (1.0 + np.exp(-v))
    return s, s * (1 - s)


def act_jacobian(h, act):
    """d act(h) / dh per multivector: (..., 8, 8), symmetric."""
    h = np.asarray(h, np.float64)
    J = np.zeros(h.shape + (8,))
    if act == "none":
        J[..., range(8), range(8)] = 1.0
        return J
    if act == "relu":
        J[..., range(8), range(8)] = 1.0
        J[..., 0, 0] = h[..., 0] > 0
        J[..., 7, 7] = h[..., 7] != 0
        return J
    f = _gelu if act == "gelu" else _sigmoid
    J[..., 0, 0] = f(h[..., 0])[1]
    J[..., 7, 7] = 1.0 / np.cosh(h[..., 7]) ** 2
    for lo in (1, 4):
        c = h[..., lo:lo + 3]
        m = np.sqrt((c * c).sum(-1) + 1e-12)
        y, dy = f(m)
        n = c / m[..., None]
        J[..., lo:lo + 3, lo:lo + 3] = (y / m)[..., None, None] * np.eye(3) + \
            (dy - y / m)[..., None, None] * n[..., :, None] * n[..., None, :]
    return J


def norm_grad(dy, x, gamma, eps=1e-6, residual=None):
    """dx, dgamma, dbeta of y_i = gamma_i x_i / rms + beta_i, and magnitudes of the sums behind each."""
    dy, x, gamma = (np.asarray(t, np.float64) for t in (dy, x, gamma))
    d = x.shape[1]
    rms = np.sqrt((x * x).sum((1, 2), keepdims=True) / d + 2 * eps)
    xh = x / rms
    gx = np.einsum("ip,tiq,pqs->tis", gamma * REVERSE, dy, TABLE, optimize=True)
    dx = (gx - xh * (gx * xh).sum((1, 2), keepdims=True) / d) / rms
    mgx = np.einsum("ip,tiq,pqs->tis", np.abs(gamma), np.abs(dy), np.abs(TABLE), optimize=True)
    mdx = (mgx + np.abs(xh) * (mgx * np.abs(xh)).sum((1, 2), keepdims=True) / d) / rms
    if residual is not None:
        dx, mdx = dx + residual, mdx + np.abs(residual)
    dgamma = np.einsum("tip,tiq,pqs->is", dy, xh * REVERSE, TABLE, optimize=True)
    mgamma = np.einsum("tip,tiq,pqs->is", np.abs(dy), np.abs(xh), np.abs(TABLE), optimize=True)
    return (dx, dgamma, dy.sum(0)), (mdx, mgamma, np.abs(dy).sum(0))


def route_grad(idx, w, g, E):
    """dlogits of the softmax over the chosen logits, and its magnitude."""
    idx, w, g = np.asarray(idx), np.asarray(w, np.float64), np.asarray(g, np.float64)
    w = w / w.sum(1, keepdims=True)
    dl = w * (g - (w * g).sum(1, keepdims=True))
    ml = w * (np.abs(g) + (w * np.abs(g)).sum(1, keepdims=True))
    out, mag = np.zeros((len(idx), E)), np.zeros((len(idx), E))
    np.put_along_axis(out, idx, dl, 1)
    np.put_along_axis(mag, idx, ml, 1)
    return out, mag


def energy_grad(x, W, dl, ml, add=None):
    """dx, dW, db of logits = share W^T + b from dlogits and their magnitudes."""
    x, W = np.asarray(x, np.float64), np.asarray(W, np.float64)
    e = np.stack([(x ** 2).sum(1)[:, GRADE == h].sum(1) for h in range(4)], 1)
    T = e.sum(1, keepdims=True) + 1e-12
    sh = e / T
    ds, ms = dl @ W, ml @ np.abs(W)
    de = (ds - (ds * sh).sum(1, keepdims=True)) / T
    me = (ms + (ms * sh).sum(1, keepdims=True)) / T
    dx, mx = 2 * x * de[:, GRADE][:, None, :], 2 * np.abs(x) * me[:, GRADE][:, None, :]
    if add is not None:
        dx, mx = dx + add, mx + np.abs(add)
    return (dx, dl.T @ sh, dl.sum(0)), (mx, ml.T @ sh, ml.sum(0))
