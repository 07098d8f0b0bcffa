"""The float64 training oracle against finite differences of the forward definitions (CPU)."""

import numpy as np
import pytest

import _train_oracle as to

STEP = 1e-6


def _numeric(f, x, g):
    """sum(g * f(x)) differentiated by central differences, value by value."""
    out = np.zeros_like(x)
    flat, res = x.reshape(-1), out.reshape(-1)
    for n in range(flat.size):
        keep = flat[n]
        flat[n] = keep + STEP
        up = (g * f(x)).sum()
        flat[n] = keep - STEP
        dn = (g * f(x)).sum()
        flat[n] = keep
        res[n] = (up - dn) / (2 * STEP)
    return out


def _close(a, b):
    # central differences: h^2 / 6 of the third derivative and 1e-16 / h of cancellation, both below 1e-8 here
    assert np.abs(a - b).max() <= 1e-7 * (1 + np.abs(b).max())


def _gp(a, b):
    return np.einsum("...p,...q,pqs->...s", a, b, to.TABLE)


def test_pauli_map_is_the_algebra():
    g = np.random.default_rng(0)
    a, b = g.standard_normal((5, 8)), g.standard_normal((5, 8))

    def mat(v):
        m = (v @ to.TO_PAULI).reshape(-1, 2, 2, 2)
        return m[..., 0] + 1j * m[..., 1]

    assert np.allclose(mat(_gp(a, b)), mat(a) @ mat(b))
    assert np.allclose(mat(a * to.REVERSE), np.conj(np.swapaxes(mat(a), 1, 2)))
    x = g.standard_normal((3, 4, 8))
    assert np.allclose(to.blade_rows(to.half_rows(x)), x)


@pytest.mark.parametrize("eps", [1e-6, 0.3])
def test_norm(eps):
    g = np.random.default_rng(1)
    x, gamma, dy = g.standard_normal((3, 4, 8)), g.standard_normal((4, 8)), g.standard_normal((3, 4, 8))

    def f(x, gamma):
        return _gp(gamma[None], x / np.sqrt((x * x).sum((1, 2), keepdims=True) / 4 + 2 * eps))

    (dx, dgamma, dbeta), _ = to.norm_grad(dy, x, gamma, eps)
    _close(dx, _numeric(lambda v: f(v, gamma), x, dy))
    _close(dgamma, _numeric(lambda v: f(x, v), gamma, dy))
    assert np.allclose(dbeta, dy.sum(0))


@pytest.mark.parametrize("act", ["none", "gelu", "relu", "sigmoid"])
def test_linear_and_activation(act):
    g = np.random.default_rng(2)
    x, W, dy = g.standard_normal((5, 3, 8)), g.standard_normal((2, 4, 3, 8)), g.standard_normal((5, 4, 8))
    offsets = [0, 2, 5]

    def activate(h):
        if act == "none":
            return h
        if act == "relu":
            return np.concatenate([np.maximum(h[..., :1], 0), h[..., 1:]], -1)
        f = to._gelu if act == "gelu" else to._sigmoid
        parts = [f(h[..., :1])[0]]
        for lo in (1, 4):
            m = np.sqrt((h[..., lo:lo + 3] ** 2).sum(-1, keepdims=True) + 1e-12)
            parts.append(h[..., lo:lo + 3] / m * f(m)[0])
        return np.concatenate(parts + [np.tanh(h[..., 7:])], -1)

    def f(x, W):
        h = activate(x)
        return np.concatenate([np.einsum("jip,riq,pqs->rjs", W[e], h[offsets[e]:offsets[e + 1]], to.TABLE)
                               for e in range(2)])

    grad, _ = to.linear_grad(to.half_rows(dy), W, offsets)
    _close(np.einsum("...ab,...a->...b", to.act_jacobian(x, act), grad), _numeric(lambda v: f(v, W), x, dy))
    dW, db, _, _ = to.weight_grad(to.half_rows(dy), to.half_rows(activate(x)), offsets)
    _close(dW, _numeric(lambda v: f(x, v), W, dy))
    assert np.allclose(db[1], dy[2:].sum(0))


@pytest.mark.parametrize("k", [1, 2, 3])
def test_router(k):
    g = np.random.default_rng(3)
    x, W, b = g.standard_normal((4, 5, 8)), g.standard_normal((6, 4)), g.standard_normal(6)
    gw = g.standard_normal((4, k))

    def logits(x, W, b):
        e = np.stack([(x ** 2).sum(1)[:, to.GRADE == h].sum(1) for h in range(4)], 1)
        return e / (e.sum(1, keepdims=True) + 1e-12) @ W.T + b

    idx = np.argsort(-logits(x, W, b), 1)[:, :k]

    def weights(lg):
        p = np.exp(lg - lg.max(1, keepdims=True))
        p = np.take_along_axis(p / p.sum(1, keepdims=True), idx, 1)
        return p / (p.sum(1, keepdims=True) + 1e-12)

    lg = logits(x, W, b)
    dl, ml = to.route_grad(idx, weights(lg), gw, 6)
    _close(dl, _numeric(weights, lg, gw))
    (dx, dW, db), _ = to.energy_grad(x, W, dl, ml)
    _close(dx, _numeric(lambda v: weights(logits(v, W, b)), x, gw))
    _close(dW, _numeric(lambda v: weights(logits(x, v, b)), W, gw))
    _close(db, _numeric(lambda v: weights(logits(x, W, v)), b, gw))
