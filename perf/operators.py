"""The operators of a training step of the bf16 layer and of its block, as cases that can be timed and compared.

Kinds of case:
  norm_grad    the gradients of CliffordLayerNorm: of its input (plus the residual branch's gradient where
               there is one), of gamma and of beta
  weight_grad  the experts' weight and bias gradients from bf16 rows grouped by expert, ragged
  input_grad   the gradient of such rows through the experts' weights and the activation in front of them,
               the weights' device layout included (a step updates them, so each step lays them out)
  router_grad  the gradient of the routing weights back to the logits, or through the grade energies to
               the tokens and to the router's weight and bias

Multivectors are 8 values in the order 1, e1, e2, e3, e12, e13, e23, e123.  Pauli half-rows hold a row of d
multivectors as the columns b = 0, 1 of their complex 2x2 matrices: (rows, 2, d, 4), the four values the real
and imaginary parts of the column's entries c = 0 and c = 1.

``own`` chooses between the plain forms (elementary torch operations in 32 bits) and this package's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def _norm(N, d, dtype, residual):
    return dict(kind="norm_grad", N=N, d=d, dtype=dtype, residual=residual)


def _rows(kind, product, N, d, F, E, k, load="even", act="none"):
    return dict(kind=kind, product=product, N=N, d=d, F=F, E=E, k=k, load=load, act=act)


def _router(form, N, d, E, k, dtype):
    return dict(kind="router_grad", form=form, N=N, d=d, E=E, k=k, dtype=dtype)


def listed():
    return [
        # the norm in front of the smallest model's layer, a batch of 2 x 128 tokens
        dict(_norm(256, 64, "f32", False), name="norm_small"),
        # a batch of odd length through a width that is no power of two, inside a block with its residual
        dict(_norm(1500, 100, "bf16", True), name="norm_ragged"),
        # the norm of the 12-layer model's block, 8 prompts of 4096 tokens, with its residual
        dict(_norm(32768, 256, "bf16", True), name="norm_large"),
        # the up product's weight gradient of the smallest model's layer (tokens gathered by their expert)
        dict(_rows("weight_grad", "up", 256, 64, 256, 8, 2), name="weight_small"),
        # the down product's of a batch of odd length, widths that are no power of two
        dict(_rows("weight_grad", "down", 1500, 100, 300, 12, 3, "skewed"), name="weight_ragged"),
        # the up product's of a large batch, expert load skewed by Zipf's law
        dict(_rows("weight_grad", "up", 8192, 128, 512, 32, 4, "zipf"), name="weight_large"),
        # the hidden rows' gradient of the smallest model's layer, through gelu
        dict(_rows("input_grad", "down", 256, 64, 256, 8, 2, "even", "gelu"), name="input_small"),
        # the same of a large batch, expert load skewed by Zipf's law
        dict(_rows("input_grad", "down", 8192, 128, 512, 32, 4, "zipf", "gelu"), name="input_large"),
        # the tokens' gradient of one layer of the 12-layer model (64 experts' weights, mildly skewed)
        dict(_rows("input_grad", "up", 4096, 256, 1024, 64, 2, "skewed"), name="input_wide"),
        # the smallest model's grade-energy router
        dict(_router("energy", 256, 64, 8, 2, "f32"), name="router_small"),
        # the router of the 12-layer model on 8 prompts of 4096 tokens
        dict(_router("energy", 32768, 256, 64, 2, "bf16"), name="router_large"),
        # a caller's own logits: the routing's part alone
        dict(_router("logits", 16384, 128, 32, 4, "f32"), name="router_logits"),
    ]


def _log_int(rng, lo, hi, odd=0.4):
    """A whole number of [lo, hi], spread over its logarithm; else rounded to a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() >= odd:
        v = max(8, (v + 4) // 8 * 8)
    return min(max(v, lo), hi)


def draw(rng):
    kind = rng.choice(["norm_grad", "weight_grad", "input_grad", "router_grad"])
    if kind == "norm_grad":
        d = _log_int(rng, 8, 1024)
        return _norm(_log_int(rng, 1, 32768 * 256 // max(d, 256)), d, rng.choice(["f32", "bf16", "bf16"]),
                     rng.random() < 0.5)
    E = rng.choice([4, 8, 12, 16, 32, 64])
    k = rng.choice([2, 2, 3, 4, 8])
    if kind == "router_grad":
        d = _log_int(rng, 8, 512)
        return _router(rng.choice(["energy", "energy", "logits"]), _log_int(rng, 1, 32768 * 256 // max(d, 256)), d, E,
                       min(k, E), rng.choice(["f32", "bf16", "bf16"]))
    k = min(rng.choice([1, k]), E)
    d, F = 2 * _log_int(rng, 8, 128), 2 * _log_int(rng, 16, 512)
    N = _log_int(rng, 1, min(8192, 8192 * 4 * 128 * 512 // (k * d * F)))
    return _rows(kind, rng.choice(["up", "down"]), N, d, F, E, k, rng.choice(["even", "skewed", "zipf"]),
                 rng.choice(["gelu", "relu", "sigmoid"]) if kind == "input_grad" and rng.random() < 0.7 else "none")


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

_MASKS = (0, 1, 2, 4, 3, 5, 6, 7)  # generators of each blade
_GRADES = (0, 1, 1, 1, 2, 2, 2, 3)
_REVERSE = (1.0, 1.0, 1.0, 1.0, -1.0, -1.0, -1.0, -1.0)


def _sign(a, b):
    """The sign of blade a times blade b, given by their generators."""
    return -1.0 if sum(bin(a >> (s + 1)).count("1") for s in range(3) if b >> s & 1) % 2 else 1.0


# _TABLE[p][q][r]: blade p times blade q is that times blade r
_TABLE = [[[_sign(a, b) if c == a ^ b else 0.0 for c in _MASKS] for b in _MASKS] for a in _MASKS]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def rn(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    return g, rn


def _logits(c, g, rn):
    """Router logits of an even, mildly skewed or Zipf-like load."""
    N, E, k = c["N"], c["E"], c["k"]
    if c["load"] != "zipf":
        return rn(N, E) + (0.5 * rn(E)[None, :] if c["load"] == "skewed" else 0.0)
    ranking = torch.randperm(E, generator=g, device="cuda")
    p = torch.arange(1, E + 1, device="cuda", dtype=torch.float64) ** -1.2
    chosen = torch.multinomial((p / p.sum()).float().expand(N, E), k, replacement=False, generator=g)
    steps = (k - torch.arange(k, device="cuda", dtype=torch.float32)).expand(N, k)
    return (0.1 * rn(N, E)).scatter_add_(1, ranking[chosen], steps)


def _grouped(c, g, rn):
    """Rows grouped by expert: their tokens, the experts' bounds on the device and their sizes on the host."""
    idx = torch.topk(_logits(c, g, rn), c["k"], dim=1).indices
    counts = torch.bincount(idx.reshape(-1), minlength=c["E"])
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    perm = (torch.argsort(idx.reshape(-1), stable=True) // c["k"]).to(torch.int32)
    return dict(perm=perm, offsets=offsets, sizes=counts.tolist())


def prepare(case, seed):
    c = case
    g, rn = _generator(seed)
    N, d = c["N"], c["d"]
    if c["kind"] == "norm_grad":
        dt = DTYPES[c["dtype"]]
        gamma = 0.1 * rn(d, 8)
        gamma[:, 0] += 1.0
        return dict(c=c, x=rn(N, d, 8).to(dt), dy=(0.02 * rn(N, d, 8)).to(dt), gamma=gamma,
                    residual=(0.02 * rn(N, d, 8)).to(dt) if c["residual"] else None,
                    table=torch.tensor(_TABLE, device="cuda"), reverse=torch.tensor(_REVERSE, device="cuda"))
    if c["kind"] == "router_grad":
        E, k = c["E"], c["k"]
        grades = torch.tensor(_GRADES, device="cuda")
        # tokens whose energy lies in other grades from one to the next
        x = (rn(N, d, 8) * torch.exp(0.7 * rn(N, 1, 4))[..., grades]).to(DTYPES[c["dtype"]])
        weight, bias = 2.0 * rn(E, 4), 0.1 * rn(E)
        logits = _signature(x.float())[1] @ weight.T + bias if c["form"] == "energy" else rn(N, E)
        p, idx = torch.topk(torch.softmax(logits, 1), k, dim=1)
        return dict(c=c, x=x, weight=weight, bias=bias, logits=logits, idx=idx.to(torch.int32),
                    w=p / (p.sum(1, keepdim=True) + 1e-12), dw=rn(N, k), grades=grades)
    F, E, P = c["F"], c["E"], N * c["k"]
    st = dict(c=c, **_grouped(c, g, rn))
    up = c["product"] == "up"
    # entries of the half-rows of multivectors of N(0, 1) values are N(0, 2)
    st["dy"] = (0.02 * rn(P, 2, F if up else d, 4)).bfloat16()
    if c["kind"] == "weight_grad":
        st["a"] = (math.sqrt(2.0) * (rn(N, 2, d, 4) if up else rn(P, 2, F, 4))).bfloat16()
        st["gather"] = st["perm"] if up else None
        return st
    d_out, d_in = (F, d) if up else (d, F)  # of the product whose input's gradient this is
    st["w"] = rn(E, d_out, d_in, 8) / math.sqrt(8.0 * d_in)
    st["h_pre"] = rn(P, d_in, 8).bfloat16() if c["act"] != "none" else None
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(state):
    c = state["c"]
    if own:
        return _run_own(c, state)
    if c["kind"] == "norm_grad":
        return _norm_grad(state["dy"], state["x"], state["gamma"], state["residual"], state["table"], state["reverse"])
    if c["kind"] == "router_grad":
        return _router_grad(state, c)
    dy = _matrices(state["dy"]).split(state["sizes"])
    if c["kind"] == "weight_grad":
        a = state["a"] if state["gather"] is None else state["a"][state["gather"].long()]
        a = _matrices(a).split(state["sizes"])
        return dict(dw=torch.stack([_weight_grad(x, y) for x, y in zip(dy, a)]),
                    db=torch.stack([_blades(x.sum(0).permute(1, 2, 0)) for x in dy]))
    w = _entries(state["w"]).permute(0, 1, 3, 2, 4)  # (E, d_out, a, d_in, c)
    m = torch.cat([_input_grad(x, y) for x, y in zip(dy, w.unbind(0))])  # (P, b, d_in, c)
    grad = _blades(m.permute(0, 2, 3, 1))
    if c["act"] != "none":
        grad = _act_grad(state["h_pre"].float(), grad, c["act"])
    return _half_rows(grad).bfloat16() if c["product"] == "down" else grad.bfloat16()


def _run_own(c, state):
    from yggdrasil_amd import ops

    if c["kind"] == "norm_grad":
        dx, dgamma, dbeta = ops.clifford_layer_norm_backward(state["dy"], state["x"], state["gamma"], EPS,
                                                             residual_grad=state["residual"])
        return dict(dx=dx, dgamma=dgamma, dbeta=dbeta)
    if c["kind"] == "router_grad":
        if c["form"] == "logits":
            return dict(dlogits=ops.route_backward(state["idx"], state["w"], state["dw"], c["E"]))
        dx, dweight, dbias = ops.route_energy_backward(state["x"], state["weight"], state["idx"], state["w"],
                                                       state["dw"])
        return dict(dx=dx, dweight=dweight, dbias=dbias)
    if c["kind"] == "weight_grad":
        dw, db = ops.grouped_weight_grad_pauli(state["dy"], state["a"], state["offsets"], c["E"],
                                               gather=state["gather"])
        return dict(dw=dw, db=db)
    adjoint = ops.prepare_adjoint_weights(state["w"], "pauli")
    return ops.pauli_grouped_input_grad(state["dy"], adjoint, state["offsets"], h_pre=state["h_pre"], act=c["act"],
                                        y_layout="pauli" if c["product"] == "down" else "blade")


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _matrices(rows):
    """Half-rows (R, 2, d, 4) as complex columns (R, b, d, c)."""
    return torch.view_as_complex(rows.float().reshape(*rows.shape[:3], 2, 2))


def _entries(w):
    """Multivectors (..., 8) as complex matrices (..., a, c)."""
    s, v1, v2, v3, b12, b13, b23, t = w.unbind(-1)
    re = torch.stack([s + v3, v1 - b13, v1 + b13, s - v3], -1)
    im = torch.stack([t + b12, b23 - v2, b23 + v2, t - b12], -1)
    return torch.complex(re, im).reshape(*w.shape[:-1], 2, 2)


def _blades(m):
    """Complex matrices (..., 2, 2) as multivectors (..., 8)."""
    (u00, v00), (u01, v01), (u10, v10), (u11, v11) = [
        (e.real, e.imag) for e in (m[..., 0, 0], m[..., 0, 1], m[..., 1, 0], m[..., 1, 1])]
    return 0.5 * torch.stack([u00 + u11, u10 + u01, v10 - v01, u00 - u11, v00 - v11, u10 - u01, v10 + v01, v00 + v11],
                             -1)


def _half_rows(x):
    """Multivectors (R, d, 8) as half-rows (R, 2, d, 4)."""
    return torch.view_as_real(_entries(x).permute(0, 3, 1, 2)).reshape(x.shape[0], 2, x.shape[1], 4)


def _weight_grad(dy, a):
    """dW_ji = sum_r M(dy_rj) M(a_ri)^H of one expert's rows: (R, b, j, a), (R, b, i, c) -> (j, i, 8)."""
    j, i = dy.shape[2], a.shape[2]
    m = dy.reshape(-1, 2 * j).T @ a.conj().reshape(-1, 2 * i)
    return _blades(m.reshape(j, 2, i, 2).permute(0, 2, 1, 3))


def _input_grad(dy, w):
    """sum_j M(W_ji)^H M(dy_rj) of one expert's rows: (R, b, j, a), (j, a, i, c) -> (R, b, i, c)."""
    j, i = w.shape[0], w.shape[2]
    return (dy.reshape(-1, 2 * j) @ w.conj().reshape(2 * j, 2 * i)).reshape(dy.shape[0], 2, i, 2)


def _act_grad(h, g, act):
    """The grade-wise activation's gradient: grade 0 by f', grades 1 and 2 by f of their length, grade 3 by tanh'."""
    if act == "relu":
        return torch.cat([g[..., :1] * (h[..., :1] > 0), g[..., 1:7], g[..., 7:] * (h[..., 7:] != 0)], -1)

    def f(v):
        if act == "sigmoid":
            s = 1.0 / (1.0 + torch.exp(-v))
            return s, s * (1.0 - s)
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (v + 0.044715 * v * v * v))
        return 0.5 * v * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * k * (1.0 + 3.0 * 0.044715 * v * v)

    def gate(v, u):
        mag = torch.sqrt((v * v).sum(-1, keepdim=True) + 1e-12)
        n = v / mag
        y, dy = f(mag)
        return (y / mag) * u + (dy - y / mag) * (n * u).sum(-1, keepdim=True) * n

    t = torch.tanh(h[..., 7:])
    return torch.cat([g[..., :1] * f(h[..., :1])[1], gate(h[..., 1:4], g[..., 1:4]), gate(h[..., 4:7], g[..., 4:7]),
                      g[..., 7:] * (1.0 - t * t)], -1)


def _norm_grad(dy, x, gamma, residual, table, reverse):
    """y_i = gamma_i x_i / rms + beta_i, rms^2 the mean over i of |x_i|^2, plus 2 eps."""
    N, d, _ = x.shape
    u, v = dy.float(), x.float()
    rms = torch.sqrt((v * v).sum(-1).mean(-1) + 2.0 * EPS)[:, None, None]
    xh = v / rms
    left = ((gamma * reverse) @ table.reshape(8, 64)).reshape(d, 8, 8)  # of the reversed gamma
    gx = torch.bmm(u.transpose(0, 1).contiguous(), left).transpose(0, 1)
    dx = (gx - xh * (gx * xh).sum((-2, -1), keepdim=True) / d) / rms
    if residual is not None:
        dx = dx + residual.float()
    pairs = torch.bmm(u.permute(1, 2, 0).contiguous(), (xh * reverse).transpose(0, 1).contiguous())  # (d, p, q)
    return dict(dx=dx.to(x.dtype), dgamma=pairs.reshape(d, 64) @ table.reshape(64, 8), dbeta=u.sum(0))


def _signature(v):
    """A token's energy in each grade, as shares of their sum, and that sum."""
    e = (v * v).sum(-2)
    e = torch.stack([e[..., 0], e[..., 1:4].sum(-1), e[..., 4:7].sum(-1), e[..., 7]], -1)
    total = e.sum(-1, keepdim=True) + 1e-12
    return total, e / total


def _router_grad(st, c):
    """w is the softmax over the chosen logits, so dlogit_s = w_s (g_s - sum_j w_j g_j) and nothing elsewhere."""
    w, g = st["w"], st["dw"]
    dl = w * (g - (w * g).sum(1, keepdim=True))
    dl = torch.zeros(c["N"], c["E"], device=w.device).scatter_(1, st["idx"].long(), dl)
    if c["form"] == "logits":
        return dict(dlogits=dl)
    v = st["x"].float()
    total, share = _signature(v)
    ds = dl @ st["weight"]
    de = (ds - (ds * share).sum(-1, keepdim=True)) / total
    return dict(dx=(2.0 * v * de[:, st["grades"]][:, None, :]).to(st["x"].dtype), dweight=dl.T @ share,
                dbias=dl.sum(0))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    c = case
    mac = 2 * 32  # a geometric product as a product of complex 2x2 matrices: 32 real multiply-adds
    N, d = c["N"], c["d"]
    if c["kind"] == "norm_grad":  # two geometric products and some 40 more operations a multivector
        es = 4 if c["dtype"] == "f32" else 2
        return dict(bytes=8 * N * d * es * (4 if c["residual"] else 3) + 3 * 32 * d, flops=N * d * (2 * mac + 40))
    if c["kind"] == "router_grad":
        E, k = c["E"], c["k"]
        if c["form"] == "logits":
            return dict(bytes=12 * N * k + 4 * N * E, flops=4 * N * k)
        es = 4 if c["dtype"] == "f32" else 2
        return dict(bytes=16 * N * d * es + 12 * N * k + 36 * E, flops=N * (40 * d + 16 * k))
    P, F, E = N * c["k"], c["F"], c["E"]
    touched = E * (1.0 - (1.0 - c["k"] / E) ** N)
    if c["kind"] == "weight_grad":
        rows = P * F + N * d if c["product"] == "up" else P * (d + F)
        return dict(bytes=16 * rows + 4 * N * c["k"] + 32 * E * (F * d + (F if c["product"] == "up" else d)),
                    flops=mac * P * d * F)
    rows = P * (d + F) + (P * (d if c["product"] == "up" else F) if c["act"] != "none" else 0)
    return dict(bytes=16 * rows + 32 * touched * F * d, flops=mac * P * d * F)


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------


def _blade_rows64(rows):
    """Half-rows (R, 2, d, 4) -> (R, d, 8): each blade's coefficient is half the trace with its matrix."""
    r = rows.double().reshape(rows.shape[0], 2, rows.shape[2], 2, 2)  # [r, b, i, c, re / im]
    re, im = r[..., 0], r[..., 1]
    return 0.5 * torch.stack([
        re[:, 0, :, 0] + re[:, 1, :, 1], re[:, 0, :, 1] + re[:, 1, :, 0], im[:, 0, :, 1] - im[:, 1, :, 0],
        re[:, 0, :, 0] - re[:, 1, :, 1], im[:, 0, :, 0] - im[:, 1, :, 1], re[:, 0, :, 1] - re[:, 1, :, 0],
        im[:, 0, :, 1] + im[:, 1, :, 0], im[:, 0, :, 0] + im[:, 1, :, 1]], -1)


def _act64(v, act):
    f = {"gelu": lambda u: 0.5 * u * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (u + 0.044715 * u ** 3))),
         "relu": lambda u: torch.clamp(u, min=0.0), "sigmoid": torch.sigmoid}[act]
    parts = [f(v[..., 0:1])]
    for lo in (1, 4):
        m = v[..., lo:lo + 3]
        mag = torch.sqrt((m * m).sum(-1, keepdim=True) + 1e-12)
        parts.append(m / mag * f(mag) if act != "relu" else m)
    return torch.cat(parts + [v[..., 7:8] if act == "relu" else torch.tanh(v[..., 7:8])], -1)


def exact(case, seed):
    with torch.enable_grad():
        return _exact(case, prepare(case, seed))


def _exact(c, st):
    dev = "cuda"
    table = torch.tensor(_TABLE, device=dev, dtype=torch.float64)
    if c["kind"] == "norm_grad":
        x, gamma = st["x"].double().requires_grad_(True), st["gamma"].double().requires_grad_(True)
        beta = torch.zeros_like(gamma).requires_grad_(True)
        xh = x / torch.sqrt((x * x).sum((-2, -1), keepdim=True) / c["d"] + 2.0 * EPS)
        y = beta.expand_as(x)
        for p in range(8):  # gamma's blade p times every blade of xh
            y = y + gamma[:, p:p + 1] * (xh @ table[p])
        dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), st["dy"].double())
        return dict(dx=dx if st["residual"] is None else dx + st["residual"].double(), dgamma=dgamma, dbeta=dbeta)
    if c["kind"] == "router_grad":
        energy = c["form"] == "energy"
        if energy:
            x = st["x"].double().requires_grad_(True)
            weight, bias = st["weight"].double().requires_grad_(True), st["bias"].double().requires_grad_(True)
            e = torch.stack([(x[..., lo:hi] ** 2).sum((-2, -1)) for lo, hi in ((0, 1), (1, 4), (4, 7), (7, 8))], -1)
            logits = (e / (e.sum(-1, keepdim=True) + 1e-12)) @ weight.T + bias
        else:
            logits = st["logits"].double().requires_grad_(True)
        p = torch.softmax(logits, 1).gather(1, st["idx"].long())
        w = p / (p.sum(1, keepdim=True) + 1e-12)
        grads = torch.autograd.grad(w, (x, weight, bias) if energy else (logits,), st["dw"].double())
        return dict(zip(("dx", "dweight", "dbias") if energy else ("dlogits",), grads))
    dy = _blade_rows64(st["dy"]).split(st["sizes"])
    if c["kind"] == "weight_grad":  # dW_ji = sum_r dy_rj ~a_ri
        a = _blade_rows64(st["a"])
        a = (a if st["gather"] is None else a[st["gather"].long()]).split(st["sizes"])
        rev = torch.tensor(_REVERSE, device=dev, dtype=torch.float64)
        dw = []
        for u, v in zip(dy, a):
            right = torch.einsum("riq,pqs->rpis", v * rev, table)  # blade p of dy meets every blade of ~a
            dw.append((u.permute(1, 0, 2).reshape(u.shape[1], -1) @ right.reshape(-1, v.shape[1] * 8)).reshape(
                u.shape[1], v.shape[1], 8))
        return dict(dw=torch.stack(dw), db=torch.stack([u.sum(0) for u in dy]))
    grads = []
    for u, w in zip(dy, st["w"].double().unbind(0)):  # y_j = sum_i W_ji x_i, so the gradient of x_i is its transpose
        j, i = w.shape[:2]
        dense = torch.einsum("jip,pqs->iqjs", w, table).reshape(i * 8, j * 8)
        grads.append((u.reshape(-1, j * 8) @ dense.T).reshape(-1, i, 8))
    grad = torch.cat(grads)
    if c["act"] != "none":
        h = st["h_pre"].double().requires_grad_(True)
        (grad,) = torch.autograd.grad(_act64(h, c["act"]), h, grad)
    if c["product"] == "up":
        return grad
    s, v1, v2, v3, b12, b13, b23, t = grad.unbind(-1)
    columns = [torch.stack([s + v3, t + b12, v1 + b13, b23 + v2], -1), torch.stack([v1 - b13, b23 - v2, s - v3, t - b12], -1)]
    return torch.stack(columns, 1)
