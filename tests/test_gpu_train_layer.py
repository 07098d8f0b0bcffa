"""GPU: a training step of the bf16 layer and of the block (norm, layer, residual) through autograd.

The layer's bf16 backward is a chain of operators that are tested on their own (``test_gpu_train_ops.py``):
here the chain is held to those operators bit for bit, and the whole to float64 autograd of the definition.

Tolerances against float64 are relative in the 2-norm: an array whose values are rounded to bf16 is off by at
most 2^-8 of its norm, products with it by as much again, and independent roundings do not add up to more than
their sum.  The longest chain (dx of a block) has 11: x_norm, its Pauli rows, W_up, h_pre, h, dy, W_down, dh,
W_up again, the slots' rows, dx.  fp32 layers: sums of at most 2^11 terms, 2^-24 each, twice through the chain.
"""

import numpy as np
import pytest
import torch

import _train_oracle as to
from _gpu_helpers import say

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8
F32 = 2.0 ** -24 * 2 ** 11


def _pkg():
    import yggdrasil_amd

    return yggdrasil_amd


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape
    return float((got - want).norm() / max(float(want.norm()), 1e-30))


def _layer(g, d, F, E, k, dtype, router="energy", act="gelu", block=False, **more):
    y = _pkg()
    cfg = y.MoEHLMConfig(d_model=d, d_ff=F, n_experts=E, top_k=k, activation=act, dtype=dtype, router=router,
                         bf16_grad=dtype == torch.bfloat16, **more)
    m = y.CliffordMoEBlockFFN(cfg, device="cuda", grad=True) if block else y.CliffordMoELayer(cfg, device="cuda")
    moe = m.moe if block else m
    n = lambda *s: g.standard_normal(s).astype(np.float32)
    moe.load_reference_weights(router_weight=2 * n(E, 4), router_bias=0.1 * n(E), w_up=n(E, F, d, 8) / np.sqrt(8 * d),
                               b_up=0.1 * n(E, F, 8), w_down=n(E, d, F, 8) / np.sqrt(8 * F), b_down=0.1 * n(E, d, 8))
    if block:
        with torch.no_grad():
            m.ffn_norm.gamma.add_(torch.from_numpy(0.3 * n(d, 8)).cuda())
            m.ffn_norm.beta.copy_(torch.from_numpy(0.1 * n(d, 8)).cuda())
    return m


def _tokens(g, B, T, d, dtype):
    x = g.standard_normal((B, T, d, 8)) * np.exp(0.7 * g.standard_normal((B, T, 1, 4)))[..., to.GRADE]
    return torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()


TABLE = torch.from_numpy(to.TABLE)


def _gp(a, b):
    return torch.einsum("...p,...q,pqs->...s", a, b, TABLE)


def _act64(v, act):
    f = {"gelu": lambda u: 0.5 * u * (1 + torch.tanh(np.sqrt(2 / np.pi) * (u + 0.044715 * u ** 3))),
         "sigmoid": torch.sigmoid, "relu": lambda u: torch.clamp(u, min=0)}[act]
    parts = [f(v[..., :1])]
    for lo in (1, 4):
        m = v[..., lo:lo + 3]
        mag = torch.sqrt((m * m).sum(-1, keepdim=True) + 1e-12)
        parts.append(m if act == "relu" else m / mag * f(mag))
    return torch.cat(parts + [v[..., 7:] if act == "relu" else torch.tanh(v[..., 7:])], -1)


def _reference(moe, x, idx, grad, logits=None, norm=None):
    """Gradients of sum(grad * layer(x)) in float64 on the routing idx: by name."""
    P = {n: p.detach().double().cpu().requires_grad_(True) for n, p in moe.named_parameters()}
    xs = x.detach().double().cpu().reshape(-1, *x.shape[2:]).requires_grad_(True)
    leaves = dict(x=xs, **P)
    h = xs
    if norm is not None:
        leaves["gamma"], leaves["beta"] = (t.detach().double().cpu().requires_grad_(True) for t in (norm.gamma, norm.beta))
        rms = torch.sqrt((xs * xs).sum((1, 2), keepdim=True) / xs.shape[1] + 2 * norm.eps)
        h = _gp(leaves["gamma"][None], xs / rms) + leaves["beta"]
    if logits is not None:
        leaves["logits"] = lg = logits.detach().double().cpu().requires_grad_(True)
    else:
        e = torch.stack([(h[..., lo:hi] ** 2).sum((1, 2)) for lo, hi in ((0, 1), (1, 4), (4, 7), (7, 8))], 1)
        lg = e / (e.sum(1, keepdim=True) + 1e-12) @ P["router_weight"].T + P["router_bias"]
    p = torch.softmax(lg, 1).gather(1, idx.long().cpu())
    w = p / (p.sum(1, keepdim=True) + 1e-12)
    out = xs * 0 if norm is None else xs
    for e in range(P["w_up"].shape[0]):
        t, s = torch.nonzero(idx.cpu() == e, as_tuple=True)
        if len(t):
            u = torch.einsum("jip,niq,pqs->njs", P["w_up"][e], h[t], TABLE) + P["b_up"][e]
            y = torch.einsum("jip,niq,pqs->njs", P["w_down"][e], _act64(u, moe.cfg.activation), TABLE) + P["b_down"][e]
            out = out.index_add(0, t, w[t, s][:, None, None] * y)
    names = list(leaves)
    grads = torch.autograd.grad(out, [leaves[n] for n in names], grad.double().cpu().reshape(out.shape), allow_unused=True)
    return out.detach(), dict(zip(names, grads))


# ---- the bf16 layer's operators ------------------------------------------------------------------


@pytest.mark.parametrize("N,d,F,E,k,act,residual,given", [
    (1, 2, 2, 1, 1, "gelu", False, True), (37, 8, 20, 4, 2, "gelu", True, True), (130, 64, 96, 8, 3, "sigmoid", False, False),
    (70, 18, 34, 5, 1, "relu", True, False), (300, 32, 24, 16, 8, "gelu", True, True), (9, 66, 130, 64, 2, "none", False, True)])
def test_backward_is_the_chain_of_its_operators(N, d, F, E, k, act, residual, given):
    ops = _pkg().ops
    g = torch.Generator(device="cuda").manual_seed(N)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, dout, res = rn(N, d, 8).bfloat16(), rn(N, d, 8).bfloat16(), rn(N, d, 8).bfloat16()
    wu, wd = rn(E, F, d, 8) / (8 * d) ** 0.5, rn(E, d, F, 8) / (8 * F) ** 0.5
    bu, bd = ops.prepare_bias(0.1 * rn(E, F, 8)), ops.prepare_bias(0.1 * rn(E, d, 8))
    kw = dict(logits=rn(N, E)) if given else dict(router_weight=rn(E, 4), router_bias=rn(E))
    pu, pd = ops.prepare_weights(wu, "pauli"), ops.prepare_weights(wd, "pauli")
    say(f"bf16 training step N={N} d={d} F={F} E={E} k={k} {act} residual={residual} logits={given}")
    out, routing, saved = ops.moe_forward_train_bf16(x, k, pu, pd, bu, bd, act, residual=res if residual else None, **kw)
    want, lite = ops.moe_forward(x, k, pu, pd, bu, bd, act, residual=res if residual else None, **kw)
    assert torch.equal(out, want)
    assert all(torch.equal(routing[n], lite[n]) for n in ("topk_idx", "topk_w", "counts", "offsets"))
    au, ad = ops.prepare_adjoint_weights(wu, "pauli"), ops.prepare_adjoint_weights(wd, "pauli")
    dx, dWu, dbu, dWd, dbd, dtw = ops.moe_backward_bf16(dout, saved, routing, au, ad, act, residual=residual,
                                                        routing_grad=True)
    # the same step by step
    idx, w, offsets = routing["topk_idx"], routing["topk_w"], routing["offsets"]
    order = torch.argsort(idx.reshape(-1).long(), stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(N * k, device="cuda")
    perm = (order // k).to(torch.int32)
    xp = ops.pauli_rows_from_blade(x)
    pre = ops.pauli_grouped_linear(xp, pu, offsets, bu, "none", x_layout="pauli", gather=perm, y_layout="blade")
    h = ops.pauli_grouped_linear(xp, pu, offsets, bu, act, x_layout="pauli", gather=perm, y_layout="pauli")
    y = ops.pauli_grouped_linear(h, pd, offsets, bd, "none", x_layout="pauli", y_layout="blade")
    f = dout.float()
    m = torch.stack([f[..., 0] + f[..., 3], f[..., 7] + f[..., 4], f[..., 1] + f[..., 5], f[..., 6] + f[..., 2],
                     f[..., 1] - f[..., 5], f[..., 6] - f[..., 2], f[..., 0] - f[..., 3], f[..., 7] - f[..., 4]], -1)
    dy = (w.reshape(-1)[order][:, None, None] * m[perm.long()]).bfloat16()  # (P, d, [column][entry])
    dy = dy.reshape(N * k, d, 2, 4).permute(0, 2, 1, 3).contiguous()
    dh = ops.pauli_grouped_input_grad(dy, ad, offsets, pre if act != "none" else None, act, y_layout="pauli")
    assert torch.equal(dWd, ops.grouped_weight_grad_pauli(dy, h, offsets, E)[0])
    assert torch.equal(dbd, ops.grouped_weight_grad_pauli(dy, h, offsets, E)[1])
    wgu = ops.grouped_weight_grad_pauli(dh, xp, offsets, E, gather=perm)
    assert torch.equal(dWu, wgu[0]) and torch.equal(dbu, wgu[1])
    rows = ops.pauli_grouped_input_grad(dh, au, offsets).float()[pos.reshape(N, k)]
    acc = f if residual else torch.zeros_like(f)
    for s in range(k):
        acc = acc + rows[:, s]
    assert torch.equal(dx, acc.bfloat16())
    terms = dout.double()[:, None] * y.double()[pos.reshape(N, k)]
    assert bool(((dtw.double() - terms.sum((2, 3))).abs() <= (8 * d + 16) * 2.0 ** -24 * terms.abs().sum((2, 3))).all())


def test_no_tokens():
    ops = _pkg().ops
    w = torch.randn(3, 6, 4, 8, device="cuda")
    pu, pd = ops.prepare_weights(w, "pauli"), ops.prepare_weights(w.transpose(1, 2).contiguous(), "pauli")
    say("bf16 training step of no tokens")
    x = torch.empty(0, 4, 8, device="cuda", dtype=torch.bfloat16)
    out, routing, saved = ops.moe_forward_train_bf16(x, 2, pu, pd, logits=torch.empty(0, 3, device="cuda"))
    got = ops.moe_backward_bf16(x, saved, routing, ops.prepare_adjoint_weights(w, "pauli"),
                                ops.prepare_adjoint_weights(w.transpose(1, 2).contiguous(), "pauli"), routing_grad=True)
    assert out.shape == (0, 4, 8) and got[5].shape == (0, 2)
    assert not any(bool(t.any()) for t in got[1:5]) and not bool(routing["counts"].any())


def test_a_token_that_is_not_finite_stays_alone():
    """NaN and infinite tokens reach their own dx and their experts' gradients, no other token and no other expert."""
    ops = _pkg().ops
    g = torch.Generator(device="cuda").manual_seed(2)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    N, d, F, E = 40, 18, 20, 6
    x, dout = rn(N, d, 8).bfloat16(), rn(N, d, 8).bfloat16()
    logits = rn(N, E)
    logits[[4, 9], 0] += 20.0  # both go to expert 0 alone
    logits[:, 0] -= 10.0
    wu, wd = rn(E, F, d, 8) / 12, rn(E, d, F, 8) / 12
    pu, pd = ops.prepare_weights(wu, "pauli"), ops.prepare_weights(wd, "pauli")
    au, ad = ops.prepare_adjoint_weights(wu, "pauli"), ops.prepare_adjoint_weights(wd, "pauli")

    def step(x, dout):
        _, r, saved = ops.moe_forward_train_bf16(x, 1, pu, pd, logits=logits)
        return ops.moe_backward_bf16(dout, saved, r, au, ad)[:5]

    say("bf16 training step with tokens that are not finite")
    clean = step(x, dout)
    x2, dout2 = x.clone(), dout.clone()
    x2[4], dout2[9] = float("nan"), float("inf")
    got = step(x2, dout2)
    keep = [t for t in range(N) if t not in (4, 9)]
    assert torch.equal(got[0][keep], clean[0][keep])
    assert all(torch.equal(a[1:], b[1:]) for a, b in zip(got[1:], clean[1:]))
    assert not bool(torch.isfinite(got[1][0]).all())


# ---- the modules ------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("router,act,B,T,d,F,E,k", [
    ("energy", "gelu", 2, 33, 32, 48, 6, 2), ("logits", "sigmoid", 1, 41, 18, 20, 8, 3), ("energy", "relu", 3, 5, 34, 64, 4, 4)])
def test_gradients_against_float64(dtype, block, router, act, B, T, d, F, E, k):
    g = np.random.default_rng(B * 100 + T)
    m = _layer(g, d, F, E, k, dtype, router=router, act=act, block=block, router_grad=True)
    moe, norm = (m.moe, m.ffn_norm) if block else (m, None)
    x = _tokens(g, B, T, d, dtype).requires_grad_(True)
    logits = torch.from_numpy(g.standard_normal((B * T, E)).astype(np.float32)).cuda().requires_grad_(router == "logits")
    lg = logits if router == "logits" else None
    grad = torch.from_numpy(g.standard_normal((B, T, d, 8)).astype(np.float32)).cuda().to(dtype)
    say(f"training step {dtype} block={block} {router} {act} B={B} T={T} d={d} F={F} E={E} k={k}")
    out = m(x, logits=lg) if block else m.moe_forward(x, logits=lg)
    out.backward(grad)
    idx = moe.last_routing["topk_idx"]
    want_out, want = _reference(moe, x, idx, grad, logits=lg, norm=norm)
    u = BF16 if dtype == torch.bfloat16 else F32
    n = 11 if dtype == torch.bfloat16 else 2
    assert _rel(out.reshape(want_out.shape), want_out) < n * u
    got = dict(x=x.grad.reshape(want["x"].shape), logits=logits.grad, **{n: p.grad for n, p in moe.named_parameters()})
    if block:
        got["gamma"], got["beta"] = norm.gamma.grad, norm.beta.grad
    # the router's gradients are differences g_s - sum w g of numbers that are this much larger
    for name, ref in want.items():
        if ref is None:
            assert got[name] is None, name
            continue
        scale = 8 if name.startswith("router") or name == "logits" else 1
        assert _rel(got[name], ref) < scale * n * u, (name, _rel(got[name], ref))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_norm_module(dt):
    g = np.random.default_rng(8)
    norm = _pkg().CliffordLayerNorm(20, device="cuda", grad=True)
    with torch.no_grad():
        norm.gamma.add_(torch.from_numpy(g.standard_normal((20, 8)).astype(np.float32)).cuda())
    x = _tokens(g, 2, 9, 20, dt).requires_grad_(True)
    dy = torch.from_numpy(g.standard_normal((2, 9, 20, 8)).astype(np.float32)).to(dt).cuda()
    say(f"norm module {dt}")
    y = norm(x.transpose(0, 1))  # not contiguous
    y.backward(dy.transpose(0, 1))
    want, _ = to.norm_grad(dy.double().cpu().numpy().reshape(18, 20, 8), x.detach().double().cpu().numpy().reshape(18, 20, 8),
                           norm.gamma.detach().double().cpu().numpy())
    for got, ref, u in ((x.grad.reshape(18, 20, 8), want[0], F32 + (BF16 if dt == torch.bfloat16 else 0)),
                        (norm.gamma.grad, want[1], F32), (norm.beta.grad, want[2], F32)):
        assert _rel(got, torch.from_numpy(ref)) < u
    assert torch.equal(norm(x.detach()).detach(), _pkg().ops.clifford_layer_norm(x.detach(), norm.gamma.detach(), norm.beta.detach()))


def test_without_asking_there_is_no_graph():
    y = _pkg()
    say("modules that do not ask for gradients")
    for dt in (torch.float32, torch.bfloat16):
        x = torch.randn(1, 6, 8, 8, device="cuda").to(dt).requires_grad_(True)
        cfg = y.MoEHLMConfig(d_model=8, d_ff=16, dtype=dt)
        assert not y.CliffordLayerNorm(8, device="cuda")(x).requires_grad
        assert not y.CliffordMoEBlockFFN(cfg, device="cuda")(x).requires_grad
        assert y.CliffordMoELayer(cfg, device="cuda").moe_forward(x).requires_grad == (dt == torch.float32)
    layer = y.CliffordMoELayer(y.MoEHLMConfig(d_model=8, d_ff=16), device="cuda")
    layer.moe_forward(torch.randn(1, 6, 8, 8, device="cuda")).sum().backward()
    assert layer.router_weight.grad is None and layer.w_up.grad is not None
    with torch.no_grad():
        m = _layer(np.random.default_rng(0), 8, 16, 4, 2, torch.bfloat16, block=True)
        assert not m(x).requires_grad


def test_graph_and_plain_outputs_agree():
    g = np.random.default_rng(5)
    for dt in (torch.float32, torch.bfloat16):
        m = _layer(g, 16, 24, 4, 2, dt, block=True)
        x = _tokens(g, 2, 40, 16, dt)
        say(f"block with and without a graph {dt}")
        with torch.no_grad():
            want = m(x)
        got = m(x)
        assert got.requires_grad
        if dt == torch.bfloat16:
            assert torch.equal(got, want)
        else:
            assert _rel(got, want.cpu()) < F32


def test_weights_changed_before_the_backward():
    g = np.random.default_rng(6)
    for block in (False, True):
        m = _layer(g, 8, 12, 4, 2, torch.bfloat16, block=block)
        x = _tokens(g, 1, 9, 8, torch.bfloat16)
        say(f"weights changed in place, block={block}")
        out = m(x) if block else m.moe_forward(x)
        with torch.no_grad():
            (m.moe if block else m).w_up.add_(1.0)
        with pytest.raises(RuntimeError, match="modified in place"):
            out.sum().backward()


@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step_captured_and_replayed(block, dtype):
    g = np.random.default_rng(7)
    m = _layer(g, 16, 24, 4, 2, dtype, block=block, router_grad=True)
    params = [p for p in m.parameters()]
    x, grad = _tokens(g, 2, 30, 16, dtype), _tokens(g, 2, 30, 16, dtype)

    def step():
        xi = x.detach().requires_grad_(True)
        out = m(xi) if block else m.moe_forward(xi)
        return (out.detach(), *torch.autograd.grad(out, [xi, *params], grad, allow_unused=True))

    say(f"training step captured, block={block} {dtype}")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    want = [None if t is None else t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(4):
        for t in got:
            if t is not None:
                t.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, want))
        other = step()
        torch.cuda.synchronize()
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(other, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_step_with_its_update(dtype):
    """A graph of forward, backward and a gradient-descent update: every replay trains the updated weights."""
    m = _layer(np.random.default_rng(10), 16, 24, 4, 2, dtype, block=True, router_grad=True)
    params = list(m.parameters())
    x, grad = (_tokens(np.random.default_rng(i), 1, 40, 16, dtype) for i in (11, 12))

    def step():
        out = m(x)
        grads = torch.autograd.grad(out, params, grad)
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.add_(g, alpha=-0.02)
        return out.detach()

    say(f"captured training steps with updates {dtype}")
    start = [p.detach().clone() for p in params]

    def restart():
        with torch.no_grad():
            for p, s in zip(params, start):
                p.copy_(s)

    want = []
    for _ in range(4):
        want.append((step().clone(), [p.detach().clone() for p in params]))
    assert not torch.equal(want[0][0], want[1][0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    restart()
    for o, ps in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and all(torch.equal(p.detach(), q) for p, q in zip(params, ps))


def test_two_steps_at_once():
    """Two batches forward before either goes back: each keeps rows of its own."""
    g = np.random.default_rng(9)
    m = _layer(g, 16, 24, 4, 2, torch.bfloat16, block=True, router_grad=True)
    xs = [_tokens(g, 1, 30 + i, 16, torch.bfloat16).requires_grad_(True) for i in range(2)]
    say("two training steps interleaved")
    alone = [torch.autograd.grad(m(x).float().sum(), [x, m.moe.w_up, m.ffn_norm.gamma, m.moe.router_weight]) for x in xs]
    outs = [m(x) for x in xs]
    for i in (0, 1):
        got = torch.autograd.grad(outs[i].float().sum(), [xs[i], m.moe.w_up, m.ffn_norm.gamma, m.moe.router_weight])
        assert all(torch.equal(a, b) for a, b in zip(got, alone[i]))


@pytest.mark.parametrize("block", [False, True])
def test_layouts_of_a_capture_stay_in_its_graph(block):
    """Weights first laid out in a capture: an eager call before any replay lays them out for itself."""
    g = np.random.default_rng(13)
    m = _layer(g, 16, 24, 4, 2, torch.bfloat16, block=block)
    x = _tokens(g, 1, 20, 16, torch.bfloat16)
    run = (lambda: m(x)) if block else (lambda: m.moe_forward(x))
    say(f"weights first laid out in a capture, block={block}")
    run()
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(1.25)
    other = _layer(np.random.default_rng(13), 16, 24, 4, 2, torch.bfloat16, block=block)
    other.load_state_dict(m.state_dict())
    want = other(x) if block else other.moe_forward(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run().detach()
    assert torch.equal(run(), want)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(run(), want)


@pytest.mark.parametrize("which", ["layer", "block", "norm"])
def test_capture_refused_while_an_eager_graph_lives(which):
    """Refused on the host; without the eager graph the same step is captured."""
    y = _pkg()
    g = np.random.default_rng(14)
    x = _tokens(g, 1, 20, 16, torch.bfloat16)
    if which == "norm":
        m = y.CliffordLayerNorm(16, device="cuda", grad=True)
    else:
        m = _layer(g, 16, 24, 4, 2, torch.bfloat16, block=which == "block")
    run = (lambda: m.moe_forward(x)) if which == "layer" else (lambda: m(x))
    say(f"a capture beside an eager graph of the {which}")
    alive = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            run()
    want = alive.detach().clone()
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run().detach()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_tokens_changed_before_the_backward():
    """A bf16 layer's backward reads its tokens for the router's gradient alone: elsewhere they may be overwritten."""
    g = np.random.default_rng(15)
    x = _tokens(g, 1, 20, 16, torch.bfloat16)
    dout = _tokens(g, 1, 20, 16, torch.bfloat16)
    for more in (dict(), dict(router_grad=True)):
        m = _layer(g, 16, 24, 4, 2, torch.bfloat16, **more)
        say(f"tokens overwritten after the forward {more}")
        want = torch.autograd.grad(m.moe_forward(x.clone()), [m.w_up, m.w_down], dout)
        y = x.clone()
        out = m.moe_forward(y)
        y.zero_()
        if more:
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(out, [m.w_up, m.w_down], dout)
        else:
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, [m.w_up, m.w_down], dout), want))
