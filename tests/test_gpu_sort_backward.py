"""Gradients of dispatch and combine against float64, and of the operators' chain from tokens to output.

Tolerances: dy is one fp32 product (2^-24 of it) and, in Pauli layouts, one sum of two; dtopk_w adds 8 d products, at most
8 d / 64 + 9 additions deep after one rounding each (a lane's chain and the sum over the wave), 2^-24 of the sum of
the magnitudes each; dx at most k + 1 additions.  A bf16 output is off by 2^-8 of its value.
"""

import numpy as np
import pytest
import torch

from _gpu_helpers import bf16_round, say

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _ops():
    from yggdrasil_amd import ops

    return ops


def _host(t):
    return t.double().cpu().numpy()


def _routed(seed, N, E, k):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _ops().route(torch.randn(N, E, generator=g, device="cuda"), k)


def _within(got, want, bound, what):
    off = np.abs(_host(got) - want) - bound - 1e-38
    assert tuple(got.shape) == want.shape and not np.isnan(off).any() and off.max(initial=-1.0) <= 0, (what, off.max())


def _entries(x):
    """(..., 8) -> (..., c, b, re / im)"""
    s, v1, v2, v3, b12, b13, b23, t = np.moveaxis(x, -1, 0)
    return np.stack([s + v3, t + b12, v1 - b13, b23 - v2, v1 + b13, b23 + v2, s - v3, t - b12], -1).reshape(*s.shape, 2, 2, 2)


SIZES = [(1, 1, 1, 1), (1, 70, 8, 8), (5, 3, 4, 2), (64, 64, 8, 2), (257, 33, 16, 4), (130, 128, 64, 3), (300, 100, 12, 5),
         (37, 512, 8, 2), (9, 600, 5, 5)]


@pytest.mark.parametrize("N,d,E,k", SIZES)
@pytest.mark.parametrize("td,ty", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("layout", ["blade", "pauli"])
def test_combine_backward(N, d, E, k, td, ty, layout):
    ops = _ops()
    r = _routed(N + d, N, E, k)
    P = N * k
    g = torch.randn(N, d, 8, device="cuda").to(DT[td])
    y = torch.randn(P, d, 8, device="cuda").to(DT[ty])
    say(f"combine_backward N={N} d={d} E={E} k={k} {td} {ty} {layout}")
    dy, dw = ops.combine_backward(g, y, r, y_layout=layout)
    G, Y, W, S = _host(g), _host(y), _host(r.topk_w), r.slot_pos.cpu().numpy()
    want = np.zeros((P, d, 8))
    want[S.reshape(-1)] = (W[:, :, None, None] * G[:, None]).reshape(P, d, 8)
    bound = U32 * np.abs(want)
    if layout == "pauli":
        e = _entries(want)
        s, v1, v2, v3, b12, b13, b23, t = np.moveaxis(np.abs(want), -1, 0)
        size = np.stack([s + v3, t + b12, v1 + b13, b23 + v2, v1 + b13, b23 + v2, s + v3, t + b12], -1).reshape(e.shape)
        bound = 3 * U32 * size
        if ty == "bf16":
            order = (0, 3, 1, 2, 4)
            want, bound = e.transpose(order).reshape(P, 2, d, 4), bound.transpose(order).reshape(P, 2, d, 4)
        else:
            order = (0, 1, 3, 4, 2)
            want, bound = e.transpose(order), bound.transpose(order)
    if ty == "bf16":
        bound = bound * (1 + U16) + U16 * np.abs(want)
    _within(dy, want, bound, "dy")
    terms = G[:, None] * Y[S]
    _within(dw, terms.sum((-2, -1)), (8 * ((d + 63) // 64) + 10) * U32 * np.abs(terms).sum((-2, -1)), "dw")
    dy2, none = ops.combine_backward(g, None, r, y_layout=layout, out_dtype=DT[ty])
    assert none is None and torch.equal(dy2, dy)


@pytest.mark.parametrize("N,d,E,k", SIZES + [(600, 17, 8, 2), (1000, 5, 4, 1)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("with_add", [False, True])
def test_dispatch_backward(N, d, E, k, dt, with_add):
    ops = _ops()
    r = _routed(N + d, N, E, k)
    dxs = torch.randn(N * k, d, 8, device="cuda").to(DT[dt])
    add = torch.randn(N, d, 8, device="cuda").to(DT[dt]) if with_add else None
    say(f"dispatch_backward N={N} d={d} E={E} k={k} {dt} add={with_add}")
    dx = ops.dispatch_backward(dxs, r, dx_add=add)
    terms = _host(dxs)[r.slot_pos.cpu().numpy()]
    want, size = terms.sum(1), np.abs(terms).sum(1)
    if with_add:
        want, size = want + _host(add), size + np.abs(_host(add))
    bound = k * U32 * size
    if dt == "bf16":
        bound = bound * (1 + U16) + U16 * np.abs(want)
    _within(dx, want, bound, "dx")


def test_more_tokens_than_one_launch():
    """Powers of two as weights, so every product is exact; the rows in reversed order."""
    ops = _ops()
    N, d, k = (1 << 22) + 7, 1, 2
    P = N * k
    say(f"sort gradients of {N} tokens")
    slots = torch.arange(P - 1, -1, -1, device="cuda", dtype=torch.int32).view(N, k)
    w = torch.exp2(-(slots % 3).float())
    r = ops.Routing(slots, w, slots[0], slots[0], slots[0], slots)
    dout = torch.randint(-8, 9, (N, d, 8), device="cuda").float()
    y = torch.randint(-8, 9, (P, d, 8), device="cuda").float()
    dy, dw = ops.combine_backward(dout, y, r)
    back = y.flip(0).view(N, k, 8)
    assert torch.equal(dy.flip(0).view(N, k, 8), w[..., None] * dout)
    assert torch.equal(dw, (dout * back).sum(-1))
    assert torch.equal(ops.dispatch_backward(y, r, dout), (dout[:, 0] + back[:, 0] + back[:, 1])[:, None])


def test_slots_outside_the_rows():
    """A caller who drops slots (a full expert) names rows outside: nothing is read or written for them."""
    ops = _ops()
    N, d, k = 40, 24, 2
    P = 50
    g = torch.Generator().manual_seed(3)
    slots = torch.full((N * k,), -1, dtype=torch.int32)
    at = torch.randperm(N * k, generator=g)[:P - 4]
    slots[at] = torch.randperm(P, generator=g)[:P - 4].to(torch.int32)
    slots[(slots < 0).nonzero()[:5, 0]] = 2 ** 31 - 1
    slots = slots.view(N, k).cuda()
    slots[7] = -1  # a token without any expert
    w = torch.rand(N, k, device="cuda")
    r = ops.Routing(torch.zeros_like(slots), w, slots[0], slots[0], slots[0], slots)
    dout, y = torch.randn(N, d, 8, device="cuda"), torch.randn(P, d, 8, device="cuda")
    say("sort gradients: slots outside the rows")
    keep = (slots >= 0) & (slots < P)
    dy = torch.full((P, d, 8), 5.0, device="cuda")
    dw = torch.full((N, k), 5.0, device="cuda")
    ops.check(ops.lib().ygg_combine_backward(dout.data_ptr(), 0, y.data_ptr(), N, k, d, P, w.data_ptr(), slots.data_ptr(),
                                             dy.data_ptr(), 0, 0, dw.data_ptr(), ops.stream_handle()))
    want = torch.full_like(dy, 5.0)
    tok = torch.arange(N, device="cuda")[:, None].expand(N, k)[keep]
    want[slots[keep].long()] = w[keep][:, None, None] * dout[tok]
    assert torch.equal(dy, want)
    assert (dw[~keep] == 0).all() and (dw[keep] != 5.0).all()
    dx = ops.dispatch_backward(y, r)
    assert (dx[7] == 0).all()
    one = torch.where(keep[:, :, None, None], y[slots.clamp(0, P - 1).long()], torch.zeros((), device="cuda"))
    assert torch.equal(dx, one[:, 0] + one[:, 1])
    none, dw0 = ops.combine_backward(dout, y[:0], r)
    assert none.shape == (0, d, 8) and (dw0 == 0).all()
    assert (ops.dispatch_backward(y[:0], r) == 0).all()


def test_chain_of_operators_against_autograd():
    """dispatch, one expert product, combine, and their gradients, as a caller chains them, against float64 autograd; the
    chain's rows are bf16, so each of its five roundings is 2^-8 of the largest value that it meets."""
    ops = _ops()
    N, d, F, E, k = 200, 32, 48, 8, 2
    torch.manual_seed(5)
    logits = torch.randn(N, E, device="cuda")
    r = ops.route(logits, k)
    x = torch.randn(N, d, 8, device="cuda").bfloat16()
    w = torch.randn(E, F, d, 8, device="cuda") / (8 * d) ** 0.5
    dout = torch.randn(N, F, 8, device="cuda").bfloat16()
    say("chain: dispatch, product, combine and back")
    xs = ops.dispatch(x, r)
    y = ops.pauli_grouped_linear(xs, ops.prepare_weights(w, "pauli"), r.offsets)
    ops.combine(y, r)
    dy, dw = ops.combine_backward(dout, y, r, y_layout="pauli")
    dxs = ops.pauli_grouped_input_grad(dy, ops.prepare_adjoint_weights(w, "pauli"), r.offsets)
    dx = ops.dispatch_backward(dxs, r)
    gw, _ = ops.grouped_weight_grad_pauli(dy, ops.pauli_rows_from_blade(xs), r.offsets, E)
    # float64: geometric products by their table
    from oracle import cl3

    table = torch.zeros(8, 8, 8, dtype=torch.float64, device="cuda")
    for p in range(8):
        for q in range(8):
            a, b = np.zeros((1, 8)), np.zeros((1, 8))
            a[0, p] = b[0, q] = 1
            table[p, q] = torch.from_numpy(np.asarray(cl3.geom_prod(a, b))[0]).cuda()
    X, Wt = x.double().requires_grad_(True), w.double().requires_grad_(True)
    tw = r.topk_w.double().requires_grad_(True)
    tok = r.perm.long()
    owner = torch.repeat_interleave(torch.arange(E, device="cuda"), r.counts.long())
    rows = []
    for e in range(E):
        dense = torch.einsum("jip,pqs->iqjs", Wt[e], table).reshape(d * 8, F * 8)
        rows.append((X[tok[owner == e]].reshape(-1, d * 8) @ dense).reshape(-1, F, 8))
    Y = torch.cat(rows)
    out = (tw[:, :, None, None] * Y[r.slot_pos.long()]).sum(1)
    gx, gW, gt = torch.autograd.grad(out, (X, Wt, tw), dout.double())
    for name, got, want in (("dx", dx, gx), ("dw", dw, gt), ("dW", gw, gW)):
        err = float((got.double() - want).abs().max() / want.abs().max())
        assert err <= 5 * U16, (name, err)


def test_captured_and_on_another_stream():
    ops = _ops()
    N, d, E, k = 300, 40, 8, 2
    r = _routed(1, N, E, k)
    g, y = torch.randn(N, d, 8, device="cuda"), torch.randn(N * k, d, 8, device="cuda")
    say("sort gradients captured")

    def step():
        dy, dw = ops.combine_backward(g, y, r)
        return dy, dw, ops.dispatch_backward(dy, r, dx_add=g)

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_empty_and_off_16_bytes():
    ops = _ops()
    r = _routed(2, 30, 4, 2)
    flat = torch.randn(30 * 8 * 8 + 1, device="cuda")
    dout = flat[1:].view(30, 8, 8)
    y = torch.randn(60 * 8 * 8 + 1, device="cuda")[1:].view(60, 8, 8)
    say("sort gradients off 16 bytes, and of no tokens")
    a, b = ops.combine_backward(dout, y, r), ops.combine_backward(dout.clone(), y.clone(), r)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(ops.dispatch_backward(y, r, dx_add=dout), ops.dispatch_backward(y.clone(), r, dx_add=dout.clone()))
    e = ops.route(torch.empty(0, 4, device="cuda"), 2)
    dy, dw = ops.combine_backward(torch.empty(0, 8, 8, device="cuda"), torch.empty(0, 8, 8, device="cuda"), e)
    assert dy.shape == (0, 8, 8) and dw.shape == (0, 2)
    assert ops.dispatch_backward(torch.empty(0, 8, 8, device="cuda"), e).shape == (0, 8, 8)


def test_refusals():
    ops = _ops()
    r = _routed(2, 30, 4, 2)
    dout, y = torch.randn(30, 8, 8, device="cuda"), torch.randn(60, 8, 8, device="cuda")
    say("sort gradients: refusals")
    for args, kwargs in (((dout[:29], y, r), {}), ((dout, y[:, :7], r), {}), ((dout.half(), y, r), {}),
                         ((dout, y, r), dict(y_layout="rows")), ((dout, y, r), dict(out_dtype=torch.bfloat16)),
                         ((dout, y.transpose(0, 1), r), {}), ((dout, y.cpu(), r), {}), ((dout[0], y, r), {})):
        with pytest.raises(ValueError):
            ops.combine_backward(*args, **kwargs)
    for args, kwargs in (((y.half(), r), {}), ((y, r), dict(dx_add=dout.bfloat16())), ((y, r), dict(dx_add=dout[:3])),
                         ((y[0], r), {}), ((y.transpose(0, 1), r), {})):
        with pytest.raises(ValueError):
            ops.dispatch_backward(*args, **kwargs)
    bad = ops.Routing(r.topk_idx, r.topk_w, r.counts, r.offsets, r.perm, r.slot_pos.long())
    with pytest.raises(ValueError):
        ops.dispatch_backward(y, bad)
