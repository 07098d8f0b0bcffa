"""dispatch, combine and their gradients for callers who drop slots (places outside the rows: a full expert) or pad the
experts' ranges: nothing is read or written for a dropped slot, and rows that no slot names are zero.

combine rounds every product and every sum to fp32, which elementary fp32 operations in its order repeat bit for bit."""

import pytest
import torch

from _gpu_helpers import say

pytestmark = pytest.mark.gpu

FAR = (-1, 2 ** 31 - 1, -2 ** 31)


def _ops():
    from yggdrasil_amd import ops

    return ops


def _dropped(seed, N, E, k, P, share=0.3):
    """A routing of N tokens into P rows, about `share` of its slots dropped, token N // 2 without any; and which slots are on."""
    g = torch.Generator().manual_seed(seed)
    idx = torch.rand(N, E, generator=g).argsort(1)[:, :k].to(torch.int32)
    on = torch.rand(N, k, generator=g) >= share
    on[N // 2] = False
    on &= (on.flatten().cumsum(0) <= P).view(N, k)
    slots = torch.tensor([*FAR, P], dtype=torch.int64)[torch.randint(0, 4, (N, k), generator=g)]
    slots[on] = torch.randperm(P, generator=g)[:int(on.sum())]
    slots = slots.clamp(max=2 ** 31 - 1).to(torch.int32).cuda()
    w = torch.rand(N, k, generator=g).cuda()
    return _ops().Routing(idx.cuda(), w, slots[0], slots[0], slots[0], slots), on.cuda()


SIZES = [(1, 1, 1, 1, 1), (40, 24, 8, 2, 50), (40, 24, 8, 2, 200), (37, 70, 16, 4, 148), (130, 5, 16, 8, 700), (33, 130, 5, 3, 20),
         (9, 300, 8, 1, 9)]


@pytest.mark.parametrize("N,d,E,k,P", SIZES)
@pytest.mark.parametrize("ty,to", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("mask,resid", [(False, False), (False, True), (True, True)])
def test_combine(N, d, E, k, P, ty, to, mask, resid):
    ops = _ops()
    r, on = _dropped(N + d, N, E, k, P)
    y = torch.full((P, d, 8), float("nan"), device="cuda", dtype=ty)  # in rows that no slot names too
    rows = r.slot_pos[on].long()
    y[rows] = torch.randn(rows.numel(), d, 8, device="cuda").to(ty)
    res = torch.randn(N, d, 8, device="cuda").to(to) if resid else None
    say(f"combine with dropped slots N={N} d={d} k={k} P={P} {ty} {to} mask={mask} resid={resid}")
    got = ops.combine(y, r, residual=res, y_mask_order=mask, out_dtype=to)
    order = torch.where(on, r.topk_idx, 2 ** 30).argsort(dim=1, stable=True)
    acc = torch.zeros(N, d, 8, device="cuda")
    for s in range(k):
        at = order[:, s:s + 1]
        here = on.gather(1, at)[:, 0]
        rows = r.slot_pos.gather(1, at)[here, 0].long()
        acc[here] = acc[here] + r.topk_w.gather(1, at)[here, 0][:, None, None] * y[rows].float()
    if mask:
        acc = acc[..., [0, 1, 2, 4, 3, 5, 6, 7]]
    if resid:
        acc = res.float() + acc
    assert torch.equal(got, acc.to(to))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_combine_of_no_rows(dt):
    ops = _ops()
    r, _ = _dropped(1, 30, 4, 2, 0)
    res = torch.randn(30, 6, 8, device="cuda").to(dt)
    none = torch.empty(0, 6, 8, device="cuda", dtype=dt)
    say("combine of no rows")
    assert (ops.combine(none, r) == 0).all() and torch.equal(ops.combine(none, r, residual=res), res)


@pytest.mark.parametrize("N,d,E,k,P", SIZES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [False, True])
def test_dispatch(N, d, E, k, P, dt, mask):
    ops = _ops()
    r, on = _dropped(N + d, N, E, k, P)
    x = torch.randn(N, d, 8, device="cuda").to(dt)
    say(f"dispatch with dropped slots N={N} d={d} k={k} P={P} {dt} mask={mask}")
    want = torch.zeros(P, d, 8, device="cuda", dtype=dt)
    tok = torch.arange(N, device="cuda")[:, None].expand(N, k)[on]
    want[r.slot_pos[on].long()] = x[tok]
    if mask:
        want = want[..., [0, 1, 2, 4, 3, 5, 6, 7]]
    assert torch.equal(ops.dispatch(x, r, mask_order=mask, rows=P), want)
    out = torch.full((P, d, 8), float("nan"), device="cuda", dtype=dt)
    assert ops.dispatch(x, r, mask_order=mask, out=out, rows=P) is out and torch.equal(out, want)
    # without the rows' number they are N k, and those that no slot names stay
    low = torch.where(on & (r.slot_pos < N * k), r.slot_pos, -1)
    out = torch.full((N * k, d, 8), 7.0, device="cuda", dtype=dt)
    ops.dispatch(x, ops.Routing(r.topk_idx, r.topk_w, r.counts, r.offsets, r.perm, low), out=out)
    named = torch.zeros(N * k, dtype=torch.bool, device="cuda")
    named[low[low >= 0].long()] = True
    assert (out[~named] == 7.0).all()
    assert torch.equal(out[low[low >= 0].long()], x[torch.arange(N, device="cuda")[:, None].expand(N, k)[low >= 0]])


@pytest.mark.parametrize("N,d,E,k,P", SIZES + [(0, 6, 4, 2, 90), (3000, 3, 16, 2, 9000), (5, 4, 4, 2, 0),
                                               (9000, 3, 16, 4, 32000)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["blade", "pauli"])
@pytest.mark.parametrize("with_y", [False, True])
def test_combine_backward(N, d, E, k, P, dt, layout, with_y):
    """Rows that no slot names have the gradient zero whatever the memory held, the others that of the entry that leaves
    the rest unwritten."""
    ops = _ops()
    r, on = _dropped(N + d, N, E, k, P) if N else (ops.route(torch.empty(0, E, device="cuda"), k), None)
    dout, y = torch.randn(N, d, 8, device="cuda").to(dt), torch.randn(P, d, 8, device="cuda").to(dt)
    say(f"combine_backward with dropped slots N={N} d={d} k={k} P={P} {dt} {layout} y={with_y}")
    shape = (P, d, 8) if layout == "blade" else (P, 2, d, 4) if dt == torch.bfloat16 else (P, d, 2, 2, 2)
    want, dw = torch.zeros(shape, device="cuda", dtype=dt), torch.full((N, k), 5.0, device="cuda")
    args = (dout.data_ptr(), ops.DTYPE_CODE[dt], y.data_ptr(), N, k, d, P, r.topk_w.data_ptr(), r.slot_pos.data_ptr())
    if N and P:
        ops.check(ops.lib().ygg_combine_backward(*args, want.data_ptr(), ops.DTYPE_CODE[dt], layout == "pauli", dw.data_ptr(),
                                                 ops.stream_handle()))
        named = torch.zeros(P, dtype=torch.bool, device="cuda")
        named[r.slot_pos[on].long()] = True
        assert (want[~named] == 0).all() and not (want[named].flatten(1) == 0).all(1).any()
    need = ops.lib().ygg_combine_backward_rows_workspace_bytes(N, k, P)
    assert need == (4 * P if N == 9000 else 0)  # (both ways to find the rows that no slot names)
    for fill in (0, 1):  # scratch and rows as an allocator may leave them: the scratch names a token of every row
        dirty = torch.full(shape, float("nan"), device="cuda", dtype=dt)
        tokens = torch.arange(P, device="cuda", dtype=torch.int32) * fill
        ops.check(ops.lib().ygg_combine_backward_rows(*args[:2], y.data_ptr() if with_y else None, *args[3:], dirty.data_ptr(),
                                                      ops.DTYPE_CODE[dt], layout == "pauli", dw.data_ptr() if with_y else None,
                                                      tokens.data_ptr(), need, ops.stream_handle()))
        assert torch.equal(dirty, want)
    dy, dw2 = ops.combine_backward(dout, y if with_y else None, r, y_layout=layout, rows=P)
    assert torch.equal(dy, want) and (dw2 is None if not with_y else not N or not P or torch.equal(dw2, dw))


def test_combine_backward_captured():
    ops = _ops()
    N, d, E, k, P = 300, 24, 8, 2, 700
    r, _ = _dropped(5, N, E, k, P)
    dout, y = torch.randn(N, d, 8, device="cuda"), torch.randn(P, d, 8, device="cuda")
    say("combine_backward with dropped slots captured")
    ops.combine_backward(dout, y, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.combine_backward(dout, y, r)
    for n in range(4):
        r.slot_pos.copy_(r.slot_pos.flip(0))  # other rows are named
        want = ops.combine_backward(dout, y, r)
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {n}"


def test_chain_with_full_and_padded_experts():
    """Experts of a fixed capacity: their ranges padded, the tokens past it dropped.  The operators from tokens to output and
    back, against float64 autograd; the chain's rows are bf16, so each of its five roundings is 2^-8 of the largest value
    that it meets."""
    ops = _ops()
    N, d, F, E, k, C = 200, 32, 48, 8, 2, 56
    P = E * C
    torch.manual_seed(7)
    full = ops.route(torch.randn(N, E, device="cuda") + torch.linspace(1, -1, E, device="cuda"), k)
    owner = torch.repeat_interleave(torch.arange(E, device="cuda"), full.counts.long())
    at = full.slot_pos.long()
    e, place = owner[at], at - full.offsets.long()[owner[at]]
    on = place < C
    assert not on.all() and int(full.counts.min()) < C
    slots = torch.where(on, e * C + place, -1).to(torch.int32)
    offsets = torch.arange(0, P + 1, C, device="cuda", dtype=torch.int32)
    r = ops.Routing(full.topk_idx, full.topk_w, full.counts, offsets, full.perm, slots)
    x = torch.randn(N, d, 8, device="cuda").bfloat16()
    w = torch.randn(E, F, d, 8, device="cuda") / (8 * d) ** 0.5
    dout = torch.randn(N, F, 8, device="cuda").bfloat16()
    say("chain with full and padded experts")
    junk = torch.full((64 << 20,), float("nan"), device="cuda")  # what the next allocations find
    del junk
    xs = ops.dispatch(x, r, rows=P)
    y = ops.pauli_grouped_linear(xs, ops.prepare_weights(w, "pauli"), offsets)
    out = ops.combine(y, r)
    dy, dw = ops.combine_backward(dout, y, r, y_layout="pauli")
    dxs = ops.pauli_grouped_input_grad(dy, ops.prepare_adjoint_weights(w, "pauli"), offsets)
    dx = ops.dispatch_backward(dxs, r)
    gw, _ = ops.grouped_weight_grad_pauli(dy, ops.pauli_rows_from_blade(xs), offsets, E)
    import numpy as np
    from oracle import cl3

    table = torch.zeros(8, 8, 8, dtype=torch.float64, device="cuda")
    for p in range(8):
        for q in range(8):
            a, b = np.zeros((1, 8)), np.zeros((1, 8))
            a[0, p] = b[0, q] = 1
            table[p, q] = torch.from_numpy(np.asarray(cl3.geom_prod(a, b))[0]).cuda()
    X, W = x.double().requires_grad_(True), w.double().requires_grad_(True)
    tw = r.topk_w.double().requires_grad_(True)
    total = torch.zeros(N, F, 8, dtype=torch.float64, device="cuda")
    for n in range(E):
        dense = torch.einsum("jip,pqs->iqjs", W[n], table).reshape(d * 8, F * 8)
        tok, slot = torch.nonzero(on & (full.topk_idx == n), as_tuple=True)
        total = total.index_add(0, tok, tw[tok, slot][:, None, None] * (X[tok].reshape(-1, d * 8) @ dense).reshape(-1, F, 8))
    gx, gW, gt = torch.autograd.grad(total, (X, W, tw), dout.double())
    for name, got, want in (("out", out, total), ("dx", dx, gx), ("dw", dw, gt), ("dW", gw, gW)):
        err = float((got.double() - want.detach()).abs().max() / want.detach().abs().max())
        assert err <= 5 * 2.0 ** -8, (name, err)


def test_refusals():
    ops = _ops()
    r, _ = _dropped(2, 30, 4, 2, 60)
    x, y = torch.randn(30, 8, 8, device="cuda"), torch.randn(60, 8, 8, device="cuda")
    say("dispatch and combine: refusals")
    other = ops.Routing(r.topk_idx[:29], r.topk_w[:29], r.counts, r.offsets, r.perm, r.slot_pos[:29])
    long = ops.Routing(r.topk_idx, r.topk_w, r.counts, r.offsets, r.perm, r.slot_pos.long())
    idx = ops.Routing(r.topk_idx[:, :1], r.topk_w, r.counts, r.offsets, r.perm, r.slot_pos)
    for args, kwargs in (((x, other), {}), ((x, long), {}), ((x[0], r), {}), ((x[..., :4].contiguous(), r), {}),
                         ((x, r), dict(out=x)), ((x, r), dict(out=y.bfloat16())), ((x, r), dict(out=y, rows=59)),
                         ((x, r), dict(out=torch.empty(60, 8, 16, device="cuda")[..., ::2])), ((x.cpu(), r), {})):
        with pytest.raises(ValueError):
            ops.dispatch(*args, **kwargs)
    for args, kwargs in (((y, long), {}), ((y, idx), {}), ((y[0], r), {}), ((y, r), dict(residual=x[:29])),
                         ((y, r), dict(residual=x.bfloat16())), ((y, r), dict(out=y)), ((y, r), dict(out_dtype=torch.half)),
                         ((y, r), dict(out=torch.empty(30, 8, 16, device="cuda")[..., ::2])), ((y.cpu(), r), {})):
        with pytest.raises(ValueError):
            ops.combine(*args, **kwargs)
