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
