"""GPU parity of the bf16 training operators against float64 (``_train_oracle``).

Tolerances: a result may be off by half a step per rounding, relative to the sum of the magnitudes
of its terms: 2^-24 for each of the fp32 additions on the longest chain to a value, and 2^-8 of the
value itself where it is rounded to bf16.  A wrong or missing term is larger than that at these sizes.
"""

import numpy as np
import pytest
import torch

import _train_oracle as to
from _gpu_helpers import bf16_round, say

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _ops():
    from yggdrasil_amd import ops

    return ops


def _bf16(a):
    return bf16_round(np.asarray(a, np.float32))


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _host(t):
    return t.detach().double().cpu().numpy()


def _within(got, want, bound, what=""):
    got = _host(got) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want) - bound
    assert not np.isnan(off).any() and off.max(initial=-1.0) <= 0, \
        (what, float(off.max()), np.unravel_index(np.argmax(off), off.shape))


def _bounds(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


# ---- weight gradient ---------------------------------------------------------------------------

WEIGHT_CASES = [
    # rows of each expert, d_in, d_out, gathered, bias
    ([1], 2, 2, False, True),
    ([0, 3, 0], 6, 4, True, True),
    ([5, 0, 64, 1], 34, 18, False, True),
    ([65, 31, 2], 64, 64, True, True),
    ([33, 129], 66, 130, True, False),
    ([0, 0], 10, 8, False, True),
    ([7, 200, 0, 190, 3], 100, 36, False, True),
    ([400], 24, 72, True, True),
    ([1] * 64, 16, 20, True, True),
    ([1300, 0, 513, 512], 6, 10, True, True),  # experts of several chunks of rows
    ([0, 1025], 70, 66, False, True),
    ([0 if e % 5 == 0 else e * 37 % 90 for e in range(62)] + [700, 1100], 10, 6, True, True),
]


@pytest.mark.parametrize("rows,d_in,d_out,gathered,bias", WEIGHT_CASES)
def test_weight_grad(rows, d_in, d_out, gathered, bias):
    ops = _ops()
    g = np.random.default_rng(len(rows) * 1000 + d_in)
    offsets = _bounds(rows)
    P, E = int(offsets[-1]), len(rows)
    n_a = P // 2 + 3 if gathered else P
    dy, a = _bf16(g.standard_normal((P, 2, d_out, 4))), _bf16(g.standard_normal((n_a, 2, d_in, 4)))
    gather = g.integers(0, n_a, P).astype(np.int32) if gathered else None
    say(f"weight grad bf16 rows={rows[:8]} d_in={d_in} d_out={d_out} gathered={gathered}")
    args = (_dev(dy, torch.bfloat16), _dev(a, torch.bfloat16), _dev(offsets), E)
    kw = dict(gather=_dev(gather) if gathered else None, with_bias=bias)
    dW, db = ops.grouped_weight_grad_pauli(*args, **kw)
    want, want_b, mW, mb = to.weight_grad(dy, a[gather] if gathered else a, offsets)
    n = max(rows)
    _within(dW, want, (4 * n + 16) * U32 * mW, "dW")
    if bias:
        _within(db, want_b, (n + 16) * U32 * mb, "db")
    else:
        assert db is None
    again = ops.grouped_weight_grad_pauli(*args, **kw)
    assert torch.equal(dW, again[0]) and (not bias or torch.equal(db, again[1]))


def test_weight_grad_rows_past_the_last_expert_and_bad_indices():
    """Rows past offsets[E] belong to no expert; offsets are clamped; a gather index outside a reads zeros."""
    ops = _ops()
    g = np.random.default_rng(5)
    dy, a = _bf16(g.standard_normal((40, 2, 12, 4))), _bf16(g.standard_normal((9, 2, 10, 4)))
    gather = g.integers(0, 9, 40).astype(np.int32)
    bad = gather.copy()
    bad[[3, 17]] = [9, -1]
    offsets = np.array([0, 11, 30], np.int32)
    say("weight grad bf16, rows past the experts, bad gather indices")
    dW, db = ops.grouped_weight_grad_pauli(_dev(dy, torch.bfloat16), _dev(a, torch.bfloat16), _dev(offsets), 2,
                                           gather=_dev(bad))
    rows = a[gather].copy()
    rows[[3, 17]] = 0
    want, want_b, mW, mb = to.weight_grad(dy, rows, offsets)
    _within(dW, want, (4 * 19 + 16) * U32 * mW)
    _within(db, want_b, (19 + 16) * U32 * mb)
    clamped = ops.grouped_weight_grad_pauli(_dev(dy, torch.bfloat16), _dev(a, torch.bfloat16),
                                            _dev(np.array([-5, 11, 4000], np.int32)), 2, gather=_dev(bad))
    want, want_b, mW, mb = to.weight_grad(dy, rows, [0, 11, 40])
    _within(clamped[0], want, (4 * 29 + 16) * U32 * mW)
    _within(clamped[1], want_b, (29 + 16) * U32 * mb)


# ---- input gradient ------------------------------------------------------------------------------

INPUT_CASES = [
    # rows of each expert, d_out (contraction), d_in, act, layout, out dtype
    ([1], 2, 1, "none", "blade", "f32"),
    ([3, 0, 2], 6, 5, "gelu", "blade", "bf16"),
    ([17, 1], 16, 34, "gelu", "pauli", "bf16"),
    ([0, 66, 5], 18, 66, "sigmoid", "pauli", "bf16"),
    ([64, 33], 64, 40, "relu", "pauli", "bf16"),
    ([31, 0, 70], 100, 64, "gelu", "blade", "f32"),
    ([129], 36, 130, "gelu", "pauli", "bf16"),
    ([12, 9], 34, 7, "none", "blade", "bf16"),
    ([1] * 64, 20, 18, "sigmoid", "blade", "bf16"),
    ([0, 0], 20, 18, "gelu", "pauli", "bf16"),
]


def _exact_weights(g, E, d_out, d_in):
    """fp32 weights whose halved matrix entries are bf16 numbers: their layout rounds nothing."""
    m = g.integers(-127, 128, (E, d_out, d_in, 8)) / 64.0
    return (m @ to.FROM_PAULI).astype(np.float32)


def _input_bound(want, grad, mag, J, d_out, pauli, rounded):
    """Half steps of the sum, of the slope (at most some 40 fp32 roundings: the exponential's argument is below
    32 and the hardware's functions are within a step) and of the stored value."""
    g_off = (4 * d_out + 16) * U32 * mag
    aJ = np.abs(J)
    off = np.einsum("...ab,...b->...a", aJ, g_off) + 2.0 ** -16 * np.einsum("...ab,...b->...a", aJ + 1.0, np.abs(grad))
    if pauli:
        m = np.transpose((off @ np.abs(to.TO_PAULI)).reshape(*off.shape[:2], 2, 2, 2), (0, 3, 1, 2, 4))
        off = m.reshape(want.shape)
    # a rounding to bf16 of a value that is off by `off` itself
    return off * (1 + U16) + (U16 * np.abs(want) if rounded else 4 * U32 * np.abs(want))


@pytest.mark.parametrize("rows,d_out,d_in,act,layout,out", INPUT_CASES)
def test_input_grad(rows, d_out, d_in, act, layout, out):
    ops = _ops()
    g = np.random.default_rng(d_out * 100 + d_in)
    offsets = _bounds(rows)
    P, E = int(offsets[-1]), len(rows)
    dy = _bf16(g.standard_normal((P, 2, d_out, 4)))
    W = _exact_weights(g, E, d_out, d_in)
    h = _bf16(1.5 * g.standard_normal((P, d_in, 8)))
    if P > 4:
        h[:3, :, 1:4] = 0.0  # no vector part: the length's epsilon alone
        h[2, :, 0] = 0.0
        h[3, :, 7] = 0.0
        h[4] *= 16
        h = _bf16(h)
    say(f"input grad rows={rows[:8]} d_out={d_out} d_in={d_in} act={act} {layout} {out}")
    adj = ops.prepare_adjoint_weights(_dev(W), "pauli")
    args = (_dev(dy, torch.bfloat16), adj, _dev(offsets))
    kw = dict(h_pre=_dev(h, torch.bfloat16) if act != "none" else None, act=act, y_layout=layout, out_dtype=DT[out])
    got = ops.pauli_grouped_input_grad(*args, **kw)
    grad, mag = to.linear_grad(dy, W, offsets)
    J = to.act_jacobian(h, act)
    want = np.einsum("...ab,...b->...a", J, grad)
    if layout == "pauli":
        want = to.half_rows(want)
    _within(got, want, _input_bound(want, grad, mag, J, d_out, layout == "pauli", got.dtype == torch.bfloat16))
    assert torch.equal(got, ops.pauli_grouped_input_grad(*args, **kw))


def test_adjoint_layout_is_that_of_the_adjoint_weights():
    ops = _ops()
    g = np.random.default_rng(9)
    W = _dev(g.standard_normal((3, 10, 7, 8)).astype(np.float32))
    say("bf16 adjoint weight layout")
    got, want = ops.prepare_adjoint_weights(W, "pauli"), ops.prepare_weights(ops.adjoint_weights(W), "pauli")
    assert torch.equal(got.data, want.data) and (got.E, got.d_out, got.d_in, got.fmt) == (3, 7, 10, "pauli")


def test_input_grad_leaves_the_rows_past_the_last_expert():
    ops = _ops()
    from yggdrasil_amd import _native as N

    g = np.random.default_rng(11)
    for d_out in (8, 40):  # both product kernels
        W, dy = _exact_weights(g, 2, d_out, 6), _bf16(g.standard_normal((50, 2, d_out, 4)))
        adj, rows = ops.prepare_adjoint_weights(_dev(W), "pauli"), _dev(dy, torch.bfloat16)
        offsets = _dev(np.array([0, 20, 33], np.int32))
        dx = torch.full((50, 6, 8), 7.0, device="cuda")
        say(f"input grad, rows past the experts, d_out={d_out}")
        N.check(N.lib().ygg_pauli_grouped_input_grad(rows.data_ptr(), 50, adj.data.data_ptr(), offsets.data_ptr(), 2,
                                                     d_out, 6, 0, None, dx.data_ptr(), 1, 0, N.stream_handle(dx.device)))
        assert bool((dx[33:] == 7.0).all()) and not bool((dx[:33] == 7.0).all())


# ---- norm ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("N,d,dt,gdt,residual", [
    (1, 1, "f32", "f32", False), (3, 5, "f32", "f32", True), (70, 64, "f32", "f32", False), (65, 64, "bf16", "bf16", True),
    (200, 100, "bf16", "bf16", True), (130, 33, "bf16", "f32", False), (31, 129, "f32", "bf16", True),
    (40, 256, "bf16", "bf16", False), (19, 300, "f32", "f32", True), (5, 1000, "bf16", "bf16", True),
    (3, 1025, "bf16", "bf16", False), (2, 4096, "f32", "f32", True), (700, 8, "bf16", "bf16", False),
    (2500, 16, "f32", "f32", False), (600, 64, "bf16", "bf16", True), (515, 100, "f32", "bf16", False),
    (300, 256, "bf16", "bf16", True), (150, 300, "f32", "f32", True), (50, 1000, "bf16", "f32", False),
    (512, 64, "f32", "f32", True), (513, 8, "f32", "f32", False), (32, 1024, "bf16", "bf16", True)])
@pytest.mark.parametrize("eps", [1e-6, 0.25])
def test_norm_backward(N, d, dt, gdt, residual, eps):
    ops = _ops()
    g = np.random.default_rng(N * 7 + d)
    rd = lambda a, t: _bf16(a) if t == "bf16" else np.asarray(a, np.float32)
    x, dy = rd(g.standard_normal((N, d, 8)), dt), rd(g.standard_normal((N, d, 8)), gdt)
    if N > 2:
        x[1] = 0.0  # a row of zeros: rms is sqrt(2 eps)
    gamma = g.standard_normal((d, 8)).astype(np.float32)
    res = rd(g.standard_normal((N, d, 8)), dt) if residual else None
    say(f"norm backward N={N} d={d} {dt}/{gdt} residual={residual} eps={eps}")
    args = (_dev(dy, DT[gdt]), _dev(x, DT[dt]), _dev(gamma), eps)
    kw = dict(residual_grad=_dev(res, DT[dt]) if residual else None)
    got = ops.clifford_layer_norm_backward(*args, **kw)
    want, mag = to.norm_grad(dy, x, gamma, eps, res)
    chain = 8 * d + 64
    _within(got[0], want[0], chain * U32 * mag[0] + (U16 * (1 + 1e-3) * np.abs(want[0]) if dt == "bf16" else 0), "dx")
    _within(got[1], want[1], (N + chain) * U32 * mag[1], "dgamma")
    _within(got[2], want[2], (N + 16) * U32 * mag[2], "dbeta")
    again = ops.clifford_layer_norm_backward(*args, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_norm_backward_of_no_tokens():
    ops = _ops()
    say("norm backward of no tokens")
    dx, dg, db = ops.clifford_layer_norm_backward(torch.empty(0, 6, 8, device="cuda"), torch.empty(0, 6, 8, device="cuda"),
                                                  torch.ones(6, 8, device="cuda"))
    assert dx.shape == (0, 6, 8) and not bool(dg.any()) and not bool(db.any())


# ---- router ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("N,d,E,k,dt,add", [
    (1, 1, 1, 1, "f32", False), (5, 3, 4, 2, "f32", True), (257, 64, 8, 2, "f32", False), (70, 100, 12, 3, "bf16", True),
    (33, 7, 64, 8, "bf16", False), (1000, 16, 64, 2, "bf16", True), (19, 300, 16, 4, "f32", True), (300, 8, 3, 3, "bf16", False),
    (40, 20, 6, 1, "f32", True), (3000, 2, 5, 2, "f32", False),
    (400, 100, 64, 8, "bf16", True), (300, 200, 16, 2, "f32", False), (120, 300, 9, 3, "bf16", True),
    (512, 64, 64, 8, "f32", True), (513, 5, 3, 2, "bf16", False), (2, 2000, 4, 4, "f32", True),
    (40003, 3, 6, 2, "f32", True)])  # (the last: more than a batch a workgroup)
def test_router_backward(N, d, E, k, dt, add):
    ops = _ops()
    g = np.random.default_rng(N + d * 3 + E)
    rd = _bf16 if dt == "bf16" else (lambda a: np.asarray(a, np.float32))
    x = rd(g.standard_normal((N, d, 8)) * np.exp(0.7 * g.standard_normal((N, 1, 4)))[..., to.GRADE])
    W = (2 * g.standard_normal((E, 4))).astype(np.float32)
    logits = g.standard_normal((N, E)).astype(np.float32)
    gw = g.standard_normal((N, k)).astype(np.float32)
    plus = rd(g.standard_normal((N, d, 8))) if add else None
    say(f"router backward N={N} d={d} E={E} k={k} {dt} add={add}")
    r = ops.route(_dev(logits), k)
    w, idx = r.topk_w.cpu().numpy(), r.topk_idx.cpu().numpy().astype(np.int64)
    dlogits = ops.route_backward(r.topk_idx, r.topk_w, _dev(gw), E)
    want, ml = to.route_grad(idx, w, gw, E)
    if k == 1:
        want, ml = np.zeros_like(want), ml
    # the weights are within 4 half steps of the softmax, whose sum of 8 is off by as much
    _within(dlogits, want, 24 * U32 * ml, "dlogits")
    got = ops.route_energy_backward(_dev(x, DT[dt]), _dev(W), r.topk_idx, r.topk_w, _dev(gw),
                                    dx_add=_dev(plus, DT[dt]) if add else None)
    want3, mag = to.energy_grad(x, W, want, ml, plus)
    chain = 8 * d + 64 + 4 * k
    _within(got[0], want3[0], chain * U32 * mag[0] + (U16 * (1 + 1e-3) * np.abs(want3[0]) if dt == "bf16" else 0), "dx")
    _within(got[1], want3[1], (N + chain) * U32 * mag[1], "dW")
    _within(got[2], want3[2], (N + 32) * U32 * mag[2], "db")
    again = ops.route_energy_backward(_dev(x, DT[dt]), _dev(W), r.topk_idx, r.topk_w, _dev(gw),
                                      dx_add=_dev(plus, DT[dt]) if add else None)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_router_backward_ignores_experts_out_of_range():
    ops = _ops()
    say("router backward, an expert index out of range")
    idx = torch.tensor([[0, 9], [1, -1]], device="cuda", dtype=torch.int32)
    w, g = torch.full((2, 2), 0.5, device="cuda"), torch.tensor([[1.0, 2.0], [3.0, 4.0]], device="cuda")
    dl = ops.route_backward(idx, w, g, 3)
    assert dl.cpu().tolist() == [[-0.25, 0.0, 0.0], [0.0, -0.25, 0.0]]
    x = torch.randn(2, 4, 8, device="cuda")
    dx, dW, db = ops.route_energy_backward(x, torch.ones(3, 4, device="cuda"), idx, w, g)
    assert bool(torch.isfinite(dx).all()) and db.cpu().tolist() == [-0.25, -0.25, 0.0]


# ---- streams, graphs, alignment ----------------------------------------------------------------------


def _one_of_each(g):
    """(name, call) of every operator on small inputs; call() returns its outputs."""
    ops = _ops()
    rows = [20, 0, 13]
    offsets, P = _dev(_bounds(rows)), 33
    dy, a = _dev(g.standard_normal((P, 2, 36, 4)), torch.bfloat16), _dev(g.standard_normal((P, 2, 24, 4)), torch.bfloat16)
    W = _dev(g.standard_normal((3, 36, 24, 8)).astype(np.float32))
    h = _dev(g.standard_normal((P, 24, 8)), torch.bfloat16)
    x, res = _dev(g.standard_normal((50, 36, 8)), torch.bfloat16), _dev(g.standard_normal((50, 36, 8)), torch.bfloat16)
    gamma = _dev(g.standard_normal((36, 8)).astype(np.float32))
    rw, gw = _dev(g.standard_normal((5, 4)).astype(np.float32)), _dev(g.standard_normal((50, 2)).astype(np.float32))
    r = ops.route(_dev(g.standard_normal((50, 5)).astype(np.float32)), 2)
    return [
        ("weight", lambda: ops.grouped_weight_grad_pauli(dy, a, offsets, 3)),
        ("input", lambda: (ops.pauli_grouped_input_grad(dy, ops.prepare_adjoint_weights(W, "pauli"), offsets, h, "gelu"),)),
        ("norm", lambda: ops.clifford_layer_norm_backward(res, x, gamma, residual_grad=res)),
        ("router", lambda: ops.route_energy_backward(x, rw, r.topk_idx, r.topk_w, gw, dx_add=res)),
        ("logits", lambda: (ops.route_backward(r.topk_idx, r.topk_w, gw, 5),)),
    ]


@pytest.mark.parametrize("which", range(5))
def test_on_another_stream(which):
    name, call = _one_of_each(np.random.default_rng(3))[which]
    say(f"{name} on a stream of its own")
    want = call()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = call()
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", range(5))
def test_captured_and_replayed(which):
    name, call = _one_of_each(np.random.default_rng(4))[which]
    say(f"{name} captured into a graph")
    want = call()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        call()
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(4):
        for t in got:
            t.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        other = call()  # the program's own work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_operands_off_their_alignment():
    ops = _ops()
    g = np.random.default_rng(6)

    def shifted(t):  # the same values one element past a 16-byte boundary
        flat = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    offsets = _dev(_bounds([9, 4]))
    dy, a = _dev(g.standard_normal((13, 2, 6, 4)), torch.bfloat16), _dev(g.standard_normal((13, 2, 10, 4)), torch.bfloat16)
    h = _dev(g.standard_normal((13, 10, 8)), torch.bfloat16)
    W = _dev(g.standard_normal((2, 6, 10, 8)).astype(np.float32))
    x, gamma = _dev(g.standard_normal((7, 10, 8)), torch.bfloat16), _dev(g.standard_normal((10, 8)).astype(np.float32))
    rw, r = _dev(g.standard_normal((4, 4)).astype(np.float32)), ops.route(_dev(g.standard_normal((7, 4)).astype(np.float32)), 2)
    gw = torch.ones(7, 2, device="cuda")
    gw[:, 0] = 3.0
    say("operands off their 16-byte alignment")
    for f in (lambda s: ops.grouped_weight_grad_pauli(s(dy), s(a), offsets, 2),
              lambda s: (ops.pauli_grouped_input_grad(s(dy), ops.prepare_adjoint_weights(s(W), "pauli"), offsets, s(h), "relu"),),
              lambda s: ops.clifford_layer_norm_backward(s(x), s(x), s(gamma), residual_grad=s(x)),
              lambda s: ops.route_energy_backward(s(x), s(rw), r.topk_idx, r.topk_w, gw, dx_add=s(x))):
        assert all(torch.equal(p, q) for p, q in zip(f(shifted), f(lambda t: t)))


@pytest.mark.parametrize("n,d", [(9, 36), (700, 36), (9, 300), (300, 300), (9, 1024), (9, 1100)])
def test_outputs_in_place(n, d):
    """dx in the place of the gradient that it adds."""
    from yggdrasil_amd import _native as N

    ops, L = _ops(), N.lib()
    g = np.random.default_rng(d)
    x, dy, res = (_dev(g.standard_normal((n, d, 8)).astype(np.float32)) for _ in range(3))
    gamma = _dev(g.standard_normal((d, 8)).astype(np.float32))
    say(f"outputs in place of inputs n={n} d={d}")
    want = ops.clifford_layer_norm_backward(dy, x, gamma, residual_grad=res)
    ws = torch.empty(L.ygg_clifford_layer_norm_backward_workspace_bytes(n, d) + 1, device="cuda", dtype=torch.uint8)
    dx, dg, db = res.clone(), torch.empty_like(gamma), torch.empty_like(gamma)
    N.check(L.ygg_clifford_layer_norm_backward(dy.data_ptr(), 0, x.data_ptr(), 0, n, d, gamma.data_ptr(), 1e-6,
                                               dx.data_ptr(), dx.data_ptr(), dg.data_ptr(), db.data_ptr(), ws.data_ptr(),
                                               ws.numel(), N.stream_handle(x.device)), "norm")
    assert all(torch.equal(p, q) for p, q in zip((dx, dg, db), want))
    rw, gw = _dev(g.standard_normal((5, 4)).astype(np.float32)), _dev(g.standard_normal((n, 2)).astype(np.float32))
    r = ops.route(_dev(g.standard_normal((n, 5)).astype(np.float32)), 2)
    want = ops.route_energy_backward(x, rw, r.topk_idx, r.topk_w, gw, dx_add=res)
    dx, dw, db = res.clone(), torch.empty_like(rw), torch.empty(5, device="cuda")
    ws = torch.empty(L.ygg_route_energy_backward_workspace_bytes(n, d, 5, 2) + 1, device="cuda", dtype=torch.uint8)
    N.check(L.ygg_route_energy_backward(x.data_ptr(), 0, n, d, rw.data_ptr(), 5, 2, r.topk_idx.data_ptr(),
                                        r.topk_w.data_ptr(), gw.data_ptr(), dx.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                                        db.data_ptr(), ws.data_ptr(), ws.numel(), N.stream_handle(x.device)), "router")
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), want))


@pytest.mark.parametrize("d", [6, 600])
def test_router_backward_of_no_tokens(d):
    ops = _ops()
    say(f"router backward of no tokens d={d}")
    i, f = torch.empty(0, 2, device="cuda", dtype=torch.int32), torch.empty(0, 2, device="cuda")
    dx, dW, db = ops.route_energy_backward(torch.empty(0, d, 8, device="cuda"), torch.ones(5, 4, device="cuda"), i, f, f)
    assert dx.shape == (0, d, 8) and dW.shape == (5, 4) and not bool(dW.any()) and not bool(db.any())
    assert ops.route_backward(i, f, f, 5).shape == (0, 5)


@pytest.mark.parametrize("n", [384, 385])
def test_few_rows_and_more_agree(n):
    """The tokens of one launch and of two: dx is a token's own, the parameters' sums differ by their order.

    dx: two orders of sums of 8 d = 320 terms, whose roundings add up to less than 2^8 half steps of the largest value;
    parameters: sums of n tokens' terms, each of at most 8 products, a half step an addition."""
    ops = _ops()
    g = np.random.default_rng(21)
    say(f"norm and router backward around the last call in one launch n={n}")
    x, dy = (_dev(g.standard_normal((n, 40, 8)).astype(np.float32)) for _ in range(2))
    gamma, rw = _dev(g.standard_normal((40, 8)).astype(np.float32)), _dev(g.standard_normal((7, 4)).astype(np.float32))
    r = ops.route(_dev(g.standard_normal((n, 7)).astype(np.float32)), 3)
    gw = _dev(g.standard_normal((n, 3)).astype(np.float32))
    for call in (lambda s: ops.clifford_layer_norm_backward(dy[s], x[s], gamma),
                 lambda s: ops.route_energy_backward(x[s], rw, r.topk_idx[s], r.topk_w[s], gw[s])):
        whole, parts = call(slice(0, n)), [call(slice(0, 200)), call(slice(200, n))]
        scale = [float(t.abs().max()) for t in whole]
        assert float((whole[0] - torch.cat([p[0] for p in parts])).abs().max()) < 2.0 ** -16 * scale[0]
        for i in (1, 2):
            assert float((whole[i] - parts[0][i] - parts[1][i]).abs().max()) < 2.0 ** -24 * n * 8 * scale[i]
