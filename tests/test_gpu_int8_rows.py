"""Rows in int8 and their products with int8 weights, against whole-number sums and float64 (``_int8_oracle``).

Tolerances: codes, scales and the integer sums are exact.  After them a value takes the conversion of the sum, two
products with scales, one addition of two entries and one of the bias, each half a step, 2^-24 of the magnitudes that
meet in it: 5 2^-24.  An activation passes an error on by at most its gain; its gate, an exponential and a reciprocal
of the hardware of an argument z below 64 wherever the gate is not below fp32's smallest, is off by 64 2^-23 of the
value.  tanh of grade 3 is 2 s - 1, s = 1 / (1 + e): e is off by 2^-23 of itself, of which e / (1 + e) <= 1 reaches
s, the sum by 2^-24, the reciprocal by 2^-23, so 2 s <= 2 by 2 (2 2^-23 + 2^-24) = 10 2^-24 whatever is left after the
subtraction.  A bf16 output is off by 2^-8 of the value.
"""

import numpy as np
import pytest
import torch

import _int8_oracle as io
from _gpu_helpers import bf16_round, say

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8


def _ops():
    from yggdrasil_amd import ops

    return ops


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _rows(g, rows, d, bf16):
    x = (g.standard_normal((rows, d, 8)) * np.exp(0.5 * g.standard_normal((rows, 1, 1)))).astype(np.float32)
    return bf16_round(x) if bf16 else x


def _weights(g, E, d_out, d_in):
    return ((g.standard_normal((E, d_out, d_in, 8)) / np.sqrt(8 * d_in)).astype(np.float32),
            (0.3 * g.standard_normal((E, d_out, 8))).astype(np.float32))


def _bounds(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def _check(got, want, size, act, bf16, what):
    y, gain = io.activate(want, act)
    bound = gain * 5 * U32 * size + (128 * U32 * np.abs(y) if act in ("gelu", "sigmoid") else 0) + 1e-30
    if act in ("gelu", "sigmoid"):
        bound[..., 7] += 10 * U32
    if bf16:
        bound = bound * (1 + U16) + U16 * np.abs(y) + 1e-38
    assert tuple(got.shape) == want.shape, what
    off = np.abs(got.double().cpu().numpy() - y) - bound
    worst = float(off.max(initial=-1.0))
    assert worst <= 0, (what, worst, np.unravel_index(off.argmax(), off.shape))  # (a NaN fails too)


# ---- quantization ------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,d", [(1, 1), (3, 5), (7, 31), (5, 32), (9, 33), (4, 64), (6, 65), (130, 100), (11, 255),
                                    (3, 257), (2, 1024), (2, 1100), (1, 2500)])
@pytest.mark.parametrize("bf16", [False, True])
def test_quantize_rows_bit_exact(rows, d, bf16):
    ops = _ops()
    g = np.random.default_rng(rows * 1000 + d)
    x = _rows(g, rows, d, bf16)
    say(f"quantize_rows rows={rows} d={d} bf16={bf16}")
    got = ops.quantize_rows(_dev(x, torch.bfloat16 if bf16 else None))
    q, s = io.quantize(x)
    assert np.array_equal(got.scale.cpu().numpy(), s)
    assert np.array_equal(got.codes.cpu().numpy(), io.codes_layout(q))
    want = (q * s.astype(np.float64)[:, None, None, None, None])
    back = got.values().double().cpu().numpy()
    assert back.shape == x.shape
    # sums of two rounded products
    assert np.abs(back[..., 0] - (want[..., 0, 0, 0] + want[..., 1, 1, 0])).max() <= 4 * U32 * 2 * np.abs(want).max()


@pytest.mark.parametrize("d", [3, 64, 100, 300, 1100])
@pytest.mark.parametrize("bf16", [False, True])
def test_quantize_rows_far_values(d, bf16):
    """Zeros, values whose sums pass the type's range, values below the smallest scale, infinities and NaN."""
    ops = _ops()
    g = np.random.default_rng(d)
    x = _rows(g, 12, d, bf16)
    x[0] = 0
    x[1] *= np.float32(2.0 ** 120)
    x[2] = np.float32(3e38)
    x[3] *= np.float32(2.0 ** -98)
    x[4] *= np.float32(2.0 ** -110)
    x[5] = np.float32(1e-40)
    x[6, d - 1, 7] = np.inf
    x[7, 0, 3] = -np.inf
    x[8, d // 2, 5] = np.nan
    x[9] = -x[9]
    x[10, :, :] = 0
    x[10, d - 1, 2] = np.float32(2.0 ** -20)
    if bf16:
        x = bf16_round(x)
    say(f"quantize_rows far values d={d} bf16={bf16}")
    got = ops.quantize_rows(_dev(x, torch.bfloat16 if bf16 else None))
    q, s = io.quantize(x)
    assert np.array_equal(got.scale.cpu().numpy(), s, equal_nan=True)
    assert np.isnan(s[6:9]).all() and np.isfinite(np.delete(s, [6, 7, 8])).all()
    assert np.array_equal(got.codes.cpu().numpy(), io.codes_layout(q))


@pytest.mark.parametrize("d,rows", [(1, (1 << 22) + 5), (257, (1 << 22) + 1)])
def test_quantize_rows_of_more_than_one_launch(d, rows):
    """More rows than a launch takes: those at the seam and at the end, as in a batch of their own."""
    ops = _ops()
    say(f"quantize_rows {rows} x {d}")
    part = _dev(_rows(np.random.default_rng(16), 64, d, True), torch.bfloat16)
    x = torch.zeros(rows, d, 8, device="cuda", dtype=torch.bfloat16)
    places = [0, (1 << 22) - 64, rows - 64]
    for at in places:
        x[at:at + 64] = part
    got = ops.quantize_rows(x)
    one = ops.quantize_rows(part)
    at = rows - 64  # (the last to be written: whole)
    assert torch.equal(got.codes[at:], one.codes) and torch.equal(got.scale[at:], one.scale)
    assert torch.equal(got.codes[:64], one.codes) and torch.equal(got.scale[:64], one.scale)
    n = at - places[1]
    assert torch.equal(got.codes[places[1]:at], one.codes[:n]) and torch.equal(got.scale[places[1]:at], one.scale[:n])
    assert int(got.codes[64:places[1]].max()) == 0 and float(got.scale[64:places[1]].max()) == float(got.scale[64:65])


def test_quantize_rows_of_nothing_and_off_16_bytes():
    ops = _ops()
    say("quantize_rows of no rows, and of a tensor off 16 bytes")
    empty = ops.quantize_rows(torch.empty((0, 40, 8), device="cuda"))
    assert empty.codes.shape == (0, 2, 2, 2, 4, 16) and empty.values().shape == (0, 40, 8)
    flat = torch.randn(6 * 40 * 8 + 1, device="cuda")
    x = flat[1:].view(6, 40, 8)
    assert x.data_ptr() % 16
    a, b = ops.quantize_rows(x), ops.quantize_rows(x.clone())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scale, b.scale)
    pw, off = ops.prepare_weights(torch.randn(1, 24, 40, 8, device="cuda"), "int8_rows"), _dev(_bounds([6]))
    off_16 = torch.empty(a.block.numel() + 4, device="cuda", dtype=torch.uint8)[4:].copy_(a.block)
    assert off_16.data_ptr() % 16
    assert torch.equal(ops.int8_grouped_linear(ops.Int8Rows(off_16, 6, 40), pw, off), ops.int8_grouped_linear(b, pw, off))


# ---- the product -------------------------------------------------------------------------------

CASES = [
    # rows of each expert, d_in, d_out, gathered, bias
    ([1], 1, 1, False, False),
    ([1], 256, 1024, True, True),
    ([0, 3, 0], 5, 7, True, True),
    ([5, 0, 64, 1], 33, 9, False, True),
    ([65, 31, 2], 64, 64, True, True),
    ([33, 129], 100, 65, True, False),
    ([128, 0, 0, 70], 130, 40, False, True),
    ([300], 31, 130, False, True),
    ([17, 16, 15, 90, 63], 96, 66, True, True),
    ([2] * 64, 32, 8, True, True),
    ([0, 0], 40, 20, False, True),
    ([700, 900, 1, 450], 70, 50, True, True),
]


@pytest.mark.parametrize("rows,d_in,d_out,gathered,with_bias", CASES)
@pytest.mark.parametrize("act,bf16", [("none", False), ("gelu", True), ("gelu", False), ("relu", True),
                                      ("sigmoid", False), ("sigmoid", True)])
def test_product(rows, d_in, d_out, gathered, with_bias, act, bf16):
    ops = _ops()
    g = np.random.default_rng(d_in * 100 + d_out + len(act))
    E, P = len(rows), sum(rows)
    N = max(1, P // 2) if gathered else P
    x = _rows(g, N, d_in, bf16)
    w, b = _weights(g, E, d_out, d_in)
    gather = g.integers(0, N, P).astype(np.int32) if gathered else None
    say(f"int8 product rows={rows} d_in={d_in} d_out={d_out} act={act} bf16={bf16}")
    pw = ops.prepare_weights(_dev(w), "int8_rows")
    pb = ops.prepare_bias(_dev(b)) if with_bias else None
    y = ops.int8_grouped_linear(ops.quantize_rows(_dev(x)), pw, _dev(_bounds(rows)), pb, act,
                                gather=None if gather is None else _dev(gather),
                                out_dtype=torch.bfloat16 if bf16 else torch.float32)
    q, s = io.quantize(x)
    want, size = io.grouped(q, s, _bounds(rows), *io.quantized_weights(w), b if with_bias else None, gather)
    _check(y, want, size, act, bf16, (rows, d_in, d_out))


def test_largest_codes_are_summed_exactly():
    """Codes of +-127 throughout: the sums' largest magnitudes, in every sign."""
    ops = _ops()
    d_in, d_out, P = 640, 40, 70
    g = np.random.default_rng(5)
    # one blade a multivector: every entry of its matrix is 0 or of one magnitude
    x = np.zeros((P, d_in, 8), np.float32)
    w = np.zeros((1, d_out, d_in, 8), np.float32)
    x[..., 0] = g.choice([-2.0, 2.0], (P, d_in))
    w[..., 0] = g.choice([-1.0, 1.0], (1, d_out, d_in))
    x[0, :, 0], w[0, 0, :, 0] = -2.0, 1.0
    x[1], w[0, 1] = 0, 0
    x[1, :, 7] = 2.0  # the pseudoscalar: the imaginary unit
    w[0, 1, :, 7] = 1.0
    say("int8 product of the largest codes")
    y = ops.int8_grouped_linear(ops.quantize_rows(_dev(x)), ops.prepare_weights(_dev(w), "int8_pauli"),
                                _dev(_bounds([P])), out_dtype=torch.float32)
    q, s = io.quantize(x)
    assert np.abs(q).max() == 127
    want, size = io.grouped(q, s, _bounds([P]), *io.quantized_weights(w), None)
    assert np.isclose(want[0, 0, 0], -2.0 * d_in, rtol=1e-5) and np.isclose(want[1, 1, 0], -2.0 * d_in, rtol=1e-5)
    _check(y, want, size, "none", False, "largest codes")


@pytest.mark.parametrize("P", [5, 4000])
def test_most_inputs_with_every_code_at_its_limit(P):
    """16384 inputs, X = 1 + i and W = 1 - i in every entry of their matrices: each product of entries adds 2 127^2 to a sum,
    and the scalar and e1 are the sum of two, 8 16384 127^2 < 2^31; Y = 4 16384 (1 + e1), or less that."""
    ops = _ops()
    d_in, d_out = 16384, 64
    x = torch.zeros(P, d_in, 8, device="cuda", dtype=torch.bfloat16)
    x[..., [0, 1, 6, 7]] = 1.0
    x[1::2] *= -1
    w = torch.zeros(1, d_out, d_in, 8, device="cuda")
    w[..., [0, 1]], w[..., [6, 7]] = 1.0, -1.0
    w[:, 2::3] *= -1
    say(f"int8 product of {P} rows of 16384 inputs")
    y = ops.int8_grouped_linear(ops.quantize_rows(x), ops.prepare_weights(w, "int8_rows"), _dev(_bounds([P])),
                                out_dtype=torch.float32).cpu()
    sign = torch.where(torch.arange(P) % 2 == 1, -1.0, 1.0)[:, None] * torch.where(torch.arange(d_out) % 3 == 2, -1.0, 1.0)
    assert (y[..., 2:] == 0).all()
    # two scales and their product, the sum's conversion and the multiply-add: half a step each
    assert float((y[..., :2] / (sign[..., None] * 4 * d_in) - 1).abs().max()) <= 5 * U32


def test_rows_that_are_not_finite_touch_no_other_row():
    ops = _ops()
    g = np.random.default_rng(8)
    rows, d_in, d_out = [40, 50], 48, 24
    x = _rows(g, 90, d_in, True)
    w, b = _weights(g, 2, d_out, d_in)
    bad = x.copy()
    bad[7, 3, 2], bad[55, 0, 0], bad[89, 47, 7] = np.nan, np.inf, -np.inf
    pw, pb, off = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b)), _dev(_bounds(rows))
    say("int8 product of rows that are not finite")
    for act in ("none", "gelu", "relu", "sigmoid"):
        y0 = ops.int8_grouped_linear(ops.quantize_rows(_dev(x)), pw, off, pb, act, out_dtype=torch.float32)
        y1 = ops.int8_grouped_linear(ops.quantize_rows(_dev(bad)), pw, off, pb, act, out_dtype=torch.float32)
        keep = torch.ones(90, dtype=torch.bool, device="cuda")
        keep[[7, 55, 89]] = False
        assert torch.equal(y0[keep], y1[keep])
        assert torch.isnan(y1[~keep]).all() and torch.isfinite(y0).all()


def test_rows_past_the_last_range_stay_and_gathers_outside_read_zeros():
    ops = _ops()
    g = np.random.default_rng(9)
    E, d_in, d_out, P, N = 3, 40, 70, 200, 50
    w, b = _weights(g, E, d_out, d_in)
    x = _dev(_rows(g, N, d_in, False))
    gather = g.integers(0, N, P).astype(np.int32)
    gather[[3, 100, 120]] = [N, -1, 2 ** 31 - 1]
    pw, pb = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b))
    rows = ops.quantize_rows(x)
    off = _dev(np.array([0, 90, 90, 150], np.int32))
    y = torch.full((P, d_out, 8), 7.0, device="cuda")
    gt = _dev(gather)
    say("int8 product: rows past the last range")
    ops.check(ops.lib().ygg_int8_grouped_linear(
        rows.codes.data_ptr(), rows.scale.data_ptr(), N, gt.data_ptr(), P, pw.data.data_ptr(), pw.scales.data_ptr(),
        pb.data_ptr(), off.data_ptr(), E, d_in, d_out, 0, y.data_ptr(), 0, ops.stream_handle()))
    assert (y[150:] == 7.0).all()
    bt = _dev(b)
    assert torch.equal(y[3], bt[0]) and torch.equal(y[100], bt[2]) and torch.equal(y[120], bt[2])
    gather[[3, 100, 120]] = 0
    whole = ops.int8_grouped_linear(rows, pw, off, pb, gather=_dev(gather), out_dtype=torch.float32)
    keep = torch.ones(150, dtype=torch.bool, device="cuda")
    keep[[3, 100, 120]] = False
    assert torch.equal(y[:150][keep], whole[:150][keep])


def test_a_row_does_not_depend_on_its_batch():
    ops = _ops()
    g = np.random.default_rng(10)
    E, d_in, d_out = 4, 128, 136
    w, b = _weights(g, E, d_out, d_in)
    pw, pb = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b))
    sizes = [900, 40, 0, 700]
    x = _dev(_rows(g, sum(sizes), d_in, True), torch.bfloat16)
    say("int8 product: a row does not depend on its batch")
    rows = ops.quantize_rows(x)
    y = ops.int8_grouped_linear(rows, pw, _dev(_bounds(sizes)), pb, "gelu")
    for first, n, e in ((0, 1, 0), (100, 7, 0), (899, 1, 0), (900, 40, 1), (1300, 200, 3)):
        few = [0] * E
        few[e] = n
        part = ops.int8_grouped_linear(ops.quantize_rows(x[first:first + n]), pw, _dev(_bounds(few)), pb, "gelu")
        assert torch.equal(part, y[first:first + n]), (first, n)


def test_large_fp32_outputs():
    """More output than the caches hold (past L2): the rows of a small batch, bit for bit; channels no multiple of four."""
    ops = _ops()
    g = np.random.default_rng(14)
    E, d_in, d_out, P = 2, 33, 511, 14000
    w, b = _weights(g, E, d_out, d_in)
    pw, pb = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b))
    x = _dev(_rows(g, P, d_in, False))
    say("int8 product of 229 MB of fp32 outputs")
    y = ops.int8_grouped_linear(ops.quantize_rows(x), pw, _dev(_bounds([6000, 8000])), pb, out_dtype=torch.float32)
    for first, n, e in ((0, 700, 0), (5700, 300, 0), (6000, 100, 1), (13300, 700, 1)):
        few = [0, 0]
        few[e] = n
        part = ops.int8_grouped_linear(ops.quantize_rows(x[first:first + n]), pw, _dev(_bounds(few)), pb,
                                       out_dtype=torch.float32)
        assert torch.equal(part, y[first:first + n]), (first, n)


def test_rows_past_2_gib():
    """Codes of more than 2 GiB and outputs of more than 4, in place: 64-bit addresses, the rows of a small batch bit for
    bit; gathered, such rows are refused."""
    ops = _ops()
    g = np.random.default_rng(15)
    E, d_in, d_out, P = 3, 260, 256, 1_100_000
    w, b = _weights(g, E, d_out, d_in)
    pw, pb = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b))
    bounds = [0, 100, 1_050_000, P]
    say("int8 product of codes past 2 GiB")
    part = _dev(_rows(g, 1000, d_in, True), torch.bfloat16)
    x = torch.zeros(P, d_in, 8, device="cuda", dtype=torch.bfloat16)
    places = [0, 500_000, 1_049_500, P - 1000]
    for at in places:
        x[at:at + 1000] = part
    rows = ops.quantize_rows(x)
    assert rows.codes.numel() > 2 ** 31 and P * d_out * 16 > 2 ** 32
    del x
    y = ops.int8_grouped_linear(rows, pw, _dev(np.array(bounds, np.int32)), pb, "relu")
    one = [ops.int8_grouped_linear(ops.quantize_rows(part), pw, _dev(_bounds([1000 if e == f else 0 for f in range(E)])), pb,
                                   "relu") for e in range(E)]
    for at in places:
        for first, e in ((0, 0), (100, 1), (1_050_000, 2)):
            lo, hi = max(at, first), min(at + 1000, bounds[e + 1])
            if lo < hi:
                assert torch.equal(y[lo:hi], one[e][lo - at:hi - at]), (at, e)
    with pytest.raises(Exception, match="2 GiB"):
        ops.int8_grouped_linear(rows, pw, _dev(np.array(bounds, np.int32)), pb,
                                gather=torch.zeros(P, device="cuda", dtype=torch.int32))


def test_on_another_stream():
    ops = _ops()
    g = np.random.default_rng(11)
    w, b = _weights(g, 2, 64, 64)
    x = _dev(_rows(g, 500, 64, True), torch.bfloat16)
    pw, pb, off = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b)), _dev(_bounds([200, 300]))
    say("int8 product on another stream")
    want = ops.int8_grouped_linear(ops.quantize_rows(x), pw, off, pb, "relu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.int8_grouped_linear(ops.quantize_rows(x), pw, off, pb, "relu")
    side.synchronize()
    assert torch.equal(got, want)


# ---- the experts, the layer and the block --------------------------------------------------------


def _layer(g, N, d, F, E, k, router="logits", act="gelu"):
    from yggdrasil_amd import CliffordMoELayer, MoEHLMConfig

    cfg = MoEHLMConfig(d_model=d, d_ff=F, n_experts=E, top_k=k, activation=act, dtype=torch.bfloat16,
                       weight_format="int8_rows", router=router)
    layer = CliffordMoELayer(cfg, device="cuda")
    with torch.no_grad():
        for p in (layer.b_up, layer.b_down):
            p.copy_(0.2 * torch.randn_like(p))
    x = _dev(_rows(g, N, d, True), torch.bfloat16).view(1, N, d, 8)
    return layer, x, _dev(g.standard_normal((1, N, E)).astype(np.float32))


@pytest.mark.parametrize("N,d,F,E,k,act", [(1, 8, 16, 4, 2, "gelu"), (40, 33, 70, 5, 3, "relu"), (300, 64, 130, 8, 2, "gelu"),
                                           (130, 130, 40, 64, 8, "sigmoid"), (2000, 32, 64, 16, 2, "gelu")])
def test_layer_is_its_operators(N, d, F, E, k, act):
    """The layer against route, quantize_rows, the two products, and combine, bit for bit; and experts() likewise."""
    ops = _ops()
    g = np.random.default_rng(N + d)
    layer, x, logits = _layer(g, N, d, F, E, k, act=act)
    say(f"int8_rows layer N={N} d={d} F={F} E={E} k={k} act={act}")
    out = layer.moe_forward(x, logits=logits, residual=x)
    r = ops.route(logits.view(N, E), k)
    wu, wd = (ops.prepare_weights(p.detach(), "int8_rows") for p in (layer.w_up, layer.w_down))
    bu, bd = ops.prepare_bias(layer.b_up.detach()), ops.prepare_bias(layer.b_down.detach())
    flat = x.view(N, d, 8)
    h = ops.int8_grouped_linear(ops.quantize_rows(flat), wu, r.offsets, bu, act, gather=r.perm)
    y = ops.int8_grouped_linear(ops.quantize_rows(h), wd, r.offsets, bd)
    assert torch.equal(out.view(N, d, 8), ops.combine(y, r, residual=flat))
    y2 = layer.experts(ops.dispatch(flat, r), r.offsets[:-1], r.counts)
    assert torch.equal(y2, y)


def test_layer_against_float64():
    """Against the float64 layer whose rows are quantized where the layer quantizes them.  h is rounded to bf16 and then to
    codes: where fp32 and float64 fall on two sides of a border, h moves by 2^-7 of its value or by a code's step, so
    the outputs are compared at BASELINE's 2e-2 for int8 weights, normwise."""
    ops = _ops()
    g = np.random.default_rng(77)
    N, d, F, E, k = 96, 40, 72, 6, 2
    layer, x, logits = _layer(g, N, d, F, E, k)
    say("int8_rows layer against float64")
    out = layer.moe_forward(x, logits=logits).view(N, d, 8).double().cpu().numpy()
    r = {n: t.cpu().numpy() for n, t in layer.last_routing.items()}
    xs = x.view(N, d, 8).float().cpu().numpy()
    w = {n: p.detach().cpu().numpy() for n, p in layer.named_parameters()}
    want = np.zeros_like(out)
    for e in range(E):
        tok, slot = np.nonzero(r["topk_idx"] == e)
        q, s = io.quantize(xs[tok])
        h = io.activate(io.product(q, s, *(v[e] for v in io.quantized_weights(w["w_up"])), w["b_up"][e])[0], "gelu")[0]
        q, s = io.quantize(bf16_round(h.astype(np.float32)))
        y = io.product(q, s, *(v[e] for v in io.quantized_weights(w["w_down"])), w["b_down"][e])[0]
        np.add.at(want, tok, r["topk_w"][tok, slot][:, None, None] * y)
    assert np.abs(out - want).max() <= 2e-2 * np.abs(want).max()


@pytest.mark.parametrize("router", ["energy", "logits", "clifford_head"])
def test_layer_and_block_routers(router):
    """Both modules with every router: the same outputs as their bf16 form up to what int8 costs (two roundings to 8 bits,
    about 1/127 of the largest value each, added over d and F terms: a tenth of the largest output is far above)."""
    from yggdrasil_amd import CliffordMoEBlockFFN, MoEHLMConfig

    torch.manual_seed(4)
    blocks = []
    for fmt in ("int8_rows", "pauli"):
        cfg = MoEHLMConfig(d_model=64, d_ff=128, n_experts=8, top_k=2, dtype=torch.bfloat16, weight_format=fmt, router=router)
        blocks.append(CliffordMoEBlockFFN(cfg, device="cuda"))
    blocks[0].load_state_dict(blocks[1].state_dict())
    x = torch.randn(2, 150, 64, 8, device="cuda").bfloat16()
    lg = torch.randn(2, 150, 8, device="cuda") if router == "logits" else None
    say(f"int8_rows block router={router}")
    a, b = (m(x, logits=lg).float() for m in blocks)
    assert torch.isfinite(a).all()
    assert float((a - b).abs().max()) <= 0.1 * float((b - x.float()).abs().max())
    out, aux = blocks[0].moe(x.view(2, 150, 512), logits=lg)
    assert out.shape == (2, 150, 512) and torch.isfinite(aux)


def test_captured_layer_replays():
    g = np.random.default_rng(12)
    layer, x, logits = _layer(g, 700, 64, 96, 8, 2)
    say("int8_rows layer captured")
    with torch.no_grad():
        want = layer.moe_forward(x, logits=logits).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.moe_forward(x, logits=logits)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.moe_forward(x, logits=logits)
        for r in range(4):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), f"replay {r}"
            assert torch.equal(layer.moe_forward(x, logits=logits), want)
            layer.moe_forward(torch.cat([x, x], 1), logits=torch.cat([logits, logits], 1))  # a larger eager call between
        layer.w_up.mul_(0.5)  # an eager call lays the weights out anew, in the place that the graph reads
        x.copy_(torch.randn_like(x.float()).bfloat16())
        want = layer.moe_forward(x, logits=logits)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", ["int8_rows", "pauli"])
def test_experts_of_any_bounds(fmt):
    """Ranges as int32, int64 or another type, and malformed ones: brought into ascending order inside the rows, in every
    format."""
    ops = _ops()
    torch.manual_seed(6)
    E, d, F, P = 4, 16, 24, 50
    wu = ops.prepare_weights(torch.randn(E, F, d, 8, device="cuda") / (8 * d) ** 0.5, fmt)
    wd = ops.prepare_weights(torch.randn(E, d, F, 8, device="cuda") / (8 * F) ** 0.5, fmt)
    x = torch.randn(P, d, 8, device="cuda").bfloat16()
    off, cnt = torch.tensor([0, 20, 20, 35], device="cuda"), torch.tensor([20, 0, 15, 15], device="cuda")
    say(f"experts of any bounds {fmt}")
    want = ops.grouped_experts(x, off, cnt, wu, wd)
    for dt in (torch.int32, torch.int16):
        assert torch.equal(ops.grouped_experts(x, off.to(dt), cnt.to(dt), wu, wd), want)
    bad_off = torch.tensor([-5, 30, 10, 35], device="cuda")
    for dt in (torch.int32, torch.int64):
        bounds = torch.empty(E + 1, device="cuda", dtype=torch.int32)
        o, c = bad_off.to(dt), torch.tensor([3, 3, 3, 2 ** 31 - 40], device="cuda").to(dt)
        ops.check(ops.lib().ygg_expert_bounds(o.data_ptr(), c.data_ptr(), o.element_size(), E, P, bounds.data_ptr(),
                                              ops.stream_handle()))
        assert bounds.tolist() == [0, 30, 30, 35, P]
    y = ops.grouped_experts(x, bad_off, torch.tensor([3, 3, 3, 15], device="cuda"), wu, wd)
    good = ops.grouped_experts(x, torch.tensor([0, 30, 30, 35], device="cuda"), torch.tensor([30, 0, 5, 15], device="cuda"),
                               wu, wd)
    assert torch.equal(y, good)
    one = ops.grouped_experts(x, torch.tensor([0, 0, 0, 0], device="cuda"), torch.tensor([0, 0, 0, 50], device="cuda"), wu, wd)
    assert torch.equal(one[35:], want[35:])  # the same expert's rows


def test_empty_batch():
    g = np.random.default_rng(13)
    layer, _, _ = _layer(g, 4, 16, 24, 4, 2)
    say("int8_rows layer of no tokens")
    out = layer.moe_forward(torch.empty(1, 0, 16, 8, device="cuda", dtype=torch.bfloat16),
                            logits=torch.empty(1, 0, 4, device="cuda"))
    assert out.shape == (1, 0, 16, 8) and int(layer.last_routing["counts"].sum()) == 0


def test_refusals():
    from yggdrasil_amd import ops

    x = torch.randn(6, 40, 8, device="cuda")
    rows = ops.quantize_rows(x)
    pw = ops.prepare_weights(torch.randn(2, 8, 40, 8, device="cuda"), "int8_rows")
    off = torch.tensor([0, 3, 6], device="cuda", dtype=torch.int32)
    say("int8 rows: refusals")
    for bad in (x[0], x.double(), x.half(), x[:, :, :4], x.transpose(0, 1)):
        with pytest.raises(ValueError):
            ops.quantize_rows(bad)
    for kwargs in (dict(offsets=off[:2]), dict(offsets=off.long()), dict(act="tanh"), dict(out_dtype=torch.float16),
                   dict(gather=torch.zeros(6, device="cuda")), dict(bias_prepared=torch.zeros(2, 7, 8, device="cuda")),
                   dict(pw=ops.prepare_weights(torch.randn(2, 8, 40, 8, device="cuda"), "pauli")),
                   dict(pw=ops.prepare_weights(torch.randn(2, 8, 41, 8, device="cuda"), "int8_rows")),
                   dict(rows=ops.Int8Rows(rows.block[:-1], 6, 40)), dict(rows=ops.Int8Rows(rows.block, 7, 40)),
                   dict(rows=ops.Int8Rows(rows.block, 6, 39)), dict(rows=ops.Int8Rows(rows.block.float(), 6, 40)),
                   dict(rows=ops.Int8Rows(rows.block.cpu(), 6, 40)), dict(offsets=off.cpu())):
        with pytest.raises(ValueError):
            ops.int8_grouped_linear(**{**dict(rows=rows, pw=pw, offsets=off), **kwargs})
    with pytest.raises(ValueError):  # fp32 rows into bf16 experts
        ops.grouped_experts(x, off[:2], torch.tensor([3, 3], device="cuda", dtype=torch.int32), pw,
                            ops.prepare_weights(torch.randn(2, 40, 8, 8, device="cuda"), "int8_rows"))
