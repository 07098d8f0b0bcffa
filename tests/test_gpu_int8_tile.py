"""The kernel for many outputs of int8 products: against whole-number sums and float64 (``_int8_oracle``), tolerances as in
``test_gpu_int8_rows``, and bit for bit against the kernel for few.  Every size says which kernel it takes."""

import functools

import numpy as np
import pytest
import torch

import _int8_oracle as io
from _gpu_helpers import say
from test_gpu_int8_rows import _bounds, _check, _dev, _layer, _ops, _rows, _weights

pytestmark = pytest.mark.gpu


def _many(P, d_out):
    assert _ops().lib().ygg_int8_product_small(P, d_out) == 0, (P, d_out)


# rows of each expert (tiles are of 64 rows: whole ones, last ones of 33 to 63 and of 1 to 32), d_in, d_out, gathered, bias
CASES = [
    ([700, 33, 1, 32, 63, 0, 64], 31, 240, True, True),
    ([1000, 17, 47], 32, 200, False, False),
    ([400, 31, 96, 129, 2], 70, 330, True, True),
    ([2100], 130, 100, False, True),
    ([5] * 64, 66, 640, True, True),
    ([300, 0, 500], 33, 257, False, True),
    ([3200], 5, 65, True, False),
    ([13000], 40, 1, True, True),
    ([9000, 5000, 33], 20, 4, False, True),
]


@functools.lru_cache(maxsize=2)
def _case(n):
    rows, d_in, d_out, gathered, with_bias = CASES[n]
    g = np.random.default_rng(100 + n)
    E, P = len(rows), sum(rows)
    N = max(1, P // 2) if gathered else P
    x = _rows(g, N, d_in, False)
    w, b = _weights(g, E, d_out, d_in)
    gather = g.integers(0, N, P).astype(np.int32) if gathered else None
    q, s = io.quantize(x)
    want, size = io.grouped(q, s, _bounds(rows), *io.quantized_weights(w), b if with_bias else None, gather)
    return x, w, b, gather, want, size


@pytest.mark.parametrize("n", range(len(CASES)))
@pytest.mark.parametrize("act", ["none", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("bf16", [False, True])
def test_product(n, act, bf16):
    ops = _ops()
    rows, d_in, d_out, _, with_bias = CASES[n]
    _many(sum(rows), d_out)
    x, w, b, gather, want, size = _case(n)
    say(f"int8 tiles rows={rows} d_in={d_in} d_out={d_out} act={act} bf16={bf16}")
    y = ops.int8_grouped_linear(ops.quantize_rows(_dev(x)), ops.prepare_weights(_dev(w), "int8_rows"), _dev(_bounds(rows)),
                                ops.prepare_bias(_dev(b)) if with_bias else None, act,
                                gather=None if gather is None else _dev(gather),
                                out_dtype=torch.bfloat16 if bf16 else torch.float32)
    _check(y, want, size, act, bf16, (rows, d_in, d_out))


@pytest.mark.parametrize("d_in", [20, 50, 100, 300])
@pytest.mark.parametrize("bf16", [False, True])
def test_gathered_rows_over_many_tiles(d_in, bf16):
    """At least eight tiles a workgroup, whole, short and cut ones, one K step a tile and several: a gathered product is the
    product of the gathered rows, and rows of each expert alone are the few-row kernel's."""
    ops = _ops()
    g = np.random.default_rng(d_in)
    E, d_out, N = 9, 520, 7000
    sizes = [9000, 31, 4033, 0, 6400, 12000, 1, 8001, 97]
    P = sum(sizes)
    _many(P, d_out)
    assert (P // 64) * ((d_out + 63) // 64) >= 8 * 512
    x = _dev(_rows(g, N, d_in, True), torch.bfloat16)
    w, b = _weights(g, E, d_out, d_in)
    pw, pb, off = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b)), _dev(_bounds(sizes))
    gather = _dev(g.integers(0, N, P).astype(np.int32))
    dt = torch.bfloat16 if bf16 else torch.float32
    say(f"int8 tiles gathered, {P} rows of {d_in}, bf16={bf16}")
    rows = ops.quantize_rows(x)
    y = ops.int8_grouped_linear(rows, pw, off, pb, "relu", gather=gather, out_dtype=dt)
    xs = x[gather.long()]
    assert torch.equal(y, ops.int8_grouped_linear(ops.quantize_rows(xs), pw, off, pb, "relu", out_dtype=dt))
    bounds = _bounds(sizes)
    for e in range(E):
        for first in (bounds[e], bounds[e + 1] - 80):
            first, last = max(first, bounds[e]), min(max(first, bounds[e]) + 80, bounds[e + 1])
            if last > first:
                assert ops.lib().ygg_int8_product_small(int(last - first), d_out) == 1
                few = [0] * E
                few[e] = last - first
                one = ops.int8_grouped_linear(ops.quantize_rows(xs[first:last]), pw, _dev(_bounds(few)), pb, "relu",
                                              out_dtype=dt)
                assert torch.equal(y[first:last], one), (e, first)


def test_rows_that_are_not_finite_touch_no_other_row():
    ops = _ops()
    g = np.random.default_rng(20)
    sizes, d_in, d_out = [410, 690], 48, 200
    _many(1100, d_out)
    x = _rows(g, 1100, d_in, True)
    w, b = _weights(g, 2, d_out, d_in)
    bad = x.copy()
    rows = [7, 409, 410, 900, 1099]
    bad[7, 3, 2], bad[409, 0, 0], bad[410, 47, 7], bad[900, 20, 4], bad[1099, 1, 1] = np.nan, np.inf, -np.inf, np.nan, np.inf
    pw, pb, off = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b)), _dev(_bounds(sizes))
    keep = torch.ones(1100, dtype=torch.bool, device="cuda")
    keep[rows] = False
    say("int8 tiles of rows that are not finite")
    for act in ("none", "gelu", "relu", "sigmoid"):
        for dt in (torch.float32, torch.bfloat16):
            y0, y1 = (ops.int8_grouped_linear(ops.quantize_rows(_dev(v)), pw, off, pb, act, out_dtype=dt) for v in (x, bad))
            assert torch.equal(y0[keep], y1[keep]) and torch.isfinite(y0).all() and torch.isnan(y1[~keep]).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rows_past_the_last_range_stay_and_gathers_outside_read_zeros(dt):
    ops = _ops()
    g = np.random.default_rng(21)
    E, d_in, d_out, P, N = 3, 40, 130, 2000, 500
    _many(P, d_out)
    w, b = _weights(g, E, d_out, d_in)
    x = _dev(_rows(g, N, d_in, False))
    gather = g.integers(0, N, P).astype(np.int32)
    outside = {3: N, 63: -1, 899: 2 ** 31 - 1, 900: -2 ** 31, 1500: N + 7}
    for r, src in outside.items():
        gather[r] = src
    pw, pb = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b))
    rows, bt = ops.quantize_rows(x), _dev(b).to(dt)
    off = _dev(np.array([0, 900, 900, 1501], np.int32))
    gt = _dev(gather)
    keep = torch.ones(1501, dtype=torch.bool, device="cuda")
    keep[list(outside)] = False
    gather[list(outside)] = 0
    say(f"int8 tiles: rows past the last range {dt}")
    for gt_ in (gt, None):
        y = torch.full((P, d_out, 8), 7.0, device="cuda", dtype=dt)
        src = rows if gt_ is not None else ops.quantize_rows(x[torch.arange(P, device="cuda") % N])
        ops.check(ops.lib().ygg_int8_grouped_linear(
            src.codes.data_ptr(), src.scale.data_ptr(), src.rows, None if gt_ is None else gt_.data_ptr(), P,
            pw.data.data_ptr(), pw.scales.data_ptr(), pb.data_ptr(), off.data_ptr(), E, d_in, d_out, 0, y.data_ptr(),
            ops.DTYPE_CODE[dt], ops.stream_handle()))
        assert (y[1501:] == 7.0).all() and (y[:1501] != 7.0).any(-1).any(-1).all()
        if gt_ is not None:
            for r in outside:
                assert torch.equal(y[r], bt[0 if r < 900 else 2]), r
            whole = ops.int8_grouped_linear(rows, pw, off, pb, gather=_dev(gather), out_dtype=dt)
            assert torch.equal(y[:1501][keep], whole[:1501][keep])


def test_on_another_stream():
    ops = _ops()
    g = np.random.default_rng(22)
    sizes = [1500, 2300]
    _many(3800, 64)
    w, b = _weights(g, 2, 64, 64)
    x = _dev(_rows(g, 3800, 64, True), torch.bfloat16)
    pw, pb, off = ops.prepare_weights(_dev(w), "int8_rows"), ops.prepare_bias(_dev(b)), _dev(_bounds(sizes))
    say("int8 tiles on another stream")
    want = ops.int8_grouped_linear(ops.quantize_rows(x), pw, off, pb, "gelu")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.int8_grouped_linear(ops.quantize_rows(x), pw, off, pb, "gelu")
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_layer_and_experts_replay():
    """Both products of the layer, and of the experts on grouped rows, on the kernel for many outputs."""
    ops = _ops()
    N, d, F, E, k = 1700, 64, 96, 8, 2
    _many(N * k, d), _many(N * k, F)
    layer, x, logits = _layer(np.random.default_rng(23), N, d, F, E, k)
    say("int8 tiles: layer and experts captured")
    with torch.no_grad():
        r = ops.route(logits.view(N, E), k)
        xs = ops.dispatch(x.view(N, d, 8), r)

        def both():
            return layer.moe_forward(x, logits=logits), layer.experts(xs, r.offsets[:-1], r.counts)

        want = [t.clone() for t in both()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        for n in range(4):
            for t in out:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), f"replay {n}"
            assert all(torch.equal(a, b) for a, b in zip(both(), want))
