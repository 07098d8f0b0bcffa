"""Weights of the int8 Pauli formats that are not finite, and more channels than one launch prepares."""

import numpy as np
import pytest
import torch

from _gpu_helpers import say
from oracle import moe
from test_gpu_int8_rows import _ops

pytestmark = pytest.mark.gpu

BAD = {(0, 3): float("nan"), (1, 0): float("inf"), (1, 23): -float("inf")}  # (expert, channel)


def _weights(E, d_out, d_in, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w = torch.randn(E, d_out, d_in, 8, generator=g, device="cuda") / (8 * d_in) ** 0.5
    bad = w.clone()
    for n, ((e, j), v) in enumerate(BAD.items()):
        bad[e, j, (7 * n) % d_in, (3 * n + 1) % 8] = v
    return w, bad


@pytest.mark.parametrize("d_in", [1, 40, 300])
@pytest.mark.parametrize("fmt", ["int8_rows", "int8_pauli"])
def test_scales_and_codes(d_in, fmt):
    """A channel that is not finite has the scale NaN and codes of zero; every other one is as without it."""
    ops = _ops()
    w, bad = _weights(2, 24, d_in)
    say(f"prepare weights that are not finite, d_in={d_in} {fmt}")
    a, b = ops.prepare_weights(w, fmt), ops.prepare_weights(bad, fmt)
    off = torch.zeros(2, 24, dtype=torch.bool, device="cuda")
    for at in BAD:
        off[at] = True
    sa, sb = a.scales.view(2, 24), b.scales.view(2, 24)
    assert torch.equal(sa[~off], sb[~off]) and torch.isnan(sb[off]).all() and torch.isfinite(sa).all()
    # [expert][8 channels][K step][U, V][g][2 jj + a][16 bytes]
    shape = (2, 3, (d_in + 31) // 32, 2, 4, 8, 32)
    ca, cb = (p.data.view(torch.int8).reshape(shape).permute(0, 1, 5, 2, 3, 4, 6).reshape(2, 24, -1) for p in (a, b))
    assert torch.equal(ca[~off], cb[~off]) and (cb[off] == 0).all()


@pytest.mark.parametrize("P", [6, 20000])
@pytest.mark.parametrize("act", ["none", "gelu", "relu", "sigmoid"])
def test_product(P, act):
    """Only the channel's own outputs are NaN, in the kernels for few and for many outputs."""
    ops = _ops()
    w, bad = _weights(2, 24, 40)
    assert ops.lib().ygg_int8_product_small(P, 24) == (P == 6)
    x = torch.randn(P, 40, 8, device="cuda").bfloat16()
    off = torch.tensor([0, P // 2, P], device="cuda", dtype=torch.int32)
    say(f"int8 product with weights that are not finite, P={P} {act}")
    rows = ops.quantize_rows(x)
    y0, y1 = (ops.int8_grouped_linear(rows, ops.prepare_weights(v, "int8_rows"), off, None, act) for v in (w, bad))
    mask = torch.zeros(P, 24, dtype=torch.bool, device="cuda")
    for e, j in BAD:
        mask[int(off[e]):int(off[e + 1]), j] = True
    assert torch.equal(y0[~mask], y1[~mask]) and torch.isnan(y1[mask]).all() and torch.isfinite(y0).all()


@pytest.mark.parametrize("fmt", ["int8_rows", "int8_pauli"])
@pytest.mark.parametrize("where", ["up", "down", "bias"])
def test_layer(fmt, where):
    """Tokens of the experts that have no such weight (or bias of a hidden channel) are as without it; the others' outputs
    hold NaN."""
    from yggdrasil_amd import CliffordMoELayer, MoEHLMConfig

    torch.manual_seed(3)
    N, d, F, E, k = 60, 32, 48, 4, 2
    layer = CliffordMoELayer(MoEHLMConfig(d_model=d, d_ff=F, n_experts=E, top_k=k, dtype=torch.bfloat16, weight_format=fmt,
                                          router="logits"), device="cuda")
    x, lg = torch.randn(1, N, d, 8, device="cuda").bfloat16(), torch.randn(1, N, E, device="cuda")
    say(f"{fmt} layer with a weight that is NaN, {where}")
    with torch.no_grad():
        want = layer.moe_forward(x, logits=lg).clone()
        if where == "bias":
            layer.b_up[1, 5, 2] = float("nan")
        else:
            (layer.w_up if where == "up" else layer.w_down)[1, 5, 3, 2] = float("nan")
        got = layer.moe_forward(x, logits=lg)
    hit = (layer.last_routing["topk_idx"] == 1).any(1)
    assert torch.equal(got[0][~hit], want[0][~hit]) and bool(hit.any()) and not bool(hit.all())
    nan = torch.isnan(got[0][hit]).all(-1)
    assert nan.all() if where != "down" else nan[:, 5].all() and torch.equal(got[0][hit][~nan], want[0][hit][~nan])


def test_bits_of_finite_weights():
    ops = _ops()
    g = np.random.default_rng(0)
    w = (g.standard_normal((2, 9, 33, 8)) * 10.0 ** g.integers(-30, 30, (2, 9, 1, 1))).astype(np.float32)
    w[1, 4] = 3.0e38  # entries past fp32's largest
    say("prepare finite weights, far ones")
    q, s = moe.quantize_int8_pauli(w)
    assert np.array_equal(ops.prepare_weights(torch.from_numpy(w).cuda(), "int8_rows").scales.cpu().numpy().ravel(),
                          np.asarray(s).ravel())


def test_more_channels_than_one_launch_prepares():
    """The most channels a product takes, of 33 experts: 2^24 and more in all.  Every expert as it is prepared alone."""
    ops = _ops()
    E, d_out = 33, 524288
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    w = torch.randn(E, d_out, 1, 8, generator=g, device="cuda")
    say(f"prepare {E * d_out} channels")
    pw = ops.prepare_weights(w, "int8_rows")
    data, scales = pw.data.view(E, -1), pw.scales.view(E, d_out)
    x = torch.randn(3, 1, 8, device="cuda").bfloat16()
    rows = ops.quantize_rows(x)
    for e in (0, 1, 15, 31, 32):
        one = ops.prepare_weights(w[e:e + 1].contiguous(), "int8_rows")
        assert torch.equal(scales[e], one.scales.view(-1)) and torch.equal(data[e], one.data.view(-1)), e
        bounds = torch.zeros(E + 1, device="cuda", dtype=torch.int32)
        bounds[e + 1:] = 3
        alone = torch.tensor([0, 3], device="cuda", dtype=torch.int32)
        assert torch.equal(ops.int8_grouped_linear(rows, pw, bounds), ops.int8_grouped_linear(rows, one, alone)), e
