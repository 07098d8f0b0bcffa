"""What the int8 rows' and the sort gradients' C entries refuse, on the CPU: their checks come before any launch."""

import os

import pytest
import torch

from yggdrasil_amd import _native as N
from yggdrasil_amd import ops

pytestmark = pytest.mark.skipif(not os.path.exists(N.LIB_PATH), reason="library not built")
P = 4096  # a pointer that no check may follow
FAR = [P + (i << 40) for i in range(8)]  # eight tensors that share nothing


def _refused(name, args, word):
    lib = N.lib()
    assert getattr(lib, name)(*args) == -1
    assert word in lib.ygg_last_error().decode(), lib.ygg_last_error()


@pytest.mark.parametrize("args,word", [
    ((FAR[0], 2, 4, 4, FAR[1], FAR[2], None), "dtype"),
    ((FAR[0], 0, -1, 4, FAR[1], FAR[2], None), "bad sizes"),
    ((FAR[0], 0, 4, 0, FAR[1], FAR[2], None), "bad sizes"),
    ((None, 0, 4, 4, FAR[1], FAR[2], None), "null"),
    ((FAR[0], 0, 4, 4, None, FAR[2], None), "null"),
    ((FAR[0], 0, 4, 4, FAR[1], None, None), "null"),
    ((FAR[0], 0, 4, 4, FAR[0] + 256, FAR[2], None), "share"),
    ((FAR[0], 0, 4, 4, FAR[1], FAR[0] + 508, None), "share"),
    ((FAR[0], 0, 4, 4, FAR[1], FAR[1] + 1020, None), "share"),
])
def test_quantize_rows(args, word):
    _refused("ygg_quantize_rows", args, word)


_LIN = [FAR[0], FAR[1], 8, None, 8, FAR[2], FAR[3], None, FAR[4], 2, 40, 24, 0, FAR[5], 1, None]


@pytest.mark.parametrize("at,value,word", [
    (0, None, "null"), (1, None, "null"), (5, None, "null"), (6, None, "null"), (8, None, "null"), (13, None, "null"),
    (2, -1, "bad sizes"), (2, 7, "7 rows"), (4, -1, "bad sizes"), (9, 0, "bad sizes"), (9, 65, "bad sizes"),
    (10, 0, "bad sizes"), (10, 16385, "bad sizes"), (11, 0, "bad sizes"), (12, 4, "activation"), (14, 2, "dtype")])
def test_product(at, value, word):
    args = list(_LIN)
    args[at] = value
    _refused("ygg_int8_grouped_linear", args, word)


@pytest.mark.parametrize("at,value", [(0, FAR[5] + 16), (1, FAR[5] + 8), (3, FAR[5] + 60), (5, FAR[5] - 8), (6, FAR[5] + 4),
                                      (7, FAR[5] + 32), (8, FAR[5] + 100)])
def test_product_in_place(at, value):
    args = list(_LIN)
    args[at] = value
    _refused("ygg_int8_grouped_linear", args, "share")


_EXP = [FAR[0], 8, FAR[1], FAR[2], None, FAR[3], FAR[4], None, FAR[5], FAR[5] + 1024, 4, 2, 40, 24, 1, FAR[6], FAR[7], 1 << 20,
        None]


@pytest.mark.parametrize("at,value,word", [
    (0, None, "null"), (2, None, "null"), (3, None, "null"), (5, None, "null"), (6, None, "null"), (8, None, "null"),
    (9, None, "null"), (15, None, "null"), (16, None, "null"), (1, -1, "bad sizes"), (11, 0, "bad sizes"),
    (11, 65, "bad sizes"), (12, 0, "bad sizes"), (13, 0, "bad sizes"), (14, 4, "activation"), (10, 2, "bytes"),
    (12, 20000, "16384"), (13, 20000, "16384"), (17, 100, "workspace"), (16, FAR[0], "share"), (16, FAR[6] + 16, "share"),
    (16, FAR[5], "share"), (16, FAR[5] + 1024, "share")])
def test_experts(at, value, word):
    args = list(_EXP)
    args[at] = value
    _refused("ygg_int8_grouped_experts", args, word)


@pytest.mark.parametrize("at", [2, 3, 4, 5, 6, 7])
@pytest.mark.parametrize("on", [_EXP[14 + 1], _EXP[14 + 2]])
def test_experts_over_their_weights(at, on):
    args = list(_EXP)
    args[at] = on + 16
    _refused("ygg_int8_grouped_experts", args, "share")


@pytest.mark.parametrize("args,word", [
    ((P, P, 4, 0, 8, P, None), "bad sizes"), ((P, P, 4, 65, 8, P, None), "bad sizes"), ((P, P, 4, 2, -1, P, None), "bad sizes"),
    ((P, P, 2, 2, 8, P, None), "bytes"), ((None, P, 4, 2, 8, P, None), "null"), ((P, None, 4, 2, 8, P, None), "null"),
    ((P, P, 4, 2, 8, None, None), "null")])
def test_bounds(args, word):
    _refused("ygg_expert_bounds", args, word)


_COMB = [FAR[0], 0, FAR[1], 8, 2, 4, 16, FAR[2], FAR[3], FAR[4], 0, 0, FAR[5], None]


@pytest.mark.parametrize("at,value,word", [
    (0, None, "null"), (7, None, "null"), (8, None, "null"), (9, None, "null"), (1, 2, "dtype"), (10, 2, "dtype"),
    (3, -1, "bad sizes"), (4, 0, "bad sizes"), (4, 9, "bad sizes"), (5, 0, "bad sizes"), (6, -1, "bad sizes"),
    (11, 2, "layout"), (2, None, "needs y_sorted"), (12, None, "needs y_sorted"), (9, FAR[0], "share"), (9, FAR[1], "share"),
    (9, FAR[2], "share"), (9, FAR[3], "share"), (12, FAR[0], "share"), (12, FAR[1], "share"), (12, FAR[2], "share"),
    (12, FAR[3], "share"), (12, FAR[4], "share")])
def test_combine_backward(at, value, word):
    args = list(_COMB)
    args[at] = value
    _refused("ygg_combine_backward", args, word)


_DISP = [FAR[0], 0, 8, 2, 4, 16, FAR[1], FAR[2], FAR[3], None]


@pytest.mark.parametrize("at,value,word", [
    (0, None, "null"), (6, None, "null"), (8, None, "null"), (1, 3, "dtype"), (2, -1, "bad sizes"), (3, 0, "bad sizes"),
    (3, 9, "bad sizes"), (4, 0, "bad sizes"), (5, -1, "bad sizes"), (8, FAR[0], "share"), (8, FAR[1], "share"),
    (8, FAR[2] + 32, "share")])
def test_dispatch_backward(at, value, word):
    args = list(_DISP)
    args[at] = value
    _refused("ygg_dispatch_backward", args, word)


def test_nothing_to_do_needs_no_gpu():
    lib = N.lib()
    assert lib.ygg_quantize_rows(None, 0, 0, 4, None, None, None) == 0
    assert lib.ygg_int8_grouped_linear(None, None, 0, None, 0, None, None, None, None, 1, 4, 4, 0, None, 0, None) == 0
    assert lib.ygg_combine_backward(None, 0, None, 0, 2, 4, 0, None, None, None, 0, 0, None, None) == 0
    assert lib.ygg_dispatch_backward(None, 0, 0, 2, 4, 0, None, None, None, None) == 0
    assert lib.ygg_int8_rows_bytes(3, 33) == 3 * 2 * 2 * 128 and lib.ygg_int8_rows_bytes(3, 0) == 0


_FWD = [P, 1, 4, 8, 8, 4, 2, 1, P, None, None, P, P, None, P, P, None, 6, None, P, P, P, P, P, P, 1 << 30, None]


@pytest.mark.parametrize("at,value,word", [(1, 0, "does not match dtype"), (12, None, "scales"), (15, None, "scales"),
                                           (25, 64, "workspace"), (4, 40000, "16384"), (3, 40000, "16384")])
def test_layer(at, value, word):
    args = list(_FWD)
    args[at] = value
    _refused("ygg_moe_forward", args, word)


def test_cpu_tensors_and_configurations():
    from yggdrasil_amd import MoEHLMConfig

    x = torch.zeros(4, 8, 8)
    z = torch.zeros(4, 2, dtype=torch.int32)
    r = ops.Routing(z, z.float(), z[0], z[0], z[0], z)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.combine_backward(x, None, r), lambda: ops.dispatch_backward(x, r)):
        with pytest.raises(ValueError):
            call()
    assert MoEHLMConfig(d_model=7, d_ff=5, dtype=torch.bfloat16, weight_format="int8_rows").weight_format == "int8_rows"
    for kwargs in (dict(dtype=torch.float32), dict(dtype=torch.bfloat16, bf16_grad=True),
                   dict(dtype=torch.bfloat16, router_grad=True)):
        with pytest.raises(ValueError):
            MoEHLMConfig(d_model=8, d_ff=16, weight_format="int8_rows", **kwargs)
