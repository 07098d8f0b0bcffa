"""What the C entries of dispatch and combine over a caller's rows refuse, on the CPU: their checks come before any launch."""

import os

import pytest

from yggdrasil_amd import _native as N

pytestmark = pytest.mark.skipif(not os.path.exists(N.LIB_PATH), reason="library not built")
P = 4096  # a pointer that no check may follow

DISPATCH = [P, 0, 8, 2, 4, 16, P, P, 0, None]  # x, dtype, N, k, d, rows, slots, out, mask order, stream
COMBINE = [P, 0, 0, 8, 2, 4, 16, P, P, P, None, P, 0, None]


def _refused(name, args, at, value, word):
    lib = N.lib()
    args = list(args)
    args[at] = value
    assert getattr(lib, name)(*args) == -1
    assert word in lib.ygg_last_error().decode() and name in lib.ygg_last_error().decode()


@pytest.mark.parametrize("at,value,word", [(0, None, "null"), (6, None, "null"), (7, None, "null"), (1, 2, "dtype"),
                                           (2, -1, "bad sizes"), (3, 0, "bad sizes"), (3, 9, "bad sizes"), (4, 0, "bad sizes"),
                                           (5, -1, "bad sizes")])
def test_dispatch(at, value, word):
    _refused("ygg_dispatch_rows", DISPATCH, at, value, word)


@pytest.mark.parametrize("at,value,word", [(0, None, "null"), (7, None, "null"), (8, None, "null"), (9, None, "null"),
                                           (11, None, "null"), (1, 2, "dtype"), (12, 2, "dtype"), (3, -1, "bad sizes"),
                                           (4, 0, "bad sizes"), (4, 9, "bad sizes"), (5, 0, "bad sizes"), (6, -1, "bad sizes")])
def test_combine(at, value, word):
    _refused("ygg_combine_rows", COMBINE, at, value, word)


FAR = [P + (i << 40) for i in range(7)]
# dout, type, y, N, k, d, P, weights, slots, dy, type, layout, dw, workspace, its bytes, stream
BIG = 1 << 18  # rows of a batch that takes scratch
BACK = [FAR[0], 0, FAR[1], BIG // 2, 2, 4, BIG, FAR[2], FAR[3], FAR[4], 0, 0, FAR[5], FAR[6], 4 * BIG, None]


@pytest.mark.parametrize("at,value,word", [
    (0, None, "null"), (7, None, "null"), (8, None, "null"), (9, None, "null"), (13, None, "workspace"), (14, 4 * BIG - 1, "workspace"), (1, 2, "dtype"),
    (10, 2, "dtype"), (3, -1, "bad sizes"), (4, 9, "bad sizes"), (5, 0, "bad sizes"), (6, -1, "bad sizes"), (11, 2, "layout"),
    (2, None, "needs y_sorted"), (12, None, "needs y_sorted"), (9, FAR[0], "share"), (13, FAR[0] + 64, "share"),
    (13, FAR[1], "share"), (13, FAR[2], "share"), (13, FAR[3], "share"), (13, FAR[4] + 4, "share"), (13, FAR[5], "share")])
def test_combine_backward(at, value, word):
    _refused("ygg_combine_backward_rows", BACK, at, value, word)
    assert N.lib().ygg_combine_backward_rows_workspace_bytes(BIG // 2, 2, BIG) == 4 * BIG
    assert N.lib().ygg_combine_backward_rows_workspace_bytes(8192, 2, 16384) == 0


def test_no_tokens_need_no_gpu():
    lib = N.lib()
    assert lib.ygg_dispatch_rows(None, 0, 0, 2, 4, 0, None, None, 0, None) == 0
    assert lib.ygg_combine_rows(None, 0, 0, 0, 2, 4, 0, None, None, None, None, None, 0, None) == 0
