"""Which kernel a product of int8 rows takes: few outputs, with the channels in groups of 16 as the kernel for them has them."""

import os

import pytest

from yggdrasil_amd import _native as N

pytestmark = pytest.mark.skipif(not os.path.exists(N.LIB_PATH), reason="library not built")


@pytest.mark.parametrize("P,d_out,small", [
    (1, 1, 1), (12500, 1, 1), (12501, 1, 0), (12500, 16, 1), (12501, 16, 0), (12500, 17, 0), (6250, 17, 1), (6251, 32, 0),
    (195, 1024, 1), (196, 1024, 0), (200000, 1, 0), (1, 524288, 0), (2 ** 31 - 1, 524288, 0), (2 ** 31 - 1, 1, 0)])
def test_rule(P, d_out, small):
    assert N.lib().ygg_int8_product_small(P, d_out) == small
