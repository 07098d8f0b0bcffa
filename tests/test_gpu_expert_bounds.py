"""Experts' ranges as a caller may have them: starts and counts far outside the rows, of 32 and 64 bits, brought into [0, P]
by their values, not by their low bits."""

import pytest
import torch

from _gpu_helpers import say

pytestmark = pytest.mark.gpu

I32, I64 = 2 ** 31, 2 ** 63


def _expected(offsets, counts, P):
    clip = [min(max(v, 0), P) for v in [*offsets, offsets[-1] + counts[-1]]]  # (whole numbers of any size)
    return [max(clip[:n + 1]) for n in range(len(clip))]


CASES32 = [([0, 20, 35], [20, 15, 15]), ([0, 30], [30, I32 - 1]), ([0, I32 - 1], [5, I32 - 1]), ([-I32, 7], [3, -I32]),
           ([-5, -I32], [1, -I32]), ([10], [I32 - 1])]
CASES64 = CASES32 + [([0, 2 ** 32 + 5], [5, 3]), ([0, -2 ** 32 + 7], [5, 3]), ([0, 40], [40, 2 ** 32]), ([2 ** 40, 3], [1, 1]),
                     ([0, I64 - 1], [5, I64 - 1]), ([0, -I64], [5, -I64]), ([4, 9], [5, I64 - 1]), ([0, 2 ** 33 + 1], [1, -2 ** 33])]


@pytest.mark.parametrize("dt,offsets,counts", [(torch.int32, *c) for c in CASES32] + [(torch.int64, *c) for c in CASES64])
def test_bounds(dt, offsets, counts):
    from yggdrasil_amd import ops

    P, E = 50, len(offsets)
    say(f"expert bounds {dt} {offsets} {counts}")
    o, c = torch.tensor(offsets, device="cuda", dtype=dt), torch.tensor(counts, device="cuda", dtype=dt)
    bounds = torch.full((E + 2,), 77, device="cuda", dtype=torch.int32)
    ops.check(ops.lib().ygg_expert_bounds(o.data_ptr(), c.data_ptr(), o.element_size(), E, P, bounds.data_ptr(),
                                          ops.stream_handle()))
    assert bounds.tolist() == [*_expected(offsets, counts, P), 77]


@pytest.mark.parametrize("fmt", ["int8_rows", "pauli"])
def test_experts_of_far_ranges(fmt):
    """A last range that starts 2^32 behind the rows is empty, and one that ends there goes to the last row."""
    from yggdrasil_amd import ops

    torch.manual_seed(8)
    E, d, F, P = 3, 16, 24, 50
    wu = ops.prepare_weights(torch.randn(E, F, d, 8, device="cuda") / (8 * d) ** 0.5, fmt)
    wd = ops.prepare_weights(torch.randn(E, d, F, 8, device="cuda") / (8 * F) ** 0.5, fmt)
    x = torch.randn(P, d, 8, device="cuda").bfloat16()

    def run(offsets, counts, dt=torch.int64):
        return ops.grouped_experts(x, torch.tensor(offsets, device="cuda"), torch.tensor(counts, device="cuda").to(dt), wu, wd)

    say(f"experts of far ranges {fmt}")
    want = run([0, 20, 50], [20, 30, 0]), run([0, 20, 30], [20, 10, 20])
    for dt in (torch.int64, torch.int32):  # one type, and two
        assert torch.equal(run([0, 20, 2 ** 32], [20, 30, 7], dt), want[0])
        assert torch.equal(run([0, 20, 2 ** 32 + 30], [20, 10, 0], dt)[:20], want[1][:20])
    assert torch.equal(run([0, 20, 30], [20, 10, 2 ** 32 - 30]), want[1])
