"""GPU: bf16 weight gradients around the number of rows up to which every expert is one chunk (252 + 96 log2(E)), with
the rows spread, all at one expert, and one expert of exactly so many.

Tolerances as in test_gpu_train_ops.py: 2^-24 for each addition on the longest chain to a value, times the sum of the
magnitudes of its terms.
"""

import numpy as np
import pytest
import torch

import _train_oracle as to
from _gpu_helpers import say
from test_gpu_train_ops import U32, _bf16, _bounds, _dev, _ops, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,few", [(1, 252), (3, 348), (8, 540), (64, 828)])
@pytest.mark.parametrize("more", [0, 1])
@pytest.mark.parametrize("load", ["spread", "one", "all but one row"])
def test_weight_grad_around_one_chunk(E, few, more, load):
    g = np.random.default_rng(E + more)
    P, d_in, d_out = few + more, 34, 66
    if load == "spread" or E == 1:
        rows = list(np.diff(np.sort(np.concatenate([[0, P], g.integers(0, P + 1, E - 1)]))))
    else:
        rows = [0] * E
        rows[E // 2], rows[0] = (P, 0) if load == "one" else (P - 1, 1)
    offsets = _bounds(rows)
    dy, a = _bf16(g.standard_normal((P, 2, d_out, 4))), _bf16(g.standard_normal((P, 2, d_in, 4)))
    gather = g.permutation(P).astype(np.int32)
    say(f"weight grad bf16 around one chunk E={E} P={P} {load}")
    n = max(rows)
    for idx in (None, gather):
        dW, db = _ops().grouped_weight_grad_pauli(_dev(dy, torch.bfloat16), _dev(a, torch.bfloat16), _dev(offsets), E,
                                                  gather=None if idx is None else _dev(idx))
        want, want_b, mW, mb = to.weight_grad(dy, a if idx is None else a[idx], offsets)
        _within(dW, want, (4 * n + 16) * U32 * mW, "dW")
        _within(db, want_b, (n + 16) * U32 * mb, "db")
