"""GPU: bf16 training steps with frozen experts: the weight gradients that nobody asks for are not computed, all others
are the same bit for bit."""

import numpy as np
import pytest
import torch

from _gpu_helpers import say
from test_gpu_train_layer import _layer, _tokens

pytestmark = pytest.mark.gpu

PAIRS = {"up": ("w_up", "b_up"), "down": ("w_down", "b_down")}


@pytest.mark.parametrize("frozen", [("up",), ("down",), ("up", "down")])
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("N", [40, 700])
def test_gradients_beside_frozen_experts(N, block, frozen):
    dtype = torch.bfloat16
    m = _layer(np.random.default_rng(40), 16, 24, 4, 2, dtype, block=block, router_grad=True)
    moe = m.moe if block else m
    x, dout = (_tokens(np.random.default_rng(41 + i), 1, N, 16, dtype) for i in range(2))

    def grads():
        xi = x.detach().requires_grad_(True)
        for p in m.parameters():
            p.grad = None
        (m(xi) if block else m.moe_forward(xi)).backward(dout)
        return dict(x=xi.grad, **{n: p.grad for n, p in m.named_parameters()})

    say(f"frozen experts {frozen}, N={N} block={block}")
    want = grads()
    off = [n for pair in frozen for n in PAIRS[pair]]
    for n in off:
        getattr(moe, n).requires_grad_(False)
    got = grads()
    for n, t in want.items():
        if n.split(".")[-1] in off:
            assert got[n] is None
        else:
            assert torch.equal(got[n], t), n


@pytest.mark.parametrize("N", [0, 30, 600])
def test_operator_without_weight_gradients(N):
    from yggdrasil_amd import ops

    g = torch.Generator(device="cuda").manual_seed(43)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    d, F, E = 18, 20, 4
    x, dout = rn(N, d, 8).bfloat16(), rn(N, d, 8).bfloat16()
    wu, wd = rn(E, F, d, 8) / 12, rn(E, d, F, 8) / 12
    say(f"bf16 backward without weight gradients, N={N}")
    _, routing, saved = ops.moe_forward_train_bf16(x, 2, ops.prepare_weights(wu, "pauli"), ops.prepare_weights(wd, "pauli"),
                                                   logits=rn(N, E))
    adj = ops.prepare_adjoint_weights(wu, "pauli"), ops.prepare_adjoint_weights(wd, "pauli")
    want = ops.moe_backward_bf16(dout, saved, routing, *adj, routing_grad=True)
    for up in (False, True):
        for down in (False, True):
            got = ops.moe_backward_bf16(dout, saved, routing, *adj, routing_grad=True, up_grad=up, down_grad=down)
            for i, on in enumerate((True, up, up, down, down, True)):
                assert torch.equal(got[i], want[i]) if on else got[i] is None
