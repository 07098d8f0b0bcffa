"""GPU: captured training steps beside eager calls of the same module, and parameters changed before a backward.

A captured step with its update changes the weights at every replay.  Eager calls between the replays -- with a
graph and without -- have to see them, which a module of its own with the same state shows.  Both run the same kernels
on the same values, so outputs and gradients are equal bit for bit.
"""

import numpy as np
import pytest
import torch

from _gpu_helpers import say
from test_gpu_train_layer import _layer, _tokens

pytestmark = pytest.mark.gpu


def _run(m, x, block):
    return m(x) if block else m.moe_forward(x)


def _eager(m, x, grad, block):
    """The output without a graph, and the output and gradients with one."""
    with torch.no_grad():
        plain = _run(m, x, block).clone()
    xi = x.detach().requires_grad_(True)
    out = _run(m, xi, block)
    grads = torch.autograd.grad(out, [xi, *m.parameters()], grad, allow_unused=True)
    return [plain, out.detach(), *(g for g in grads if g is not None)]


@pytest.mark.parametrize("block,dtype", [(False, torch.bfloat16), (True, torch.bfloat16), (True, torch.float32)])
def test_eager_calls_between_replays_with_updates(block, dtype):
    make = lambda: _layer(np.random.default_rng(20), 16, 24, 4, 2, dtype, block=block, router_grad=True)
    m = make()
    params = list(m.parameters())
    x, grad = (_tokens(np.random.default_rng(i), 1, 40, 16, dtype) for i in (21, 22))

    def step():
        grads = torch.autograd.grad(_run(m, x, block), params, grad)
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.add_(g.sign(), alpha=-0.02)  # (of bounded length: the values stay finite)

    say(f"eager calls between replays with updates, block={block} {dtype}")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = _eager(m, x, grad, block)
        other = make()
        other.load_state_dict(m.state_dict())
        want = _eager(other, x, grad, block)
        assert len(got) == len(want)
        same = [torch.equal(a, b) for a, b in zip(got, want)]
        assert all(same), same
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_parameters_changed_between_forward_and_backward():
    """An fp32 layer's backward lays out and routes anew: it refuses parameters that its forward did not see."""
    m = _layer(np.random.default_rng(23), 16, 24, 4, 2, torch.float32, router_grad=True)
    x = _tokens(np.random.default_rng(24), 1, 30, 16, torch.float32)
    say("fp32 layer, parameters changed before the backward")
    for p in (m.router_weight, m.w_down):
        out = m.moe_forward(x)
        with torch.no_grad():
            p.mul_(1.5)
        with pytest.raises(RuntimeError, match="modified in place"):
            out.sum().backward()
    m.moe_forward(x).sum().backward()
