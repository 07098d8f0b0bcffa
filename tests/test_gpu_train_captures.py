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


@pytest.mark.parametrize("block,dtype", [(False, torch.bfloat16), (True, torch.bfloat16), (True, torch.float32),
                                         (False, torch.float32)])
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


def test_captured_step_of_an_fp32_layer_with_its_update():
    """Every replay trains the weights of the replay before, also where the layouts were fresh at the capture."""
    m = _layer(np.random.default_rng(25), 16, 24, 4, 2, torch.float32, router_grad=True)
    params = list(m.parameters())
    x, grad = (_tokens(np.random.default_rng(i), 1, 40, 16, torch.float32) for i in (26, 27))

    def step():
        out = m.moe_forward(x)
        grads = torch.autograd.grad(out, params, grad)
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.add_(g.sign(), alpha=-0.02)
        return out.detach()

    say("captured training steps of an fp32 layer with updates")
    start = [p.detach().clone() for p in params]

    def restart():
        with torch.no_grad():
            for p, s in zip(params, start):
                p.copy_(s)

    want = [(step().clone(), [p.detach().clone() for p in params]) for _ in range(4)]
    assert not torch.equal(want[0][0], want[1][0])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    restart()
    with torch.no_grad():
        m.moe_forward(x)  # the layouts of these weights are there now
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    restart()
    for o, ps in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and all(torch.equal(p.detach(), q) for p, q in zip(params, ps))


@pytest.mark.parametrize("graph_of", ["training", "inference"])
def test_weights_first_laid_out_in_a_capture(graph_of):
    """An eager call before any replay lays the weights out for itself."""
    m, other = (_layer(np.random.default_rng(28), 16, 24, 4, 2, torch.float32) for _ in range(2))
    x = _tokens(np.random.default_rng(29), 1, 20, 16, torch.float32)

    def run(layer):
        with torch.set_grad_enabled(graph_of == "training"):
            return layer.moe_forward(x).detach()

    say(f"fp32 weights first laid out in a capture ({graph_of})")
    run(m)
    with torch.no_grad():
        for p in m.parameters():
            p.mul_(1.25)
    other.load_state_dict(m.state_dict())
    want = run(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(m)
    assert torch.equal(run(m), want)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(run(m), want)


@pytest.mark.parametrize("block,dtype,router", [(False, torch.float32, "energy"), (True, torch.bfloat16, "energy"),
                                                (False, torch.float32, "clifford_head")])
def test_an_inference_graph_follows_the_weights(block, dtype, router):
    """New weights, once an eager call has laid them out, are those of the graph's next replays."""
    m = _layer(np.random.default_rng(30), 16, 24, 4, 2, dtype, block=block, router=router)
    x = _tokens(np.random.default_rng(31), 1, 20, 16, dtype)
    say(f"an inference graph beside new weights, block={block} {dtype} {router}")
    with torch.no_grad():
        _run(m, x, block)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _run(m, x, block)
        moe = m.moe if block else m
        for _ in range(3):
            moe.w_up.mul_(1.5)
            moe.b_down.add_(0.25)
            want = _run(m, x, block).clone()
            other = [torch.full((n,), 255, device="cuda", dtype=torch.uint8) for n in (4096, 65536, 1 << 20) for _ in range(8)]
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            fresh = _layer(np.random.default_rng(30), 16, 24, 4, 2, dtype, block=block, router=router)
            fresh.load_state_dict(m.state_dict())
            assert torch.equal(_run(fresh, x, block), want)
            del other


@pytest.mark.parametrize("block,dtype", [(False, torch.float32), (False, torch.bfloat16), (True, torch.bfloat16)])
def test_a_graph_writes_no_memory_that_eager_calls_free(block, dtype):
    """After an eager call of more tokens, whose workspace takes the place of the module's, replays leave every other
    tensor as it is."""
    m = _layer(np.random.default_rng(32), 16, 24, 4, 2, dtype, block=block)
    x, more = (_tokens(np.random.default_rng(33 + i), 1, n, 16, dtype) for i, n in enumerate((20, 2000)))
    say(f"a graph beside an eager call of more tokens, block={block} {dtype}")
    with torch.no_grad():
        want = _run(m, x, block).clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _run(m, x, block)
        _run(m, more, block)
        others = [torch.full((n,), 7, device="cuda", dtype=torch.uint8)
                  for n in (512, 4096, 20000, 65536, 200000, 1 << 20) for _ in range(8)]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and all(bool((t == 7).all()) for t in others)


def test_a_captured_fp32_step_is_refused_beside_an_eager_graph():
    """Refused on the host, before any gradient is added; the forward alone is captured, and without the eager graph
    the whole step."""
    m = _layer(np.random.default_rng(35), 16, 24, 4, 2, torch.float32)
    x, grad = (_tokens(np.random.default_rng(i), 1, 20, 16, torch.float32) for i in (36, 37))
    experts = [m.w_up, m.b_up, m.w_down, m.b_down]
    say("an fp32 step captured beside an eager graph")
    alive = m.moe_forward(x)
    want = [alive.detach().clone(), *(t.clone() for t in torch.autograd.grad(alive, experts, grad, retain_graph=True))]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m.moe_forward(x).detach()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(m.moe_forward(x), experts, grad)
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.moe_forward(x)
        got = [out.detach(), *torch.autograd.grad(out, experts, grad)]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", ["layer", "block", "norm"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_are_not_differentiated_again(which, dtype):
    import yggdrasil_amd as y

    g = np.random.default_rng(38)
    m = (y.CliffordLayerNorm(16, device="cuda", grad=True) if which == "norm" else
         _layer(g, 16, 24, 4, 2, dtype, block=which == "block", router_grad=True))
    x = _tokens(g, 1, 20, 16, dtype).requires_grad_(True)
    params = list(m.parameters())
    say(f"gradients with create_graph, {which} {dtype}")
    out = m.moe_forward(x) if which == "layer" else m(x)
    dout = torch.ones_like(out)
    want = torch.autograd.grad(out, [x, *params], dout, retain_graph=True)
    got = torch.autograd.grad(out, [x, *params], dout, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for t in got:
        with pytest.raises(RuntimeError, match="differentiated again"):
            (t.sum() + x.float().sum()).backward(retain_graph=True)
