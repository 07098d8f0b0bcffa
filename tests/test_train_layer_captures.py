"""Which parameters a layer's calls and its backward use, around a captured training step and otherwise, on the CPU:
the layouts are copies of the weights here, a capture is one that says so, and a replay changes values without the
version counters, as the replays of a graph do."""

import copy

import pytest
import torch

from yggdrasil_amd import layers
from yggdrasil_amd.ops import PreparedWeights


@pytest.fixture
def capturing(monkeypatch):
    now = [False]

    def lay_out(w, fmt="pauli_f32"):
        return PreparedWeights(w.detach().clone(), None, fmt, *w.shape[:3])

    monkeypatch.setattr(layers.ops, "prepare_weights", lay_out)
    monkeypatch.setattr(layers.ops, "prepare_adjoint_weights", lay_out)
    monkeypatch.setattr(layers.ops, "prepare_bias", lambda b: b.detach().clone())
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0])
    return now


def _layer(dtype=torch.bfloat16):
    return layers.CliffordMoELayer(layers.MoEHLMConfig(d_model=4, d_ff=6, n_experts=3, dtype=dtype,
                                                       bf16_grad=dtype == torch.bfloat16))


def _replay(layer):
    v = layer.w_up._version, layer.b_up._version
    layer.w_up.data.add_(1.0)
    layer.b_up.data.add_(1.0)
    assert (layer.w_up._version, layer.b_up._version) == v


def _fresh(layer):
    p = layer._get_prepared()
    return (torch.equal(p["w_up"].data, layer.w_up) and torch.equal(p["b_up"], layer.b_up) and
            torch.equal(layer._get_adjoint()["w_up"].data, layer.w_up))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_eager_calls_between_replays_use_the_present_weights(capturing, dtype):
    layer = _layer(dtype)
    assert _fresh(layer) and layer._get_prepared() is layer._get_prepared()
    capturing[0] = True
    layers._step_layouts(layer)
    capturing[0] = False
    for _ in range(3):
        assert _fresh(layer)
        _replay(layer)
    assert _fresh(layer)
    other = copy.deepcopy(layer)  # parameters of its own, which no graph updates
    assert _fresh(other) and other._get_prepared() is other._get_prepared()


def _autograd(monkeypatch):
    """The layer's node around a forward and a backward that only hand x and dout on."""
    none = torch.zeros(0)
    monkeypatch.setattr(layers, "_train_forward", lambda layer, flat, res, logits, prep, workspace=None:
                        (2 * flat, (none, none, none, none)))
    monkeypatch.setattr(layers, "_train_backward", lambda layer, prep, flat, logits, kept, dout, residual, experts=None:
                        (2 * dout, *(torch.zeros_like(getattr(layer, n)) for n in ("w_up", "b_up", "w_down", "b_down")),
                         None, None, None))
    monkeypatch.setattr(layers.ops, "stream_handle", lambda dev: 0)
    return lambda layer, x, logits=None: layers._MoEFunction.apply(
        x, None, layer.w_up, layer.b_up, layer.w_down, layer.b_down, layer.router_weight, layer.router_bias, layer, None,
        None, logits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters_changed_between_forward_and_backward(capturing, monkeypatch, dtype):
    run = _autograd(monkeypatch)
    layer, x = _layer(dtype), torch.ones(5, 4, 8)
    for name in ("w_up", "b_up", "w_down", "b_down", "router_weight", "router_bias"):
        out = run(layer, x)
        with torch.no_grad():
            getattr(layer, name).add_(1.0)
        with pytest.raises(RuntimeError, match="modified in place"):
            out.sum().backward()
    out = run(layer, x, torch.zeros(5, 3))  # with the caller's logits the router's parameters are not read
    with torch.no_grad():
        layer.router_weight.add_(1.0)
    out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_of_a_capture_are_found_by_nothing_else(capturing, dtype):
    layer = _layer(dtype)
    before = layer._get_prepared(), layer._get_adjoint()
    with torch.no_grad():
        layer.w_up.add_(1.0)
    capturing[0] = True
    inference = layer._get_prepared()  # stale: laid out in the capture
    capturing[0] = False
    after = layer._get_prepared()
    assert after is not inference and after is not before[0] and after is layer._get_prepared()
    capturing[0] = True
    step = layers._step_layouts(layer)
    capturing[0] = False
    assert step is not after and layer._get_prepared() is not step


def test_layouts_that_a_capture_reads_are_written_over(capturing):
    """An inference graph reads the layouts that it found at every replay: new ones take their place in memory."""
    layer = _layer(torch.float32)
    layer._get_prepared()
    capturing[0] = True
    read = layer._get_prepared()
    assert layer._get_prepared() is read
    capturing[0] = False
    for _ in range(3):
        with torch.no_grad():
            layer.w_up.add_(1.0)
            layer.b_down.sub_(2.0)
        new = layer._get_prepared()
        assert _fresh(layer) and new is layer._get_prepared()
        for n in ("w_up", "w_down"):
            assert new[n].data.data_ptr() == read[n].data.data_ptr() and torch.equal(read[n].data, getattr(layer, n))
        assert new["b_down"].data_ptr() == read["b_down"].data_ptr() and torch.equal(read["b_down"], layer.b_down)
    capturing[0] = True  # and without a capture they are not
    layer = _layer(torch.float32)
    capturing[0] = False
    old = layer._get_prepared()
    with torch.no_grad():
        layer.w_up.add_(1.0)
    assert layer._get_prepared()["w_up"].data.data_ptr() != old["w_up"].data.data_ptr()


def test_a_captured_backward_reads_layouts_of_its_own(capturing, monkeypatch):
    """The forward's layouts reach an fp32 backward, and the adjoint ones are the graph's."""
    layer, seen = _layer(torch.float32), []
    layer._get_adjoint()
    monkeypatch.setattr(layers, "_train_forward", lambda layer, flat, res, logits, prep, workspace=None:
                        (2 * flat, (torch.zeros(0),) * 4))
    monkeypatch.setattr(layers.ops, "moe_backward", lambda x, k, up, up_adj, down, down_adj, dout, *a, **kw:
                        seen.append((up, up_adj)) or (dout, *(torch.zeros_like(p) for p in (
                            layer.w_up, layer.b_up, layer.w_down, layer.b_down)), None))
    monkeypatch.setattr(layers.ops, "stream_handle", lambda dev: 7)
    for now in (True, False):
        capturing[0] = now
        prep = layers._step_layouts(layer)
        out = layers._MoEFunction.apply(torch.ones(5, 4, 8), None, layer.w_up, layer.b_up, layer.w_down, layer.b_down,
                                        layer.router_weight, layer.router_bias, layer, prep, None,
                                        None)
        out.sum().backward()
        assert seen[-1][0] is prep["w_up"] and (seen[-1][1] is layer._adjoint["w_up"]) == (not now)
    del out


def test_a_graph_has_a_workspace_of_its_own(capturing):
    """What a graph writes is no tensor that a later eager call may free."""
    layer, dev = _layer(torch.float32), torch.device("cpu")
    take = lambda need: layers._call_workspace(layer, need, dev, capturing[0])
    ws = take(100)
    assert ws.numel() == 100 and take(50) is ws
    capturing[0] = True
    own = take(50), take(500)
    assert own[0] is not ws and own[1].numel() == 500 and layer._workspace is ws
    capturing[0] = False
    assert take(100) is ws and take(101) is not ws


def test_a_captured_fp32_backward_is_refused_while_an_eager_graph_lives(capturing, monkeypatch):
    """Its forward may be captured beside one: it carries a graph that nobody asked for."""
    run, x = _autograd(monkeypatch), torch.ones(5, 4, 8)
    layer, other = _layer(torch.float32), _layer(torch.float32)
    alive = run(layer, x)
    alive.sum().backward()
    capturing[0] = True
    run(other, x).sum().backward()
    out = run(layer, x)
    with pytest.raises(RuntimeError, match="still alive"):
        out.sum().backward()
    del alive
    run(layer, x).sum().backward()
    # parameters without gradients have none to add
    capturing[0] = False
    for p in layer.parameters():
        p.requires_grad_(False)
    alive = run(layer, x.requires_grad_(True))
    capturing[0] = True
    run(layer, x).sum().backward()
    del alive


def _first_order_only(out, inputs):
    """The gradients of `out` for an incoming one that is a constant, and for one that is not: each equal to the plain
    gradients, and each refusing to be differentiated."""
    want = torch.autograd.grad(out, inputs, torch.ones_like(out), retain_graph=True)
    assert not any(t.requires_grad for t in want)
    for dout in (torch.ones_like(out), torch.ones_like(out, requires_grad=True)):
        got = torch.autograd.grad(out, inputs, dout, retain_graph=True, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for t in got:
            with pytest.raises(RuntimeError, match="differentiated again"):
                (t.sum() + inputs[0].sum()).backward(retain_graph=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_are_not_differentiated_again(capturing, monkeypatch, dtype):
    run = _autograd(monkeypatch)
    layer, x = _layer(dtype), torch.ones(5, 4, 8, requires_grad=True)
    _first_order_only(run(layer, x), [x, layer.w_up, layer.b_down])
    monkeypatch.setattr(layers.ops, "clifford_layer_norm", lambda x, gamma, beta, eps, out_dtype=None: 2 * x)
    monkeypatch.setattr(layers.ops, "clifford_layer_norm_backward", lambda dy, x, gamma, eps, residual_grad=None:
                        (2 * dy, torch.zeros_like(gamma), torch.zeros_like(gamma)))
    norm = layers.CliffordLayerNorm(4, grad=True)
    _first_order_only(norm(x), [x, norm.gamma, norm.beta])
    # a residual's gradient is the incoming one, with its graph
    res = torch.ones(5, 4, 8, requires_grad=True)
    out = layers._MoEFunction.apply(x, res, layer.w_up, layer.b_up, layer.w_down, layer.b_down, layer.router_weight,
                                    layer.router_bias, layer, None, None, None)
    a = torch.tensor(3.0, requires_grad=True)
    dres, = torch.autograd.grad(out, [res], a * torch.ones_like(out), create_graph=True)
    assert torch.autograd.grad(dres.sum(), [a])[0] == dres.numel()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bf16_training_step_takes_no_inference_workspace(capturing, monkeypatch, dtype):
    seen = []
    monkeypatch.setattr(layers.ops, "moe_workspace_bytes", lambda *a: 1000)
    monkeypatch.setattr(layers, "_train_forward", lambda layer, flat, res, logits, prep, workspace=None:
                        seen.append(workspace) or (2 * flat, (torch.zeros(0),) * 4))
    monkeypatch.setattr(layers.ops, "stream_handle", lambda dev: 0)
    layer = _layer(dtype)
    layer.moe_forward(torch.ones(1, 5, 4, 8, dtype=dtype))
    kept = layer.__dict__["_workspace"]
    assert (kept is None and seen == [None]) if dtype == torch.bfloat16 else seen[0] is kept and kept.numel() == 1000


@pytest.mark.parametrize("frozen", [("w_up", "b_up"), ("w_down", "b_down"), ("w_up", "b_up", "w_down", "b_down"), ("w_up",)])
def test_frozen_experts_have_no_weight_products(capturing, monkeypatch, frozen):
    seen = []
    monkeypatch.setattr(layers, "_train_forward", lambda layer, flat, res, logits, prep, workspace=None:
                        (2 * flat, (torch.zeros(0),) * 4))
    monkeypatch.setattr(layers.ops, "stream_handle", lambda dev: 0)

    def backward(dout, rows, routing, up, down, act, residual, routing_grad, up_grad, down_grad):
        seen.append((up_grad, down_grad))
        z = lambda n, want: torch.zeros_like(getattr(layer, n)) if want else None
        return dout, z("w_up", up_grad), z("b_up", up_grad), z("w_down", down_grad), z("b_down", down_grad), None

    monkeypatch.setattr(layers.ops, "moe_backward_bf16", backward)
    layer = _layer()
    for n in frozen:
        getattr(layer, n).requires_grad_(False)
    x = torch.ones(1, 5, 4, 8, dtype=torch.bfloat16, requires_grad=True)
    layer.moe_forward(x).sum().backward()
    assert seen == [(not {"w_up", "b_up"} <= set(frozen), not {"w_down", "b_down"} <= set(frozen))] and x.grad is not None
    assert [n for n in ("w_up", "b_up", "w_down", "b_down") if getattr(layer, n).grad is None] == sorted(frozen, key=(
        "w_up", "b_up", "w_down", "b_down").index)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_router_head_that_a_capture_read(capturing, dtype):
    """An fp32 head is the parameter itself, which no new layout writes; one of another type is a copy, which is."""
    layer = layers.CliffordMoELayer(layers.MoEHLMConfig(d_model=4, d_ff=6, n_experts=3, router="clifford_head"))
    layer.head_weight = torch.nn.Parameter(layer.head_weight.detach().to(dtype))
    layer._get_prepared()
    capturing[0] = True
    read = layer._get_prepared()["head"]
    capturing[0] = False
    first = layer.head_weight
    kept = first.detach().clone()
    with torch.no_grad():
        other = torch.nn.Parameter(2 * first)
        other.add_(1.0)
    layer.head_weight = other  # replaced, not changed in place
    new = layer._get_prepared()["head"]
    assert torch.equal(first, kept) and torch.equal(new, other.float())
    assert (new is read) == (dtype == torch.float64)


def test_layouts_of_a_single_product_in_captures(capturing):
    """CliffordLinear: a capture's own layouts where its weights had changed, the module's written over where not."""
    lin = layers.CliffordLinear(4, 6)
    lin._prepared()
    capturing[0] = True
    read = lin._prepared()
    capturing[0] = False
    with torch.no_grad():
        lin.weight.add_(1.0)
    new = lin._prepared()
    assert new["w"].data.data_ptr() == read["w"].data.data_ptr() and torch.equal(read["w"].data[0], lin.weight)
    with torch.no_grad():
        lin.weight.add_(1.0)
    capturing[0] = True
    own = lin._prepared()
    capturing[0] = False
    assert own["w"] is not lin._prepared()["w"] and torch.equal(lin._prepared()["w"].data[0], lin.weight)


def test_layouts_of_inference_mode_that_a_capture_reads(capturing):
    """Made and captured in inference mode, written over outside of it."""
    layer = _layer(torch.float32)
    with torch.inference_mode():
        layer._get_prepared()
        capturing[0] = True
        read = layer._get_prepared()
        capturing[0] = False
    with torch.no_grad():
        layer.w_up.add_(1.0)
    new = layer._get_prepared()
    assert new["w_up"].data.data_ptr() == read["w_up"].data.data_ptr() and torch.equal(new["w_up"].data, layer.w_up)
