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


@pytest.mark.parametrize("block", [False, True])
def test_eager_calls_between_replays_use_the_present_weights(capturing, block):
    layer = _layer()
    assert _fresh(layer) and layer._get_prepared() is layer._get_prepared()
    capturing[0] = True
    layers._step_layouts(layer, block)
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
    monkeypatch.setattr(layers, "_train_backward", lambda layer, flat, logits, kept, dout, residual, block=False:
                        (2 * dout, *(torch.zeros_like(getattr(layer, n)) for n in ("w_up", "b_up", "w_down", "b_down")),
                         None, None, None))
    monkeypatch.setattr(layers.ops, "stream_handle", lambda dev: 0)
    return lambda layer, x, logits=None: layers._MoEFunction.apply(
        x, None, layer.w_up, layer.b_up, layer.w_down, layer.b_down, layer.router_weight, layer.router_bias, layer, None,
        logits)


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
