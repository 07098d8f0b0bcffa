"""Which weight layouts a layer's calls use around a captured training step, on the CPU: the layouts are copies of the
weights here, a capture is one that says so, and a replay changes values without the version counters, as the replays
of a graph do."""

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
