"""What the training operators refuse, on the CPU: the C entries' checks come before any launch, and the Python
entries take no CPU tensors."""

import os

import pytest
import torch

from yggdrasil_amd import _native as N
from yggdrasil_amd import ops

pytestmark = pytest.mark.skipif(not os.path.exists(N.LIB_PATH), reason="library not built")
P = 4096  # a pointer that no check may follow


def _refused(name, args, word):
    lib = N.lib()
    assert getattr(lib, name)(*args) == -1
    assert word in lib.ygg_last_error().decode(), lib.ygg_last_error()


@pytest.mark.parametrize("args,word", [
    ((P, 2, P, 0, 4, 4, P, 1e-6, None, P, P, P, P, 1 << 20, None), "dy dtype"),
    ((P, 0, P, 5, 4, 4, P, 1e-6, None, P, P, P, P, 1 << 20, None), "x dtype"),
    ((P, 0, P, 0, -1, 4, P, 1e-6, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, P, 0, 4, 0, P, 1e-6, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, P, 0, 4, 4097, P, 1e-6, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, P, 0, 0x7fff0001, 4, P, 1e-6, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, P, 0, 4, 4, P, -1.0, None, P, P, P, P, 1 << 20, None), "eps"),
    ((P, 0, P, 0, 4, 4, None, 1e-6, None, P, P, P, P, 1 << 20, None), "null"),
    ((None, 0, P, 0, 4, 4, P, 1e-6, None, P, P, P, P, 1 << 20, None), "null"),
    ((P, 0, P, 0, 4, 4, P, 1e-6, None, P, P, P, P, 1 << 20, None), "dx is dy"),
    ((P, 0, P, 0, 4000, 4, P, 1e-6, None, P, P, P, P, 8, None), "workspace"),
    ((P, 0, P, 0, 4000, 4, P, 1e-6, None, P, P, P, None, 1 << 20, None), "workspace"),
])
def test_norm_backward(args, word):
    _refused("ygg_clifford_layer_norm_backward", args, word)


@pytest.mark.parametrize("args,word", [
    ((P, P, 8, None, P, 8, 2, 3, 4, P, P, P, 1 << 30, None), "bad sizes"),
    ((P, P, 8, None, P, 8, 2, 4, 5, P, P, P, 1 << 30, None), "bad sizes"),
    ((P, P, 8, None, P, 8, 65, 4, 4, P, P, P, 1 << 30, None), "bad sizes"),
    ((P, P, 8, None, P, -1, 2, 4, 4, P, P, P, 1 << 30, None), "bad sizes"),
    ((P, P, 7, None, P, 8, 2, 4, 4, P, P, P, 1 << 30, None), "7 rows"),
    ((P, P, 8, None, None, 8, 2, 4, 4, P, P, P, 1 << 30, None), "null"),
    ((P, P, 8, None, P, 8, 2, 4, 4, None, P, P, 1 << 30, None), "null"),
    ((None, P, 8, None, P, 8, 2, 4, 4, P, P, P, 1 << 30, None), "null"),
])
def test_weight_grad(args, word):
    _refused("ygg_grouped_weight_grad_pauli_bf16", args, word)


@pytest.mark.parametrize("args,word", [
    ((P, 8, P, P, 2, 4, 4, 1, None, P, 0, 1, None), "null"),        # an activation without its input
    ((P, 8, P, P, 2, 3, 4, 0, None, P, 0, 1, None), "bad sizes"),   # odd contraction
    ((P, 8, P, P, 2, 4, 3, 0, None, P, 0, 1, None), "bad sizes"),   # odd Pauli rows out
    ((P, 8, P, P, 0, 4, 4, 0, None, P, 0, 1, None), "bad sizes"),
    ((P, 8, P, P, 65, 4, 4, 0, None, P, 0, 1, None), "bad sizes"),
    ((P, 8, P, P, 2, 4, 4, 4, P, P, 0, 1, None), "activation"),
    ((P, 8, P, P, 2, 4, 4, 0, None, P, 2, 1, None), "layout"),
    ((P, 8, P, P, 2, 4, 4, 0, None, P, 0, 0, None), "dtype"),
    ((P, 8, P, P, 2, 4, 4, 0, None, P, 1, 3, None), "dtype"),
    ((P, 8, P, P, 2, 1 << 15, 1 << 14, 0, None, P, 0, 1, None), "2 GiB"),
])
def test_input_grad(args, word):
    _refused("ygg_pauli_grouped_input_grad", args, word)


def test_adjoint_weights():
    _refused("ygg_prepare_adjoint_weights_bf16", (P, 2, 3, 4, P, None), "even")
    _refused("ygg_prepare_adjoint_weights_bf16", (None, 2, 4, 4, P, None), "null")


@pytest.mark.parametrize("args,word", [
    ((P, P, P, 4, 65, 2, P, None), "bad sizes"),
    ((P, P, P, 4, 4, 9, P, None), "bad sizes"),
    ((P, P, P, 4, 2, 3, P, None), "bad sizes"),
    ((P, P, P, -1, 4, 2, P, None), "bad sizes"),
    ((P, None, P, 4, 4, 2, P, None), "null"),
])
def test_route_backward(args, word):
    _refused("ygg_route_backward", args, word)


@pytest.mark.parametrize("args,word", [
    ((P, 3, 4, 4, P, 4, 2, P, P, P, None, P, P, P, P, 1 << 20, None), "dtype"),
    ((P, 0, 4, 0, P, 4, 2, P, P, P, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, 4, 4, P, 65, 2, P, P, P, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, 4, 4, P, 4, 5, P, P, P, None, P, P, P, P, 1 << 20, None), "bad sizes"),
    ((P, 0, 4, 4, None, 4, 2, P, P, P, None, P, P, P, P, 1 << 20, None), "null"),
    ((P, 0, 4, 4, P, 4, 2, P, P, P, None, P, None, P, P, 1 << 20, None), "null"),
    ((P, 0, 4000, 4, P, 4, 2, P, P, P, None, P, P, P, None, 0, None), "workspace"),
])
def test_route_energy_backward(args, word):
    _refused("ygg_route_energy_backward", args, word)


_FWD = [P, 4, 8, 8, 4, 2, 1, P, None, None, P, None, P, None, None, P, P, P, P, P, P, 1 << 30, P, 1 << 30, None]


@pytest.mark.parametrize("at,value,word", [
    (1, -1, "bad sizes"), (2, 7, "bad sizes"), (3, 7, "bad sizes"), (4, 65, "bad sizes"), (5, 5, "bad sizes"),
    (5, 9, "bad sizes"), (6, 4, "activation"), (0, None, "null"), (7, None, "need logits"), (10, None, "null"),
    (18, None, "null"), (20, None, "null"), (21, 64, "keep rows"), (23, 8, "workspace"), (1, 1 << 30, "2^31")])
def test_forward_train_bf16(at, value, word):
    args = list(_FWD)
    args[at] = value
    _refused("ygg_moe_forward_train_bf16", args, word)


_BWD = [4, 8, 8, 4, 2, 1, P, P, 0, P, P, 1 << 30, P, P, P, P, P, P, P, None, P, 1 << 30, None]


@pytest.mark.parametrize("at,value,word", [
    (0, -1, "bad sizes"), (1, 7, "bad sizes"), (2, 0, "bad sizes"), (3, 0, "bad sizes"), (4, 5, "bad sizes"),
    (5, -1, "activation"), (6, None, "null"), (9, None, "null"), (10, None, "null"), (11, 64, "kept rows"),
    (14, None, "null"), (16, None, "null"), (21, 8, "workspace")])
def test_backward_bf16(at, value, word):
    args = list(_BWD)
    args[at] = value
    _refused("ygg_moe_backward_bf16", args, word)


def test_config():
    import yggdrasil_amd as y

    for kw in (dict(bf16_grad=True), dict(dtype=torch.bfloat16, weight_format="int8", bf16_grad=True),
               dict(dtype=torch.bfloat16, router_grad=True), dict(router="clifford_head", router_grad=True)):
        with pytest.raises(ValueError):
            y.MoEHLMConfig(d_model=8, d_ff=16, **kw)
    with pytest.raises(ValueError, match="grad"):
        y.CliffordMoEBlockFFN(y.MoEHLMConfig(d_model=8, d_ff=16, dtype=torch.bfloat16), grad=True)
    assert not y.MoEHLMConfig(d_model=8, d_ff=16).router_grad


def test_no_cpu_path():
    x, w = torch.zeros(3, 4, 8), torch.zeros(3, 2)
    i, h = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2, 4, 4, dtype=torch.bfloat16)
    o = torch.zeros(3, dtype=torch.int32)
    adj = ops.PreparedWeights(torch.zeros(1, dtype=torch.uint8), None, "pauli", 2, 4, 4)
    for f in (lambda: ops.clifford_layer_norm_backward(x, x, torch.zeros(4, 8)),
              lambda: ops.grouped_weight_grad_pauli(h, h, o, 2),
              lambda: ops.pauli_grouped_input_grad(h, adj, o),
              lambda: ops.prepare_adjoint_weights(torch.zeros(2, 4, 4, 8), "pauli"),
              lambda: ops.route_backward(i, w, w, 4),
              lambda: ops.route_energy_backward(x, torch.zeros(4, 4), i, w, w)):
        with pytest.raises(ValueError, match="GPU only"):
            f()


def test_workspace_sizes_of_bad_sizes_are_zero():
    lib = N.lib()
    assert lib.ygg_clifford_layer_norm_backward_workspace_bytes(-1, 4) == 0
    assert lib.ygg_clifford_layer_norm_backward_workspace_bytes(4, 5000) == 0
    assert lib.ygg_grouped_weight_grad_pauli_bf16_workspace_bytes(-1, 2, 4, 4) == 0
    assert lib.ygg_route_energy_backward_workspace_bytes(-1, 4, 4, 2) == 0


def test_launches_go_to_the_tensors_device(monkeypatch):
    """An operator called while another device is current runs with its tensors' device current."""
    seen, current = [], [0]

    class Device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            self.was, current[0] = current[0], self.d

        def __exit__(self, *exc):
            current[0] = self.was

    class Tensor:
        def get_device(self):
            return 3

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)

    @ops._on_its_device
    def op(t, more, key=None):
        seen.append((current[0], more, key))
        return "done"

    assert op(Tensor(), 5, key=6) == "done" and seen == [(3, 5, 6)] and current == [0]
    current[0] = 3
    assert op(Tensor(), 7) == "done" and seen[1] == (3, 7, None)


def test_tensors_of_two_devices_are_refused():
    class Tensor:
        is_cuda = True

        def __init__(self, n):
            self.device = torch.device("cuda", n)

        def get_device(self):
            return self.device.index

        def is_contiguous(self):
            return True

    a, b = Tensor(0), Tensor(1)
    assert ops._one_device(a, None, a) == a.device
    with pytest.raises(ValueError, match="one device"):
        ops._one_device(a, b)


def test_operators_take_their_arguments_by_name():
    w = torch.zeros(1, 4, 4, 8)
    with pytest.raises(ValueError, match="GPU only"):
        ops.prepare_adjoint_weights(w=w)
    with pytest.raises(ValueError, match="GPU only"):
        ops.grouped_weight_grad_pauli(E=1, dy_pauli=w, a_pauli=w, offsets=w)
    with pytest.raises(TypeError):
        ops.prepare_adjoint_weights()


def test_a_workspace_that_does_not_hold_its_bytes_is_not_used():
    dev = torch.device("cpu")
    one = torch.empty(256, dtype=torch.uint8)
    assert ops._workspace(one, 256, dev) is one
    assert ops._workspace(one, 257, dev).numel() == 257
    assert ops._workspace(torch.empty(1, dtype=torch.uint8).expand(256), 256, dev).is_contiguous()
    assert ops._workspace(one[4:], 64, dev).data_ptr() != one[4:].data_ptr()
    assert ops._workspace(one, 64, torch.device("cuda", 0) if torch.cuda.is_available() else torch.device("meta")) is not one


def test_a_capture_is_refused_while_an_eager_graph_lives(monkeypatch):
    """The graphs are found by their autograd nodes, which live as long as any output does."""
    from yggdrasil_amd import layers

    capturing, stream = [False], [0]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(layers.ops, "stream_handle", lambda dev: stream[0])

    class Node(torch.autograd.Function):
        @staticmethod
        def forward(ctx, w, module):
            layers._note_graph(ctx, None, module)
            return 2 * w

        @staticmethod
        def backward(ctx, g):
            return 2 * g, None

    a, b = torch.nn.Linear(2, 2), torch.nn.Linear(2, 2)
    loss = Node.apply(a.weight, a).sum()
    loss.backward()
    capturing[0] = True
    Node.apply(b.weight, b)
    with pytest.raises(RuntimeError, match="still alive"):
        Node.apply(a.weight, a)
    del loss
    Node.apply(a.weight, a)
    capturing[0], stream[0] = False, 7  # a graph of another stream can join a capture
    loss = Node.apply(a.weight, a).sum()
    capturing[0] = True
    Node.apply(a.weight, a)


@pytest.mark.parametrize("N,d,F", [(2000, 18, 300000), (2000, 300000, 18), (1 << 20, 32, 125204)])
def test_a_training_step_has_the_weight_gradients_limits(N, d, F):
    """A chunk of 1024 rows of 300000 multivectors passes 2^32 bytes: refused before the forward, as by the operator."""
    big = 1 << 62
    for at, name, args in ((1, "ygg_moe_forward_train_bf16", _FWD), (0, "ygg_moe_backward_bf16", _BWD)):
        args = list(args)
        args[at:at + 3] = N, d, F
        for i, v in enumerate(args):
            if v == 1 << 30:
                args[i] = big
        _refused(name, args, "2 GiB")
    _refused("ygg_grouped_weight_grad_pauli_bf16", (P, P, 2 * N, None, P, 2 * N, 4, F, d, P, P, P, big, None), "2 GiB")


def test_a_weight_gradient_beyond_a_launch_is_refused():
    big = 1 << 62
    _refused("ygg_grouped_weight_grad_pauli_bf16", (P, P, 1 << 30, None, P, 1 << 30, 4, 4096, 4096, P, P, P, big, None), "launch")


M = 1 << 20  # a megabyte apart


@pytest.mark.parametrize("dx,residual,dgamma,dbeta,word", [
    (1 * M, None, 9 * M, 10 * M, "dx is dy"), (1 * M + 480, None, 9 * M, 10 * M, "dx is dy"),
    (2 * M, None, 9 * M, 10 * M, "dx is x"), (2 * M - 16, None, 9 * M, 10 * M, "dx is x"),
    (2 * M + 1008, 2 * M + 4096, 9 * M, 10 * M, "dx is x"),
    (4 * M, 4 * M + 16, 9 * M, 10 * M, "residual_grad"), (4 * M, None, 3 * M, 10 * M, "gamma"),
    (4 * M, None, 9 * M, 3 * M + 96, "gamma"), (4 * M, 4 * M, 3 * M - 32, 10 * M, "gamma")])
@pytest.mark.parametrize("N", [8, 4000])
def test_norm_gradients_in_the_place_of_their_inputs(N, dx, residual, dgamma, dbeta, word):
    """dy bf16 at 1 MiB, x fp32 at 2, gamma at 3: 8 or 4000 tokens of 4 multivectors."""
    _refused("ygg_clifford_layer_norm_backward", (1 * M, 1, 2 * M, 0, N, 4, 3 * M, 1e-6, residual, dx, dgamma, dbeta,
                                                  32 * M, 1 << 24, None), word)


@pytest.mark.parametrize("dx,add,dw,db,word", [
    (1 * M, None, 9 * M, 10 * M, "dx is x"), (1 * M + 1008, 4 * M, 9 * M, 10 * M, "dx is x"),
    (4 * M, 4 * M - 16, 9 * M, 10 * M, "dx_add"), (4 * M, 4 * M, 2 * M, 10 * M, "router_w"),
    (4 * M, None, 9 * M, 2 * M + 60, "router_w")])
@pytest.mark.parametrize("N", [8, 4000])
def test_router_gradients_in_the_place_of_their_inputs(N, dx, add, dw, db, word):
    _refused("ygg_route_energy_backward", (1 * M, 0, N, 4, 2 * M, 4, 2, 5 * M, 6 * M, 7 * M, add, dx, dw, db, 32 * M, 1 << 24,
                                           None), word)


def test_other_gradients_in_the_place_of_their_inputs():
    for at in (1 * M, 2 * M, 3 * M, 3 * M + 60):
        _refused("ygg_route_backward", (1 * M, 2 * M, 3 * M, 8, 4, 2, at, None), "shares memory")
    for act, at in ((0, 1 * M), (1, 1 * M + 64), (1, 4 * M), (1, 4 * M + 496), (1, 4 * M - 16)):
        _refused("ygg_pauli_grouped_input_grad", (1 * M, 8, 2 * M, 3 * M, 2, 4, 4, act, 4 * M, at, 1, 1, None), "shares memory")


def test_weights_prepared_on_another_device_are_refused(monkeypatch):
    class Tensor:
        is_cuda = True

        def __init__(self, n):
            self.device = torch.device("cuda", n)

        def get_device(self):
            return self.device.index

        def is_contiguous(self):
            return True

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    a = Tensor(0)
    here, there = (ops.PreparedWeights(Tensor(n), None, "pauli", 2, 4, 4) for n in (0, 1))
    routing = dict(topk_w=a, offsets=a)
    for f in (lambda: ops.pauli_grouped_input_grad(a, there, a),
              lambda: ops.moe_forward_train_bf16(a, 2, here, there), lambda: ops.moe_forward_train_bf16(a, 2, there, here),
              lambda: ops.moe_backward_bf16(a, a, routing, here, there), lambda: ops.moe_backward_bf16(a, a, routing, there, here)):
        with pytest.raises(ValueError, match="one device"):
            f()


@pytest.mark.parametrize("at", [15, 16, 17, 18])
def test_a_weights_gradient_without_its_biases(at):
    args = list(_BWD)
    args[at] = None
    _refused("ygg_moe_backward_bf16", args, "together")


@pytest.mark.parametrize("E,few", [(1, 252), (2, 348), (3, 348), (4, 444), (8, 540), (15, 540), (16, 636), (32, 732), (64, 828)])
def test_weight_gradients_of_few_rows_take_no_workspace(E, few):
    """252 + 96 log2(E) rows and fewer are one chunk an expert; one row more has planes."""
    need = lambda P: N.lib().ygg_grouped_weight_grad_pauli_bf16_workspace_bytes(P, E, 64, 256)
    assert need(1) == need(few) == 0 and need(few + 1) > 0
