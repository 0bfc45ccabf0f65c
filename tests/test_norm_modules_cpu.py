"""Layer norm as a module and in the graph, without a GPU: which modules are converted, what the graph's node keeps, what
it says where it has no derivative."""
import pytest
import torch

import sv3d
from sv3d import norm


def test_conversion_leaves_layers_alone_that_the_kernel_does_not_compute():
    N = torch.nn.LayerNorm
    half_double = N(4)
    half_double.bias = torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))
    m = torch.nn.ModuleList([N(4), N(4, dtype=torch.float64), N(4, bias=False, dtype=torch.float64), half_double,
                             N(4, elementwise_affine=False), N(4, dtype=torch.bfloat16), N(4).half(), N((0, 4)),
                             N((1 << 24) + 1, elementwise_affine=False)])
    assert sv3d.convert_layer_norm(m) == 4
    assert [type(x) is norm.LayerNorm for x in m] == [True, False, False, False, True, True, True, False, False]
    x = torch.randn(3, 4, dtype=torch.float64)
    for k in (1, 2):
        assert m[k](x).dtype == torch.float64


def meta(*shape):
    return torch.empty(shape, device="meta")


def test_hooks_on_saved_tensors_see_all_that_the_graph_keeps():
    """x, weight, bias and both statistics of the rows; what the hooks hand back is what the backward takes."""
    packed, unpacked = [], []

    def pack(t):
        packed.append(t)
        return t

    def unpack(t):
        unpacked.append(t)
        return t

    x, w, b = (t.requires_grad_() for t in (meta(6, 8), meta(8), meta(8)))
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = norm.layer_norm(x, 8, w, b)
    assert [tuple(t.shape) for t in packed] == [(6, 8), (8,), (8,), (6,), (6,)]
    assert [t.shape for t in torch.autograd.grad(y, (x, w, b), meta(6, 8))] == [x.shape, w.shape, b.shape]
    assert len(unpacked) == len(packed)


def test_refusals_of_a_second_derivative_say_who_asks_for_one():
    x = meta(2, 8).requires_grad_()
    with pytest.raises(RuntimeError, match=r"second derivative.*create_graph=True.*torch\.func"):
        torch.autograd.grad(norm.layer_norm(x, 8), x, meta(2, 8), create_graph=True)
    with pytest.raises(RuntimeError, match=r"torch\.func"):
        torch.func.grad(lambda t: norm.layer_norm(t, 8).sum())(meta(2, 8))
