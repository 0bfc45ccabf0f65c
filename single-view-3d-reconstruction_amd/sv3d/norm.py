"""Layer norm on the device: entry point of the operators `sv3d::layer_norm`, `sv3d::layer_norm_stats` and `sv3d::layer_norm_backward`
(csrc/torch_train_ops.cpp over the functions of the same names in include/sv3d_hip.h), and the module over it.
The transformer camera head of the reference's network (nnutils/mesh_net.py:468-536) is made of blocks that each
end in one.  GPU tensors only.
"""
import math

import torch

from .ops import call


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """`torch.nn.functional.layer_norm`: normalises over the last `len(normalized_shape)` dimensions of `x`
    (float32, float16 or bfloat16; any strides, without a copy where rows are contiguous and evenly spaced), then
    scales and shifts by `weight` and `bias` (of x's type or float32).  Statistics and arithmetic are float32, and so are the
    sums of the weights' gradients until they are joined in float64; the result has x's type, under autocast float32 (as
    torch's).  Differentiable once in x, weight and bias, by `backward` and `torch.autograd.grad` (`create_graph=True` and
    `torch.func.grad`, which sets it, raise)."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    return call("layer_norm", x, shape, weight, bias, eps, torch.is_autocast_enabled("cuda"))


class LayerNorm(torch.nn.LayerNorm):
    """`torch.nn.LayerNorm` on the kernel: same arguments, parameters and state dict."""

    def forward(self, x):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)


_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _computable(m):
    """Whether the kernel has the layer's type and size (a layer without weights takes the type of what it is given)."""
    size = math.prod(m.normalized_shape)
    return 0 < size <= 1 << 24 and all(p is None or p.dtype in _TYPES for p in (m.weight, m.bias))


def convert_layer_norm(module):
    """Turns every `torch.nn.LayerNorm` inside `module` (or `module` itself) into this `LayerNorm`, in place:
    parameters, hooks and state dict stay.  Subclasses are left alone, and so are layers that the kernel does not compute:
    with float64 weights, or over none or more than 2^24 elements.  Returns the number of layers changed."""
    found = [m for m in module.modules() if type(m) is torch.nn.LayerNorm and _computable(m)]
    for m in found:
        m.__class__ = LayerNorm
    return len(found)
