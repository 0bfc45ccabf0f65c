"""sv3d: MI355X-native hot path (soft rasterizer + Chamfer NN, the mesh / texture stages either side of
them, and the training step's layer norm and optimizer) behind a C ABI.

`sv3d._lib` binds libsv3d_hip.so; `sv3d.ops`, `sv3d.meshreg`, `sv3d.texture`, `sv3d.norm` and `sv3d.optim` expose it as
PyTorch-ROCm custom ops (namespace `sv3d::`), all registered by importing this package.
"""
from . import _lib
from .ops import chamfer_nn, face_gather, face_gather_n, project_gather, render, soft_rasterize
from . import meshreg, norm, optim, texture
from .meshreg import flatten_loss, laplacian_loss, mesh_spmv
from .norm import LayerNorm, convert_layer_norm, layer_norm
from .texture import dt, dt_barrier, texture_sample

__all__ = ["_lib", "chamfer_nn", "face_gather", "face_gather_n", "project_gather", "render", "soft_rasterize",
           "meshreg", "norm", "optim", "texture", "LayerNorm", "convert_layer_norm", "layer_norm", "flatten_loss", "laplacian_loss", "mesh_spmv", "dt", "dt_barrier",
           "texture_sample"]
