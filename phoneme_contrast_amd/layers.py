"""Layers that run as single libpcx calls outside the whole-network plans: layer norm.

`layer_norm` / `LayerNorm` normalise the trailing axes of a float32, bfloat16 or float16 tensor and are
differentiable (csrc/layernorm.hip: one kernel forward, two backward, float32 statistics and sums, each output
rounded once, results that repeat bit by bit; csrc/torch_ops.cpp: the torch operator around them).  The networks use
the same kernels for the projection head's `projection_norm: layer` (phoneme_contrast_amd.models).  There is no CPU
path: a CPU tensor raises.
"""
import numbers

import torch.nn as nn

from . import _lib


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the trailing `normalized_shape` axes (biased variance).

    x: float32, bfloat16 or float16 on a ROCm GPU, any leading axes and any strides (evenly spaced rows of adjacent
    values are read in place); weight, bias: `normalized_shape`, both of x's type or both float32.  The result has x's
    type, the gradients their tensors' types.  Up to 32768 values per row.  The gradient is not differentiable again;
    forward-mode derivatives and torch.func.grad raise."""
    _lib.require_gpu(x, weight, bias, what="layer_norm")
    shape = (normalized_shape,) if isinstance(normalized_shape, numbers.Integral) else normalized_shape
    return _lib.torch_ops().layer_norm(x, shape, weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm (same constructor, parameters and state_dict) on `layer_norm`."""

    def forward(self, x):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)
