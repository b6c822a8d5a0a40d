"""Layers that run as single libpcx calls outside the whole-network plans: layer norm.

`layer_norm` / `LayerNorm` normalise the trailing axes of a float32, bfloat16 or float16 tensor and are
differentiable (csrc/layernorm.hip: one kernel forward, two backward, float32 statistics and sums, each output
rounded once, results that repeat bit by bit).  The networks use the same kernels for the projection head's
`projection_norm: layer` (phoneme_contrast_amd.models).  There is no CPU path: a CPU tensor raises.
"""
import functools
import math
import numbers

import torch
import torch.nn as nn

from . import _lib

MAX_DIM = 32768  # values per row


def _rows(t, D):
    """[..., D] as (tensor, rows, row stride): a view where the rows are evenly spaced with adjacent values, else a copy."""
    rows = t.numel() // D
    if t.is_contiguous():
        return t, rows, D
    try:
        v = t.view(rows, D)
    except RuntimeError:
        v = None
    if v is None or (D > 1 and v.stride(1) != 1) or (rows > 1 and v.stride(0) < D):
        return t.contiguous(), rows, D
    return v, rows, max(v.stride(0), D)


def _address(t):
    return t.data_ptr() if t is not None else None


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, D, eps):
        xr, rows, xs = _rows(x, D)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        wt = weight if weight is not None else bias
        dt = _lib.DTYPES[x.dtype]
        wdt = _lib.DTYPES[wt.dtype] if wt is not None else dt
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if any(ctx.needs_input_grad) else None
        with _lib.on_device(x):
            _lib.check(_lib.lib().pcx_layernorm_forward(dt, wdt, rows, D, xr.data_ptr(), xs, _address(w), _address(b),
                                                        eps, y.data_ptr(), _address(stats), _lib.raw_stream(x)),
                       "pcx_layernorm_forward")
        ctx.save_for_backward(x, w, stats)
        ctx.cfg = (D, eps, dt, wdt, weight is not None, None if wt is None else wt.shape,
                   None if wt is None else wt.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # create_graph: the gradient itself is not differentiable, and says so if asked
            return _layernorm_backward_once(ctx, dy)
        return _layernorm_backward(ctx, dy)


def _layernorm_backward(ctx, dy):
    x, w, stats = ctx.saved_tensors
    D, eps, dt, wdt, has_w, wshape, wtype = ctx.cfg
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    xr, rows, xs = _rows(x, D)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
    dw = torch.empty(wshape, dtype=wtype, device=x.device) if need_w else None
    db = torch.empty(wshape, dtype=wtype, device=x.device) if need_b else None
    if rows == 0:
        return dx, (dw.zero_() if need_w else None), (db.zero_() if need_b else None), None, None
    dyr, _, ds = _rows(dy, D)
    ws, nws = None, 0
    if need_w or need_b:
        nws = _workspace_bytes(dt, rows, D)
        ws = torch.empty(nws, dtype=torch.uint8, device=x.device)
    with _lib.on_device(x):
        _lib.check(_lib.lib().pcx_layernorm_backward(dt, wdt, rows, D, xr.data_ptr(), xs, _address(w), eps,
                                                     stats.data_ptr(), dyr.data_ptr(), ds, _address(dx), _address(dw),
                                                     _address(db), _address(ws), nws, _lib.raw_stream(x)),
                   "pcx_layernorm_backward")
    return dx, dw, db, None, None


_layernorm_backward_once = torch.autograd.function.once_differentiable(_layernorm_backward)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(dt, rows, D):
    return _lib.lib().pcx_layernorm_workspace_bytes(dt, rows, D)


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the trailing `normalized_shape` axes (biased variance).

    x: float32, bfloat16 or float16 on a ROCm GPU, any leading axes and any strides (rows of adjacent values are read
    in place); weight, bias: `normalized_shape`, both of x's type or both float32.  The result has x's type, the
    gradients their tensors' types.  Up to 32768 values per row."""
    shape = (int(normalized_shape),) if isinstance(normalized_shape, numbers.Integral) else tuple(normalized_shape)
    _lib.require_gpu(x, weight, bias, what="layer_norm")
    if x.dtype not in _lib.DTYPES:
        raise ValueError(f"layer_norm: float32, bfloat16 or float16 expected, got {x.dtype}")
    if not shape or x.shape[-len(shape):] != shape:
        raise ValueError(f"layer_norm: input of shape {tuple(x.shape)} does not end in {shape}")
    D = math.prod(shape)
    if not 1 <= D <= MAX_DIM:
        raise ValueError(f"layer_norm: rows of 1 to {MAX_DIM} values supported, got {shape}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.shape != shape:
            raise ValueError(f"layer_norm: {name} of shape {tuple(t.shape)}, {shape} expected")
        if t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"layer_norm: {name} must be {x.dtype} or float32, got {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"layer_norm: {name} is on {t.device}, the input on {x.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight ({weight.dtype}) and bias ({bias.dtype}) must have one type")
    if not 0.0 < float(eps) < 1e30:
        raise ValueError(f"layer_norm: eps must be positive, got {eps}")
    return _LayerNormFn.apply(x, weight, bias, D, float(eps))


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm (same constructor, parameters and state_dict) on `layer_norm`."""

    def forward(self, x):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)
