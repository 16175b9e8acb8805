"""Layer norm over the last dimension (csrc/glx_layernorm.hip), beside the training BatchNorms of spconv.core and conv2d.

    y = (x - mean) / sqrt(var + eps) * weight + bias          (biased variance, statistics in fp32)

fp32, bf16 and fp16 rows of any width; weights of the rows' type or fp32.  The backward pass gives the gradients of the rows,
the weight and the bias in two launches with fixed summation orders: the same bits every time.  Once differentiable."""
import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib


def _rows(t, width):
    """t as (rows, width) with unit stride inside a row: a view where the strides allow it -> (tensor, elements between rows)."""
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1):
        return t, t.stride(0)
    t = t.contiguous().view(-1, width)
    return t, width


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        width = x.shape[-1]
        x2, ld = _rows(x, width)
        rows = x2.shape[0]
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        keep = any(ctx.needs_input_grad)
        mean = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if keep else None
        wt = _lib.dtype_code((weight if weight is not None else bias if bias is not None else x).dtype)
        _lib.call_on(x.device, "glx_layer_norm_forward", x2, ctypes.c_int64(ld), _lib.dtype_code(x.dtype), weight, bias, wt,
                     ctypes.c_int64(rows), ctypes.c_int64(width), ctypes.c_float(eps), y, mean, rstd)
        if keep:
            ctx.save_for_backward(x, weight, mean, rstd)
            ctx.wt, ctx.wdtype = wt, (weight if weight is not None else bias if bias is not None else x).dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, weight, mean, rstd = ctx.saved_tensors
        width = x.shape[-1]
        x2, ld = _rows(x, width)
        g2, ldg = _rows(gy, width)
        rows, dev = x2.shape[0], x.device
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(width, dtype=ctx.wdtype, device=dev) if ctx.needs_input_grad[1] else None
        db = torch.empty(width, dtype=ctx.wdtype, device=dev) if ctx.needs_input_grad[2] else None
        ws = None
        if dw is not None or db is not None:
            ws = torch.empty(_lib.query("glx_layer_norm_workspace_bytes", ctypes.c_int64(rows), ctypes.c_int64(width)),
                             dtype=torch.uint8, device=dev)
        _lib.call_on(dev, "glx_layer_norm_backward", g2, ctypes.c_int64(ldg), x2, ctypes.c_int64(ld), _lib.dtype_code(x.dtype),
                     weight, ctx.wt, mean, rstd, ctypes.c_int64(rows), ctypes.c_int64(width), dx, dw, db, ws,
                     _lib.size_arg(ws.numel() if ws is not None else 0))
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x (..., width) fp32 / bf16 / fp16 device tensor, weight / bias (width,) of x's type or fp32, either may be None
    -> x's shape and type.  Rows of a 2-D tensor may be any number of elements apart."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm: x needs a last dimension of at least one value, got shape %s" % (tuple(x.shape),))
    if x.dtype not in _lib.DTYPE_CODES:
        raise ValueError("layer_norm: x must be float32, bfloat16 or float16, got %s" % x.dtype)
    if not float(eps) >= 0.0:
        raise ValueError("layer_norm: eps must not be negative, got %r" % (eps,))
    given = [(n, t) for n, t in (("weight", weight), ("bias", bias)) if t is not None]
    for n, t in given:
        if tuple(t.shape) != (x.shape[-1],):
            raise ValueError("layer_norm: %s must have shape (%d,), got %s" % (n, x.shape[-1], tuple(t.shape)))
        if t.dtype not in (x.dtype, torch.float32) or t.dtype != given[0][1].dtype:
            raise ValueError("layer_norm: weight and bias must share one type, x's (%s) or float32; %s is %s" % (x.dtype, n, t.dtype))
    _lib.check_device("layer_norm", x, weight, bias)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    return _LayerNorm.apply(x, weight, bias, float(eps))


class LayerNorm(nn.Module):
    """Layer norm with learnt scale and offset, rows of `width` values."""

    def __init__(self, width, eps=1e-5, affine=True):
        super().__init__()
        self.width, self.eps = int(width), float(eps)
        self.weight = nn.Parameter(torch.ones(self.width)) if affine else None
        self.bias = nn.Parameter(torch.zeros(self.width)) if affine else None

    def forward(self, x):
        if x.shape[-1] != self.width:
            raise ValueError("LayerNorm(%d): got rows of %d values" % (self.width, x.shape[-1]))
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return "%d, eps=%g, affine=%s" % (self.width, self.eps, self.weight is not None)
