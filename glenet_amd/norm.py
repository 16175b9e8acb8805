"""Layer norm over the last dimension (csrc/glx_layernorm.hip, bound in csrc/host/glx_torch.cpp), beside the training
BatchNorms of spconv.core and conv2d.

    y = (x - mean) / sqrt(var + eps) * weight + bias          (biased variance, statistics in fp32)

fp32, bf16 and fp16 rows of any width; weights of the rows' type or fp32.  The backward pass gives the gradients of the rows,
the weight and the bias in one or two launches with fixed summation orders: the same bits every time.  Once differentiable, in
reverse mode: an input with a forward-mode tangent is refused."""
import torch
from torch import nn

from . import _lib


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x (..., width) fp32 / bf16 / fp16 device tensor, weight / bias (width,) of x's type or fp32, either may be None
    -> x's shape and type.  Rows of a 2-D tensor may be any number of elements apart."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm: x needs a last dimension of at least one value, got shape %s" % (tuple(x.shape),))
    if x.dtype not in _lib.DTYPE_CODES:
        raise ValueError("layer_norm: x must be float32, bfloat16 or float16, got %s" % x.dtype)
    if not float(eps) >= 0.0:
        raise ValueError("layer_norm: eps must not be negative, got %r" % (eps,))
    first = weight if weight is not None else bias
    for n, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError("layer_norm: %s must have shape (%d,), got %s" % (n, x.shape[-1], tuple(t.shape)))
        if t.dtype not in (x.dtype, torch.float32) or t.dtype != first.dtype:
            raise ValueError("layer_norm: weight and bias must share one type, x's (%s) or float32; %s is %s" % (x.dtype, n, t.dtype))
    _lib.check_device("layer_norm", x, weight, bias)
    return _lib.torch_ops().layer_norm.default(x, weight, bias, float(eps))


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
