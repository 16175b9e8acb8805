"""Cross attention of stacked frames (csrc/glx_attention.hip, csrc/glx_attention_bwd.hip, bound in csrc/host/glx_torch.cpp),
beside the operators of pcdet_ops.pointnet2.pointnet2_stack that gather a frame's points at query points: here every query
weighs ALL of its frame's encoder states (points, voxels, RoI grid points; another number of them per frame) by
softmax(scale q k^T).

Two layouts.  Stacked, as (N1 + N2 + .., H, D) with int32 counts per frame on the device (no read-back: the call can be
recorded), or a padded batch (B, L, H, D).  key_mask says which encoder states take part; what the
others hold, NaN included, reaches no result."""
import math

import torch

from . import _lib


def _counts(c):
    if c.numel() == 0:
        return c.new_zeros(1, dtype=torch.int32)              # no frames: one empty frame
    if c.dtype == torch.int64:
        c = c.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return c.contiguous()


def cross_attention(q, k, v, q_batch_cnt=None, k_batch_cnt=None, key_mask=None, scale=None):
    """softmax(scale q k^T) v, every query over its own frame's encoder states.

    q (M1 + M2 + .., H, D), k / v (N1 + N2 + .., Hkv, D) with q_batch_cnt / k_batch_cnt (B,) int32 device counts, or
    q (B, M, H, D), k / v (B, N, Hkv, D) without counts; float32, bfloat16 or float16, D <= 128, H a multiple of Hkv (query
    heads j H / Hkv .. share key head j).  Any strides between rows and heads.
    key_mask (N1 + N2 + ..,) or (B, N) bool, True = attended: what a masked state holds does not matter, its gradients are 0.
    scale: default 1 / sqrt(D).
    -> q's shape and type.  A query whose frame has no state left gives 0 and no gradients, and so do rows behind the last
    frame (counts that reach beyond the tensors are cut there).  Gradients have the same bits every
    time.  Once differentiable, in reverse mode: an input with a forward-mode tangent is refused.

    Scores, softmax and sums in fp32.  Of 16-bit tensors the softmax' weights are rounded to their type in front of their product with
    v, and the weights and the scores' gradients in front of theirs in the backward pass, which together leave 1.4 times the error that
    rounding the results alone would; few rows (single queries: the time is the keys') keep the weights to twice the bits in the forward
    pass, heads of up to 32 channels in the backward pass."""
    who = "cross_attention"
    if q.dtype not in _lib.DTYPE_CODES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("%s: q, k, v must share one type, float32, bfloat16 or float16; got %s, %s, %s" % (who, q.dtype, k.dtype, v.dtype))
    stacked = q_batch_cnt is not None or k_batch_cnt is not None
    dims = 3 if stacked else 4
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise ValueError("%s: expected %s, got shapes %s, %s, %s" % (
            who, "(rows, heads, dim) with counts" if stacked else "(frames, rows, heads, dim) without counts", tuple(q.shape),
            tuple(k.shape), tuple(v.shape)))
    if k.shape != v.shape or k.shape[-1] != q.shape[-1] or (not stacked and k.shape[0] != q.shape[0]):
        raise ValueError("%s: q %s, k %s and v %s do not belong together" % (who, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    heads, dim, kvh = q.shape[-2], q.shape[-1], k.shape[-2]
    if not 1 <= dim <= 128 or kvh < 1 or heads < 1 or heads % kvh:
        raise ValueError("%s: %d heads of %d over %d key heads (dim 1 .. 128, heads a multiple of key heads)" % (who, heads, dim, kvh))
    if stacked:
        for n, c in (("q_batch_cnt", q_batch_cnt), ("k_batch_cnt", k_batch_cnt)):
            if c is None or c.dim() != 1 or c.dtype not in (torch.int32, torch.int64) or c.shape != q_batch_cnt.shape:
                raise ValueError("%s: %s must be an integer tensor (frames,) beside the other side's" % (who, n))
        q_batch_cnt, k_batch_cnt = _counts(q_batch_cnt), _counts(k_batch_cnt)
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != k.shape[:-2]:
            raise ValueError("%s: key_mask must be bool of shape %s, got %s %s" % (who, tuple(k.shape[:-2]), key_mask.dtype, tuple(key_mask.shape)))
        key_mask = key_mask.contiguous()
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("%s: scale %r" % (who, scale))
    _lib.check_device(who, q, k, v, q_batch_cnt, k_batch_cnt, key_mask)
    if q.numel() // dim >= 1 << 31 or k.numel() // dim >= 1 << 31:
        raise ValueError("%s: more than 2^31 rows x heads" % who)
    return _lib.torch_ops().cross_attention.default(q, k, v, q_batch_cnt, k_batch_cnt, key_mask, scale)
