"""Cross attention of stacked frames (csrc/glx_attention.hip, csrc/glx_attention_bwd.hip), beside the operators of
pcdet_ops.pointnet2.pointnet2_stack that gather a frame's points at query points: here every query weighs ALL of its frame's
encoder states (points, voxels, RoI grid points; another number of them per frame) by softmax(scale q k^T).

Two layouts.  Stacked, as (N1 + N2 + .., H, D) with int32 counts per frame on the device (no read-back: the call can be
recorded), or a padded batch (B, L, H, D).  key_mask says which encoder states take part; masked ones are never read."""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib


class _Attention(ctypes.Structure):        # glx_attention
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "out", "lse", "key_mask", "q_cnt", "k_cnt")]
                + [(n, ctypes.c_int64) for n in ("q_rows", "k_rows", "q_len", "k_len", "q_stride", "q_head_stride", "k_stride",
                                                 "k_head_stride", "v_stride", "v_head_stride")]
                + [(n, ctypes.c_int32) for n in ("frames", "heads", "kv_heads", "dim", "dtype")] + [("scale", ctypes.c_float)])


def _stack(t):
    """(.., rows, heads, dim) as stacked rows with unit stride inside a head -> (tensor, row stride, head stride)."""
    if t.dim() == 4:
        b, n = t.shape[:2]
        if b > 1 and n > 0 and t.stride(0) != n * t.stride(1):
            t = t.contiguous()
        row = t.stride(1) if n != 1 else t.stride(0)       # one row per frame: the frames' stride is the rows'
    else:
        row = t.stride(0)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
        row = t.shape[-2] * t.shape[-1]
    return t, row, t.stride(-2)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _descriptor(q, k, v, q_cnt, k_cnt, key_mask, scale, out, lse):
    d = _Attention()
    d.q, d.k, d.v, d.out, d.lse, d.key_mask, d.q_cnt, d.k_cnt = (_ptr(t) for t in (q[0], k[0], v[0], out, lse, key_mask, q_cnt, k_cnt))
    heads, dim = q[0].shape[-2:]
    d.q_rows, d.k_rows = q[0].numel() // (heads * dim), k[0].numel() // (k[0].shape[-2] * dim)
    if q_cnt is None:
        d.frames, d.q_len, d.k_len = q[0].shape[0], q[0].shape[1], k[0].shape[1]
    else:
        d.frames = q_cnt.shape[0]
    _, d.q_stride, d.q_head_stride = q
    _, d.k_stride, d.k_head_stride = k
    _, d.v_stride, d.v_head_stride = v
    d.heads, d.kv_heads, d.dim, d.dtype, d.scale = heads, k[0].shape[-2], dim, _lib.dtype_code(q[0].dtype), scale
    return d


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_cnt, k_cnt, key_mask, scale):
        dev = q.device
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        keep = any(ctx.needs_input_grad)
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=dev) if keep else None
        d = _descriptor(_stack(q), _stack(k), _stack(v), q_cnt, k_cnt, key_mask, scale, out, lse)
        n = _lib.query("glx_attention_workspace_bytes", ctypes.byref(d))
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n > 256 else None
        _lib.call_on(dev, "glx_attention_forward", ctypes.byref(d), ws, _lib.size_arg(n))
        if keep:
            ctx.save_for_backward(q, k, v, q_cnt, k_cnt, key_mask, out, lse)
            ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, q_cnt, k_cnt, key_mask, out, lse = ctx.saved_tensors
        dev = q.device
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) if need else None
                      for t, need in zip((q, k, v), ctx.needs_input_grad))
        g, gs, gh = _stack(go)
        sq, sk, sv = _stack(q), _stack(k), _stack(v)
        d = _descriptor(sq, sk, sv, q_cnt, k_cnt, key_mask, ctx.scale, out, lse)
        n = _lib.query("glx_attention_backward_workspace_bytes", ctypes.byref(d))
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.call_on(dev, "glx_attention_backward", ctypes.byref(d), g, ctypes.c_int64(gs), ctypes.c_int64(gh), dq, dk, dv, ws,
                     _lib.size_arg(n))
        return dq, dk, dv, None, None, None, None


def cross_attention(q, k, v, q_batch_cnt=None, k_batch_cnt=None, key_mask=None, scale=None):
    """softmax(scale q k^T) v, every query over its own frame's encoder states.

    q (M1 + M2 + .., H, D), k / v (N1 + N2 + .., Hkv, D) with q_batch_cnt / k_batch_cnt (B,) int32 device counts, or
    q (B, M, H, D), k / v (B, N, Hkv, D) without counts; float32, bfloat16 or float16, D <= 128, H a multiple of Hkv (query
    heads j H / Hkv .. share key head j).  Any strides between rows and heads.
    key_mask (N1 + N2 + ..,) or (B, N) bool, True = attended: what a masked state holds does not matter, its gradients are 0.
    scale: default 1 / sqrt(D).
    -> q's shape and type.  A query whose frame has no state left gives 0 and no gradients, and so do rows behind the last
    frame (counts that reach beyond the tensors are cut there).  Scores, softmax and sums in fp32; gradients have the same bits
    every time.  Once differentiable."""
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
        q_batch_cnt, k_batch_cnt = (c.to(torch.int32).contiguous() if c.numel() else c.new_zeros(1, dtype=torch.int32)
                                    for c in (q_batch_cnt, k_batch_cnt))           # (no frames: one empty frame)
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
    return _CrossAttention.apply(q, k, v, q_batch_cnt, k_batch_cnt, key_mask, scale)
