"""Norms after and before a block, fused with the block's gate and the residual's scale:

    r = residual_scale x + gate N_after(y),        h = N_before(r)

x: the residual stream, y: the block's output, h: what the next block reads.  The post-norm of BertGatedLinearUnitMLP
(reference: bert/src/bert_layers.py:506) is the case without gate, scale and N_after, of which h alone goes on; this one also
serves pre-norm and sandwich-norm blocks, and has gradients.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

_NONE, _CHANNEL, _SEQUENCE, _TOKEN = 0, 1, 2, 3
_PARAMS = ("after_weight", "after_bias", "before_weight", "before_bias")


def _rows(t, n):
    """t as rows of n contiguous columns, read in place where its strides allow it."""
    t = t.reshape(-1, n)
    return t if t.stride(1) == 1 or n == 1 else t.contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _args(x, y, gate, kind, seq_len, scale, params, eps, rms):
    n = x.shape[-1]
    a = _lib.ResidualNormArgs()
    a.rows, a.n = x.shape[0], n
    a.seq_len = seq_len
    a.x_dtype, a.y_dtype = ops._dt(x), ops._dt(y)
    a.gate_kind, a.rms, a.eps = kind, rms, eps
    a.x, a.ldx, a.y, a.ldy = x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0)
    if kind:
        a.gate, a.gate_dtype = gate.data_ptr(), ops._dt(gate)
        a.ldg = gate.stride(0)
    if isinstance(scale, torch.Tensor):
        a.scale_channel = scale.data_ptr()
    else:
        a.scale = scale
    a.after_weight, a.after_bias, a.before_weight, a.before_bias = (_ptr(p) for p in params)
    a.norm_after, a.norm_before = params[0] is not None, params[2] is not None
    return a


def _forward(a, x, y, shape, stats):
    r = torch.empty(shape, dtype=x.dtype, device=x.device)
    h = torch.empty(shape, dtype=y.dtype, device=x.device) if a.norm_before else None
    a.r, a.h, a.stats = r.data_ptr(), _ptr(h), _ptr(stats)
    ops._launch("m2_residual_norm_fwd", x, _lib.lib().m2_residual_norm_fwd, C.byref(a))
    return r, h


class _ResidualNorm(torch.autograd.Function):
    """Tensors in, in this order: x, y, gate, scale (tensor or None), the four parameters; then plain values."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, after_weight, after_bias, before_weight, before_bias, number, kind, seq_len, eps, rms):
        n = x.shape[-1]
        params = (after_weight, after_bias, before_weight, before_bias)
        x2, y2 = _rows(x, n), _rows(y, n)
        g2 = _rows(gate, n) if kind else None
        a = _args(x2, y2, g2, kind, seq_len, scale if scale is not None else number, params, eps, rms)
        stats = torch.empty((a.rows, 4), dtype=torch.float32, device=x.device)
        out = _forward(a, x2, y2, x.shape, stats)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, gate, scale, *params, stats)
        ctx.plain = (number, kind, seq_len, eps, rms)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_r, d_h):
        x, y, gate, scale, *params, stats = ctx.saved_tensors
        number, kind, seq_len, eps, rms = ctx.plain
        if d_r is None and d_h is None:
            return (None,) * 13
        n, dev = x.shape[-1], x.device
        x2, y2 = _rows(x, n), _rows(y, n)
        g2 = _rows(gate, n) if kind else None
        a = _args(x2, y2, g2, kind, seq_len, scale if scale is not None else number, params, eps, rms)
        a.stats = stats.data_ptr()
        d_r = d_r.contiguous() if d_r is not None else None
        d_h = d_h.contiguous() if d_h is not None else None
        want = ctx.needs_input_grad
        like = (x, y, gate, scale, *params)
        out = [torch.empty(t.shape, dtype=t.dtype, device=dev) if w and t is not None else None for t, w in zip(like, want)]
        if a.rows == 0:                                        # nothing to launch: sums over no rows
            return (*[t.zero_() if t is not None else None for t in out], None, None, None, None, None)
        g = _lib.ResidualNormGrads()
        g.d_r, g.d_h = _ptr(d_r), _ptr(d_h)
        g.d_x, g.d_y, g.d_gate, g.d_scale, g.d_after_weight, g.d_after_bias, g.d_before_weight, g.d_before_bias = (_ptr(t) for t in out)
        work = torch.empty(_lib.lib().m2_residual_norm_workspace(a.rows, seq_len, n, kind) // 4, dtype=torch.float32, device=dev)
        g.workspace = work.data_ptr()
        ops._launch("m2_residual_norm_bwd", x, _lib.lib().m2_residual_norm_bwd, C.byref(a), C.byref(g), launches=2)
        return (*out, None, None, None, None, None)


def _vector(name, what, t, n, dev):
    if t is None:
        return None
    if t.shape != (n,) or t.device != dev or not t.is_floating_point():
        raise ValueError(f"{name}: {what} has {n} values on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.dtype != torch.float32:
        t = t.float()
    return t.contiguous()


def gated_residual_norm(x, y, *, gate=None, residual_scale=1.0, after_weight=None, after_bias=None, before_weight=None, before_bias=None,
                        eps=1e-12, rms=False):
    """(r, h) with r = residual_scale * x + gate * N_after(y) and h = N_before(r), in one launch.

    x, y            (..., D), float32 or bfloat16 each, D <= 8192; r has x's type, h has y's
    gate            None, (D,), (B, 1, D) for x (B, L, D), or x's shape; float32 or bfloat16
    residual_scale  a number or a tensor (D,)
    after_weight, after_bias    of N_after, (D,); without a weight N_after(y) = y
    before_weight, before_bias  of N_before, (D,); without a weight h is None
    rms             RMS norms instead of LayerNorms

    Statistics and sums are float32; r and h are rounded once each (h is that of the unrounded r).  Differentiable in every tensor."""
    name = "gated_residual_norm"
    if x.dim() < 1 or x.shape != y.shape:
        raise ValueError(f"{name}: x and y have one shape, got {tuple(x.shape)} and {tuple(y.shape)}")
    n, dev = x.shape[-1], x.device
    if not x.is_cuda or y.device != dev or (gate is not None and gate.device != dev):
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    for t in (x, y, gate):
        if t is not None and t.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"{name}: tensors are float32 or bfloat16, got {t.dtype}")
    if n == 0:
        raise ValueError(f"{name}: rows without columns")
    if (after_bias is not None and after_weight is None) or (before_bias is not None and before_weight is None):
        raise ValueError(f"{name}: a norm's bias needs its weight")
    if not eps >= 0:
        raise ValueError(f"{name}: eps {eps}")
    rows = x.numel() // n
    kind, seq_len = _NONE, max(rows, 1)
    if gate is not None:
        if gate.shape == (n,):
            kind, gate = _CHANNEL, gate.contiguous()
        elif gate.shape == x.shape:
            kind = _TOKEN
        elif x.dim() == 3 and gate.shape == (x.shape[0], 1, n):
            kind, seq_len = _SEQUENCE, max(x.shape[1], 1)
        else:
            raise ValueError(f"{name}: a gate is ({n},), (B, 1, {n}) or {tuple(x.shape)}, got {tuple(gate.shape)}")
    params = [_vector(name, what, t, n, dev) for what, t in zip(_PARAMS, (after_weight, after_bias, before_weight, before_bias))]
    scale, number = None, 1.0
    if isinstance(residual_scale, torch.Tensor):
        scale = _vector(name, "residual_scale", residual_scale, n, dev)
    else:
        number = float(residual_scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, y, gate, scale, *params)):
        return _ResidualNorm.apply(x, y, gate, scale, *params, number, kind, seq_len, float(eps), bool(rms))
    x2, y2 = _rows(x, n), _rows(y, n)
    a = _args(x2, y2, _rows(gate, n) if kind else None, kind, seq_len, scale if scale is not None else number, params, float(eps), bool(rms))
    return _forward(a, x2, y2, x.shape, None)
