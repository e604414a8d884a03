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
_VECTORS = ("residual_scale", "after_weight", "after_bias", "before_weight", "before_bias")
_TYPES = {torch.float32: _lib.M2_F32, torch.bfloat16: _lib.M2_BF16}


def _rows(t, n):
    """The rows of t, which _evenly() gave, and the distance between them."""
    if t.is_contiguous():
        return t, n
    t = t.view(-1, n)
    return t, t.stride(0)


def _evenly(t):
    """t, or a copy: rows of adjacent columns a fixed distance apart.  Made before the gradient's function takes it, so that there is one copy."""
    if t.is_contiguous():
        return t
    n = t.shape[-1]
    if t.stride(-1) == 1 or n == 1:
        try:
            t.view(-1, n)
            return t
        except RuntimeError:
            pass
    return t.contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _args(x, y, gate, kind, seq_len, scale, number, params, eps, rms):
    """The arguments, and the tensors that they point to."""
    n = x.shape[-1]
    (x, ldx), (y, ldy), (gate, ldg) = _rows(x, n), _rows(y, n), _rows(gate, n) if kind else (None, 0)
    w1, b1, w2, b2 = params
    a = _lib.ResidualNormArgs(
        x.numel() // n, seq_len, n, _TYPES[x.dtype], _TYPES[y.dtype], _TYPES[gate.dtype] if kind else 0, kind, rms, w1 is not None, w2 is not None,
        eps, number, x.data_ptr(), ldx, y.data_ptr(), ldy, gate.data_ptr() if kind else None, ldg, _ptr(scale), _ptr(w1), _ptr(b1), _ptr(w2), _ptr(b2))
    return a, (x, y, gate)


def _forward(a, x, y, stats):
    r = x.new_empty(x.shape)
    h = y.new_empty(x.shape) if a.norm_before else None
    a.r, a.h, a.stats = r.data_ptr(), _ptr(h), _ptr(stats)
    ops._launch("m2_residual_norm_fwd", x, _lib.lib().m2_residual_norm_fwd, C.byref(a), launches=None)
    return r, h


class _ResidualNorm(torch.autograd.Function):
    """Tensors in, in this order: x, y, gate, scale (tensor or None), the four parameters; then plain values."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, after_weight, after_bias, before_weight, before_bias, number, kind, seq_len, eps, rms):
        params = (after_weight, after_bias, before_weight, before_bias)
        a, keep = _args(x, y, gate, kind, seq_len, scale, number, params, eps, rms)  # noqa: F841
        stats = torch.empty((a.rows, 4), dtype=torch.float32, device=x.device)
        out = _forward(a, x, y, stats)
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
        n = x.shape[-1]
        a, keep = _args(x, y, gate, kind, seq_len, scale, number, params, eps, rms)  # noqa: F841
        a.stats = stats.data_ptr()
        d_r = d_r.contiguous() if d_r is not None else None
        d_h = d_h.contiguous() if d_h is not None else None
        want = ctx.needs_input_grad
        out = [t.new_empty(t.shape) if w and t is not None else None for t, w in zip((x, y, gate, scale, *params), want)]
        if a.rows == 0:                                        # nothing to launch: sums over no rows
            return (*[t.zero_() if t is not None else None for t in out], None, None, None, None, None)
        size = ops._on_device(x.get_device(), _lib.lib().m2_residual_norm_workspace, a.rows, seq_len, n, kind)
        work = stats.new_empty(size // 4)
        g = _lib.ResidualNormGrads(_ptr(d_r), _ptr(d_h), *(_ptr(t) for t in out), work.data_ptr(), size)
        ops._launch("m2_residual_norm_bwd", x, _lib.lib().m2_residual_norm_bwd, C.byref(a), C.byref(g), launches=None)
        return (*out, None, None, None, None, None)


def _vector(name, what, t, n, dev):
    if t.shape != (n,) or t.get_device() != dev or not t.is_floating_point():
        raise ValueError(f"{name}: {what} has {n} values on device {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def gated_residual_norm(x, y, *, gate=None, residual_scale=1.0, after_weight=None, after_bias=None, before_weight=None, before_bias=None,
                        eps=1e-12, rms=False):
    """(r, h) with r = residual_scale * x + gate * N_after(y) and h = N_before(r), in one launch.

    x, y            (..., D), float32 or bfloat16 each, D <= 8192; r has x's type, h has y's.  Rows a fixed distance apart are
                    read in place, others (x[:, :-1] of a batch) are copied first
    gate            None, (D,), (B, 1, D) for x (B, L, D), or x's shape; float32 or bfloat16
    residual_scale  a number or a tensor (D,)
    after_weight, after_bias    of N_after, (D,); without a weight N_after(y) = y
    before_weight, before_bias  of N_before, (D,); without a weight h is None
    rms             RMS norms instead of LayerNorms

    Statistics and sums are float32; r and h are rounded once each (h is that of the unrounded r).  Differentiable in every tensor."""
    name = "gated_residual_norm"
    if x.dim() < 1 or x.shape != y.shape:
        raise ValueError(f"{name}: x and y have one shape, got {tuple(x.shape)} and {tuple(y.shape)}")
    n, dev = x.shape[-1], x.get_device()
    if dev < 0 or y.get_device() != dev or (gate is not None and gate.get_device() != dev):
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    if x.dtype not in _TYPES or y.dtype not in _TYPES or (gate is not None and gate.dtype not in _TYPES):
        raise TypeError(f"{name}: tensors are float32 or bfloat16, got {x.dtype}, {y.dtype}{'' if gate is None else f' and {gate.dtype}'}")
    if n == 0:
        raise ValueError(f"{name}: rows without columns")
    if (after_bias is not None and after_weight is None) or (before_bias is not None and before_weight is None):
        raise ValueError(f"{name}: a norm's bias needs its weight")
    eps = float(eps)
    if not eps >= 0:
        raise ValueError(f"{name}: eps {eps}")
    kind, seq_len = _NONE, 1
    if gate is not None:
        if gate.shape == (n,):
            kind, gate = _CHANNEL, gate.contiguous()
        elif gate.shape == x.shape:
            kind = _TOKEN
        elif x.dim() == 3 and gate.shape == (x.shape[0], 1, n):
            kind, seq_len = _SEQUENCE, max(x.shape[1], 1)
        else:
            raise ValueError(f"{name}: a gate is ({n},), (B, 1, {n}) or {tuple(x.shape)}, got {tuple(gate.shape)}")
    x, y = _evenly(x), _evenly(y)
    if kind > _CHANNEL:
        gate = _evenly(gate)
    tensors = [x, y, gate, residual_scale if isinstance(residual_scale, torch.Tensor) else None, after_weight, after_bias, before_weight, before_bias]
    for i in range(3, 8):
        if tensors[i] is not None:
            tensors[i] = _vector(name, _VECTORS[i - 3], tensors[i], n, dev)
    number = float(residual_scale) if tensors[3] is None else 1.0
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return _ResidualNorm.apply(*tensors, number, kind, seq_len, eps, bool(rms))
    a, keep = _args(x, y, gate, kind, seq_len, tensors[3], number, tensors[4:], eps, bool(rms))  # noqa: F841
    return _forward(a, x, y, None)
