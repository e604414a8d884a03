"""Dropout from a counter-based generator, with a mask that is never stored: what nn.Dropout does behind the reference's blocks in training
(bert/src/bert_layers.py:487, 505), with the residual's sum in the same launch.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

_TYPES = {torch.float32: _lib.M2_F32, torch.bfloat16: _lib.M2_BF16}


def _drop(x, residual, threshold, seed):
    y = x.new_empty(x.shape)
    a = _lib.DropoutArgs(x.numel(), threshold, _TYPES[x.dtype], x.data_ptr(), residual.data_ptr() if residual is not None else None, y.data_ptr())
    if isinstance(seed, torch.Tensor):
        a.seed = seed.data_ptr()
    else:
        a.key = seed
    ops._launch("m2_dropout", x, _lib.lib().m2_dropout, C.byref(a), launches=None)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed):
        ctx.threshold = threshold
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
        ctx.number = None if isinstance(seed, torch.Tensor) else seed
        return _drop(x, residual, threshold, seed)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        seed = ctx.saved_tensors[0] if ctx.number is None else ctx.number
        return (_drop(d_y.contiguous(), None, ctx.threshold, seed) if ctx.needs_input_grad[0] else None, d_y if ctx.needs_input_grad[1] else None, None, None)


def dropout(x, p, seed, *, residual=None):
    """residual + x / (1 - p) where an element is kept, residual elsewhere, for x and residual (None: 0) of one shape and type, float32 or
    bfloat16; sums are float32, rounded once.  An element that is dropped is 0 whatever it was.

    p      0 to 1, rounded to a multiple of 2^-16 (1 / (1 - p) is that p's; p = 1 drops all)
    seed   an integer, or an int64 tensor (2,) on x's device that holds a seed and the number of the call, read when the kernel runs: a
           captured graph that changes the number (seed[1] += 1) after its backward pass drops other elements in every replay.  Use every pair once:
           calls with the same seed (an integer has call number 0) and number drop the same places.

    Whether element i of x (counted in its shape's order, whatever its strides) is kept is decided by Philox 4x32-10 with the key `seed`
    and the counter (i // 8, number of the call), 16 bits for each element: the same for every type, GPU and grid.  The gradient makes the mask again.
    Differentiable in x and residual."""
    name = "dropout"
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{name}: p is a probability, got {p}")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name}: x is float32 or bfloat16, got {x.dtype}")
    dev = x.get_device()
    if dev < 0 or (residual is not None and residual.get_device() != dev):
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{name}: residual is {x.dtype} {tuple(x.shape)}, got {residual.dtype} {tuple(residual.shape)}")
    if isinstance(seed, torch.Tensor):
        if seed.shape != (2,) or seed.dtype != torch.long or seed.get_device() != dev or not seed.is_contiguous():
            raise ValueError(f"{name}: a seed is an integer or (2,) int64 on {x.device}, got {seed.dtype} {tuple(seed.shape)} on {seed.device}")
    else:
        seed = int(seed)
        if not -(1 << 63) <= seed < 1 << 64:
            raise ValueError(f"{name}: seed {seed} has more than 64 bits")
        seed &= (1 << 64) - 1
    ops._no_tangents(name, x, residual)
    threshold = round(p * 65536)
    x = x.contiguous()
    residual = residual.contiguous() if residual is not None else None
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, threshold, seed)
    return _drop(x, residual, threshold, seed)
