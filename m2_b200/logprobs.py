"""Log probabilities of given tokens, with entropy and the best alternatives, from logits: what the loss of the reference's
masked-LM head computes behind its decoder (bert/src/bert_layers.py, BertForMaskedLM), and its scoring.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """logprob, entropy (...) float32; top_logprob float32 and top_id int64 (..., top), best first."""
    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_id: torch.Tensor


_TYPES = {torch.float32: _lib.M2_F32, torch.bfloat16: _lib.M2_BF16}


def _readable(logits):
    """logits as they are read in place, or a copy of them: adjacent logits, and at most two leading dimensions with strides of
    their own (a batch's texts without their last row, logits[:, :-1])."""
    if logits.is_contiguous():
        return logits
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        return logits.contiguous()
    if logits.dim() <= 3:
        return logits
    try:
        return logits.view(-1, *logits.shape[-2:])
    except RuntimeError:
        return logits.contiguous()


def _strides(x):
    """From row to row, rows of a group (0: all rows are one), from group to group."""
    if x.is_contiguous() or x.dim() == 1:
        return x.shape[-1], 0, 0
    return (x.stride(0), 0, 0) if x.dim() == 2 else (x.stride(1), x.shape[1], x.stride(0))


def _forward(x, targets, top, ignore_index, want_stats):
    """The results and, where they are wanted, what the gradient needs besides."""
    ld, group, ld_group = _strides(x)
    shape, V = targets.shape, x.shape[-1]
    n = targets.numel()
    logprob = torch.empty(shape, dtype=torch.float32, device=x.device)
    entropy = torch.empty_like(logprob)
    best, ids = logprob.new_empty((*shape, top)), targets.new_empty((*shape, top))
    stats = logprob.new_empty((n, 2)) if want_stats else None
    a = _lib.TokenLogprobsArgs(n, V, top, _TYPES[x.dtype], x.data_ptr(), ld, targets.data_ptr(), ignore_index, logprob.data_ptr(), entropy.data_ptr(),
                               stats.data_ptr() if want_stats else None, best.data_ptr(), ids.data_ptr(), group, ld_group)
    ops._launch("m2_token_logprobs_fwd", x, _lib.lib().m2_token_logprobs_fwd, C.byref(a), launches=None)
    return TokenLogprobs(logprob, entropy, best, ids), stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, top, ignore_index):
        out, stats = _forward(x, targets, top, ignore_index, True)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(out.top_id)
        ctx.save_for_backward(x, targets, stats, out.entropy, out.top_id)
        ctx.ignore_index = ignore_index
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprob, d_entropy, d_top, _):
        x, targets, stats, entropy, ids = ctx.saved_tensors
        ld, group, ld_group = _strides(x)
        keep = [t.contiguous() if t is not None else None for t in (d_logprob, d_entropy, d_top)]
        d = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        V = x.shape[-1]
        a = _lib.TokenLogprobsBwdArgs(targets.numel(), V, ids.shape[-1], _TYPES[x.dtype], x.data_ptr(), ld, targets.data_ptr(), ctx.ignore_index,
                                      stats.data_ptr(), entropy.data_ptr(), ids.data_ptr(), *(t.data_ptr() if t is not None else None for t in keep),
                                      d.data_ptr(), V, group, ld_group)
        ops._launch("m2_token_logprobs_bwd", x, _lib.lib().m2_token_logprobs_bwd, C.byref(a), launches=None)
        return d, None, None, None


def token_logprobs(logits, targets, *, top=0, ignore_index=-100):
    """TokenLogprobs of logits (..., V), float32 or bfloat16, and targets (...), integers: log softmax(logits) at the target, the
    entropy of softmax(logits), and the `top` (<= 32) best ids with their log probabilities, best first; equal logits go by
    ascending id.  The logits are read once, in place where a row's lie side by side and the leading dimensions have at most two
    strides (logits[:, :-1] of a batch); others are copied first.  Everything is summed in float32.

    Rows whose target is `ignore_index` are not read: zeros, ids -1, no gradient.  A target outside 0 .. V-1 gives NaN and sets
    M2_DEV_BAD_INDEX (ops.device_status()).  Logits of -inf have probability 0; where a row has no others its log probabilities
    are -inf, its entropy and its gradient 0.  Differentiable in logits, through logprob, entropy and top_logprob."""
    name = "token_logprobs"
    if logits.dim() < 1 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"{name}: one target for each row of logits, got {tuple(targets.shape)} and {tuple(logits.shape)}")
    V = logits.shape[-1]
    if logits.dtype not in _TYPES:
        raise TypeError(f"{name}: logits are float32 or bfloat16, got {logits.dtype}")
    if targets.dtype != torch.long and (targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool):
        raise TypeError(f"{name}: targets are integers, got {targets.dtype}")
    if not logits.is_cuda or targets.get_device() != logits.get_device():
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    top = int(top)
    if V == 0 or not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"{name}: {top} alternatives of {V} logits (0 to {MAX_TOP}, no more than there are)")
    if targets.dtype != torch.long or not targets.is_contiguous():
        targets = targets.to(torch.long).contiguous()
    x = _readable(logits)
    if x.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(x, targets, top, int(ignore_index)))
    return _forward(x, targets, top, int(ignore_index), False)[0]
