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


def _rows(logits):
    t = logits.reshape(-1, logits.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _forward(x, targets, top, ignore_index, shape):
    n, dev = x.shape[0], x.device
    logprob, entropy = (torch.empty(shape, dtype=torch.float32, device=dev) for _ in range(2))
    best = torch.empty((*shape, top), dtype=torch.float32, device=dev)
    ids = torch.empty((*shape, top), dtype=torch.long, device=dev)
    stats = torch.empty((n, 2), dtype=torch.float32, device=dev)
    a = _lib.TokenLogprobsArgs()
    a.rows, a.vocab, a.top, a.dtype = n, x.shape[1], top, ops._dt(x)
    a.logits, a.ld, a.targets, a.ignore_index = x.data_ptr(), x.stride(0), targets.data_ptr(), ignore_index
    a.logprob, a.entropy, a.stats, a.top_logprob, a.top_id = logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(), best.data_ptr(), ids.data_ptr()
    ops._launch("m2_token_logprobs_fwd", x, _lib.lib().m2_token_logprobs_fwd, C.byref(a))
    return TokenLogprobs(logprob, entropy, best, ids), stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, ignore_index):
        x = _rows(logits)
        out, stats = _forward(x, targets, top, ignore_index, logits.shape[:-1])
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(out.top_id)
        ctx.save_for_backward(logits, targets, stats, out.entropy, out.top_id)
        ctx.ignore_index = ignore_index
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprob, d_entropy, d_top, _):
        logits, targets, stats, entropy, ids = ctx.saved_tensors
        x = _rows(logits)
        keep = [t.contiguous() if t is not None else None for t in (d_logprob, d_entropy, d_top)]
        d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a = _lib.TokenLogprobsBwdArgs()
        a.rows, a.vocab, a.top, a.dtype = x.shape[0], x.shape[1], ids.shape[-1], ops._dt(x)
        a.logits, a.ld, a.targets, a.ignore_index = x.data_ptr(), x.stride(0), targets.data_ptr(), ctx.ignore_index
        a.stats, a.entropy, a.top_id = stats.data_ptr(), entropy.data_ptr(), ids.data_ptr()
        a.d_logprob, a.d_entropy, a.d_top_logprob = (t.data_ptr() if t is not None else None for t in keep)
        a.d_logits, a.ldd = d.data_ptr(), x.shape[1]
        ops._launch("m2_token_logprobs_bwd", x, _lib.lib().m2_token_logprobs_bwd, C.byref(a))
        return d, None, None, None


def token_logprobs(logits, targets, *, top=0, ignore_index=-100):
    """TokenLogprobs of logits (..., V), float32 or bfloat16, and targets (...), integers: log softmax(logits) at the target, the
    entropy of softmax(logits), and the `top` (<= 32) best ids with their log probabilities, best first; equal logits go by
    ascending id.  The logits are read once; everything is summed in float32.

    Rows whose target is `ignore_index` are not read: zeros, ids -1, no gradient.  A target outside 0 .. V-1 gives NaN and sets
    M2_DEV_BAD_INDEX (ops.device_status()).  Logits of -inf have probability 0; where a row has no others its log probabilities
    are -inf, its entropy and its gradient 0.  Differentiable in logits, through logprob, entropy and top_logprob."""
    name = "token_logprobs"
    if logits.dim() < 1 or targets.shape != logits.shape[:-1]:
        raise ValueError(f"{name}: one target for each row of logits, got {tuple(targets.shape)} and {tuple(logits.shape)}")
    V = logits.shape[-1]
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name}: logits are float32 or bfloat16, got {logits.dtype}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise TypeError(f"{name}: targets are integers, got {targets.dtype}")
    if not logits.is_cuda or targets.device != logits.device:
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    top = int(top)
    if V == 0 or not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"{name}: {top} alternatives of {V} logits (0 to {MAX_TOP}, no more than there are)")
    targets = targets.to(torch.long).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top, int(ignore_index)))
    return _forward(_rows(logits), targets, top, int(ignore_index), logits.shape[:-1])[0]
