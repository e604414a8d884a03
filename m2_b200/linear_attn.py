"""Linear attention with a decay for each head: a causal sequence mixer whose state has a fixed size, beside the long
convolutions of MonarchMixerSequenceMixing (the reference's only mixer, bert/src/mm/monarch_mixer_sequence_mixer.py:100-154).

    S_t = exp(log_decay[h]) S_{t-1} + k_t v_t^T,        o_t = scale q_t^T S_t

linear_attention() takes whole sequences (prompts, training: it has gradients), linear_attention_step() one token of each.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops


_TYPES = {torch.float32: _lib.M2_F32, torch.bfloat16: _lib.M2_BF16}


def _check(name, q, k, v, log_decay, dims):
    """(B, H, kv heads, dk, dv) of q (B, [L,] H, dk), k and v."""
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != dims or len(ks) != dims or len(vs) != dims:
        raise ValueError(f"{name}: q, k and v have {dims} dimensions, got {tuple(qs)}, {tuple(ks)} and {tuple(vs)}")
    B, (H, dk), (K, dv) = qs[0], qs[-2:], vs[-2:]
    if dk == 0 or dv == 0 or ks[:-2] != qs[:-2] or ks[-2] != K or ks[-1] != dk or vs[:-2] != qs[:-2] or K == 0 or H % K:
        raise ValueError(f"{name}: shapes {tuple(qs)}, {tuple(ks)} and {tuple(vs)} of q, k and v do not belong together")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"{name}: q, k and v are all float32 or all bfloat16, got {q.dtype}, {k.dtype} and {v.dtype}")
    if log_decay.shape != (H,):
        raise ValueError(f"{name}: log_decay has one value for each of the {H} heads, got shape {tuple(log_decay.shape)}")
    if log_decay.is_complex():
        raise TypeError(f"{name}: log_decay holds real numbers, got {log_decay.dtype}")
    dev = q.get_device()
    if dev < 0 or k.get_device() != dev or v.get_device() != dev or log_decay.get_device() != dev:
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name}: the decay is a constant of the head and has no gradient; pass log_decay.detach()")
    return B, H, K, dk, dv


def _state(name, s, what, shape, dev):
    if s.shape != shape or s.dtype != torch.float32 or s.get_device() != dev:
        raise ValueError(f"{name}: {what} is a float32 tensor {tuple(shape)} on device {dev}, got {s.dtype} {tuple(s.shape)} on {s.device}")


def _packed(t):
    """t with contiguous channels."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _decay(log_decay):
    return log_decay if log_decay.dtype == torch.float32 and log_decay.is_contiguous() else ops._f32c(log_decay)


def _args(q, k, v, log_decay, scale, initial, lengths, o=None, state=None):
    B, L, H, dk = q.shape
    K, dv = v.shape[2:]
    return _lib.LinearAttentionArgs(
        B, L, H, K, dk, dv, _TYPES[q.dtype], scale, q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3],
        log_decay.data_ptr(), lengths.data_ptr() if lengths is not None else None, initial.data_ptr() if initial is not None else None,
        o.data_ptr() if o is not None else None, state.data_ptr() if state is not None else None)


def _workspace(a, dev, backward):
    n = ops._on_device(dev.index, _lib.lib().m2_linear_attention_workspace, a.batch, a.seq_len, a.heads, a.kv_heads, a.dk, a.dv, a.dtype, backward)
    w = torch.empty(n // 4, dtype=torch.float32, device=dev) if n else None
    if w is not None:
        a.workspace, a.workspace_bytes = w.data_ptr(), n
    return w


def _forward(q, k, v, log_decay, scale, initial, lengths, want_state):
    B, L, H, dk = q.shape
    dv = v.shape[3]
    o = q.new_empty((B, L, H, dv))
    state = torch.empty((B, H, dk, dv), dtype=torch.float32, device=q.device) if want_state else None
    a = _args(q, k, v, log_decay, scale, initial, lengths, o, state)
    work = _workspace(a, q.device, 0)  # noqa: F841  (alive until the launch)
    ops._launch("m2_linear_attention_fwd", q, _lib.lib().m2_linear_attention_fwd, C.byref(a), launches=None)
    return o, state


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, initial, lengths, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, initial, lengths)
        ctx.scale = scale
        return _forward(q, k, v, log_decay, scale, initial, lengths, want_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o, d_state):
        q, k, v, log_decay, initial, lengths = ctx.saved_tensors
        B, L, H, dk = q.shape
        if d_o is None and d_state is None:
            return (None,) * 8
        d_o = torch.zeros((B, L, H, v.shape[3]), dtype=q.dtype, device=q.device) if d_o is None else _packed(d_o)
        a = _args(q, k, v, log_decay, ctx.scale, initial, lengths)
        dq, dk_, dv_ = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
        d_initial = initial.new_empty(initial.shape) if initial is not None else None
        if d_state is not None:
            d_state = d_state.contiguous()
        g = _lib.LinearAttentionGrads(d_o.data_ptr(), *d_o.stride()[:3], d_state.data_ptr() if d_state is not None else None,
                                      dq.data_ptr(), dk_.data_ptr(), dv_.data_ptr(), d_initial.data_ptr() if d_initial is not None else None)
        work = _workspace(a, q.device, 1)  # noqa: F841
        ops._launch("m2_linear_attention_bwd", q, _lib.lib().m2_linear_attention_bwd, C.byref(a), C.byref(g), launches=None)
        return dq, dk_, dv_, None, None, d_initial, None, None


def linear_attention(q, k, v, log_decay, *, scale=None, initial_state=None, lengths=None, return_state=False):
    """o (B, L, H, dv) for q (B, L, H, dk), k (B, L, K, dk), v (B, L, K, dv), all float32 or all bfloat16, any strides
    (contiguous channels are read in place); K divides H, head h reads key head h // (H // K); dk, dv <= 128.

    log_decay      (H,) float: log of the factor by which a head's state fades with every token, <= 0; a constant, not trained
    scale          default dk ** -0.5
    initial_state  None (zero) or (B, H, dk, dv) float32: what earlier calls left
    lengths        None or (B,) integers: tokens of every sequence.  What lies behind them is not read; rows of o behind them
                   are zero and the state is that behind the last token
    return_state   also return the state behind the last token, (B, H, dk, dv) float32

    Sums and states are float32, and o is rounded once.  bfloat16: operands of the tensor cores that are no bfloat16 numbers (the
    weights scale (q_i . k_j) exp(log_decay (i - j)), the copy of the state that q meets) keep 16 bits; float32 tensors have
    float32 products throughout.  Two calls give the same bits, with or without the state; those of a text go by the batch it is
    in, as a long axis is cut where sequences and heads do not fill the GPU, and the parts' sums are then added in another order.

    A NaN or an infinity in v[:, t] reaches, besides the tokens after t, outputs of up to 63 tokens before it.  An infinity in k
    or v becomes an infinity or NaN in the channels of the state that it meets, and so in later outputs.
    Differentiable in q, k, v and initial_state."""
    name = "linear_attention"
    B, H, K, dk, dv = _check(name, q, k, v, log_decay, 4)
    scale = dk ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -100 <= abs(scale) <= 2.0 ** 100:
        raise ValueError(f"{name}: scale {scale}")
    if initial_state is not None:
        _state(name, initial_state, "initial_state", (B, H, dk, dv), q.get_device())
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if lengths.shape != (B,) or lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool or lengths.device != q.device:
            raise ValueError(f"{name}: lengths are ({B},) integers on {q.device}, got {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
        lengths = lengths.to(torch.long).contiguous()
    q, k, v = _packed(q), _packed(k), _packed(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (initial_state is not None and initial_state.requires_grad)):
        o, state = _LinearAttention.apply(q, k, v, _decay(log_decay), scale, initial_state, lengths, return_state)
    else:
        o, state = _forward(q, k, v, _decay(log_decay), scale, initial_state, lengths, return_state)
    return (o, state) if return_state else o


def linear_attention_step(q, k, v, log_decay, state, *, scale=None):
    """One token of each sequence: q (B, H, dk), k (B, K, dk), v (B, K, dv) -> o (B, H, dv).  `state` (B, H, dk, dv) float32,
    its last two dimensions packed, is updated in place.  It has no gradient: linear_attention(initial_state=...) has."""
    name = "linear_attention_step"
    B, H, K, dk, dv = _check(name, q, k, v, log_decay, 3)
    _state(name, state, "state", (B, H, dk, dv), q.get_device())
    s_b, s_h, s_i, s_j = state.stride()
    size = dk * dv
    if (s_j != 1 and dv > 1) or (s_i != dv and dk > 1) or (H > 1 and s_h < size) or (B > 1 and s_b < size) or \
            (B > 1 and H > 1 and s_b < H * s_h and s_h < B * s_b):
        raise ValueError(f"{name}: state is updated in place: its last two dimensions are packed and no two heads overlap, got strides {state.stride()}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or linear_attention with initial_state")
    scale = dk ** -0.5 if scale is None else float(scale)
    if not 2.0 ** -100 <= abs(scale) <= 2.0 ** 100:
        raise ValueError(f"{name}: scale {scale}")
    q, k, v, ld = _packed(q), _packed(k), _packed(v), _decay(log_decay)
    o = q.new_empty((B, H, dv))
    a = _lib.LinearAttentionStepArgs(
        B, H, K, dk, dv, _TYPES[q.dtype], scale, q.data_ptr(), *q.stride()[:2], k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2],
        ld.data_ptr(), state.data_ptr(), s_b, s_h, o.data_ptr())
    ops._launch("m2_linear_attention_step", q, _lib.lib().m2_linear_attention_step, C.byref(a), launches=None)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return o
