"""Short causal convolution of every channel with its own taps, in front of a selective scan: beside the short convolution inside the reference's mixer
(bert/src/mm/monarch_mixer_sequence_mixer.py:118-121), which has three taps around a token.

    v_t = bias + sum_i weight[d, i] x_{t - W + 1 + i},        y_t = v_t or silu(v_t)

causal_conv() takes whole sequences (prompts, training: it has gradients), causal_conv_step() one token of each.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops

MAX_TAPS = 8
_TYPES = {torch.float32: _lib.M2_F32, torch.bfloat16: _lib.M2_BF16}


def _packed(t):
    """t with contiguous channels."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _vector(name, what, t, shape, dev):
    """t, a parameter of this shape, as packed float32."""
    if t.shape != shape or t.get_device() != dev or not t.is_floating_point():
        raise ValueError(f"{name}: {what} is {tuple(shape)} on device {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if t.dtype != torch.float32:
        t = t.float()
    return t if t.is_contiguous() else t.contiguous()


def _lengths(name, lengths, B, like):
    if lengths is None:
        return None
    if lengths.shape != (B,) or lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool or lengths.device != like.device:
        raise ValueError(f"{name}: lengths are ({B},) integers on {like.device}, got {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
    return lengths.to(torch.long).contiguous()


def _check(name, x, weight, bias, activation, dims):
    if x.dim() != dims or weight.dim() != 2 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"{name}: x has {dims} dimensions and weight is (D, W), got {tuple(x.shape)} and {tuple(weight.shape)}")
    D, W = weight.shape
    if D == 0 or not 1 <= W <= MAX_TAPS:
        raise ValueError(f"{name}: {D} channels, {W} taps (1 to {MAX_TAPS})")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name}: x is float32 or bfloat16, got {x.dtype}")
    if activation not in (None, "silu"):
        raise ValueError(f"{name}: activation {activation!r} (None or 'silu')")
    dev = x.get_device()
    if dev < 0 or weight.get_device() != dev:
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    return _vector(name, "weight", weight, (D, W), dev), _vector(name, "bias", bias, (D,), dev) if bias is not None else None


def _args(x, weight, bias, silu, state, lengths, y=None, state_out=None):
    B, L, D = x.shape
    return _lib.CausalConvArgs(B, L, D, weight.shape[1], silu, _TYPES[x.dtype], x.data_ptr(), *x.stride()[:2], weight.data_ptr(), _ptr(bias),
                               _ptr(lengths), _ptr(state), _ptr(y), _ptr(state_out))


def _forward(x, weight, bias, silu, state, lengths, want_state):
    y = x.new_empty(x.shape)
    state_out = x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2])) if want_state else None
    a = _args(x, weight, bias, silu, state, lengths, y, state_out)
    ops._launch("m2_causal_conv_fwd", x, _lib.lib().m2_causal_conv_fwd, C.byref(a), launches=None)
    return y, state_out


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, silu, lengths, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu = silu
        return _forward(x, weight, bias, silu, state, lengths, want_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y, d_state):
        x, weight, bias, state, lengths = ctx.saved_tensors
        if d_y is None and d_state is None:
            return (None,) * 7
        B, L, D = x.shape
        d_y = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if d_y is None else _packed(d_y)
        d_state = d_state.contiguous() if d_state is not None else None
        want = ctx.needs_input_grad
        d_x = x.new_empty(x.shape)
        d_w = weight.new_empty(weight.shape) if want[1] else None
        d_b = bias.new_empty(bias.shape) if bias is not None and want[2] else None
        d_before = state.new_empty(state.shape) if state is not None and want[3] else None
        if B == 0:
            return d_x, *(t.zero_() if t is not None else None for t in (d_w, d_b)), d_before, None, None, None
        a = _args(x, weight, bias, ctx.silu, state, lengths)
        size = ops._on_device(x.get_device(), _lib.lib().m2_causal_conv_workspace, B, L, D, weight.shape[1])
        work = torch.empty(size // 4, dtype=torch.float32, device=x.device)
        g = _lib.CausalConvGrads(d_y.data_ptr(), *d_y.stride()[:2], _ptr(d_state), d_x.data_ptr(), _ptr(d_before), _ptr(d_w), _ptr(d_b), work.data_ptr(), size)
        ops._launch("m2_causal_conv_bwd", x, _lib.lib().m2_causal_conv_bwd, C.byref(a), C.byref(g), launches=None)
        return d_x, d_w, d_b, d_before, None, None, None


def causal_conv(x, weight, bias=None, *, activation=None, initial_state=None, lengths=None, return_state=False):
    """y (B, L, D) for x (B, L, D), float32 or bfloat16, any strides (contiguous channels are read in place).

    weight         (D, W), W <= 8 taps, the last of which meets the token itself; bias None or (D,)
    activation     None or "silu"
    initial_state  None (zeros) or (B, W - 1, D) of x's type, oldest first: the inputs in front of x, what earlier calls left
    lengths        None or (B,) integers: tokens of every sequence.  What lies behind them is not read, and y is zero there
    return_state   also return the last W - 1 inputs of every sequence (those of initial_state among them where it is shorter)

    Products and sums are float32, y is rounded once.  Differentiable in x, weight, bias and initial_state; two runs give the same bits."""
    name = "causal_conv"
    weight, bias = _check(name, x, weight, bias, activation, 3)
    B, L, D = x.shape
    W = weight.shape[1]
    if initial_state is not None:
        if initial_state.shape != (B, W - 1, D) or initial_state.dtype != x.dtype or initial_state.device != x.device:
            raise ValueError(f"{name}: initial_state is {x.dtype} {(B, W - 1, D)} on {x.device}, got {initial_state.dtype} {tuple(initial_state.shape)} on {initial_state.device}")
        initial_state = initial_state.contiguous()
    lengths = _lengths(name, lengths, B, x)
    ops._no_tangents(name, x, weight, bias, initial_state)
    x = _packed(x)
    silu = activation is not None
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (initial_state is not None and initial_state.requires_grad)):
        y, state = _CausalConv.apply(x, weight, bias, initial_state, silu, lengths, return_state)
    else:
        y, state = _forward(x, weight, bias, silu, initial_state, lengths, return_state)
    return (y, state) if return_state else y


def causal_conv_step(x, state, weight, bias=None, *, activation=None):
    """One token of each sequence: x (B, D) -> y (B, D).  `state` (B, W - 1, D) of x's type, its last two dimensions packed, loses its oldest
    input and takes x, in place.  It has no gradient: causal_conv(initial_state=...) has."""
    name = "causal_conv_step"
    weight, bias = _check(name, x, weight, bias, activation, 2)
    (B, D), W = x.shape, weight.shape[1]
    if state.shape != (B, W - 1, D) or state.dtype != x.dtype or state.device != x.device:
        raise ValueError(f"{name}: state is {x.dtype} {(B, W - 1, D)} on {x.device}, got {state.dtype} {tuple(state.shape)} on {state.device}")
    s_b, s_i, s_d = state.stride()
    if W > 1 and ((s_d != 1 and D > 1) or (s_i != D and W > 2) or (B > 1 and s_b < (W - 1) * D)):
        raise ValueError(f"{name}: state is updated in place: its last two dimensions are packed and no two sequences overlap, got strides {state.stride()}")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or state.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or causal_conv with initial_state")
    ops._no_tangents(name, x, state, weight, bias)
    x = _packed(x)
    y = x.new_empty((B, D))
    a = _lib.CausalConvStepArgs(B, D, W, activation is not None, _TYPES[x.dtype], x.data_ptr(), x.stride(0), weight.data_ptr(), _ptr(bias), state.data_ptr(), s_b,
                                y.data_ptr())
    ops._launch("m2_causal_conv_step", x, _lib.lib().m2_causal_conv_step, C.byref(a), launches=None)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return y
