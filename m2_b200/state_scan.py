"""Selective state space scan: a causal sequence mixer whose channels have states of a fixed size, faded and fed by the token itself; beside
linear_attention and the long convolutions of MonarchMixerSequenceMixing (the reference's only mixer, bert/src/mm/monarch_mixer_sequence_mixer.py:100-154).

    s_t = softplus(delta_t + delta_bias),      h_t[d, n] = exp(s_t[d] a[d, n]) h_{t-1}[d, n] + s_t[d] x_t[d] b_t[n],
    y_t[d] = (sum_n c_t[n] h_t[d, n] + skip[d] x_t[d]) silu(gate_t[d])

selective_scan() takes whole sequences (prompts, training: it has gradients), selective_scan_step() one token of each.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .linear_attn import _state
from .short_conv import _TYPES, _lengths, _packed, _ptr, _vector

MAX_STATES = 64


def _check(name, x, delta, a, b, c, skip, gate, delta_bias, dims):
    """b and c as (B, [L,] G, N), and the parameters as packed float32."""
    if x.dim() != dims or delta.shape != x.shape or (gate is not None and gate.shape != x.shape):
        raise ValueError(f"{name}: x, delta and gate have one shape of {dims} dimensions, got {tuple(x.shape)}, {tuple(delta.shape)}"
                         f"{'' if gate is None else f' and {tuple(gate.shape)}'}")
    D = x.shape[-1]
    if a.dim() != 2 or a.shape[0] != D or D == 0 or not 1 <= a.shape[1] <= MAX_STATES:
        raise ValueError(f"{name}: a is ({D}, N) with 1 to {MAX_STATES} states, got {tuple(a.shape)}")
    N = a.shape[1]
    if b.shape != c.shape or b.dim() not in (dims, dims + 1) or b.shape[:dims - 1] != x.shape[:-1] or b.shape[-1] != N:
        raise ValueError(f"{name}: b and c are {(*x.shape[:-1], N)} or {(*x.shape[:-1], 'G', N)}, got {tuple(b.shape)} and {tuple(c.shape)}")
    if b.dim() == dims:
        b, c = b.unsqueeze(-2), c.unsqueeze(-2)
    G = b.shape[-2]
    if G == 0 or D % G:
        raise ValueError(f"{name}: {G} groups of b and c do not divide {D} channels")
    dtype, dev = x.dtype, x.get_device()
    if dtype not in _TYPES or delta.dtype != dtype or b.dtype != dtype or c.dtype != dtype or (gate is not None and gate.dtype != dtype):
        raise TypeError(f"{name}: x, delta, b, c and gate are all float32 or all bfloat16, got {dtype}, {delta.dtype}, {b.dtype}, {c.dtype}"
                        f"{'' if gate is None else f' and {gate.dtype}'}")
    if dev < 0 or a.get_device() != dev or delta.get_device() != dev or b.get_device() != dev or c.get_device() != dev or \
            (gate is not None and gate.get_device() != dev):
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    return (b, c, _vector(name, "a", a, (D, N), dev), _vector(name, "skip", skip, (D,), dev) if skip is not None else None,
            _vector(name, "delta_bias", delta_bias, (D,), dev) if delta_bias is not None else None)


def _wants_gradient(tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _two(t):
    return t.stride()[:2] if t is not None else (0, 0)


def _args(x, delta, a, b, c, skip, gate, bias, softplus, initial, lengths, y=None, state=None):
    B, L, D = x.shape
    return _lib.SelectiveScanArgs(
        B, L, D, a.shape[1], b.shape[2], softplus, _TYPES[x.dtype], x.data_ptr(), *_two(x), delta.data_ptr(), *_two(delta), _ptr(gate), *_two(gate),
        b.data_ptr(), *b.stride()[:3], c.data_ptr(), *c.stride()[:3], a.data_ptr(), _ptr(skip), _ptr(bias), _ptr(lengths), _ptr(initial), _ptr(y), _ptr(state))


def _workspace(a, dev, backward):
    n = ops._on_device(dev.index, _lib.lib().m2_selective_scan_workspace, a.batch, a.seq_len, a.dim, a.states, a.groups, backward)
    w = torch.empty(n // 4, dtype=torch.float32, device=dev) if n else None
    if w is not None:
        a.workspace, a.workspace_bytes = w.data_ptr(), n
    return w


def _saves(a, saves):
    a.saves, a.saves_bytes = saves.data_ptr(), saves.numel() * 4


def _forward(x, delta, a, b, c, skip, gate, bias, softplus, initial, lengths, want_state, train):
    B, L, D = x.shape
    y = x.new_empty(x.shape)
    state = torch.empty((B, D, a.shape[1]), dtype=torch.float32, device=x.device) if want_state else None
    args = _args(x, delta, a, b, c, skip, gate, bias, softplus, initial, lengths, y, state)
    saves = None
    if train:
        n = ops._on_device(x.get_device(), _lib.lib().m2_selective_scan_saves, B, L, D, a.shape[1], b.shape[2])
        saves = torch.empty(n // 4, dtype=torch.float32, device=x.device)
        _saves(args, saves)
    work = _workspace(args, x.device, 0)  # noqa: F841  (alive until the launch)
    ops._launch("m2_selective_scan_fwd", x, _lib.lib().m2_selective_scan_fwd, C.byref(args), launches=None)
    return y, state, saves


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, a, b, c, skip, gate, bias, initial, softplus, lengths, want_state):
        ctx.set_materialize_grads(False)
        y, state, saves = _forward(x, delta, a, b, c, skip, gate, bias, softplus, initial, lengths, want_state, True)
        ctx.save_for_backward(x, delta, a, b, c, skip, gate, bias, initial, lengths, saves)
        ctx.softplus = softplus
        return y, state

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y, d_state):
        x, delta, a, b, c, skip, gate, bias, initial, lengths, saves = ctx.saved_tensors
        if d_y is None and d_state is None:
            return (None,) * 12
        d_y = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if d_y is None else _packed(d_y)
        d_state = d_state.contiguous() if d_state is not None else None
        want = ctx.needs_input_grad
        full = [t.new_empty(t.shape) if t is not None else None for t in (x, delta, gate, b, c)]
        own = [t.new_empty(t.shape) if w and t is not None else None for t, w in ((a, want[2]), (skip, want[5]), (bias, want[7]), (initial, want[8]))]
        if x.shape[0] == 0:
            own = [t.zero_() if t is not None else None for t in own]
        else:
            args = _args(x, delta, a, b, c, skip, gate, bias, ctx.softplus, initial, lengths)
            _saves(args, saves)
            work = _workspace(args, x.device, 1)  # noqa: F841
            g = _lib.SelectiveScanGrads(d_y.data_ptr(), *_two(d_y), _ptr(d_state), *(_ptr(t) for t in full), *(_ptr(t) for t in own))
            ops._launch("m2_selective_scan_bwd", x, _lib.lib().m2_selective_scan_bwd, C.byref(args), C.byref(g), launches=None)
        d_x, d_delta, d_gate, d_b, d_c = full
        d_a, d_skip, d_bias, d_initial = own
        return d_x, d_delta, d_a, d_b, d_c, d_skip, d_gate, d_bias, d_initial, None, None, None


def selective_scan(x, delta, a, b, c, *, skip=None, gate=None, delta_bias=None, softplus=False, initial_state=None, lengths=None, return_state=False):
    """y (B, L, D) for x, delta (B, L, D) and b, c (B, L, N) or (B, L, G, N), all float32 or all bfloat16, any strides (contiguous channels and
    states are read in place); channel d reads group d // (D // G), N <= 64.

    a              (D, N) float: exp(s a) fades a state with every token; < 0 for states that do not grow.  An infinity counts as float32's
                   largest number, so that a step of 0 changes nothing
    skip           None or (D,): x's own share of y;   gate  None or x's shape and type: y is multiplied by silu(gate)
    delta_bias     None or (D,), added to delta;       softplus  whether the step s is softplus of that sum, or the sum itself
    initial_state  None (zero) or (B, D, N) float32: what earlier calls left
    lengths        None or (B,) integers: tokens of every sequence.  What lies behind them is not read; rows of y behind them
                   are zero and the state is that behind the last token
    return_state   also return the state behind the last token, (B, D, N) float32

    Steps, states and sums are float32, y is rounded once.  Two calls give the same bits; those of a text go by the batch it is in, as a long
    axis is cut where sequences and channels do not fill the GPU.  Differentiable in every tensor but lengths; for the gradient the state is kept
    every 32 tokens in float32."""
    name = "selective_scan"
    b, c, a, skip, delta_bias = _check(name, x, delta, a, b, c, skip, gate, delta_bias, 3)
    B, L, D = x.shape
    if initial_state is not None:
        _state(name, initial_state, "initial_state", (B, D, a.shape[1]), x.get_device())
        initial_state = initial_state.contiguous()
    lengths = _lengths(name, lengths, B, x)
    x, delta, b, c, gate = _packed(x), _packed(delta), _packed(b), _packed(c), _packed(gate) if gate is not None else None
    tensors = (x, delta, a, b, c, skip, gate, delta_bias, initial_state)
    ops._no_tangents(name, *tensors)
    if _wants_gradient(tensors):
        y, state = _SelectiveScan.apply(*tensors, bool(softplus), lengths, return_state)
    else:
        y, state, _ = _forward(*tensors[:8], bool(softplus), initial_state, lengths, return_state, False)
    return (y, state) if return_state else y


def selective_scan_step(x, delta, a, b, c, state, *, skip=None, gate=None, delta_bias=None, softplus=False):
    """One token of each sequence: x, delta, gate (B, D), b, c (B, N) or (B, G, N) -> y (B, D).  `state` (B, D, N) float32, its last two
    dimensions packed, is updated in place.  It has no gradient: selective_scan(initial_state=...) has."""
    name = "selective_scan_step"
    b, c, a, skip, delta_bias = _check(name, x, delta, a, b, c, skip, gate, delta_bias, 2)
    (B, D), N = x.shape, a.shape[1]
    _state(name, state, "state", (B, D, N), x.get_device())
    s_b, s_d, s_n = state.stride()
    if (s_n != 1 and N > 1) or (s_d != N and D > 1) or (B > 1 and s_b < D * N):
        raise ValueError(f"{name}: state is updated in place: its last two dimensions are packed and no two sequences overlap, got strides {state.stride()}")
    if _wants_gradient((x, delta, a, b, c, skip, gate, delta_bias, state)):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or selective_scan with initial_state")
    ops._no_tangents(name, x, delta, a, b, c, skip, gate, delta_bias, state)
    x, delta, b, c, gate = _packed(x), _packed(delta), _packed(b), _packed(c), _packed(gate) if gate is not None else None
    y = x.new_empty((B, D))
    args = _lib.SelectiveScanStepArgs(
        B, D, N, b.shape[1], bool(softplus), _TYPES[x.dtype], x.data_ptr(), x.stride(0), delta.data_ptr(), delta.stride(0), _ptr(gate),
        gate.stride(0) if gate is not None else 0, b.data_ptr(), *b.stride()[:2], c.data_ptr(), *c.stride()[:2], a.data_ptr(), _ptr(skip), _ptr(delta_bias),
        state.data_ptr(), s_b, y.data_ptr())
    ops._launch("m2_selective_scan_step", x, _lib.lib().m2_selective_scan_step, C.byref(args), launches=None)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return y
