"""One step of a beam search: the best of all (beam, token) pairs from logits, behind the decoder and beside token_logprobs, and the states of the
chosen beams (of linear_attention, selective_scan, causal_conv) moved to their places.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib, ops

MAX_BEAMS = 32
_TYPES = {torch.float32: _lib.M2_F32, torch.bfloat16: _lib.M2_BF16}


class BeamStep(NamedTuple):
    """score float32; beam, the one that is continued, and token, int64; finished, bool, or None without end_id: all (B, keep), best first."""
    score: torch.Tensor
    beam: torch.Tensor
    token: torch.Tensor
    finished: Optional[torch.Tensor]


def beam_select(logits, scores, *, keep=None, finished=None, end_id=None):
    """The `keep` (default K, at most 32) best continuations of each text by scores[b, k] + log softmax(logits[b, k])[token], for logits
    (B, K, V), float32 or bfloat16 (rows of adjacent logits are read in place, once), and scores (B, K), taken as float32; K <= 32.

    end_id    None, or the id that ends a text: `finished` of the result says which beams have ended with this token or before
    finished  None or (B, K) bool: an ended beam has one continuation, end_id at its own score; its logits are not read

    A beam's tokens go by their logits, equal ones by ascending id; beams go by the sums in 64 bits, equal ones by ascending beam.  A
    score of -inf is no candidate (a text's first step: scores 0, -inf, -inf ... where all its beams are alike); where there are fewer
    than `keep`, the rest are beam 0, token end_id (0 without it), score -inf.  NaN goes before all.  It has no gradient."""
    name = "beam_select"
    if logits.dim() != 3 or scores.shape != logits.shape[:2]:
        raise ValueError(f"{name}: logits are (B, K, V) and scores (B, K), got {tuple(logits.shape)} and {tuple(scores.shape)}")
    B, K, V = logits.shape
    if logits.dtype not in _TYPES:
        raise TypeError(f"{name}: logits are float32 or bfloat16, got {logits.dtype}")
    if not scores.is_floating_point():
        raise TypeError(f"{name}: scores are real numbers, got {scores.dtype}")
    dev = logits.get_device()
    if dev < 0 or scores.get_device() != dev or (finished is not None and finished.get_device() != dev):
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    keep = K if keep is None else int(keep)
    if V == 0 or not 1 <= K <= MAX_BEAMS or not 1 <= keep <= MAX_BEAMS:
        raise ValueError(f"{name}: {keep} of {K} beams (1 to {MAX_BEAMS} each) and {V} logits")
    if end_id is not None and not 0 <= int(end_id) < 1 << 62:
        raise ValueError(f"{name}: end_id {end_id}")
    if finished is not None:
        if end_id is None:
            raise ValueError(f"{name}: finished beams need an end_id")
        if finished.shape != (B, K) or finished.dtype != torch.bool:
            raise ValueError(f"{name}: finished is ({B}, {K}) bool, got {finished.dtype} {tuple(finished.shape)}")
        finished = finished.contiguous()
    if torch.is_grad_enabled() and (logits.requires_grad or scores.requires_grad):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad(), or pass detached tensors")
    ops._no_tangents(name, logits, scores)
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    scores = (scores if scores.dtype == torch.float32 else scores.float()).contiguous()
    score = scores.new_empty((B, keep))
    beam, token = (torch.empty((B, keep), dtype=torch.long, device=logits.device) for _ in range(2))
    done = torch.empty((B, keep), dtype=torch.bool, device=logits.device) if end_id is not None else None
    size = _lib.lib().m2_beam_select_workspace(B, K, V, keep)
    work = torch.empty(size, dtype=torch.uint8, device=logits.device)
    a = _lib.BeamSelectArgs(B, K, V, keep, _TYPES[logits.dtype], logits.data_ptr(), *logits.stride()[:2], scores.data_ptr(),
                            finished.data_ptr() if finished is not None else None, -1 if end_id is None else int(end_id), score.data_ptr(), beam.data_ptr(),
                            token.data_ptr(), done.data_ptr() if done is not None else None, work.data_ptr(), size)
    ops._launch("m2_beam_select", logits, _lib.lib().m2_beam_select, C.byref(a), launches=None)
    return BeamStep(score, beam, token, done)


def _apart(states, rows):
    """Whether no element belongs to two of the states, each (pointer, bytes of a row, distance of rows), of `rows` rows."""
    order, last = sorted(states), 0
    for p, row, step in order:
        if p < last and row:
            break
        last = p + step * (rows - 1) + row if row else last
    else:
        return True                                            # one behind the other
    order = [s for s in order if s[1]]
    ends = [p + step * (rows - 1) + row for p, row, step in order]
    for i, (p, row, step) in enumerate(order):
        for q, row2, step2 in order[i + 1:]:
            if q >= ends[i]:
                break
            at = (q - p) % step                                # rows of one cache, side by side
            if step != step2 or at < row or at + row2 > step:
                return False
    return True


def reorder_states(states, beam):
    """In each tensor of `states`, (B * K, ...), row b K + k becomes what row b K + beam[b, k] was, in place and in one launch for all that are
    laid out alike; beam (B, K) int64 as beam_select gives it, K <= 32.  Every row is packed; rows of one tensor lie a fixed distance
    apart, and share no memory with beam.  An entry of beam outside 0 .. K-1 is clamped and sets M2_DEV_BAD_INDEX (ops.device_status())."""
    name = "reorder_states"
    states = [states] if isinstance(states, torch.Tensor) else list(states)
    if beam.dim() != 2 or beam.dtype != torch.long:
        raise ValueError(f"{name}: beam is (B, K) int64, got {beam.dtype} {tuple(beam.shape)}")
    B, K = beam.shape
    if not 1 <= K <= MAX_BEAMS:
        raise ValueError(f"{name}: {K} beams (1 to {MAX_BEAMS})")
    dev = beam.get_device()
    if dev < 0 or [s for s in states if s.get_device() != dev]:
        raise RuntimeError(f"{name}: m2_b200 kernels need CUDA tensors of one device; there is no CPU fallback")
    ops._no_tangents(name, *states)
    rows, numbers, grad = B * K, [], torch.is_grad_enabled()
    for s in states:
        if s.dim() < 1 or s.shape[0] != rows:
            raise ValueError(f"{name}: states have B * K = {rows} rows, got {tuple(s.shape)}")
        if grad and s.requires_grad:
            raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")
        if rows == 0:
            continue
        n = s.nbytes // rows
        if s.is_contiguous():
            numbers.append((s.data_ptr(), n, n))
            continue
        step = s.stride(0) * s.element_size()
        if not s[0].is_contiguous() or (rows > 1 and step < n):
            raise ValueError(f"{name}: a state is changed in place: its rows are packed and do not overlap, got {tuple(s.shape)} with strides {s.stride()}")
        numbers.append((s.data_ptr(), n, step if rows > 1 else n))
    beam = beam.contiguous()
    if not _apart(numbers + [(beam.data_ptr(), 8, 8)] if rows else [], rows):        # beam is read while states are written
        raise ValueError(f"{name}: two states, or a state and beam, share memory")
    if not numbers:
        return
    table = (_lib.BeamState * len(numbers))(*numbers)
    a = _lib.ReorderStatesArgs(B, K, len(numbers), beam.data_ptr(), table)
    ops._launch("m2_reorder_states", beam, _lib.lib().m2_reorder_states, C.byref(a), launches=None)
    torch.autograd.graph.increment_version([s for s in states if not s.is_inference()])
