"""Beam search: the best continuations over beams x vocabulary, and the beams' states after them (B200, sm_100a).

* ``beam_select(logits, scores, k, finished, end_token)``: per request the ``k``
  best of ``scores[w] + log_softmax(logits[w])`` over its beams and the vocabulary
  (``ta_beam_select``).
* ``beam_reorder(states, parents)``: each kept beam's row of a state tensor, taken
  from its parent (``ta_beam_reorder``).
"""
from __future__ import annotations

import torch

from . import _lib
from ._launch import DTYPES, check_status_tensor, launch, overlap, ptr

MAX_BEAMS = MAX_K = 32
_LOGITS = {**DTYPES, torch.float32: _lib.DTYPE_F32}


def beam_select(logits, scores, k=None, finished=None, end_token=-1):
    """``(scores, parents, tokens)``, each ``[R, k]``: every request's best candidates, best first.

    ``logits`` ``[R, W, V]`` or ``[R * W, V]`` (bfloat16, float16 or float32),
    ``scores`` ``[R, W]`` float32.  Candidate (w, t) scores ``scores[r, w] +
    logits[r, w, t] - logsumexp(logits[r, w])``; ``parents`` (w) and ``tokens`` (t)
    are int64, ties go to the lowest ``w * V + t``.  Scores are compared in 64
    bits and returned in 32.  ``k`` defaults to W.  A beam marked in ``finished``
    (bool ``[R, W]``) offers ``end_token`` alone, at its unchanged score.  A beam
    score of -inf (an unused beam) and a logit of -inf (a token ruled out) leave
    candidates at -inf, which come last; a NaN logit counts as -inf, one
    above 131072 (+inf) as that.  Up to 32
    beams and candidates.
    """
    if scores.dim() != 2 or scores.dtype != torch.float32:
        raise ValueError("beam_select: scores must be float32 [R, W]")
    r, w = scores.shape
    if logits.dim() not in (2, 3) or logits.shape[:-1].numel() != r * w or \
            (logits.dim() == 3 and logits.shape[:2] != (r, w)):
        raise ValueError("beam_select: logits must be [R, W, V] or [R * W, V]")
    vocab = logits.shape[-1]
    device = logits.device
    if not logits.is_cuda or scores.device != device or (finished is not None and finished.device != device):
        raise ValueError("beam_select: all tensors must be CUDA tensors on one device")
    if logits.dtype not in _LOGITS:
        raise ValueError("beam_select: logits must be bfloat16, float16 or float32")
    k = w if k is None else k
    if not 1 <= w <= MAX_BEAMS or not 1 <= k <= MAX_K or vocab < 1 or k > w * vocab:
        raise ValueError(f"beam_select: 1 to {MAX_BEAMS} beams, k from 1 to {MAX_K} and at most W * V")
    if finished is not None:
        if finished.dtype != torch.bool or finished.shape != (r, w):
            raise ValueError("beam_select: finished must be bool [R, W]")
        if not 0 <= end_token < vocab:
            raise ValueError("beam_select: finished beams need an end_token within the vocabulary")
        finished = finished.contiguous()
    if logits.dim() == 3:
        if r > 1 and logits.stride(0) != w * logits.stride(1):
            logits = logits.contiguous()
        stride = logits.stride(1)
        if w == 1 and r > 1:
            stride = logits.stride(0)
    else:
        stride = logits.stride(0)
    if vocab > 1 and logits.stride(-1) != 1:
        logits, stride = logits.contiguous(), vocab
    scores = scores.contiguous()
    best = torch.empty((r, k), device=device, dtype=torch.float32)
    chosen = torch.empty((2, r, k), device=device, dtype=torch.int64)
    parents, tokens = chosen[0], chosen[1]
    if r == 0:
        return best, parents, tokens
    dtype = _LOGITS[logits.dtype]
    size = _lib.load().ta_beam_workspace_bytes(r, w, vocab, k, dtype)
    workspace = torch.empty(size, device=device, dtype=torch.uint8)
    launch("ta_beam_select", device, logits.data_ptr(), stride, scores.data_ptr(), ptr(finished), r, w, vocab, k,
           end_token, dtype, best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), workspace.data_ptr(), size)
    return best, parents, tokens


def beam_reorder(states, parents, out=None, status=None):
    """``out[r, i] = states[r, parents[r, i]]``: the kept beams' rows of a state tensor ``[R, W, ...]``.

    ``parents`` int64 ``[R, K]`` (any request stride) with values in ``[0, W)``;
    ``out`` ``[R, K, ...]`` contiguous, of ``states``' dtype, must not overlap
    ``states``.  A parent outside the beams leaves its row as it is and is
    recorded in ``status`` (int32, one element).
    """
    if states.dim() < 2 or parents.dim() != 2 or parents.shape[0] != states.shape[0]:
        raise ValueError("beam_reorder wants states [R, W, ...] and parents [R, K]")
    if parents.dtype != torch.int64:
        raise ValueError("beam_reorder: parents must be int64")
    device = states.device
    if not states.is_cuda or parents.device != device or (out is not None and out.device != device):
        raise ValueError("beam_reorder: all tensors must be CUDA tensors on one device")
    check_status_tensor("beam_reorder", status, device)
    r, w = states.shape[:2]
    kept = parents.shape[1]
    if w == 0 and r * kept:
        raise ValueError("beam_reorder: no beams to take rows from")
    if not states[:1, :1].is_contiguous():                # the rows themselves
        states = states.contiguous()
    if kept > 1 and parents.stride(1) != 1:
        parents = parents.contiguous()
    shape = (r, kept, *states.shape[2:])
    if out is None:
        out = torch.empty(shape, device=device, dtype=states.dtype)
    elif out.shape != shape or out.dtype != states.dtype or not out.is_contiguous():
        raise ValueError("beam_reorder: out must be contiguous [R, K, ...] of the states' dtype")
    elif overlap(out, states) or overlap(out, parents):
        raise ValueError("beam_reorder: out overlaps an input")
    if out.numel() == 0:
        return out
    size = states.element_size()
    row_bytes = out[0, 0].numel() * size
    launch("ta_beam_reorder", device, states.data_ptr(), states.stride(0) * size, states.stride(1) * size, r, w,
           row_bytes, parents.data_ptr(), parents.stride(0), kept, out.data_ptr(), ptr(status))
    return out
