"""Rotary positions of q and k, fused with their norms and the append to the pools (B200, sm_100a).

* ``rotary_frequencies(rotary_dim, base, scaling, length)``: the pairs'
  frequencies and the attention factor, plain or stretched for a long context.
* ``rotary_append(q, k, v, positions, inv_freq, kp, vp, targets, ...)``: one launch
  (``ta_rotary_append``) that replaces a layer's q/k RMSNorm, rotary embedding and
  ``append_kv``: q comes back normalised and turned, k and v go into the pools.

Serving only: no gradient is recorded.
"""
from __future__ import annotations

import math

import torch

from ._launch import DTYPES, check_pools, check_status_tensor, launch, overlap, ptr, rows16

HEAD_DIMS = (32, 64, 128)


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, length=None, device=None):
    """``(inv_freq [rotary_dim / 2] float32, attention_factor)`` of a rotary embedding.

    ``inv_freq[i] = base^(-2 i / rotary_dim)``, changed for contexts beyond the
    trained one by ``scaling``, a dict with ``"type"``:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"dynamic"``: the base raised so that a context of ``length`` tokens
      (``original`` where it is shorter) turns the slowest pair as far as the
      trained context of ``original`` tokens did, ``factor`` times stretched;
    * ``"yarn"``: pairs with more than ``beta_fast`` (32) turns over ``original``
      tokens keep their frequency, those with fewer than ``beta_slow`` (1) are
      divided by ``factor``, a linear ramp over the pairs between; the attention
      factor is ``0.1 ln(factor) + 1``;
    * ``"bands"``: as ``"yarn"`` but with the ramp linear in the number of turns,
      between ``low`` and ``high`` turns, and attention factor 1.

    Computed in 64 bits, rounded once.
    """
    if rotary_dim <= 0 or rotary_dim % 2 or not base > 0:
        raise ValueError("rotary_frequencies: rotary_dim must be even and positive, base positive")
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    kind = None if scaling is None else scaling.get("type")
    attention_factor = 1.0
    if kind is None and scaling is not None:
        raise ValueError("rotary_frequencies: scaling needs a type")
    factor = 1.0 if kind is None else float(scaling["factor"])
    if not factor >= 1.0:
        raise ValueError("rotary_frequencies: factor must be at least 1")
    if kind == "dynamic":
        if rotary_dim <= 2:
            raise ValueError("rotary_frequencies: dynamic scaling wants more than one pair")
        original = scaling["original"]
        stretch = factor * max(length or original, original) / original - (factor - 1)
        base = base * stretch ** (rotary_dim / (rotary_dim - 2))
    freq = base ** -exponent
    if kind is None or kind == "dynamic":
        pass
    elif kind == "linear":
        freq = freq / factor
    elif kind == "yarn":
        fast, slow, original = scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0), scaling["original"]

        def pair_with(turns):
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_with(fast)), 0)
        high = min(math.ceil(pair_with(slow)), rotary_dim - 1)
        ramp = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        attention_factor = 0.1 * math.log(factor) + 1.0
    elif kind == "bands":
        turns = scaling["original"] * freq / (2 * math.pi)
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if not high > low:
            raise ValueError("rotary_frequencies: high must exceed low")
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    else:
        raise ValueError(f"rotary_frequencies: unknown scaling {kind!r}")
    return freq.float().to(device or "cpu"), attention_factor


def rotary_append(q, k, v, positions, inv_freq, kp, vp, targets, interleaved=False, attention_factor=1.0,
                  q_weight=None, k_weight=None, eps=1e-6, out=None, status=None, tails=None):
    """Norm and turn ``q`` and ``k``, append ``k`` and ``v`` to the pools; returns the new q ``[N, HQ, D]``.

    ``q`` ``[N, HQ, D]``, ``k`` and ``v`` ``[N, HK, D]`` (any token and head
    strides, e.g. slices of one projection), ``positions`` int64 ``[N]``,
    ``inv_freq`` float32 ``[rotary_dim / 2]`` with ``rotary_dim`` a multiple of 16
    up to ``D`` (32, 64 or 128), ``targets`` int64 pool positions ``[N]``.  Pair i
    is elements ``(i, i + rotary_dim / 2)``, or ``(2i, 2i + 1)`` when
    ``interleaved``; its angle is ``positions * inv_freq[i]``, exact for far
    positions.  ``q_weight`` / ``k_weight`` ``[D]``, where given, apply an RMSNorm
    (``eps``) over each head first.  All arithmetic is in 32 bits (angles 64),
    rounded once.

    Targets must be distinct; ``-1`` stores nothing (padding tokens), other
    positions outside the pools are skipped and recorded in ``status``.
    ``tails = (cached_plan, count, offset)`` also sets a ``CachedDecodePlan``'s tail
    lengths, as in ``append_kv``.  ``out`` may be ``q`` itself where that is
    contiguous.
    """
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError("rotary_append wants q [N, HQ, D] and k, v [N, HK, D]")
    n, hq, dim = q.shape
    hk = k.shape[1]
    device = q.device
    if not q.is_cuda:
        raise ValueError("rotary_append: all tensors must be CUDA tensors on one device")
    if dim not in HEAD_DIMS:
        raise ValueError(f"rotary_append: head_dim must be one of {HEAD_DIMS}")
    check_pools("rotary_append", kp, vp, device)
    if kp.shape[0] != hk or kp.shape[2] != dim:
        raise ValueError(f"rotary_append: pools must be [{hk}, T, {dim}], got {tuple(kp.shape)}")
    dtype = q.dtype
    if dtype not in DTYPES or any(t.dtype != dtype for t in (k, v, kp, vp)):
        raise ValueError("rotary_append: q, k, v and the pools must share one dtype, bfloat16 or float16")
    rot = 2 * inv_freq.numel()
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or rot > dim or rot % 16:
        raise ValueError("rotary_append: inv_freq must be float32 [rotary_dim / 2], rotary_dim a multiple of 16 up to D")
    for name, t in (("positions", positions), ("targets", targets)):
        if t.dtype != torch.int64 or t.shape != (n,):
            raise ValueError(f"rotary_append: {name} must be int64 [N]")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype != dtype or w.shape != (dim,)):
            raise ValueError("rotary_append: norm weights must be [D] of the inputs' dtype")
    if any(t is not None and t.device != device for t in (k, v, positions, inv_freq, targets, q_weight, k_weight, out)):
        raise ValueError("rotary_append: all tensors must be CUDA tensors on one device")
    check_status_tensor("rotary_append", status, device)
    q, k, v = rows16(q), rows16(k), rows16(v)
    positions, targets, inv_freq = positions.contiguous(), targets.contiguous(), inv_freq.contiguous()
    q_weight, k_weight = (w if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0)
                          else w.clone(memory_format=torch.contiguous_format) for w in (q_weight, k_weight))
    if out is None:
        out = torch.empty((n, hq, dim), device=device, dtype=dtype)
    else:
        if out.shape != (n, hq, dim) or out.dtype != dtype or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("rotary_append: out must be contiguous [N, HQ, D] of the inputs' dtype, 16-byte aligned")
        same = out.data_ptr() == q.data_ptr() and q.is_contiguous()
        if any(overlap(out, t) for t in (k, v, kp, vp)) or (overlap(out, q) and not same):
            raise ValueError("rotary_append: out overlaps an input")
    klen = tail_ids = count = None
    offset = num_tails = num_jobs = 0
    if tails is not None:
        cached, count_t, offset = tails
        p = cached.prepared
        if count_t.device != device or count_t.dtype != torch.int64 or count_t.numel() < 1:
            raise ValueError("rotary_append: the step count must be an int64 tensor of at least one element "
                             "on the pools' device")
        if p.klen.device != device or cached.tail_indices.device != device or cached.tail_indices.dtype != torch.int32:
            raise ValueError("rotary_append: the cached plan lives on another device than the pools")
        klen, tail_ids, count = p.klen.data_ptr(), cached.tail_indices.data_ptr(), count_t.data_ptr()
        num_tails, num_jobs = cached.tail_indices.numel(), p.layout.num_jobs
        status = p.status if status is None else status
    launch("ta_rotary_append", device, q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
           v.data_ptr(), v.stride(0), v.stride(1), positions.data_ptr(), inv_freq.data_ptr(), rot, int(interleaved),
           float(attention_factor), ptr(q_weight), ptr(k_weight), float(eps), out.data_ptr(), kp.data_ptr(),
           vp.data_ptr(), targets.data_ptr(), n, hq, hk, kp.shape[1], dim, DTYPES[dtype], klen, tail_ids, num_tails,
           count, int(offset), num_jobs, ptr(status))
    return out
