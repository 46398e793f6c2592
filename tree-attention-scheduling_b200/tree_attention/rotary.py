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

from ._lib import ops


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
    klen = tail_ids = count = None
    offset = num_jobs = 0
    if tails is not None:
        cached, count, offset = tails
        p = cached.prepared
        klen, tail_ids, num_jobs = p.klen, cached.tail_indices, p.layout.num_jobs
        status = p.status if status is None else status
    return ops().rotary_append(q, k, v, positions, inv_freq, kp, vp, targets, interleaved, attention_factor, q_weight,
                               k_weight, eps, out, status, klen, tail_ids, count, offset, num_jobs)
