"""Attention of chunks of new tokens over pages of the pools (B200, sm_100a).

* ``path_table(paths, device)``: request paths (lists of pool positions) as the
  page table of page size 1 and the sequences' lengths.
* ``chunk_attention(q, kp, vp, table, kv_lens, cu_q, ...)``: a ragged batch of
  chunks -- whole prompts, parts of prompts after a cached prefix, single tokens --
  each over its own pages of the resident ``[HK, T, D]`` pools (``ta_chunk_attention``).

``attention_matrix`` answers one token of every request of a planned tree; this
answers any number of tokens of any sequences without a plan, from tensors on the
device alone, so a captured call follows its lengths and tables.  Serving only: no
gradient is recorded.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from ._launch import DTYPES, check_pools, check_status_tensor, launch, overlap, ptr, rows16

HEAD_DIMS = (32, 64, 128)


def path_table(paths, device):
    """``(table [B, longest] int32, kv_lens [B] int32)`` of sequences given as lists of pool positions."""
    lens = np.fromiter((len(p) for p in paths), dtype=np.int32, count=len(paths))
    table = np.full((len(paths), max(1, int(lens.max(initial=0)))), -1, dtype=np.int32)
    for row, path in zip(table, paths):
        row[:len(path)] = path
    return torch.from_numpy(table).to(device), torch.from_numpy(lens).to(device)


def chunk_attention(q, kp, vp, table, kv_lens, cu_q, page_size=1, scale=None, causal=True, out=None, out_lse=None,
                    status=None):
    """Attention of ``q`` ``[N, HQ, D]`` over each sequence's pages; returns the output ``[N, HQ, D]``.

    Sequence b's queries are rows ``cu_q[b]`` to ``cu_q[b + 1]`` (``cu_q`` int32
    ``[B + 1]``, rising), its keys the first ``kv_lens[b]`` (int32 ``[B]``) of its
    pages, its new tokens' own included: key j lies at pool position
    ``table[b, j // page_size] * page_size + j % page_size`` (``table`` int32
    ``[B, W]``, rows contiguous; ``page_size`` a power of two; entries past a
    sequence's last page are not read).  Row i of n sees the keys up to its own,
    ``kv_lens[b] - n + i + 1`` of them, or all when not ``causal``.  ``scale``
    defaults to ``D ** -0.5``.

    A row without keys gets 0 and an LSE of -inf.  ``out_lse`` (``[N, HQ]``
    float32) receives the natural-log LSE.  With ``out`` given, rows behind the
    last sequence stay as they are (else they are not defined).  K and V of keys
    below ``kv_lens`` must be finite; positions past them may hold anything.
    Lengths beyond the table and positions outside the pools are recorded in
    ``status`` (int32, one element) and not followed.
    """
    if q.dim() != 3 or kp.dim() != 3:
        raise ValueError("q must be [N, HQ, D] and the pools [HK, T, D]")
    n, hq, dim = q.shape
    device, dtype = q.device, q.dtype
    if not q.is_cuda:
        raise ValueError("chunk_attention: all tensors must be CUDA tensors on one device")
    check_pools("chunk_attention", kp, vp, device)
    hk, tokens, kdim = kp.shape
    if dim not in HEAD_DIMS or kdim != dim:
        raise ValueError(f"chunk_attention: head_dim must be one of {HEAD_DIMS} and that of the pools")
    if dtype not in DTYPES or kp.dtype != dtype or vp.dtype != dtype:
        raise ValueError("q, K and V must share one dtype, bfloat16 or float16")
    if hk == 0 or hq == 0 or hq % hk:
        raise ValueError("Query heads must be divisible by KV heads")
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError("chunk_attention: page_size must be a power of two")
    b = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    if kv_lens.dtype != torch.int32 or b < 0 or cu_q.dtype != torch.int32 or cu_q.shape != (b + 1,):
        raise ValueError("chunk_attention: kv_lens must be int32 [B] and cu_q int32 [B + 1]")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != b or (table.shape[1] > 1
                                                                                  and table.stride(1) != 1):
        raise ValueError("chunk_attention: table must be int32 [B, W] with contiguous rows")
    if any(t.device != device for t in (table, kv_lens, cu_q)):
        raise ValueError("chunk_attention: all tensors must be CUDA tensors on one device")
    if scale is None:
        scale = dim ** -0.5
    elif not (scale > 0 and scale < float("inf")):
        raise ValueError("chunk_attention: scale must be positive")
    check_status_tensor("chunk_attention", status, device)
    q = rows16(q)
    kv_lens, cu_q = kv_lens.contiguous(), cu_q.contiguous()
    if out is None:
        out = torch.empty((n, hq, dim), device=device, dtype=dtype)
    elif out.shape != (n, hq, dim) or out.dtype != dtype or out.device != device or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError("chunk_attention: out must be contiguous [N, HQ, D] like q, 16-byte aligned")
    elif any(overlap(out, t) for t in (q, kp, vp)):
        raise ValueError("chunk_attention: out overlaps an input")
    if out_lse is not None and (out_lse.shape != (n, hq) or out_lse.dtype != torch.float32
                                or out_lse.device != device or not out_lse.is_contiguous()):
        raise ValueError("chunk_attention: out_lse must be contiguous float32 [N, HQ] on q's device")
    if n == 0 or b == 0:
        return out
    width = table.shape[1]
    workspace, size = None, _workspace_bytes(device, n, b, hq, hk, dim, width, page_size)
    if size:
        workspace = torch.empty(size, device=device, dtype=torch.uint8)
    launch("ta_chunk_attention", device, q.data_ptr(), q.stride(0), q.stride(1), kp.data_ptr(), vp.data_ptr(), tokens,
           table.data_ptr(), table.stride(0), width, page_size, kv_lens.data_ptr(), cu_q.data_ptr(), b, n, hq, hk, dim,
           DTYPES[dtype], scale, int(causal), out.data_ptr(), ptr(out_lse), ptr(workspace), size, ptr(status))
    return out


def _workspace_bytes(device, *sizes):
    lib = _lib.load()
    if device.index == torch.cuda.current_device():
        return lib.ta_chunk_workspace_bytes(*sizes)
    with torch.cuda.device(device.index):
        return lib.ta_chunk_workspace_bytes(*sizes)
