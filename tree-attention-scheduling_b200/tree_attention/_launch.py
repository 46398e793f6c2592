"""Shared pieces of the kernel entry points: dtype codes, row layout, aliasing and the launch itself."""
from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def launch(name, device, *args):
    """Call the library's ``name`` with ``args`` and the current stream of ``device``; raise on an error code.

    The launch goes to ``device`` whatever the current device is.
    """
    fn = getattr(_lib.load(), name)
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch.cuda.current_stream(index).cuda_stream)
    if rc:
        _lib.check(rc, name)


def rows16(x):
    """``x`` ``[N, H, D]`` itself where its rows can be read in 16-byte pieces, else a contiguous copy."""
    st, sh, sd = x.stride()
    if sd != 1 or st % 8 or sh % 8 or x.data_ptr() % 16:
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _span(x):
    """Byte range ``[first, end)`` that ``x``'s elements lie in."""
    last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
    return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()


def overlap(a, b):
    """Whether the memory ranges of two tensors of one device meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def check_pools(what, kp, vp, device):
    """The resident ``[HK, T, D]`` pools as every operator on them wants them."""
    if kp.dim() != 3 or vp.shape != kp.shape or not (kp.is_contiguous() and vp.is_contiguous()):
        raise ValueError(f"{what} wants contiguous [HK, T, D] pools of one shape")
    if kp.device != device or vp.device != device:
        raise ValueError(f"{what}: all tensors must be CUDA tensors on one device")
    if kp.data_ptr() % 16 or vp.data_ptr() % 16:
        raise ValueError(f"{what}: the pools must be 16-byte aligned")


def check_status_tensor(what, status, device):
    if status is not None and (status.device != device or status.dtype != torch.int32 or status.numel() < 1):
        raise ValueError(f"{what}: status must be an int32 CUDA tensor on the pools' device")


def ptr(x):
    return None if x is None else x.data_ptr()
