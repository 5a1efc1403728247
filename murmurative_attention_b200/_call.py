"""Shared pieces of the operators' host side: element types, devices, the C call."""
from __future__ import annotations

import ctypes

import torch

from . import _lib

DTYPES = {torch.float32: _lib.MURM_F32, torch.float16: _lib.MURM_F16, torch.bfloat16: _lib.MURM_BF16}


def dtype_code(t: torch.Tensor, name: str) -> int:
    """The C ABI's code of a CUDA tensor's dtype; other dtypes raise TypeError, CPU tensors RuntimeError."""
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"murmurative CUDA kernels require CUDA tensors; {name} is on {t.device}")
    return code


def same_device(t: torch.Tensor, dev: torch.device, name: str) -> None:
    if t.device != dev:
        raise RuntimeError(f"{name} must be on {dev}, got {t.device}")


def call(fn, args: ctypes.Structure, dev: torch.device) -> None:
    """Enqueues one C call on the current stream of ``dev``."""
    if dev.index == torch.cuda.current_device():
        _lib.check(fn(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream))
        return
    with torch.cuda.device(dev):
        _lib.check(fn(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream))
