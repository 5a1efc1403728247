"""Linear layer with bias, activation and residual in the matrix product's epilogue.

``fused_linear`` is a block's projections and feed-forward products around ``slot_murmurate``:
``act(x W^T + b) + residual`` without a pass over memory for anything but the product. The
compute is ``murm_linear_fwd`` / ``_bwd`` (murm_linear.cu, murm_gemm.cu).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._call import call, dtype_code, same_device

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor the C ABI reads in place: unit inner stride, rows that do not overlap."""
    ok = (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] == 1 or t.stride(0) >= t.shape[1])
    return t if ok else t.contiguous()


def _stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _workspace(fn, args, dev) -> Optional[torch.Tensor]:
    n = ctypes.c_size_t()
    _lib.check(fn(ctypes.byref(args), ctypes.byref(n)))
    if not n.value:
        return None
    ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), n.value
    return ws


def _forward(x, weight, bias, residual, act, save):
    """x [M, K], weight [N, K], residual [M, N] -> (out [M, N], slope or None)."""
    lib = _lib.load_library()
    x, weight = _rows(x), _rows(weight)
    M, K = x.shape
    N = weight.shape[0]
    out = torch.empty(M, N, dtype=x.dtype, device=x.device)
    slope = torch.empty_like(out) if save and act else None
    if not out.numel():
        return out, slope
    if bias is not None:
        bias = bias.contiguous()
    a = _lib.LinearArgs(M, K, N, dtype_code(x, "x"), act, x.data_ptr(), _stride(x), weight.data_ptr(),
                        _stride(weight), bias.data_ptr() if bias is not None else None)
    if residual is not None:
        residual = _rows(residual)
        a.residual, a.r_stride = residual.data_ptr(), _stride(residual)
    a.out, a.out_stride = out.data_ptr(), N
    if slope is not None:
        a.slope = slope.data_ptr()
    ws = _workspace(lib.murm_linear_workspace, a, x.device)  # noqa: F841  (alive until the call is enqueued)
    call(lib.murm_linear_fwd, a, x.device)
    return out, slope


def _backward(x, weight, slope, go, act, need_x, need_w, need_b):
    lib = _lib.load_library()
    x, weight, go = _rows(x), _rows(weight), _rows(go.to(x.dtype))
    M, K = x.shape
    N = weight.shape[0]
    dev = x.device
    gx = torch.empty(M, K, dtype=x.dtype, device=dev) if need_x else None
    gw = torch.empty(N, K, dtype=x.dtype, device=dev) if need_w else None
    gb = torch.empty(N, dtype=x.dtype, device=dev) if need_b else None
    ptr = lambda t: t.data_ptr() if t is not None else None
    a = _lib.LinearBwdArgs(M, K, N, dtype_code(x, "x"), act, x.data_ptr(), _stride(x), weight.data_ptr(),
                           _stride(weight), ptr(slope), go.data_ptr(), _stride(go), ptr(gx), K, ptr(gw), K, ptr(gb))
    ws = _workspace(lib.murm_linear_bwd_workspace, a, dev)  # noqa: F841
    call(lib.murm_linear_bwd, a, dev)
    return gx, gw, gb


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        out, slope = _forward(x, weight, bias, residual, act, True)
        ctx.save_for_backward(x, weight, slope)
        ctx.act = act
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go):
        x, weight, slope = ctx.saved_tensors
        need = ctx.needs_input_grad
        gx = gw = gb = None
        if need[0] or need[1] or need[2]:
            gx, gw, gb = _backward(x, weight, slope, go, ctx.act, need[0], need[1], need[2])
        return gx, gw, gb, go if need[3] else None, None


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 activation: str = "none", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x W^T + bias) + residual.

    Args:
        x: [..., K]; weight: [N, K]; bias: [N]; residual: broadcastable to [..., N]. One dtype: fp16,
           bf16 or fp32 (fp32 products keep fp32 accuracy). Any strides; rows with a unit inner
           stride are read in place.
        activation: "none", "relu", "silu", "gelu" (error function) or "gelu_tanh".

    Returns [..., N]. Differentiable with respect to x, weight, bias and residual; the backward reads
    x, weight and the activation's slopes, which the forward saves in x's dtype (not for "none").
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    dtype_code(x, "x")
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise RuntimeError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if N < 1 or K < 1:
        raise RuntimeError(f"weight must not be empty, got {tuple(weight.shape)}")
    dev, dt = x.device, x.dtype
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is None:
            continue
        if t.dtype != dt:
            raise TypeError(f"{name} must have x's dtype {dt}, got {t.dtype}")
        same_device(t, dev, name)
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != N):
        raise RuntimeError(f"bias must be [N={N}], got {tuple(bias.shape)}")
    shape = x.shape[:-1] + (N,)
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if residual is not None:
        if residual.shape != shape:
            try:
                residual = residual.expand(shape)
            except RuntimeError:
                raise RuntimeError(f"residual must broadcast to {list(shape)}, got {list(residual.shape)}") from None
        if residual.dim() != 2:
            residual = residual.reshape(-1, N)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        out = _FusedLinear.apply(x2, weight, bias, residual, act)
    else:
        out, _ = _forward(x2, weight, bias, residual, act, False)
    return out if x.dim() == 2 else out.view(shape)
