"""Linear layer with bias, activation and residual in the matrix product's epilogue.

``fused_linear`` is a block's projections and feed-forward products around ``slot_murmurate``:
``act(x W^T + b) + residual`` without a pass over memory for anything but the product. The
compute is ``murm_linear_fwd`` / ``_bwd`` (murm_linear.cu, murm_gemm.cu), the host side is compiled
(murm_torch.cpp).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 activation: str = "none", residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x W^T + bias) + residual.

    Args:
        x: [..., K]; weight: [N, K]; bias: [N]; residual: broadcastable to [..., N]. One dtype: fp16,
           bf16 or fp32 (fp32 products keep fp32 accuracy; where an operand holds an infinity the
           result is not finite, but may be NaN instead of an infinity). Any strides; rows with a
           unit inner stride are read in place.
        activation: "none", "relu", "silu", "gelu" (error function) or "gelu_tanh".

    Returns [..., N]. Differentiable (once) with respect to x, weight, bias and residual; the backward
    reads x, weight and the activation's slopes, which the forward saves in two bytes per element of
    16-bit outputs and four of fp32 ones (none without an activation).

    Other dtypes raise TypeError, an unknown activation ValueError, CPU tensors, shapes that do not fit and
    torch.jit.trace RuntimeError, forward-mode differentiation NotImplementedError. torch.compile, make_fx and
    other dispatch modes see a registered operator.
    """
    if _native.traced():
        from .torch_ops import fused_linear as registered
        return registered(x, weight, bias, activation, residual)
    return _native.binding().fused_linear(x, weight, bias, activation, residual)
