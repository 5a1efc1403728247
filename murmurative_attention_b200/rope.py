"""Per-head norms of queries and keys with the position rotation in the same pass, and the
rotation alone by positions of one or several axes.

``qk_norm_rope`` sits between the projections and ``slot_murmurate`` (or the six-argument
``functional.slot_murmurate``, whose token keys it treats alongside the queries); ``rotary`` is
the rotation without the norm, for images and video as well. Both read tensors [B, H, N, d] in
place, with any strides of a unit inner stride: the [B, N, H, d] memory of a projection costs no
transpose copy, and results keep the input's layout. The compute is ``murm_norm_rope_fwd`` /
``_bwd`` (murm_rope.cu), one launch for q and k together; the host side is compiled
(murm_torch.cpp).
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _native


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6, base: float = 10000.0, rotary_dim: Optional[int] = None,
                 interleaved: bool = False, sections: Optional[Sequence[int]] = None, spectrum: str = "shared",
                 freqs: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """RMS norm of every head's queries and keys, then their rotation by position, in one pass.

    Args:
        q: [B, Hq, N, d]; k: [B, Hk, N, d] of the same dtype, or None (slot_murmurate's own token
           keys are its queries). fp16, bf16 or fp32, d even and at most 256, unit inner stride.
        positions: int64, int32 or float32, [N] or [B, N]; with ``sections``, [N, A] or [B, N, A].
        q_weight, k_weight: gains [d], fp32 or of q's dtype; None: no gain.
        eps, base, rotary_dim, interleaved, sections, spectrum, freqs: as in :func:`rotary`, eps is
           added to the mean square.

    Returns (q, k) normed and rotated, in the inputs' layouts (k None when it was None).
    Differentiable (once) with respect to q, k and the gains.

    Other dtypes raise TypeError, an unknown spectrum ValueError, CPU tensors, shapes that do not fit and
    torch.jit.trace RuntimeError, forward-mode differentiation NotImplementedError. torch.compile, make_fx and
    other dispatch modes see a registered operator.
    """
    if _native.traced():
        oq, ok = torch.ops.murmurative_attention.qk_norm_rope(q, k, positions, q_weight, k_weight, eps, base, rotary_dim,
                                                              interleaved, sections, spectrum, freqs)
        return oq, ok if k is not None else None
    return _native.binding().qk_norm_rope(q, k, positions, q_weight, k_weight, eps, base, rotary_dim, interleaved,
                                          sections, spectrum, freqs)


def rotary(x: torch.Tensor, positions: torch.Tensor, *, base: float = 10000.0, rotary_dim: Optional[int] = None,
           interleaved: bool = False, sections: Optional[Sequence[int]] = None, spectrum: str = "shared",
           freqs: Optional[torch.Tensor] = None, inverse: bool = False) -> torch.Tensor:
    """Rotates the rows of x [B, H, N, d] by their tokens' positions.

    Args:
        positions: int64, int32 or float32, [N] or [B, N]; with ``sections``, [N, A] or [B, N, A],
           one position per axis (for instance time, height, width).
        rotary_dim: the leading elements that turn (even, default d); the rest pass through.
        interleaved: pairs are neighbours (2i, 2i+1) instead of (i, i + rotary_dim/2).
        sections: number of pairs of each axis, in the order of the pairs; they add up to
           rotary_dim/2. None: one axis.
        spectrum: "shared": pair i turns at base^(-2i/rotary_dim) whatever its axis; "own": the j-th
           of an axis's s pairs turns at base^(-j/s).
        freqs: float32 [rotary_dim/2] frequencies (radians per position) instead of base's.
        inverse: turn the other way.

    Returns a tensor in x's layout. Differentiable with respect to x (the inverse rotation).
    """
    if _native.traced():
        return torch.ops.murmurative_attention.rotary(x, positions, base, rotary_dim, interleaved, sections, spectrum,
                                                      freqs, inverse)
    return _native.binding().rotary(x, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, inverse)
