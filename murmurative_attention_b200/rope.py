"""Per-head norms of queries and keys with the position rotation in the same pass, and the
rotation alone by positions of one or several axes.

``qk_norm_rope`` sits between the projections and ``slot_murmurate`` (or the six-argument
``functional.slot_murmurate``, whose token keys it treats alongside the queries); ``rotary`` is
the rotation without the norm, for images and video as well. Both read tensors [B, H, N, d] in
place, with any strides of a unit inner stride: the [B, N, H, d] memory of a projection costs no
transpose copy, and results keep the input's layout. The compute is ``murm_norm_rope_fwd`` /
``_bwd`` (murm_rope.cu), one launch for q and k together.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib
from ._call import call, dtype_code, same_device

_POSITION_TYPES = {torch.int64: _lib.MURM_POS_I64, torch.int32: _lib.MURM_POS_I32, torch.float32: _lib.MURM_POS_F32}
_SPECTRA = {"shared": 0, "own": 1}


class _Rotation(NamedTuple):
    """Everything about a call except its rows, gains and frequencies."""
    positions: torch.Tensor
    freqs: Optional[torch.Tensor]
    rotary_dim: int
    sections: Tuple[int, ...]
    own: int
    interleaved: int
    base: float
    eps: float


def _check_rows(t: torch.Tensor, name: str) -> None:
    dtype_code(t, name)
    if t.dim() != 4:
        raise RuntimeError(f"{name} must be 4-D [B, H, N, head_dim], got shape {tuple(t.shape)}")


def _rotation(x, positions, base, rotary_dim, sections, spectrum, interleaved, freqs, eps=0.0) -> _Rotation:
    """Checks the rotation's arguments against rows x [B, H, N, d]."""
    B, _, N, d = x.shape
    rd = d if rotary_dim is None else int(rotary_dim)
    if rd < 0 or rd > d or rd % 2:
        raise RuntimeError(f"rotary_dim must be even and in 0..{d}, got {rd}")
    if spectrum not in _SPECTRA:
        raise ValueError(f"spectrum must be 'shared' or 'own', got {spectrum!r}")
    if not torch.is_tensor(positions) or positions.dtype not in _POSITION_TYPES:
        raise TypeError("positions must be an int64, int32 or float32 tensor")
    same_device(positions, x.device, "positions")
    sec = () if sections is None else tuple(int(s) for s in sections)
    want = (N,) if sections is None else (N, len(sec))
    if sections is not None:
        if not 1 <= len(sec) <= 4 or min(sec) < 0 or sum(sec) != rd // 2:
            raise RuntimeError(f"sections must be 1 to 4 counts of pairs that add up to rotary_dim/2 = {rd // 2}, "
                               f"got {sec}")
    shape = tuple(positions.shape)
    if shape != want and shape != (B,) + want and shape != (1,) + want:
        raise RuntimeError(f"positions must be {list(want)} or {[B] + list(want)}, got {list(shape)}")
    if freqs is not None:
        if freqs.dtype != torch.float32 or tuple(freqs.shape) != (rd // 2,):
            raise RuntimeError(f"freqs must be a float32 tensor of rotary_dim/2 = {rd // 2} elements")
        same_device(freqs, x.device, "freqs")
        freqs = freqs.contiguous()
    return _Rotation(positions, freqs, rd, sec, _SPECTRA[spectrum], 1 if interleaved else 0, float(base), float(eps))


def _weight(w: Optional[torch.Tensor], x: torch.Tensor, name: str) -> Optional[torch.Tensor]:
    if w is None:
        return None
    dtype_code(w, name)
    if w.dtype != x.dtype and w.dtype != torch.float32:
        raise TypeError(f"{name} must be float32 or {x.dtype}, got {w.dtype}")
    if tuple(w.shape) != (x.shape[3],):
        raise RuntimeError(f"{name} must be [head_dim={x.shape[3]}], got {tuple(w.shape)}")
    same_device(w, x.device, name)
    return w.contiguous()


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 else t.contiguous()


def _args(x: torch.Tensor, rot: _Rotation, normalize: int, inverse: int) -> "_lib.NormRopeArgs":
    a = _lib.NormRopeArgs()
    a.batch, _, a.tokens, a.head_dim = x.shape
    a.rotary_dim, a.dtype, a.normalize = rot.rotary_dim, dtype_code(x, "x"), normalize
    a.interleaved, a.inverse, a.own_spectrum = rot.interleaved, inverse, rot.own
    a.eps, a.base = rot.eps, rot.base
    p = rot.positions
    st = p.stride()
    if rot.sections:
        a.axes = len(rot.sections)
        a.sections[:a.axes] = rot.sections
    else:
        a.axes = 1
        st += (0,)
    if len(st) == 2:
        st = (0,) + st
    elif p.shape[0] == 1:
        st = (0,) + st[1:]
    a.position_type, a.positions, a.position_stride[:] = _POSITION_TYPES[p.dtype], p.data_ptr(), st
    if rot.freqs is not None:
        a.freqs = rot.freqs.data_ptr()
    return a


def _fill(r: "_lib.HeadRows", x: torch.Tensor, out: torch.Tensor, weight: Optional[torch.Tensor] = None,
          grad: Optional[torch.Tensor] = None, grad_weight: Optional[torch.Tensor] = None) -> None:
    r.x, r.x_stride[:] = x.data_ptr(), x.stride()[:3]
    r.out, r.out_stride[:] = out.data_ptr(), out.stride()[:3]
    r.heads = x.shape[1]
    if weight is not None:
        r.weight, r.weight_dtype = weight.data_ptr(), dtype_code(weight, "weight")
    if grad is not None:
        r.grad, r.grad_stride[:] = grad.data_ptr(), grad.stride()[:3]
    if grad_weight is not None:
        r.grad_weight = grad_weight.data_ptr()


def _norm_rope_forward(q, k, q_weight, k_weight, rot: _Rotation):
    a = _args(q, rot, 1, 0)
    outs = []
    for rows, x, w in ((a.q, q, q_weight), (a.k, k, k_weight)):
        out = None
        if x is not None:
            x = _unit(x)
            out = torch.empty_like(x)
            _fill(rows, x, out, w)
        outs.append(out)
    if q.numel() or (k is not None and k.numel()):
        call(_lib.load_library().murm_norm_rope_fwd, a, q.device)
    return outs


def _norm_rope_backward(rows, rot: _Rotation):
    """rows: per tensor (x, weight, grad_out) or None; returns [(grad_x, grad_weight) or None]."""
    lib = _lib.load_library()
    first = next(r for r in rows if r is not None)[0]
    a = _args(first, rot, 1, 0)
    res, sums = [], False
    keep = []  # copies that must outlive the call
    for dst, r in zip((a.q, a.k), rows):
        if r is None:
            res.append(None)
            continue
        x, w, go = r
        if not x.numel():  # no rows: an empty gradient, and gain gradients that are sums of nothing
            res.append((torch.empty_like(x), torch.zeros_like(w) if w is not None else None))
            continue
        x, go = _unit(x), _unit(go.to(x.dtype))
        gx = torch.empty_like(x)
        gw = torch.empty_like(w) if w is not None else None
        sums = sums or gw is not None
        _fill(dst, x, gx, w, go, gw)
        keep.append((x, go))
        res.append((gx, gw))
    if sums:
        ws = torch.empty(lib.murm_norm_rope_workspace(), dtype=torch.uint8, device=first.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    if keep:
        call(lib.murm_norm_rope_bwd, a, first.device)
    return res


def _rotate(x: torch.Tensor, rot: _Rotation, inverse: int) -> torch.Tensor:
    x = _unit(x)
    out = torch.empty_like(x)
    if x.numel():
        a = _args(x, rot, 0, inverse)
        _fill(a.q, x, out)
        call(_lib.load_library().murm_norm_rope_fwd, a, x.device)
    return out


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, rot):
        ctx.save_for_backward(q, k, q_weight, k_weight, rot.positions, rot.freqs)
        ctx.rot = rot._replace(positions=None, freqs=None)
        return tuple(_norm_rope_forward(q, k, q_weight, k_weight, rot))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, qw, kw, positions, freqs = ctx.saved_tensors
        rot = ctx.rot._replace(positions=positions, freqs=freqs)
        need = ctx.needs_input_grad
        rows = []
        for x, w, g, want in ((q, qw, gq, need[0] or need[2]), (k, kw, gk, need[1] or need[3])):
            rows.append(None if x is None or not want else (x, w, torch.zeros_like(x) if g is None else g))
        res = _norm_rope_backward(rows, rot)
        (dq, dqw), (dk, dkw) = (r if r is not None else (None, None) for r in res)
        return dq, dk, dqw, dkw, None


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rot, inverse):
        ctx.save_for_backward(rot.positions, rot.freqs)
        ctx.rot, ctx.inverse = rot._replace(positions=None, freqs=None), inverse
        return _rotate(x, rot, inverse)

    @staticmethod
    def backward(ctx, g):
        positions, freqs = ctx.saved_tensors
        rot = ctx.rot._replace(positions=positions, freqs=freqs)
        return _RotaryFn.apply(g, rot, 1 - ctx.inverse), None, None


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
    Differentiable with respect to q, k and the gains.
    """
    _check_rows(q, "q")
    if k is not None:
        _check_rows(k, "k")
        if k.dtype != q.dtype:
            raise TypeError(f"q and k must share a dtype, got {q.dtype} and {k.dtype}")
        same_device(k, q.device, "k")
        if k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]:
            raise RuntimeError(f"k must be [B={q.shape[0]}, Hk, N={q.shape[2]}, d={q.shape[3]}], got {tuple(k.shape)}")
    elif k_weight is not None:
        raise RuntimeError("k_weight given without k")
    q_weight, k_weight = _weight(q_weight, q, "q_weight"), _weight(k_weight, q, "k_weight")
    rot = _rotation(q, positions, base, rotary_dim, sections, spectrum, interleaved, freqs, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRope.apply(q, k, q_weight, k_weight, rot)
    return tuple(_norm_rope_forward(q, k, q_weight, k_weight, rot))


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
    _check_rows(x, "x")
    rot = _rotation(x, positions, base, rotary_dim, sections, spectrum, interleaved, freqs)
    if x.requires_grad and torch.is_grad_enabled():
        return _RotaryFn.apply(x, rot, 1 if inverse else 0)
    return _rotate(x, rot, 1 if inverse else 0)
