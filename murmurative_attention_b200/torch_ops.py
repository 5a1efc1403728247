"""``torch.ops.murmurative_attention``: the reference's op namespace over this library.

The reference registers seven operator schemas in the namespace ``murmurative_attention``
(torch-ext/torch_binding.cpp:6-33) with CUDA kernels (:35-43), and its Python layer fetches
them as ``torch.ops.murmurative_attention`` (src/murmurative/ops.py:30-38). Importing this
module defines the same seven schemas, with the same names, argument names and results, and
implements them for CUDA tensors on the per-phase C ABI (murm_ops.cu, through
``functional``): callers of the reference's ops find them here unchanged.

    slot_select_attend, slot_select_attend_backward, slot_update (in place),
    slot_update_backward, slot_diffusion (in place), slot_diffusion_backward,
    slot_update_diffuse (in place)

It also defines the north-star operation of this library as an operator with autograd:

    slot_murmurate(Tensor q, Tensor slots_k, Tensor slots_v, int rounds=3, int top_k=7,
                   bool causal=False, float alpha=0.9, float gamma=0.15, float? scale=None)
        -> (Tensor out, Tensor indices, Tensor weights)

built from ``slot_murmurate_fwd`` (which also returns the block the backward reads) and
``slot_murmurate_bwd``, both on the fused tensor-core C ABI, and the block's operators around it
with their gradients (``fused_linear_fwd`` / ``_bwd``, ``qk_norm_rope`` / ``_bwd``, ``rotary``), which
``fused_linear``, ``qk_norm_rope`` and ``rotary`` call while torch.compile traces them. Every operator has a fake
(meta) implementation, so FakeTensor tracing and ``torch.compile(fullgraph=True)`` see
through them; the sizes the fakes need come from the library's host-only size functions.
There is no CPU kernel: like the reference's ops, these run on CUDA tensors only.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib, _native, functional, ops

NS = "murmurative_attention"

# The reference's schemas (torch-ext/torch_binding.cpp:7-32), verbatim: an interface.
REFERENCE_SCHEMAS = {
    "slot_select_attend": "slot_select_attend(Tensor query, Tensor slot_keys, Tensor slot_values, "
                          "Tensor? mask, bool causal, Tensor? position_bias, float? scale, int effective_M) -> "
                          "(Tensor, Tensor, Tensor)",
    "slot_select_attend_backward": "slot_select_attend_backward(Tensor grad_output, Tensor grad_weights, "
                                   "Tensor query, Tensor slot_keys, Tensor slot_values, Tensor indices, "
                                   "Tensor weights, float? scale) -> (Tensor, Tensor, Tensor)",
    "slot_update": "slot_update(Tensor(a!) slot_keys, Tensor(b!) slot_values, Tensor token_keys, "
                   "Tensor token_values, Tensor indices, Tensor weights, float alpha) -> ()",
    "slot_update_backward": "slot_update_backward(Tensor grad_new_sk, Tensor grad_new_sv, Tensor token_keys, "
                            "Tensor token_values, Tensor indices, Tensor weights, float alpha) -> "
                            "(Tensor, Tensor, Tensor, Tensor, Tensor)",
    "slot_diffusion": "slot_diffusion(Tensor(a!) slot_keys, Tensor(b!) slot_values, float gamma) -> ()",
    "slot_diffusion_backward": "slot_diffusion_backward(Tensor grad_new_keys, Tensor grad_new_values, "
                               "float gamma) -> (Tensor, Tensor)",
    "slot_update_diffuse": "slot_update_diffuse(Tensor(a!) slot_keys, Tensor(b!) slot_values, Tensor token_keys, "
                           "Tensor token_values, Tensor indices, Tensor weights, float alpha, float gamma) -> ()",
}
NORTH_STAR_SCHEMAS = {
    "slot_murmurate_fwd": "slot_murmurate_fwd(Tensor q, Tensor slots_k, Tensor slots_v, int rounds, int top_k, "
                          "bool causal, float alpha, float gamma, float? scale) -> "
                          "(Tensor, Tensor, Tensor, Tensor)",
    "slot_murmurate_bwd": "slot_murmurate_bwd(Tensor? grad_out, Tensor? grad_weights, Tensor q, Tensor saved, "
                          "int slots, int rounds, int top_k, bool causal, float alpha, float gamma, "
                          "float? scale) -> (Tensor, Tensor, Tensor)",
    "slot_murmurate": "slot_murmurate(Tensor q, Tensor slots_k, Tensor slots_v, int rounds=3, int top_k=7, "
                      "bool causal=False, float alpha=0.9, float gamma=0.15, float? scale=None) -> "
                      "(Tensor, Tensor, Tensor)",
}

_ROTATION = ("float eps, float base, int? rotary_dim, bool interleaved, int[]? sections, str spectrum, "
             "Tensor? freqs")
BLOCK_SCHEMAS = {
    "fused_linear_fwd": "fused_linear_fwd(Tensor x, Tensor weight, Tensor? bias, str activation, Tensor? residual, "
                        "bool save=True) -> (Tensor, Tensor)",
    "fused_linear_bwd": "fused_linear_bwd(Tensor grad_out, Tensor x, Tensor weight, Tensor slope, str activation, "
                        "bool need_x=True, bool need_weight=True, bool need_bias=True) -> (Tensor, Tensor, Tensor)",
    "qk_norm_rope": f"qk_norm_rope(Tensor q, Tensor? k, Tensor positions, Tensor? q_weight, Tensor? k_weight, "
                    f"{_ROTATION}) -> (Tensor, Tensor)",
    "qk_norm_rope_bwd": f"qk_norm_rope_bwd(Tensor grad_q, Tensor grad_k, Tensor q, Tensor? k, Tensor positions, "
                        f"Tensor? q_weight, Tensor? k_weight, {_ROTATION}, bool[4] need=[True, True, True, True]) -> "
                        "(Tensor, Tensor, Tensor, Tensor)",
    "rotary": "rotary(Tensor x, Tensor positions, float base, int? rotary_dim, bool interleaved, int[]? sections, "
              "str spectrum, Tensor? freqs, bool inverse) -> Tensor",
}

_LIB = torch.library.Library(NS, "DEF")
for _schema in list(REFERENCE_SCHEMAS.values()) + list(NORTH_STAR_SCHEMAS.values()) + list(BLOCK_SCHEMAS.values()):
    _LIB.define(_schema)


def _q(name: str) -> str:
    return f"{NS}::{name}"


# ---------------------------------------------------------------------------
# The reference's seven operators (CUDA kernels = adapters onto the per-phase C ABI)
# ---------------------------------------------------------------------------
@torch.library.impl(_q("slot_select_attend"), "CUDA", lib=_LIB)
def _select_attend_cuda(query, slot_keys, slot_values, mask, causal, position_bias, scale, effective_M):
    with torch.no_grad():
        return functional.slot_select_attend(query, slot_keys, slot_values, mask, causal, position_bias, scale,
                                             effective_M)


@torch.library.register_fake(_q("slot_select_attend"), lib=_LIB)
def _select_attend_fake(query, slot_keys, slot_values, mask, causal, position_bias, scale, effective_M):
    B, H, N, D = query.shape
    return (query.new_empty(B, H, N, D), query.new_empty(B, H, N, 7, dtype=torch.float32),
            query.new_empty(B, H, N, 7, dtype=torch.int64))


@torch.library.impl(_q("slot_select_attend_backward"), "CUDA", lib=_LIB)
def _select_attend_bwd_cuda(grad_output, grad_weights, query, slot_keys, slot_values, indices, weights, scale):
    return functional.select_attend_backward(grad_output, grad_weights, query, slot_keys, slot_values, indices,
                                             weights, scale)


@torch.library.register_fake(_q("slot_select_attend_backward"), lib=_LIB)
def _select_attend_bwd_fake(grad_output, grad_weights, query, slot_keys, slot_values, indices, weights, scale):
    B, H, N, D = query.shape
    M = slot_keys.shape[2]
    return query.new_empty(B, H, N, D), query.new_empty(B, H, M, D), query.new_empty(B, H, M, D)


@torch.library.impl(_q("slot_update"), "CUDA", lib=_LIB)
def _update_cuda(slot_keys, slot_values, token_keys, token_values, indices, weights, alpha):
    with torch.no_grad():
        nk, nv = functional.slot_update(token_keys, token_values, slot_keys, slot_values, indices, weights, alpha)
        slot_keys.copy_(nk)
        slot_values.copy_(nv)


@torch.library.register_fake(_q("slot_update"), lib=_LIB)
def _update_fake(slot_keys, slot_values, token_keys, token_values, indices, weights, alpha):
    return None


@torch.library.impl(_q("slot_update_backward"), "CUDA", lib=_LIB)
def _update_bwd_cuda(grad_new_sk, grad_new_sv, token_keys, token_values, indices, weights, alpha):
    return functional.slot_update_backward(grad_new_sk, grad_new_sv, token_keys, token_values, indices, weights,
                                           alpha, grad_new_sk.shape[2])


@torch.library.register_fake(_q("slot_update_backward"), lib=_LIB)
def _update_bwd_fake(grad_new_sk, grad_new_sv, token_keys, token_values, indices, weights, alpha):
    B, H, N, D = token_keys.shape
    M = grad_new_sk.shape[2]
    return (token_keys.new_empty(B, H, N, D), token_keys.new_empty(B, H, N, D), token_keys.new_empty(B, H, M, D),
            token_keys.new_empty(B, H, M, D), token_keys.new_empty(B, H, N, 7, dtype=torch.float32))


@torch.library.impl(_q("slot_diffusion"), "CUDA", lib=_LIB)
def _diffusion_cuda(slot_keys, slot_values, gamma):
    with torch.no_grad():
        nk, nv = functional.slot_diffusion(slot_keys, slot_values, gamma)
        slot_keys.copy_(nk)
        slot_values.copy_(nv)


@torch.library.register_fake(_q("slot_diffusion"), lib=_LIB)
def _diffusion_fake(slot_keys, slot_values, gamma):
    return None


@torch.library.impl(_q("slot_diffusion_backward"), "CUDA", lib=_LIB)
def _diffusion_bwd_cuda(grad_new_keys, grad_new_values, gamma):
    return functional.slot_diffusion_backward(grad_new_keys, grad_new_values, gamma)


@torch.library.register_fake(_q("slot_diffusion_backward"), lib=_LIB)
def _diffusion_bwd_fake(grad_new_keys, grad_new_values, gamma):
    return torch.empty_like(grad_new_keys), torch.empty_like(grad_new_values)


@torch.library.impl(_q("slot_update_diffuse"), "CUDA", lib=_LIB)
def _update_diffuse_cuda(slot_keys, slot_values, token_keys, token_values, indices, weights, alpha, gamma):
    with torch.no_grad():
        nk, nv = functional.slot_update(token_keys, token_values, slot_keys, slot_values, indices, weights, alpha)
        nk, nv = functional.slot_diffusion(nk, nv, gamma)
        slot_keys.copy_(nk)
        slot_values.copy_(nv)


@torch.library.register_fake(_q("slot_update_diffuse"), lib=_LIB)
def _update_diffuse_fake(slot_keys, slot_values, token_keys, token_values, indices, weights, alpha, gamma):
    return None


# ---------------------------------------------------------------------------
# The north-star operator with autograd (fused tensor-core C ABI)
# ---------------------------------------------------------------------------
def _out_layout(q: Tensor) -> Tensor:
    """The output's layout: q's own strides when the C ABI reads and writes them in place (unit
    inner stride, non-negative strides that are multiples of 8 elements), else contiguous."""
    st = q.stride()
    ok = st[-1] == 1 and all(s > 0 and s % 8 == 0 for s in st[:3])
    return torch.empty_strided(q.shape, st, dtype=q.dtype, device=q.device) if ok else \
        torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _shape(q, M, rounds, top_k, causal, alpha, gamma, scale):
    return ops._make_shape(q, M, rounds, top_k, causal, alpha, gamma, scale)


@torch.library.impl(_q("slot_murmurate_fwd"), "CUDA", lib=_LIB)
def _fwd_cuda(q, slots_k, slots_v, rounds, top_k, causal, alpha, gamma, scale):
    if top_k != _lib.TOP_K:
        raise ValueError(f"top_k must be {_lib.TOP_K} (the reference hard-codes k=7), got {top_k}")
    out, idx, w, saved, _ = ops._forward(q, slots_k, slots_v, rounds, top_k, causal, alpha, gamma, scale,
                                         out=_out_layout(q))
    return out, idx, w, saved


@torch.library.register_fake(_q("slot_murmurate_fwd"), lib=_LIB)
def _fwd_fake(q, slots_k, slots_v, rounds, top_k, causal, alpha, gamma, scale):
    B, H, N, D = q.shape
    saved_b, _, _ = ops.slot_murmurate_sizes(_shape(q, slots_k.shape[2], rounds, top_k, causal, alpha, gamma, scale))
    return (_out_layout(q), q.new_empty(B, H, N, 7, dtype=torch.int64), q.new_empty(B, H, N, 7, dtype=torch.float32),
            q.new_empty(saved_b, dtype=torch.uint8))


@torch.library.impl(_q("slot_murmurate_bwd"), "CUDA", lib=_LIB)
def _bwd_cuda(grad_out, grad_weights, q, saved, slots, rounds, top_k, causal, alpha, gamma, scale):
    shape = _shape(q, slots, rounds, top_k, causal, alpha, gamma, scale)
    B, H, _, D = q.shape
    go = grad_out if grad_out is not None else torch.zeros_like(q)
    return ops._backward(q, go, grad_weights, saved, shape, (B, H, slots, D), gq=_out_layout(q))


@torch.library.register_fake(_q("slot_murmurate_bwd"), lib=_LIB)
def _bwd_fake(grad_out, grad_weights, q, saved, slots, rounds, top_k, causal, alpha, gamma, scale):
    B, H, _, D = q.shape
    return _out_layout(q), q.new_empty(B, H, slots, D), q.new_empty(B, H, slots, D)


def _fwd_setup(ctx, inputs, output):
    q, slots_k, slots_v, rounds, top_k, causal, alpha, gamma, scale = inputs
    _, _, _, saved = output
    ctx.save_for_backward(q, saved)
    ctx.args = (slots_k.shape[2], rounds, top_k, causal, alpha, gamma, scale)
    ctx.slot_dtypes = (slots_k.dtype, slots_v.dtype)


def _fwd_backward(ctx, grad_out, grad_idx, grad_w, grad_saved):
    q, saved = ctx.saved_tensors
    gq, gsk, gsv = torch.ops.murmurative_attention.slot_murmurate_bwd(grad_out, grad_w, q, saved, *ctx.args)
    return gq, gsk, gsv, None, None, None, None, None, None


torch.library.register_autograd(_q("slot_murmurate_fwd"), _fwd_backward, setup_context=_fwd_setup, lib=_LIB)


@torch.library.impl(_q("slot_murmurate"), "CompositeImplicitAutograd", lib=_LIB)
def _slot_murmurate(q, slots_k, slots_v, rounds=3, top_k=7, causal=False, alpha=0.9, gamma=0.15, scale=None):
    out, idx, w, _ = torch.ops.murmurative_attention.slot_murmurate_fwd(q, slots_k, slots_v, rounds, top_k, causal,
                                                                         alpha, gamma, scale)
    return out, idx, w


def slot_murmurate(q: Tensor, slots_k: Tensor, slots_v: Tensor, rounds: int = 3, top_k: int = 7,
                   causal: bool = False, *, alpha: float = 0.9, gamma: float = 0.15,
                   scale: Optional[float] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """``torch.ops.murmurative_attention.slot_murmurate``: the same operation and results as
    ``murmurative_attention_b200.slot_murmurate``, as a registered operator (traceable by
    torch.compile)."""
    return torch.ops.murmurative_attention.slot_murmurate(q, slots_k, slots_v, rounds, top_k, causal, alpha, gamma,
                                                          scale)


# ---------------------------------------------------------------------------
# The block's operators (compiled binding over the C ABI)
# ---------------------------------------------------------------------------
@torch.library.impl(_q("fused_linear_fwd"), "CUDA", lib=_LIB)
def _linear_fwd_cuda(x, weight, bias, activation, residual, save=True):
    return _native.binding().linear_fwd(x, weight, bias, activation, residual, save)


_LINEAR_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def _refuse(bad: bool, message: str, kind=RuntimeError) -> None:
    if bad:
        raise kind(message)


def _like(t: Optional[Tensor], x: Tensor, name: str) -> None:
    if t is not None:
        _refuse(t.dtype != x.dtype, f"{name} must have x's dtype {x.dtype}, got {t.dtype}", TypeError)
        _refuse(t.device != x.device, f"{name} must be on {x.device}, got {t.device}")


def _check_linear(x, weight, activation, bias=None):
    """What the compiled binding refuses of the linear operators' arguments, for their fakes: a trace fails
    where the call would."""
    _refuse(activation not in _ACTIVATIONS, f"activation must be one of {', '.join(_ACTIVATIONS)}, got '{activation}'",
            ValueError)
    _refuse(x.dtype not in _LINEAR_DTYPES, f"x must be float32, float16 or bfloat16, got {x.dtype}", TypeError)
    _refuse(x.dim() != 2 or weight.dim() != 2 or weight.shape[1] != x.shape[1],
            f"x must be [M, K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    _refuse(weight.shape[0] < 1 or weight.shape[1] < 1, f"weight must not be empty, got {tuple(weight.shape)}")
    _like(weight, x, "weight")
    _like(bias, x, "bias")
    _refuse(bias is not None and (bias.dim() != 1 or bias.shape[0] != weight.shape[0]),
            f"bias must be [N={weight.shape[0]}], got {tuple(bias.shape) if bias is not None else None}")


def _check_outputs(t: Tensor, x: Tensor, weight: Tensor, name: str) -> None:
    _refuse(t.dim() != 2 or t.shape[0] != x.shape[0] or t.shape[1] != weight.shape[0],
            f"{name} must be [M={x.shape[0]}, N={weight.shape[0]}], got {tuple(t.shape)}")


@torch.library.register_fake(_q("fused_linear_fwd"), lib=_LIB)
def _linear_fwd_fake(x, weight, bias, activation, residual, save=True):
    _check_linear(x, weight, activation, bias)
    if residual is not None:
        _like(residual, x, "residual")
        _check_outputs(residual, x, weight, "residual")
    out = x.new_empty(x.shape[0], weight.shape[0])
    if activation == "none" or not save:
        return out, x.new_empty(0)
    return out, torch.empty_like(out, dtype=torch.float32 if x.dtype == torch.float32 else torch.int16)


@torch.library.impl(_q("fused_linear_bwd"), "CUDA", lib=_LIB)
def _linear_bwd_cuda(grad_out, x, weight, slope, activation, need_x=True, need_weight=True, need_bias=True):
    return _native.binding().linear_bwd(grad_out, x, weight, slope, activation, need_x, need_weight, need_bias)


@torch.library.register_fake(_q("fused_linear_bwd"), lib=_LIB)
def _linear_bwd_fake(grad_out, x, weight, slope, activation, need_x=True, need_weight=True, need_bias=True):
    _check_linear(x, weight, activation)
    _like(grad_out, x, "grad_out")
    _check_outputs(grad_out, x, weight, "grad_out")
    if activation != "none":
        kind = torch.float32 if x.dtype == torch.float32 else torch.int16
        _refuse(slope.dtype != kind, f"slope must be {kind} beside {x.dtype}, got {slope.dtype}", TypeError)
        _refuse(slope.device != x.device, f"slope must be on {x.device}, got {slope.device}")
        _check_outputs(slope, x, weight, "slope")
    return tuple(x.new_empty(shape if need else 0) for shape, need in
                 ((x.shape, need_x), (weight.shape, need_weight), (weight.shape[0], need_bias)))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, activation, residual, _ = inputs
    ctx.save_for_backward(x, weight, output[1])
    ctx.activation = activation
    ctx.mark_non_differentiable(output[1])


def _linear_backward(ctx, grad_out, grad_slope):
    x, weight, slope = ctx.saved_tensors
    need = ctx.needs_input_grad
    grads = [None, None, None]
    if any(need[:3]):
        grads = torch.ops.murmurative_attention.fused_linear_bwd(grad_out, x, weight, slope, ctx.activation, *need[:3])
    return tuple(g if n else None for g, n in zip(grads, need)) + (None, grad_out if need[4] else None, None)


torch.library.register_autograd(_q("fused_linear_fwd"), _linear_backward, setup_context=_linear_setup, lib=_LIB)


def fused_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], activation: str,
                 residual: Optional[Tensor]) -> Tensor:
    """The registered form of ``fused_linear`` (same operation; traceable by torch.compile)."""
    _refuse(x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1],
            f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    shape = x.shape[:-1] + (weight.shape[0],)
    x2 = x.reshape(-1, x.shape[-1])
    r2 = residual.expand(shape).reshape(-1, shape[-1]) if residual is not None else None
    save = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))
    out, _ = torch.ops.murmurative_attention.fused_linear_fwd(x2, weight, bias, activation, r2, save)
    return out.view(shape)


def _unit_layout(t: Tensor) -> Tensor:
    """An empty tensor as the rotation's results are laid out: like the rows when their inner stride is 1
    and the copy's is too (rows that overlap have no layout to keep)."""
    out = torch.empty_like(t if t.stride(3) == 1 else t.contiguous())
    return out if out.stride(3) == 1 else torch.empty_like(t, memory_format=torch.contiguous_format)


@torch.library.impl(_q("qk_norm_rope"), "CUDA", lib=_LIB)
def _qk_cuda(q, k, positions, q_weight, k_weight, *rotation):
    with torch.no_grad():
        oq, ok = _native.binding().qk_norm_rope(q, k, positions, q_weight, k_weight, *rotation)
    return oq, ok if ok is not None else q.new_empty(0)


@torch.library.register_fake(_q("qk_norm_rope"), lib=_LIB)
def _qk_fake(q, k, positions, q_weight, k_weight, *rotation):
    return _unit_layout(q), _unit_layout(k) if k is not None else q.new_empty(0)


@torch.library.impl(_q("qk_norm_rope_bwd"), "CUDA", lib=_LIB)
def _qk_bwd_cuda(grad_q, grad_k, q, k, positions, q_weight, k_weight, *rotation):
    return _native.binding().qk_bwd(grad_q, grad_k, q, k, positions, q_weight, k_weight, *rotation)


@torch.library.register_fake(_q("qk_norm_rope_bwd"), lib=_LIB)
def _qk_bwd_fake(grad_q, grad_k, q, k, positions, q_weight, k_weight, eps, base, rotary_dim, interleaved, sections,
                 spectrum, freqs, need=(True,) * 4):
    for g, t, name in ((grad_q, q, "grad_q"), (grad_k, k, "grad_k")):
        if t is not None:
            _like(g, t, name)
            _refuse(g.shape != t.shape, f"{name} must be {tuple(t.shape)}, got {tuple(g.shape)}")
    none = q.new_empty(0)
    gains = [w is not None and n for w, n in zip((q_weight, k_weight), need[2:])]
    return (_unit_layout(q) if need[0] or gains[0] else none,
            _unit_layout(k) if k is not None and (need[1] or gains[1]) else none,
            torch.empty_like(q_weight) if gains[0] else none, torch.empty_like(k_weight) if gains[1] else none)


def _qk_setup(ctx, inputs, output):
    q, k, positions, q_weight, k_weight, eps, base, rotary_dim, interleaved, sections, spectrum, freqs = inputs
    ctx.save_for_backward(q, k, positions, q_weight, k_weight, freqs)
    ctx.rotation = (eps, base, rotary_dim, interleaved, sections, spectrum)


def _qk_backward(ctx, grad_q, grad_k):
    q, k, positions, q_weight, k_weight, freqs = ctx.saved_tensors
    need = ctx.needs_input_grad
    gq, gk, gqw, gkw = torch.ops.murmurative_attention.qk_norm_rope_bwd(
        grad_q if grad_q is not None else torch.zeros_like(q),
        grad_k if grad_k is not None else torch.zeros_like(k if k is not None else q), q, k, positions, q_weight,
        k_weight, *ctx.rotation, freqs, [need[0], need[1], need[3], need[4]])
    return (gq if need[0] else None, gk if need[1] else None, None, gqw if need[3] else None,
            gkw if need[4] else None) + (None,) * 7


torch.library.register_autograd(_q("qk_norm_rope"), _qk_backward, setup_context=_qk_setup, lib=_LIB)


@torch.library.impl(_q("rotary"), "CUDA", lib=_LIB)
def _rotary_cuda(x, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, inverse):
    with torch.no_grad():
        return _native.binding().rotary(x, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, inverse)


@torch.library.register_fake(_q("rotary"), lib=_LIB)
def _rotary_fake(x, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, inverse):
    return _unit_layout(x)


def _rotary_setup(ctx, inputs, output):
    x, positions, base, rotary_dim, interleaved, sections, spectrum, freqs, inverse = inputs
    ctx.save_for_backward(positions, freqs)
    ctx.rotation = (base, rotary_dim, interleaved, sections, spectrum)
    ctx.inverse = inverse


def _rotary_backward(ctx, grad):
    positions, freqs = ctx.saved_tensors
    return (torch.ops.murmurative_attention.rotary(grad, positions, *ctx.rotation, freqs, not ctx.inverse),) + (None,) * 8


torch.library.register_autograd(_q("rotary"), _rotary_backward, setup_context=_rotary_setup, lib=_LIB)
