"""The compiled torch binding of the block operators (csrc/murm_torch.cpp).

``binding()`` imports ``_murm_torch.so`` once and hands it the C ABI's functions from the library
``_lib`` has loaded, so both run on one library instance. As with the library there is no
fallback: a missing build raises RuntimeError.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_FUNCTIONS = ("murm_linear_fwd", "murm_linear_bwd", "murm_linear_workspace", "murm_linear_bwd_workspace",
              "murm_norm_rope_fwd", "murm_norm_rope_bwd", "murm_norm_rope_workspace", "murm_last_error_message",
              "murm_status_string")
_binding = None


def traced() -> bool:
    """Whether this call is being traced (torch.compile, torch.export) or a dispatch mode watches it (make_fx,
    fake tensors, counters of operations): then it has to be a registered operator, since the binding runs
    below the dispatcher and a mode would see nothing of it but the allocation of its results."""
    return torch.compiler.is_compiling() or torch._C._len_torch_dispatch_stack() > 0


def binding():
    global _binding
    if _binding is None:
        lib = _lib.load_library()
        try:
            from . import _murm_torch
        except ImportError as e:
            raise RuntimeError("murmurative_attention_b200: torch binding not built or built for another torch "
                               f"({e}). Build it with:  python -m murmurative_attention_b200.build") from e
        _murm_torch.bind({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _FUNCTIONS})
        _binding = _murm_torch
    return _binding
