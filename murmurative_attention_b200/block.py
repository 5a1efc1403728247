"""A pre-norm block around ``slot_murmurate``: every matrix product, residual addition, query norm and
rotation runs on this library's kernels (the norms over the model's width are torch's).

    x = x + o_proj(slot_murmurate(rotated, normed q_proj(norm(x))))
    x = x + down(act(up(norm(x))))

The reference's layer (README.md:82-102) is the first line without norms, rotation and residual. The
projections' epilogues hold the bias, the activation and the residual (``fused_linear``); the heads'
queries are normed and rotated in the projection's own [B, N, H, d] memory (``qk_norm_rope``, or
``rotary`` alone without ``qk_norm``), with one position per token or, for images and video, one per
axis. ``step`` is the same block for one token per sequence over a resident slot pool
(``decode.SlotPool``): the products take their few-row kernels there.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
import torch.nn as nn

from .decode import SlotPool
from .linear import fused_linear
from .ops import slot_murmurate
from .rope import qk_norm_rope, rotary
from .torch_ops import slot_murmurate as slot_murmurate_op


class MurmurativeBlock(nn.Module):
    def __init__(self, dim: int = 256, heads: int = 4, slots: int = 256, rounds: int = 3, causal: bool = False, *,
                 ffn_dim: Optional[int] = None, activation: str = "gelu", qk_norm: bool = True,
                 rope_base: float = 10000.0, sections: Optional[Sequence[int]] = None, spectrum: str = "shared",
                 device=None, dtype=None):
        super().__init__()
        if dim % heads:
            raise ValueError(f"Embedding dimension D ({dim}) must be divisible by num_heads ({heads})")
        self.dim, self.heads, self.slots, self.rounds, self.causal = dim, heads, slots, rounds, causal
        self.head_dim, self.activation = dim // heads, activation
        self.rope = dict(base=rope_base, sections=None if sections is None else tuple(sections), spectrum=spectrum)
        kw = dict(device=device, dtype=dtype)
        ffn_dim = 4 * dim if ffn_dim is None else ffn_dim
        self.norm1, self.norm2 = nn.RMSNorm(dim, **kw), nn.RMSNorm(dim, **kw)
        self.q_proj = nn.Linear(dim, dim, bias=False, **kw)
        self.o_proj = nn.Linear(dim, dim, bias=False, **kw)
        self.q_norm = nn.Parameter(torch.ones(self.head_dim, **kw)) if qk_norm else None
        self.slot_embeddings = nn.Parameter(torch.randn(heads, slots, self.head_dim, **kw))
        self.up, self.down = nn.Linear(dim, ffn_dim, **kw), nn.Linear(ffn_dim, dim, **kw)

    def _queries(self, h: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """[B, N, D] -> [B, H, N, d], normed and rotated, in the projection's memory layout."""
        B, N, _ = h.shape
        q = fused_linear(h, self.q_proj.weight).view(B, N, self.heads, self.head_dim).transpose(1, 2)
        if self.q_norm is None:
            return rotary(q, positions, **self.rope)
        return qk_norm_rope(q, None, positions, self.q_norm, **self.rope)[0]

    def _feed_forward(self, x: torch.Tensor) -> torch.Tensor:
        h = fused_linear(self.norm2(x), self.up.weight, self.up.bias, activation=self.activation)
        return fused_linear(h, self.down.weight, self.down.bias, residual=x)

    def forward(self, x: torch.Tensor, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x: [B, N, D]; positions: [N] or [B, N] (with ``sections``, [N, A] or [B, N, A]), by default
        0..N-1 (one axis only)."""
        B, N, D = x.shape
        if positions is None:
            if self.rope["sections"] is not None:
                raise ValueError("positions of several axes have to be given")
            positions = torch.arange(N, device=x.device)
        q = self._queries(self.norm1(x), positions)
        slots_k = self.slot_embeddings.unsqueeze(0).expand(B, -1, -1, -1)
        op = slot_murmurate_op if torch.compiler.is_compiling() else slot_murmurate
        attn, _, _ = op(q, slots_k, torch.zeros_like(slots_k), rounds=self.rounds, causal=self.causal)
        x = fused_linear(attn.transpose(1, 2).reshape(B, N, D), self.o_proj.weight, residual=x)
        return self._feed_forward(x)

    def new_pool(self, batch: int) -> SlotPool:
        """Slot pools at a sequence's beginning."""
        return SlotPool.from_embeddings(self.slot_embeddings, torch.zeros_like(self.slot_embeddings), batch)

    @torch.no_grad()
    def step(self, x: torch.Tensor, pool: SlotPool, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token per sequence, x [B, D]: its ``rounds`` rounds of select, attend and slot update on the
        pool, the attended values summed over them as in ``forward``; then the pool's positions advance. Tokens
        so take all their rounds one after another, where ``forward`` runs each round over all tokens.
        positions: [B, 1] (with ``sections`` [B, 1, A]), by default the pool's."""
        if positions is None:
            if self.rope["sections"] is not None:
                raise ValueError("positions of several axes have to be given")
            positions = pool.positions.unsqueeze(1)
        q = self._queries(self.norm1(x).unsqueeze(1), positions)[:, :, 0]
        attn = None if self.rounds else torch.zeros_like(q)
        for _ in range(self.rounds):
            attn = pool.step(q, q, q, attn, causal=self.causal, gamma=0.15, advance=False)
        pool.positions += 1
        x = fused_linear(attn.reshape(x.shape), self.o_proj.weight, residual=x)
        return self._feed_forward(x)
