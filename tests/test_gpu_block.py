"""The block's operators together: ``MurmurativeBlock`` forward, gradients and single-token steps against
the same block written in plain torch around ``slot_murmurate`` itself, the registered operators under
torch.compile, and the example.

Both sides call the same slot operator on queries that differ by roundings; a token whose 7th and 8th
slots are closer than that may pick another one, so the slot operator's result is compared through
inputs (the queries) and outputs (from the same queries), never across a selection. fp32 tolerances:
the plain side's products of K <= 512 fp32 terms and this library's differ by at most
(K/16 + 16) 2^-23 * 4 of their scale, some 2e-5, passed through the next products once more: 1e-4.
"""
import pytest
import torch

import examples.video_block as example
from murmurative_attention_b200 import MurmurativeBlock, fused_linear, qk_norm_rope, rotary, slot_murmurate

pytestmark = pytest.mark.gpu
TOL = dict(atol=1e-4, rtol=1e-4)


def plain_queries(block, h, positions):
    B, N, D = h.shape
    q = (h @ block.q_proj.weight.t()).view(B, N, block.heads, block.head_dim).transpose(1, 2)
    if block.q_norm is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * block.q_norm
    half = block.head_dim // 2
    freq = torch.tensor([block.rope["base"] ** (-i / half) for i in range(half)], device=h.device, dtype=torch.float64)
    p = positions.double()
    if block.rope["sections"] is None:
        p = p.unsqueeze(-1)
        axis = [0] * half
    else:
        axis = [a for a, s in enumerate(block.rope["sections"]) for _ in range(s)]
    if p.dim() == 2:
        p = p.unsqueeze(0)
    angle = p[:, None, :, axis] * freq
    c, s = angle.cos().float(), angle.sin().float()
    a, b = q[..., :half], q[..., half:]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def plain_rest(block, x, attn):
    """From the slot operator's output [B, H, N, d] on."""
    B, N, D = x.shape
    x = x + attn.transpose(1, 2).reshape(B, N, D) @ block.o_proj.weight.t()
    h = torch.nn.functional.gelu(block.norm2(x) @ block.up.weight.t() + block.up.bias)
    return x + h @ block.down.weight.t() + block.down.bias


@pytest.mark.parametrize("qk_norm", [True, False])
@pytest.mark.parametrize("sections", [None, (4, 2, 2)])
def test_block_matches_plain_torch(qk_norm, sections):
    torch.manual_seed(0)
    B, N, D, H = 2, 40, 64, 4
    block = MurmurativeBlock(D, H, slots=32, rounds=2, qk_norm=qk_norm, sections=sections, device="cuda",
                             dtype=torch.float32)
    x = torch.randn(B, N, D, device="cuda")
    pos = torch.arange(N, device="cuda") if sections is None else torch.randint(0, 9, (B, N, 3), device="cuda")
    h = block.norm1(x)
    q = block._queries(h, pos)
    torch.testing.assert_close(q, plain_queries(block, h, pos), **TOL)
    slots = block.slot_embeddings.unsqueeze(0).expand(B, -1, -1, -1)
    attn = slot_murmurate(q, slots, torch.zeros_like(slots), rounds=2)[0]
    torch.testing.assert_close(block(x, pos), plain_rest(block, x, attn), **TOL)
    # gradients: of the queries' side and of the rest, each from one and the same upstream gradient
    g = torch.randn(B, H, N, D // H, device="cuda")
    ps = [p for p in (block.q_proj.weight, block.q_norm) if p is not None]
    for a, b in zip(torch.autograd.grad(block._queries(h, pos), ps, g, retain_graph=True),
                    torch.autograd.grad(plain_queries(block, h, pos), ps, g, retain_graph=True)):
        torch.testing.assert_close(a, b, atol=1e-3 * float(b.abs().max()), rtol=1e-3)
    ps = [block.o_proj.weight, block.up.weight, block.up.bias, block.down.weight, block.down.bias]
    go = torch.randn(B, N, D, device="cuda")
    for a, b in zip(torch.autograd.grad(block(x, pos), ps, go),
                    torch.autograd.grad(plain_rest(block, x, attn), ps, go)):
        torch.testing.assert_close(a, b, atol=1e-3 * float(b.abs().max()), rtol=1e-3)


def test_step_is_the_block_on_one_token():
    """From a fresh pool, a non-causal step is one round over one token: the same selection on the same
    keys, so forward (rounds = 1) and step agree."""
    torch.manual_seed(1)
    B, D, H = 3, 64, 4
    block = MurmurativeBlock(D, H, slots=32, rounds=1, device="cuda", dtype=torch.float32)
    x = torch.randn(B, D, device="cuda")
    pool = block.new_pool(B)
    y = block.step(x, pool)
    with torch.no_grad():
        want = block(x.unsqueeze(1), torch.zeros(B, 1, dtype=torch.int64, device="cuda"))[:, 0]
    torch.testing.assert_close(y, want, **TOL)
    assert torch.equal(pool.positions.cpu(), torch.ones(B, dtype=torch.int64))
    again = block.step(x, pool)  # the pool has moved and so has the position
    assert bool(again.isfinite().all()) and not torch.equal(again, y)


def test_positions_are_needed_with_sections():
    block = MurmurativeBlock(64, 4, slots=32, sections=(4, 4), device="cuda")
    with pytest.raises(ValueError):
        block(torch.randn(1, 5, 64, device="cuda"))
    with pytest.raises(ValueError):
        block.step(torch.randn(1, 64, device="cuda"), block.new_pool(1))


def test_registered_operators_under_compile():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 64, generator=g).cuda().requires_grad_(True)
    w = torch.randn(64, 64, generator=g).cuda().requires_grad_(True)
    b = torch.randn(64, generator=g).cuda().requires_grad_(True)
    gain = torch.randn(16, generator=g).cuda().requires_grad_(True)
    pos = torch.arange(6).cuda()

    def f(x, w, b, gain):
        h = fused_linear(x, w, b, activation="gelu", residual=x)
        q = h.view(2, 6, 4, 16).transpose(1, 2)
        q, k = qk_norm_rope(q, q[:, :2], pos, gain, None, rotary_dim=8)
        return rotary(q, pos, interleaved=True), k, qk_norm_rope(q, None, pos)[0]

    want = f(x, w, b, gain)
    grads = torch.autograd.grad(sum(o.square().sum() for o in want), (x, w, b, gain))
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x, w, b, gain)
    got_grads = torch.autograd.grad(sum(o.square().sum() for o in got), (x, w, b, gain))
    for a, c in zip(got + got_grads, want + grads):
        torch.testing.assert_close(a, c)


def test_example_learns_and_decodes():
    losses = example.train(steps=12)
    assert losses[-1] < 0.8 * losses[0]
    out = example.decode(tokens=4)
    assert out.shape == (4, 2, 256) and bool(out.isfinite().all())
