"""The saved slopes beside 16-bit tensors, where they are small: an activation's tail has a gradient of its
own, within the rounding of its type and not of a step near one.

One input per output (W the identity), so that dx is the product dy act'(z) rounded as an operand and
nothing else. Tolerances, u_T = 2^-11 (fp16), 2^-8 (bf16): a slope below 2^-7 (fp16), 2^-8 (bf16) is
saved within u_T of itself (fp16 in steps of 2^-24 below 2^-14), dz adds u_T of its own (fp16 likewise), dx
none; act' itself is computed within 2^-12 of its value in the tails, from z = -2 down (gelu's normal
distribution, by a formula of absolute error 1.5e-7, is 2e-4 of the slope off at -9, less nearer zero; the
exponents' rounding 2^-19), and within 2^-20 elsewhere, the slope's zero between -2 and 0 among it. A slope
above is within 2^-16, and the two roundings u_T and 2^-20 of the function. All beside dy's magnitude.
"""
import math

import pytest
import torch

from murmurative_attention_b200 import fused_linear
from test_gpu_linear import U

pytestmark = pytest.mark.gpu


def slope64(z, act):
    """act'(z), from forms that do not cancel in the tails (1 + erf(z / sqrt 2) has no digits left at -9)."""
    if act == "silu":
        return torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))
    if act == "gelu":
        return 0.5 * torch.special.erfc(-z / 2 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * math.pi) ** 0.5
    u, du = (8 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3), (8 / math.pi) ** 0.5 * (1 + 0.134145 * z * z)
    return torch.sigmoid(u) * (1 + z * torch.sigmoid(-u) * du)


SMALL = {torch.float16: 2.0 ** -7, torch.bfloat16: 2.0 ** -8}
RANGE = {"silu": (-20.0, 20.0), "gelu": (-9.0, 9.0), "gelu_tanh": (-6.0, 6.0)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("n,rows", [(1, 4001), (64, 3000), (72, 5), (63, 700)])
def test_tails_have_their_gradient(dtype, act, n, rows):
    """Few-row kernel, tensor tiles, with and without 16-byte rows; every code path that saves or reads slopes."""
    g = torch.Generator().manual_seed(51)
    lo, hi = RANGE[act]
    x = (torch.rand(rows, n, generator=g) * (hi - lo) + lo).to(dtype).cuda().requires_grad_(True)
    go = (torch.rand(rows, n, generator=g) + 0.5).to(dtype).cuda()
    eye = torch.eye(n, device="cuda", dtype=dtype)
    dx, = torch.autograd.grad(fused_linear(x, eye, activation=act), x, go)
    z = x.detach().double()
    slope = slope64(z, act)
    dy, s, u = go.double(), slope.abs(), U[dtype]
    steps = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -80
    small = u * s + torch.where(z < -2, 2.0 ** -12 * s, torch.full_like(s, 2.0 ** -20)) + steps
    tol = dy * torch.where(s < 0.99 * SMALL[dtype], small, 2.0 ** -16 + 2.0 ** -20)
    tol = tol + u * (dy * s + tol) + steps
    err = (dx.double() - dy * slope).abs()
    assert bool((err <= tol).all()), f"worst excess {float((err - tol).max()):.3e}"
    if dtype == torch.bfloat16 and act != "gelu_tanh":  # no tail is lost
        assert bool((dx[z < -2] != 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(3, 64), (300, 65), (300, 64)])
def test_zero_and_nan_slopes(dtype, rows, n):
    """relu's slopes are 0 and 1 exactly; a far tail's is 0; a NaN's reaches its own elements alone."""
    g = torch.Generator().manual_seed(52)
    x = torch.randn(rows, n, generator=g).to(dtype).cuda().requires_grad_(True)
    go = torch.randn(rows, n, generator=g).to(dtype).cuda()
    eye = torch.eye(n, device="cuda", dtype=dtype)
    dx, = torch.autograd.grad(fused_linear(x, eye, activation="relu"), x, go)
    assert torch.equal(dx, torch.where(x > 0, go, torch.zeros_like(go)))
    far = torch.full((rows, n), -300.0, device="cuda", dtype=dtype)
    far[1, 3] = float("nan")
    for act in ("silu", "gelu", "gelu_tanh"):
        z = far.clone().requires_grad_(True)
        dz, = torch.autograd.grad(fused_linear(z, eye, activation=act), z, go)
        assert bool(dz[1].isnan().all())  # the product's row: NaN times the identity's zeros
        keep = [i for i in range(rows) if i != 1]
        assert bool((dz[keep] == 0).all())
