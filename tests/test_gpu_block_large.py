"""The block operators where offsets pass 32 bits: rows far apart, and more than 2^31 elements.

The large tensors are compared on some rows, the first and last among them; upstream gradients are
zero on the others, which then add nothing to the sums over rows. Tolerances are those of the small
sizes (tests/test_gpu_linear.py, tests/test_gpu_rope.py): per row they do not depend on the number
of rows, and rows of zeros add no rounding to a sum.
"""
import pytest
import torch

from murmurative_attention_b200 import fused_linear, qk_norm_rope, rotary
from test_gpu_linear import check as check_linear
from test_gpu_rope import U, close_rows, frequencies, rotate

pytestmark = pytest.mark.gpu


def far_apart(t, stride):
    """t's rows [M, K], `stride` elements apart."""
    m, k = t.shape
    base = torch.empty((m - 1) * stride + k, dtype=t.dtype, device="cuda")
    view = base.as_strided((m, k), (stride, 1))
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype,odd", [(torch.float16, 0), (torch.float16, 1), (torch.float32, 0)])
def test_linear_rows_far_apart(dtype, odd):
    """Row 299 begins past element 2^31; with `odd` the rows are not 16-byte aligned."""
    g = torch.Generator().manual_seed(21)
    m, k, n = 300, 264, 200
    stride = (1 << 23) - odd
    assert (m - 1) * stride > 1 << 31
    x = far_apart(torch.randn(m, k, generator=g).to(dtype), stride).requires_grad_(True)
    w = (torch.randn(n, k, generator=g) * k ** -0.5).to(dtype).cuda().requires_grad_(True)
    b = torch.randn(n, generator=g).to(dtype).cuda().requires_grad_(True)
    r = far_apart(torch.randn(m, n, generator=g).to(dtype), stride).requires_grad_(True)
    go = far_apart(torch.randn(m, n, generator=g).to(dtype), stride)
    out = fused_linear(x, w, b, activation="silu", residual=r)
    check_linear(x, w, b, r, go, "silu", out, torch.autograd.grad(out, (x, w, b, r), go))


def test_linear_more_than_2_31_outputs():
    m, k, n = 530_000, 24, 4104
    assert m * n > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(22)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).bfloat16().requires_grad_(True)
    b = torch.randn(n, generator=g, device="cuda").bfloat16().requires_grad_(True)
    edge = (1 << 31) // n  # the row that holds element 2^31
    rows = torch.cat([torch.arange(40), torch.arange(edge - 20, edge + 20), torch.arange(m - 40, m)]).cuda()
    go = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    go[rows] = torch.randn(len(rows), n, generator=g, device="cuda").bfloat16()
    out = fused_linear(x, w, b, activation="gelu_tanh")
    dx, dw, db = torch.autograd.grad(out, (x, w, b), go)
    check_linear(x[rows], w, b, None, go[rows], "gelu_tanh", out[rows], (dx[rows], dw, db))
    rest = torch.ones(m, dtype=torch.bool, device="cuda")
    rest[rows] = False
    assert bool((dx[rest] == 0).all())


def rope_reference(x, w, go, pos, eps):
    """Forward, dx with its scale, and the terms of dw, in 64 bits; x, go [1, H, n, d], pos [1, n]."""
    d = x.shape[-1]
    freq, axis = frequencies(d)
    x, w, go = x.double().cpu(), w.detach().double().cpu(), go.double().cpu()
    p3 = pos.cpu()[:, :, None]
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    out = rotate(x * r * w, p3, d, freq, axis, False)
    gg = rotate(go, p3, d, freq, axis, False, -1.0)
    h = gg * w
    dx = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
    scale = (r * h).abs().amax(-1, keepdim=True) * 2 + dx.abs().amax(-1, keepdim=True)
    return out, dx, scale, gg * x * r


def check_rope(q, w, go, pos, out, dx, dw, eps):
    want, wdx, scale, terms = rope_reference(q, w, go, pos, eps)
    close_rows(out, want, q.dtype)
    close_rows(dx, wdx, q.dtype, scale)
    wsum = terms.sum((0, 1, 2))
    tol = (U[q.dtype] * wsum.abs() + (terms[..., 0].numel() + 32) * 2.0 ** -24 * terms.abs().sum((0, 1, 2))
           + 2.0 ** -25)
    assert bool(((dw.double().cpu() - wsum).abs() <= tol).all())


@pytest.mark.parametrize("axis", ["head", "token"])
def test_rope_rows_far_apart(axis):
    """Heads, then tokens, whose last one begins past element 2^31."""
    g = torch.Generator().manual_seed(23)
    H, N, d, eps = 5, 9, 64, 1e-6
    strides = (0, (1 << 29) + 64, d, 1) if axis == "head" else (0, d, (1 << 28) + 64, 1)
    base = torch.empty(strides[1] * (H - 1) + strides[2] * (N - 1) + d, dtype=torch.bfloat16, device="cuda")
    q = base.as_strided((1, H, N, d), strides).copy_(torch.randn(1, H, N, d, generator=g)).requires_grad_(True)
    w = torch.randn(d, generator=g).bfloat16().cuda().requires_grad_(True)
    go = torch.randn(1, H, N, d, generator=g).bfloat16().cuda()
    pos = torch.randint(0, 100000, (1, N), generator=g).cuda()
    out, _ = qk_norm_rope(q, None, pos, w, eps=eps)
    dx, dw = torch.autograd.grad(out, (q, w), go)
    check_rope(q.detach(), w, go, pos, out.detach(), dx, dw, eps)
    freq, ax = frequencies(d)
    close_rows(rotary(q.detach(), pos), rotate(q.detach().double().cpu(), pos.cpu()[:, :, None], d, freq, ax, False),
               torch.bfloat16)


def test_rope_more_than_2_31_elements():
    H, N, d, eps = 16, 1_050_000, 128, 1e-6
    assert H * N * d > 1 << 31
    g = torch.Generator(device="cuda").manual_seed(24)
    q = torch.randn(1, N, H, d, generator=g, device="cuda", dtype=torch.bfloat16).transpose(1, 2).requires_grad_(True)
    w = torch.randn(d, generator=g, device="cuda").bfloat16().requires_grad_(True)
    edge = (1 << 31) // (H * d)
    rows = torch.cat([torch.arange(5), torch.arange(edge - 3, edge + 3), torch.arange(N - 5, N)]).cuda()
    pos = torch.arange(N, device="cuda").unsqueeze(0)
    go = torch.zeros(1, N, H, d, device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    go[:, :, rows] = torch.randn(1, H, len(rows), d, generator=g, device="cuda").bfloat16()
    out, _ = qk_norm_rope(q, None, pos, w, eps=eps)
    dx, dw = torch.autograd.grad(out, (q, w), go)
    check_rope(q.detach()[:, :, rows], w, go[:, :, rows], pos[:, rows], out.detach()[:, :, rows], dx[:, :, rows], dw, eps)
    freq, ax = frequencies(d)
    turned = rotary(q.detach(), pos)[:, :, rows]
    close_rows(turned, rotate(q.detach()[:, :, rows].double().cpu(), pos[:, rows].cpu()[:, :, None], d, freq, ax, False),
               torch.bfloat16)
