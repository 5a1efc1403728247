"""fp32 products of a long K, in each of the three products: no sum of many terms in one accumulator.

As in test_gpu_linear.py::test_fp32_long_sums, segments of at most 1024 terms whose errors add up like
independent ones: 64 bits within the bound of one such sum everywhere and 2^-20 of the norm overall
(a plain fp32 sum of this length loses 2^-21 and more); joining n segments adds a rounding each,
n 2^-24 of the running sum, in the elementwise bound.
"""
import pytest
import torch

from murmurative_attention_b200 import fused_linear
from test_gpu_linear import make, within

pytestmark = pytest.mark.gpu


def close(got, a, b, rows=None):
    """got [M, N] against a [M, K] b [N, K]^T in 64 bits."""
    a, b = a.double(), b.double()
    want = a @ b.t()
    s, k = (a.square() @ b.square().t()).sqrt(), a.shape[1]
    within(got, want, (1024 / 16 + 16 + k / 1024) * 2.0 ** -23 * 4 * s, torch.float32)
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -20


@pytest.mark.parametrize("rows,k,n", [(40000, 64, 64), (70000, 24, 129), (131072, 40, 72), (33000, 130, 257)])
def test_weight_gradient_over_many_rows(rows, k, n):
    """dW sums over the rows; odd sizes too (a residual's place, rows no copy engine can address)."""
    g = torch.Generator().manual_seed(41)
    x, go = make((rows, k), torch.float32, g), make((rows, n), torch.float32, g)
    w = make((n, k), torch.float32, g).requires_grad_(True)
    dw, = torch.autograd.grad(fused_linear(x, w), w, go)
    close(dw, go.t(), x.t())


@pytest.mark.parametrize("k", [16384, 20001, 40000])
def test_forward_and_input_gradient_of_a_long_row(k):
    g = torch.Generator().manual_seed(42)
    m, n = 300, 264
    x, w = make((m, k), torch.float32, g), make((n, k), torch.float32, g, k ** -0.5)
    b, r = make((1, n), torch.float32, g)[0], make((m, n), torch.float32, g)
    plain = fused_linear(x, w)
    close(plain, x, w)
    y = fused_linear(x, w, b, activation="relu", residual=r)  # the same sums, an epilogue behind them
    torch.testing.assert_close(y, torch.relu(plain + b) + r, rtol=2.0 ** -22, atol=2.0 ** -22)
    xs = make((m, n), torch.float32, g).requires_grad_(True)  # dx sums over the outputs
    dx, = torch.autograd.grad(fused_linear(xs, w.t().contiguous()), xs, x)
    close(dx, x, w)


@pytest.mark.parametrize("rows", [65536, 65537])
def test_many_tiles_keep_their_segments(rows):
    """4096 x 4096 on both sides of a tile row more; compared on some rows."""
    g = torch.Generator(device="cuda").manual_seed(43)
    x = torch.randn(rows, 4096, generator=g, device="cuda")
    w = torch.randn(4096, 4096, generator=g, device="cuda") / 64
    got = fused_linear(x, w)
    pick = torch.cat([torch.arange(40), torch.arange(rows - 40, rows)]).cuda()
    close(got[pick], x[pick], w)


def test_results_repeat():
    g = torch.Generator().manual_seed(44)
    x = make((5000, 100), torch.float32, g).requires_grad_(True)
    w = make((3000, 100), torch.float32, g).requires_grad_(True)
    go = make((5000, 3000), torch.float32, g)
    res = [torch.autograd.grad(fused_linear(x, w, activation="silu"), (x, w), go) for _ in range(3)]
    assert all(torch.equal(a, b) for r in res[1:] for a, b in zip(res[0], r))
