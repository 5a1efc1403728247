"""``fused_linear`` against its definition in 64 bits: forward, gradients (against the formula's and
against differences), layouts, special values, refusals.

Tolerances, u_T = 2^-24, 2^-11, 2^-8 the rounding of the result's type:
- a product's sum of K terms adds up in 32 bits, 16 terms to a step, each step rounding (or
  cutting) the running sum by at most 2^-23 of it. Running sums of signed terms stay below about
  4 sqrt(sum of squares of the terms) =: 4 S, so E = (K/16 + 16) 2^-23 4 S. Terms of one sign reach
  further: there S is the sum of magnitudes.
- an activation passes z's error on with a slope of at most 1.13 and adds 2^-20 max(|z|, 1) of its own.
- dz = dy act'(z), the slope computed from z (act'' is at most 0.8) and saved within 2^-16 beside 16-bit
  tensors, 2^-24 of itself beside fp32: |dy| (0.8 E + 2^-20 + that), plus u_T |dz| as the operand of the
  16-bit products. relu's slope may differ where |z| <= E.
- sums of dz take the sum of its errors, and a column sum depth * 2^-24 of the sum of magnitudes.
fp16 results below 2^-14 are rounded to multiples of 2^-24.
"""
import pytest
import torch

from murmurative_attention_b200 import fused_linear

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "silu", "gelu", "gelu_tanh"]


def act64(z, act):
    z = z.detach().requires_grad_(True)
    f = torch.nn.functional
    y = {"none": lambda t: t * 1, "relu": f.relu, "silu": f.silu, "gelu": f.gelu,
         "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[act](z)
    slope, = torch.autograd.grad(y.sum(), z)
    return y.detach(), slope


def sum_error(a, b):
    """E for the product a [M, K] b [N, K]^T."""
    k = a.shape[1]
    return (k / 16 + 16) * 2.0 ** -23 * 4 * (a.square() @ b.square().t()).sqrt()


def within(got, want, tol, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    tol = tol + U[dtype] * (want.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"worst excess {float((err - tol).max()):.3e}"


def check(x, w, b, r, go, act, out, grads):
    dt = x.dtype
    X, W = x.detach().double(), w.detach().double()
    z = X @ W.t()
    if b is not None:
        z = z + b.detach().double()
    E = sum_error(X, W)
    y, slope = act64(z, act)
    if r is not None:
        y = y + r.detach().double()
    fn = 0.0 if act == "none" else 2.0 ** -20 * z.abs().clamp(min=1)
    within(out.detach(), y, 1.13 * E + fn + 2.0 ** -24 * y.abs(), dt)
    if grads is None:
        return
    dy = go.double()
    dz = dy * slope
    if act == "none":
        Edz = torch.zeros_like(dz)
    elif act == "relu":
        Edz = torch.where(z.abs() <= E, dy.abs(), torch.zeros_like(dz))
    else:
        Edz = dy.abs() * (0.8 * E + 2.0 ** -20 + (U[dt] * slope.abs() if dt == torch.float32 else 2.0 ** -16))
    Eop = Edz + (U[dt] * (dz.abs() + Edz) if act != "none" else 0)
    if dt == torch.float16:
        Eop = Eop + 2.0 ** -25
    within(grads[0], dz @ W, Eop @ W.abs() + sum_error(dz, W.t()), dt)
    within(grads[1], dz.t() @ X, Eop.t() @ X.abs() + sum_error(dz.t(), X.t()), dt)
    if b is not None:
        within(grads[2], dz.sum(0), Edz.sum(0) + (dz.shape[0] + 16) * 2.0 ** -24 * dz.abs().sum(0), dt)
    if r is not None:
        assert torch.equal(grads[-1], go)


def make(shape, dtype, g, scale=1.0, pad=0):
    """Random rows; with pad, a view at an odd offset into wider rows."""
    m, k = shape
    t = (torch.randn(m, k + pad, generator=g) * scale).to(dtype).cuda()
    return t[:, pad:] if pad else t


SHAPES = [  # rows, in, out
    (1, 64, 64), (1, 1, 1), (4, 1024, 1024), (7, 100, 36), (33, 257, 129), (128, 64, 256), (200, 72, 520),
    (300, 1001, 77), (5, 8, 8), (260, 512, 384), (513, 96, 1000), (3, 4096, 40), (2048, 64, 64), (16, 1000, 24),
    (9, 48, 2056), (1100, 130, 136), (65, 320, 640),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_matches_definition(dtype, act):
    g = torch.Generator().manual_seed(2)
    for i, (m, k, n) in enumerate(SHAPES):
        pad = (0, 0, 3)[i % 3]
        x, w = make((m, k), dtype, g, 1.0, pad), make((n, k), dtype, g, k ** -0.5, (0, 5)[i % 2])
        b = make((1, n), dtype, g)[0] if i % 4 else None
        r = make((m, n), dtype, g, 1.0, pad) if i % 2 else None
        go = make((m, n), dtype, g, 0.5, (0, 0, 0, 1)[i % 4])
        leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
        out = fused_linear(x, w, b, activation=act, residual=r)
        with torch.no_grad():
            assert torch.equal(out, fused_linear(x, w, b, activation=act, residual=r))
        check(x, w, b, r, go, act, out, torch.autograd.grad(out, leaves, go))


@pytest.mark.parametrize("dtype", DTYPES)
def test_larger_products(dtype):
    """Several tiles each way, partial ones at both edges, long sums in each of the three products."""
    g = torch.Generator().manual_seed(4)
    for m, k, n in [(1000, 1024, 1032), (4100, 520, 264), (777, 1001, 1111), (150, 264, 4096), (31, 2048, 2048),
                    (8200, 128, 120)]:
        x, w, b = make((m, k), dtype, g), make((n, k), dtype, g, k ** -0.5), make((1, n), dtype, g)[0]
        r, go = make((m, n), dtype, g), make((m, n), dtype, g, 0.5)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        out = fused_linear(x, w, b, activation="gelu", residual=r)
        check(x, w, b, r, go, "gelu", out, torch.autograd.grad(out, leaves, go))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_row_count(dtype):
    """Few rows take kernels of their own: every count up to past their reach."""
    g = torch.Generator().manual_seed(6)
    k, n = 264, 200
    w, b = make((n, k), dtype, g, k ** -0.5), make((1, n), dtype, g)[0]
    for m in list(range(1, 36)) + [63, 64, 65, 127, 128, 129, 255, 256, 257]:
        x, r = make((m, k), dtype, g), make((m, n), dtype, g)
        check(x, w, b, r, None, "silu", fused_linear(x, w, b, activation="silu", residual=r), None)


@pytest.mark.parametrize("m,k,n", [(955, 2064, 3224), (300, 4000, 520), (40, 9000, 130), (4200, 1100, 4100)])
def test_fp32_long_sums(m, k, n):
    """No running sum takes more than 1024 terms: E of such sums, added over the parts like independent
    errors, is below E of one sum of 1024 terms for S over all of them; 64 bits within it everywhere and
    2^-20 of the norm overall (a plain fp32 sum of this length loses about 2^-21)."""
    g = torch.Generator().manual_seed(31)
    x, w = make((m, k), torch.float32, g), make((n, k), torch.float32, g, k ** -0.5)
    want = x.double() @ w.double().t()
    got = fused_linear(x, w)
    s = (x.double().square() @ w.double().square().t()).sqrt()
    within(got, want, (1024 / 16 + 16 + k / 1024) * 2.0 ** -23 * 4 * s, torch.float32)
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -20


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n,pad", [(263, 131, 0), (264, 200, 3), (1030, 1, 0), (17, 515, 2)])
def test_every_row_count_without_alignment(dtype, k, n, pad):
    """Rows that are not 16-byte aligned, one output, fewer columns than a warp's share."""
    g = torch.Generator().manual_seed(7)
    w, b = make((n, k), dtype, g, k ** -0.5, pad), make((1, n), dtype, g)[0]
    for m in list(range(1, 20)) + [31, 32, 33, 48, 49, 80, 100, 128, 300]:
        x, r = make((m, k), dtype, g, 1.0, pad), make((m, n), dtype, g, 1.0, pad)
        check(x, w, b, r, None, "gelu", fused_linear(x, w, b, activation="gelu", residual=r), None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [64, 65])
def test_nan_reaches_its_rows_gradient_alone(dtype, n):
    for rows in (3, 300):
        for act in ("silu", "gelu", "gelu_tanh"):
            g = torch.Generator().manual_seed(9)
            x, w = make((rows, 40), dtype, g), make((n, 40), dtype, g, 0.1)
            x[1, 7] = float("nan")
            x.requires_grad_(True)
            dx, = torch.autograd.grad(fused_linear(x, w, activation=act), x, torch.ones(rows, n, device="cuda").to(dtype))
            assert bool(dx[1].isnan().all()) and bool(dx[0].isfinite().all()) and bool(dx[2:].isfinite().all())


def test_last_columns_of_a_row_may_be_special():
    """An infinity or NaN beside an odd row's end stays out of it; one in its last column counts."""
    for dtype in DTYPES:
        wide = torch.ones(3, 40, device="cuda", dtype=dtype)
        wide[:, 33:] = float("nan")
        w = torch.ones(5, 33, device="cuda", dtype=dtype)
        assert bool((fused_linear(wide[:, :33], w) == 33).all())
        x = torch.ones(3, 33, device="cuda", dtype=dtype)
        x[1, 32] = float("inf")
        got = fused_linear(x, w)
        assert bool((got[0] == 33).all()) and bool((got[2] == 33).all()) and not bool(got[1].isfinite().any())


def test_fp32_keeps_fp32_accuracy():
    """Terms of one sign, values with full mantissas and of mixed magnitudes."""
    g = torch.Generator().manual_seed(8)
    for m, k, n in [(70, 600, 90), (300, 256, 264), (2, 512, 512)]:
        x = (torch.rand(m, k, generator=g) + 0.5) * 10.0 ** torch.randint(-6, 6, (m, 1), generator=g).float()
        w = torch.rand(n, k, generator=g) + 0.5
        got = fused_linear(x.cuda(), w.cuda()).double().cpu()
        want = x.double() @ w.double().t()
        assert float(((got - want).abs() / want).max()) <= (k / 16 + 16) * 2.0 ** -23


def test_gradient_matches_differences():
    """<grad, v> against (L(t + h v) - L(t - h v)) / 2h through the kernel in fp32, h = 2^-6: the
    third derivative leaves about h^2 / 6 and the rounding 2^-24 / h, both below 1e-3 of the norms."""
    g = torch.Generator().manual_seed(10)
    m, k, n = 20, 48, 40
    ts = [torch.randn(s, generator=g).cuda() * c for s, c in (((m, k), 1), ((n, k), k ** -0.5), ((n,), 1), ((m, n), 1))]
    go = torch.randn(m, n, generator=g).cuda()
    f = lambda t, act: (fused_linear(t[0], t[1], t[2], activation=act, residual=t[3]).double() * go.double()).sum()
    for act in ("none", "silu", "gelu", "gelu_tanh"):
        leaves = [t.clone().requires_grad_(True) for t in ts]
        grads = torch.autograd.grad(fused_linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3]),
                                    leaves, go)
        h = 2.0 ** -6
        for i, t in enumerate(ts):
            v = torch.randn(t.shape, generator=g).cuda()
            up, dn = list(ts), list(ts)
            up[i], dn[i] = t + h * v, t - h * v
            diff = (f(up, act) - f(dn, act)) / (2 * h)
            direct = (grads[i].double() * v.double()).sum()
            assert abs(float(diff - direct)) <= 1e-3 * float(grads[i].double().norm() * v.double().norm())


def test_leading_dims_broadcast_residual_and_views():
    g = torch.Generator().manual_seed(12)
    dt = torch.bfloat16
    x = torch.randn(2, 3, 5, 64, generator=g).to(dt).cuda()
    w = torch.randn(48, 64, generator=g).to(dt).cuda()
    r = torch.randn(5, 48, generator=g).to(dt).cuda()
    flat = fused_linear(x.view(-1, 64), w, residual=r.expand(2, 3, 5, 48).reshape(-1, 48))
    assert torch.equal(fused_linear(x, w, residual=r), flat.view(2, 3, 5, 48))
    assert torch.equal(fused_linear(x.transpose(0, 1), w), fused_linear(x, w).transpose(0, 1))
    assert torch.equal(fused_linear(x[0, 0, 0], w), fused_linear(x, w)[0, 0, 0])
    # a weight stored transposed, and rows all the same (stride 0)
    assert torch.equal(fused_linear(x, w.t().contiguous().t()), fused_linear(x, w))
    one = x[:1, :1, :1].expand(2, 3, 5, 64)
    assert torch.equal(fused_linear(one, w), fused_linear(one.contiguous(), w))
    rr = r.clone().requires_grad_(True)
    out = fused_linear(x, w, residual=rr)
    gr, = torch.autograd.grad(out.float().sum(), rr)
    assert gr.shape == rr.shape and bool((gr.float() == 6).all())  # the sum over the broadcast
    # an expanded scalar gradient
    ww = w.clone().requires_grad_(True)
    gw, = torch.autograd.grad(fused_linear(x, ww).sum(), ww)
    want = x.double().sum((0, 1, 2)).expand(48, 64)
    within(gw, want, (30 / 16 + 16) * 2.0 ** -23 * x.double().abs().sum((0, 1, 2)).expand(48, 64), dt)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [3, 300])
def test_special_values_stay_in_their_row(dtype, rows):
    g = torch.Generator().manual_seed(14)
    x, w = make((rows, 72), dtype, g), make((80, 72), dtype, g, 0.1)
    clean = fused_linear(x, w, activation="relu")
    bad = x.clone()
    bad[1, 5] = float("nan")
    bad[2, 6] = float("inf")
    got = fused_linear(bad, w, activation="relu")
    assert bool(got[1].isnan().all())
    keep = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    assert not bool(fused_linear(bad, w)[2].isfinite().any())


def test_empty_and_determinism():
    w = torch.randn(64, 32, device="cuda", requires_grad=True)
    b = torch.randn(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 32, device="cuda", requires_grad=True)
    out = fused_linear(x, w, b, activation="silu")
    assert out.shape == (0, 64)
    gx, gw, gb = torch.autograd.grad(out, (x, w, b), torch.empty(0, 64, device="cuda"))
    assert gx.shape == (0, 32) and bool((gw == 0).all()) and bool((gb == 0).all())
    g = torch.Generator().manual_seed(16)
    for dt in DTYPES:
        xs = make((3000, 136), dt, g).requires_grad_(True)
        ws = make((72, 136), dt, g).requires_grad_(True)
        bs = make((1, 72), dt, g)[0].requires_grad_(True)
        go = make((3000, 72), dt, g)
        res = []
        for _ in range(2):
            o = fused_linear(xs, ws, bs, activation="gelu_tanh")
            res.append((o.detach(),) + torch.autograd.grad(o, (xs, ws, bs), go))
        assert all(torch.equal(p, q) for p, q in zip(*res))


def test_partial_gradients_and_other_stream():
    g = torch.Generator().manual_seed(18)
    x, w = make((50, 64), torch.float16, g), make((40, 64), torch.float16, g, 0.1)
    b = make((1, 40), torch.float16, g)[0]
    go = make((50, 40), torch.float16, g)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(fused_linear(*full, activation="silu"), full, go)
    for i in range(3):
        ts = [t.clone() for t in (x, w, b)]
        ts[i].requires_grad_(True)
        got, = torch.autograd.grad(fused_linear(*ts, activation="silu"), ts[i], go)
        assert torch.equal(got, want[i])
    s = torch.cuda.Stream()
    ref = fused_linear(x, w, b)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = fused_linear(x, w, b)
    s.synchronize()
    assert torch.equal(got, ref)


def test_refusals():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    with pytest.raises(TypeError):
        fused_linear(x.double(), w.double())
    with pytest.raises(TypeError):
        fused_linear(x, w.half())
    with pytest.raises(RuntimeError):
        fused_linear(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError):
        fused_linear(x, w.cpu())
    with pytest.raises(RuntimeError):
        fused_linear(x, w[:, :8])
    with pytest.raises(RuntimeError):
        fused_linear(x, w, torch.randn(16, device="cuda"))
    with pytest.raises(RuntimeError):
        fused_linear(x, w, residual=torch.randn(4, 9, device="cuda"))
    with pytest.raises(TypeError):
        fused_linear(x, w, residual=torch.randn(4, 8, device="cuda").half())
    with pytest.raises(ValueError):
        fused_linear(x, w, activation="swish")
    with pytest.raises(RuntimeError):
        fused_linear(x, w[:0])
