"""``qk_norm_rope`` and ``rotary`` against their definitions in 64 bits: forward, gradients (against
the formula's and against differences), layouts, positions, refusals.

Tolerances. A result is computed in 32 bits and rounded once to its type: u_T |y| for that rounding
(u_T = 2^-24, 2^-11, 2^-8) plus the 32-bit chain's error. The chain is some 20 operations of 2^-24
relative error each (mean square, rsqrt, gain, two products and a sum; sine and cosine to 2^-22 with
the angle's reduction), relative to the largest element of the row: 2^-19 of the row's maximum. fp16
results below 2^-14 are rounded to multiples of 2^-24. Sums over rows add depth * 2^-24 of the sum of
the terms' magnitudes, with a depth of at most the number of rows.
"""
import pytest
import torch

from murmurative_attention_b200 import qk_norm_rope, rotary

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def close_rows(got, want, dtype, scale=None):
    """got within the rounding of its type and 2^-19 of the row's scale (default: its maximum)."""
    scale = want.abs().amax(-1, keepdim=True) if scale is None else scale
    tol = U[dtype] * want.abs() + 2.0 ** -19 * scale + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (got.double().cpu() - want).abs()
    assert got.dtype == dtype
    assert bool((err <= tol).all()), f"worst excess {float((err - tol).max()):.3e}"


def frequencies(rd, sections=None, spectrum="shared", base=10000.0):
    half = rd // 2
    if sections is None:
        return torch.tensor([base ** (-i / half) for i in range(half)], dtype=torch.float64), [0] * half
    f, axis = [], []
    for a, s in enumerate(sections):
        for j in range(s):
            f.append(base ** (-j / s) if spectrum == "own" else base ** (-len(f) / half))
            axis.append(a)
    return torch.tensor(f, dtype=torch.float64), axis


def rotate(x, positions, rd, freq, axis, interleaved, sign=1.0):
    """Rotation of x [B, H, N, d] (64 bits); positions [B, N, A]."""
    angle = sign * positions.double()[:, None, :, axis] * freq
    c, s = angle.cos(), angle.sin()
    y = x.clone()
    i = torch.arange(rd // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y


def make(B, H, N, d, dtype, layout, g, scale=1.0):
    if layout == "token":
        return (torch.randn(B, N, H, d, generator=g) * scale).to(dtype).transpose(1, 2)
    if layout == "strided":  # rows of a wider buffer at an odd offset: no vector alignment
        return (torch.randn(B, H, N, 2 * d + 3, generator=g) * scale).to(dtype)[..., 3:3 + d]
    return (torch.randn(B, H, N, d, generator=g) * scale).to(dtype)


def cuda(t):
    """The tensor on the GPU with the same strides."""
    base = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
    return base.copy_(t)


SHAPES = [  # B, Hq, Hk, N, d, rotary_dim
    (1, 1, 1, 1, 64, 64), (2, 4, 1, 1, 64, 64), (1, 16, 4, 33, 64, 64), (2, 3, 3, 7, 128, 128), (1, 2, 2, 5, 16, 16),
    (1, 5, 1, 9, 80, 40), (2, 2, 1, 300, 72, 72), (1, 3, 2, 11, 96, 48), (1, 2, 1, 6, 2, 2), (1, 3, 1, 4, 10, 6),
    (1, 2, 2, 3, 256, 256), (1, 1, 1, 3, 254, 2), (1, 2, 1, 5, 64, 0), (3, 1, 7, 1021, 32, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["token", "head", "strided"])
def test_norm_rope_matches_definition(dtype, interleaved, layout):
    g = torch.Generator().manual_seed(3)
    eps = 1e-5
    for B, Hq, Hk, N, d, rd in SHAPES:
        q, k = make(B, Hq, N, d, dtype, layout, g), make(B, Hk, N, d, dtype, layout, g, 30.0)
        qw, kw = (torch.randn(d, generator=g).to(dtype) for _ in range(2))
        gq, gk = make(B, Hq, N, d, dtype, "token", g), make(B, Hk, N, d, dtype, "head", g)
        pos = torch.randint(0, 200000, (B, N), generator=g)
        args = [cuda(t).requires_grad_(True) for t in (q, k, qw, kw)]
        oq, ok = qk_norm_rope(args[0], args[1], pos.cuda(), args[2], args[3], eps=eps, rotary_dim=rd,
                              interleaved=interleaved)
        with torch.no_grad():  # the path without autograd is the same
            assert torch.equal(oq, qk_norm_rope(args[0], args[1], pos.cuda(), args[2], args[3], eps=eps,
                                                rotary_dim=rd, interleaved=interleaved)[0])
        grads = torch.autograd.grad((oq, ok), args, (cuda(gq), cuda(gk)))
        freq, axis = frequencies(rd)
        for x, w, go, o, dx, dw in ((q, qw, gq, oq, grads[0], grads[2]), (k, kw, gk, ok, grads[1], grads[3])):
            x, w, go = x.double(), w.double(), go.double()
            r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
            p3 = pos[:, :, None]
            close_rows(o.detach(), rotate(x * r * w, p3, rd, freq, axis, interleaved), dtype)
            gg = rotate(go, p3, rd, freq, axis, interleaved, -1.0)
            h = gg * w
            want = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
            # the two terms may cancel: the error is relative to them, not to their difference
            close_rows(dx, want, dtype, (r * h).abs().amax(-1, keepdim=True) * 2 + want.abs().amax(-1, keepdim=True))
            terms = gg * x * r
            wsum = terms.sum((0, 1, 2))
            rows = terms.shape[0] * terms.shape[1] * terms.shape[2]
            tol = U[dtype] * wsum.abs() + (rows + 32) * 2.0 ** -24 * terms.abs().sum((0, 1, 2)) + 2.0 ** -25
            assert dw.dtype == dtype and bool(((dw.double().cpu() - wsum).abs() <= tol).all())


def test_gradient_matches_differences():
    """<dL/dx, v> against (L(x + h v) - L(x - h v)) / 2h through the kernel itself in fp32: h = 2^-7
    leaves h^2 |third derivative| ~ 6e-5 and 2^-24 / h ~ 8e-6 per element, relative."""
    g = torch.Generator().manual_seed(5)
    B, H, N, d = 2, 3, 5, 64
    q, k = (torch.randn(B, H, N, d, generator=g).cuda() for _ in range(2))
    ws = [torch.randn(d, generator=g).cuda() for _ in range(2)]
    pos = torch.arange(N).cuda()
    go = [torch.randn(B, H, N, d, generator=g).cuda() for _ in range(2)]
    inputs = [q, k] + ws

    def loss(ts):
        return sum((o.double() * w.double()).sum() for o, w in zip(qk_norm_rope(ts[0], ts[1], pos, ts[2], ts[3]), go))

    leaves = [t.clone().requires_grad_(True) for t in inputs]
    grads = torch.autograd.grad(qk_norm_rope(leaves[0], leaves[1], pos, leaves[2], leaves[3]), leaves, go)
    h = 2.0 ** -7
    for i in range(4):
        v = torch.randn(inputs[i].shape, generator=g).cuda()
        up, dn = list(inputs), list(inputs)
        up[i], dn[i] = inputs[i] + h * v, inputs[i] - h * v
        diff = (loss(up) - loss(dn)) / (2 * h)
        direct = (grads[i].double() * v.double()).sum()
        size = grads[i].double().norm() * v.double().norm()
        assert abs(float(diff - direct)) <= 1e-3 * float(size)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spectrum", ["shared", "own"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_axes_match_definition(dtype, spectrum, interleaved):
    g = torch.Generator().manual_seed(7)
    for B, H, N, d, rd, sections in [(2, 3, 60, 64, 64, (8, 12, 12)), (1, 1, 1, 72, 72, (0, 18, 18)),
                                     (2, 2, 31, 128, 96, (16, 16, 8, 8)), (1, 4, 17, 10, 6, (1, 2)),
                                     (1, 2, 9, 32, 32, (16,)), (1, 2, 9, 32, 32, (0, 0, 16))]:
        for layout in ("token", "strided"):
            x, go = make(B, H, N, d, dtype, layout, g), make(B, H, N, d, dtype, "token", g)
            pos = torch.randint(-50, 3000, (B, N, len(sections)), generator=g)
            xd = cuda(x).requires_grad_(True)
            out = rotary(xd, pos.cuda(), rotary_dim=rd, sections=sections, spectrum=spectrum, interleaved=interleaved)
            dx, = torch.autograd.grad(out, xd, cuda(go))
            freq, axis = frequencies(rd, sections, spectrum)
            close_rows(out.detach(), rotate(x.double(), pos, rd, freq, axis, interleaved), dtype)
            close_rows(dx, rotate(go.double(), pos, rd, freq, axis, interleaved, -1.0), dtype)


def test_positions_types_broadcast_and_range():
    g = torch.Generator().manual_seed(9)
    B, H, N, d = 2, 2, 6, 64
    x = torch.randn(B, H, N, d, generator=g)
    freq, axis = frequencies(d)
    far = torch.arange(N) + (1 << 33)  # past 32 bits: a 64-bit product of 2^33 and f keeps 2^-20 of a radian
    for pos in (torch.arange(N), torch.arange(N, dtype=torch.int32) - 3, torch.linspace(0, 7.5, N),
                torch.arange(N) + 1000000):
        want = rotate(x.double(), pos.view(1, N, 1).expand(B, N, 1), d, freq, axis, False)
        for p in (pos, pos.view(1, N), pos.expand(B, N), pos.expand(B, N).contiguous()):
            close_rows(rotary(x.cuda(), p.cuda()), want, torch.float32)
    # frequency products at 2^33 agree to about 2^33 * 2^-52 * 16 rad between two orders of evaluation
    got = rotary(x.cuda(), far.cuda()).double().cpu()
    want = rotate(x.double(), far.view(1, N, 1).expand(B, N, 1), d, freq, axis, False)
    assert float((got - want).abs().max()) <= 2.0 ** -13 * float(x.abs().max())


def test_own_frequencies_and_inverse():
    g = torch.Generator().manual_seed(11)
    x = torch.randn(1, 2, 8, 64, generator=g)
    f = torch.rand(32, generator=g)
    pos = torch.arange(8)
    y = rotary(x.cuda(), pos.cuda(), freqs=f.cuda())
    close_rows(y, rotate(x.double(), pos.view(1, 8, 1), 64, f.double(), [0] * 32, False), torch.float32)
    back = rotary(y, pos.cuda(), freqs=f.cuda(), inverse=True)
    assert float((back.cpu() - x).abs().max()) <= 2.0 ** -19 * float(x.abs().max())


def test_rows_of_zeros_and_special_values():
    x = torch.zeros(1, 1, 4, 64)
    x[0, 0, 1] = 1.0
    x[0, 0, 2, 5] = float("nan")
    x[0, 0, 3, 7] = float("inf")
    y = qk_norm_rope(x.cuda(), None, torch.zeros(4, dtype=torch.int64).cuda())[0].cpu()
    assert bool((y[0, 0, 0] == 0).all())
    torch.testing.assert_close(y[0, 0, 1], torch.ones(64), rtol=1e-6, atol=0)
    assert bool(y[0, 0, 2].isnan().all())  # the mean square is NaN
    # an infinite element: its own quotient is inf * 0, the others' are 0
    assert bool(y[0, 0, 3, 7].isnan()) and bool((y[0, 0, 3, :7] == 0).all())
    # a neighbour's row is not touched
    gx = torch.ones_like(x).cuda()
    xd = x.cuda().requires_grad_(True)
    dx, = torch.autograd.grad(qk_norm_rope(xd, None, torch.zeros(4, dtype=torch.int64).cuda(), eps=1e-6)[0], xd, gx)
    assert bool(dx[0, 0, :2].isfinite().all())


def test_empty_and_missing_tensors():
    pos = torch.zeros(0, dtype=torch.int64).cuda()
    q = torch.empty(2, 3, 0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    o, none = qk_norm_rope(q, None, pos, w)
    assert o.shape == q.shape and none is None
    dq, dw = torch.autograd.grad(o, (q, w), torch.empty_like(o))
    assert dq.shape == q.shape and bool((dw == 0).all())
    assert rotary(torch.empty(0, 3, 5, 64, device="cuda"), torch.arange(5).cuda()).shape == (0, 3, 5, 64)


def test_gradient_of_one_input_and_broadcast_gradients():
    g = torch.Generator().manual_seed(13)
    q, k = torch.randn(1, 2, 5, 64, generator=g).cuda(), torch.randn(1, 1, 5, 64, generator=g).cuda()
    w = torch.randn(64, generator=g).cuda()
    pos = torch.arange(5).cuda()
    full = [t.clone().requires_grad_(True) for t in (q, k, w)]
    a, b = qk_norm_rope(full[0], full[1], pos, full[2], full[2])  # one gain for both: gradients add
    want = torch.autograd.grad(a.sum() + b.sum(), full)
    kk = k.clone().requires_grad_(True)
    _, ok = qk_norm_rope(q, kk, pos, w, w)
    assert torch.equal(torch.autograd.grad(ok.sum(), kk)[0], want[1])  # an expanded scalar gradient
    sep = [w.clone().requires_grad_(True) for _ in range(2)]
    a, b = qk_norm_rope(q, k, pos, sep[0], sep[1])
    gw = torch.autograd.grad(a.sum() + b.sum(), sep)
    torch.testing.assert_close(gw[0] + gw[1], want[2])


def test_fp32_gains_on_16_bit_rows_and_determinism():
    g = torch.Generator().manual_seed(17)
    q = torch.randn(2, 8, 700, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_(True)
    w = torch.randn(64, generator=g).cuda().requires_grad_(True)
    pos = torch.arange(700).cuda()
    go = torch.randn(2, 8, 700, 64, generator=g).to(torch.bfloat16).cuda()
    res = []
    for _ in range(2):
        o, _ = qk_norm_rope(q, None, pos, w)
        res.append((o.detach(),) + torch.autograd.grad(o, (q, w), go))
    assert res[0][2].dtype == torch.float32
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_other_stream():
    x = torch.randn(1, 4, 512, 64, device="cuda")
    pos = torch.arange(512, device="cuda")
    want = rotary(x, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rotary(x, pos)
    s.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    x = torch.randn(1, 2, 4, 64, device="cuda")
    pos = torch.arange(4, device="cuda")
    with pytest.raises(TypeError):
        rotary(x.double(), pos)
    with pytest.raises(RuntimeError):
        rotary(x.cpu(), pos)
    with pytest.raises(RuntimeError):
        rotary(x[0], pos)
    with pytest.raises(TypeError):
        rotary(x, pos.short())
    with pytest.raises(RuntimeError):
        rotary(x, pos[:3])
    with pytest.raises(RuntimeError):
        rotary(x, pos, rotary_dim=65)
    with pytest.raises(RuntimeError):
        rotary(x, pos, rotary_dim=66)
    with pytest.raises(RuntimeError):
        rotary(x, pos.view(4, 1).expand(4, 2), sections=(16, 15))
    with pytest.raises(ValueError):
        rotary(x, pos, spectrum="both")
    with pytest.raises(RuntimeError):
        rotary(torch.randn(1, 2, 4, 63, device="cuda"), pos, rotary_dim=62)
    with pytest.raises(RuntimeError):
        rotary(torch.randn(1, 2, 4, 260, device="cuda"), pos)
    with pytest.raises(RuntimeError):
        rotary(x, pos, base=-1.0)
    with pytest.raises(TypeError):
        qk_norm_rope(x, x.half(), pos)
    with pytest.raises(RuntimeError):
        qk_norm_rope(x, x[:, :, :3], pos)
    with pytest.raises(TypeError):
        qk_norm_rope(x, None, pos, torch.ones(64, device="cuda", dtype=torch.float16))
    with pytest.raises(RuntimeError):
        qk_norm_rope(x, None, pos, torch.ones(32, device="cuda"))
    with pytest.raises(RuntimeError):
        qk_norm_rope(x, None, pos, None, torch.ones(64, device="cuda"))
