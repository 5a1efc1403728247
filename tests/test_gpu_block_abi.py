"""The block operators' C ABI on a GPU, where it takes more than the Python functions hand it."""
import ctypes

import pytest
import torch

from murmurative_attention_b200 import _lib, rotary

pytestmark = pytest.mark.gpu
CODES = {torch.float32: _lib.MURM_F32, torch.float16: _lib.MURM_F16, torch.bfloat16: _lib.MURM_BF16}
NAN = float("nan")


def set_rows(rows, x, out):
    rows.x, rows.out, rows.heads = x.data_ptr(), out.data_ptr(), x.shape[1]
    for i in range(3):
        rows.x_stride[i], rows.out_stride[i] = x.stride(i), out.stride(i)


def rope_args(x, pos, **kw):
    B, _, N, d = x.shape
    a = _lib.NormRopeArgs(batch=B, tokens=N, head_dim=d, rotary_dim=d, dtype=CODES[x.dtype], axes=1, eps=1e-6, base=1e4,
                          position_type=_lib.MURM_POS_I64)
    a.positions = pos.data_ptr() if pos is not None else None
    a.position_stride[1] = 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def run(a):
    assert _lib.load_library().murm_norm_rope_fwd(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("N,d", [(1, 64), (37, 72), (300, 128), (5, 10)])
@pytest.mark.parametrize("hq,hk", [(4, 1), (3, 7), (0, 2), (2, 0)])
def test_rotation_alone_takes_q_and_k(dtype, N, d, hq, hk):
    """Without the norm, every row of q and k: bit for bit what each gives by itself, with either absent."""
    g = torch.Generator().manual_seed(1)
    q, k = (torch.randn(2, h, N, d, generator=g).to(dtype).cuda() for h in (hq, hk))
    pos = torch.randint(0, 100000, (N,), generator=g).cuda()
    oq, ok = torch.full_like(q, NAN), torch.full_like(k, NAN)
    a = rope_args(q, pos)
    if hq:
        set_rows(a.q, q, oq)
    if hk:
        set_rows(a.k, k, ok)
    run(a)
    for x, o in ((q, oq), (k, ok)):
        assert torch.equal(o, rotary(x, pos))


@pytest.mark.parametrize("dtype", list(CODES))
def test_nothing_rotated_needs_no_positions(dtype):
    """rotary_dim = 0: positions may be NULL, in the norm's forward and backward and in the rotation alone."""
    lib, st = _lib.load_library(), torch.cuda.current_stream().cuda_stream
    x = torch.randn(2, 3, 70, 64, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
    zeros = torch.zeros(70, dtype=torch.int64, device="cuda")
    res = []
    for pos in (zeros, None):
        out = torch.full_like(x, NAN)
        a = rope_args(x, pos, normalize=1, rotary_dim=0)
        set_rows(a.q, x, out)
        run(a)
        gx = torch.full_like(x, NAN)
        set_rows(a.q, x, gx)
        a.q.grad, a.q.grad_stride = x.data_ptr(), a.q.x_stride
        assert lib.murm_norm_rope_bwd(ctypes.byref(a), st) == 0
        torch.cuda.synchronize()
        res.append((out, gx))
    assert all(torch.equal(p, q) and bool(p.isfinite().all()) for p, q in zip(*res))
    copy = torch.full_like(x, NAN)
    a = rope_args(x, None, rotary_dim=0)
    set_rows(a.q, x, copy)
    run(a)
    assert torch.equal(copy, x)


def test_bias_gradient_of_the_widest_layer():
    """Column offsets pass 2^31 in the last block; one row, so that the sums are its elements."""
    n = (1 << 31) - 1032
    go = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    go.view(torch.int16).copy_(torch.arange(1 << 14, device="cuda", dtype=torch.int16).repeat((n >> 14) + 1)[:n])
    gb = torch.full_like(go, NAN)
    a = _lib.LinearBwdArgs(rows=1, in_features=1, out_features=n, dtype=_lib.MURM_BF16, grad_out=go.data_ptr(), go_stride=n,
                           grad_bias=gb.data_ptr())
    need = ctypes.c_size_t(0)
    lib = _lib.load_library()
    assert lib.murm_linear_bwd_workspace(ctypes.byref(a), ctypes.byref(need)) == 0 and need.value == 0
    assert lib.murm_linear_bwd(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(gb, go)
