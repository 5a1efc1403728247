"""Refusals of the block operators without a GPU: fake CUDA tensors go through the compiled binding's
checks (which raise before anything is allocated or launched) and through the registered operators' fakes,
which have to refuse while tracing what the eager call refuses."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from murmurative_attention_b200 import _lib, _native, fused_linear, qk_norm_rope, rotary, torch_ops

NS = torch.ops.murmurative_attention


@pytest.fixture
def fake():
    with FakeTensorMode():
        yield lambda *shape, dtype=torch.bfloat16, device="cuda": torch.empty(shape, dtype=dtype, device=device)


# x [4, 64], weight [32, 64] bf16 and one thing wrong
LINEAR = [
    (dict(weight=(32, 128)), RuntimeError), (dict(weight=(32, 32)), RuntimeError), (dict(weight=(64,)), RuntimeError),
    (dict(weight=(32, 64), weight_dtype=torch.float32), TypeError), (dict(weight_device="cpu"), RuntimeError),
    (dict(weight=(0, 64)), RuntimeError),
    (dict(bias=(4,)), RuntimeError), (dict(bias=(1, 32)), RuntimeError), (dict(bias=(32,), bias_dtype=torch.float32), TypeError),
    (dict(bias=(32,), bias_device="cpu"), RuntimeError),
    (dict(residual=(3, 32)), RuntimeError), (dict(residual=(4, 31)), RuntimeError),
    (dict(residual=(4, 32), residual_dtype=torch.float32), TypeError), (dict(residual=(4, 32), residual_device="cpu"), RuntimeError),
    (dict(activation="swish"), ValueError), (dict(x_dtype=torch.float64, weight_dtype=torch.float64), TypeError),
]


def linear_args(fake, c):
    make = lambda name, default: fake(*c.get(name, default), dtype=c.get(f"{name}_dtype", torch.bfloat16),
                                      device=c.get(f"{name}_device", "cuda"))
    return (make("x", (4, 64)), make("weight", (32, 64)), make("bias", ()) if "bias" in c else None,
            c.get("activation", "gelu"), make("residual", ()) if "residual" in c else None)


@pytest.mark.parametrize("case,error", LINEAR)
def test_linear_refused_everywhere(fake, case, error):
    args = linear_args(fake, case)
    for call in (NS.fused_linear_fwd, torch_ops.fused_linear, _native.binding().fused_linear, _native.binding().linear_fwd):
        with pytest.raises(error):
            call(*args)


@pytest.mark.parametrize("case,error", [
    (dict(go=(4, 31)), RuntimeError), (dict(go=(3, 32)), RuntimeError), (dict(go_dtype=torch.float32), TypeError),
    (dict(go_device="cpu"), RuntimeError), (dict(slope=(4, 31)), RuntimeError), (dict(slope=(0,)), RuntimeError),
    (dict(slope_dtype=torch.bfloat16), TypeError), (dict(slope_device="cpu"), RuntimeError),
    (dict(weight=(32, 128)), RuntimeError), (dict(weight_device="cpu"), RuntimeError), (dict(activation="swish"), ValueError),
])
def test_linear_gradients_refused(fake, case, error):
    x, w, _, act, _ = linear_args(fake, case)
    go = fake(*case.get("go", (4, 32)), dtype=case.get("go_dtype", torch.bfloat16), device=case.get("go_device", "cuda"))
    slope = fake(*case.get("slope", (4, 32)), dtype=case.get("slope_dtype", torch.int16),
                 device=case.get("slope_device", "cuda"))
    for call in (NS.fused_linear_bwd, _native.binding().linear_bwd):
        with pytest.raises(error):
            call(go, x, w, slope, act)


@pytest.mark.parametrize("case,error", [
    (dict(gq=(1, 2, 4, 64)), RuntimeError), (dict(gq=(1, 2, 5, 32)), RuntimeError), (dict(gk=(1, 2, 5, 64)), RuntimeError),
    (dict(gq_dtype=torch.float32), TypeError), (dict(gk_device="cpu"), RuntimeError),
])
def test_norm_rope_gradients_refused(fake, case, error):
    q, k, pos = fake(1, 2, 5, 64), fake(1, 1, 5, 64), fake(5, dtype=torch.int64)
    gq = fake(*case.get("gq", (1, 2, 5, 64)), dtype=case.get("gq_dtype", torch.bfloat16))
    gk = fake(*case.get("gk", (1, 1, 5, 64)), device=case.get("gk_device", "cuda"))
    rest = (None, None, 1e-6, 1e4, None, False, None, "shared", None)
    for call in (NS.qk_norm_rope_bwd, _native.binding().qk_bwd):
        with pytest.raises(error):
            call(gq, gk, q, k, pos, *rest)


def test_what_fits_is_traced(fake):
    x, w, b, r = fake(4, 64), fake(32, 64), fake(32), fake(4, 32)
    out, slope = NS.fused_linear_fwd(x, w, b, "gelu", r)
    assert out.shape == slope.shape == (4, 32) and slope.dtype == torch.int16
    assert [t.shape for t in NS.fused_linear_bwd(out, x, w, slope, "gelu")] == [(4, 64), (32, 64), (32,)]
    assert torch_ops.fused_linear(fake(2, 3, 64), w, b, "none", fake(3, 32)).shape == (2, 3, 32)


@pytest.mark.parametrize("kw,status", [
    (dict(), 0), (dict(positions=4100, position_type=_lib.MURM_POS_I32), 0),
    (dict(positions=4100), 1), (dict(positions=4098, position_type=_lib.MURM_POS_F32), 1), (dict(freqs=4098), 1),
    (dict(weight=4097), 1), (dict(weight=4098), 0), (dict(weight=4098, weight_dtype=_lib.MURM_F32), 1),
])
def test_norm_rope_pointers_are_aligned(kw, status):
    """No batch: a call that passes the checks launches nothing."""
    a = _lib.NormRopeArgs(batch=0, tokens=4, head_dim=64, rotary_dim=64, dtype=_lib.MURM_F16, normalize=1, axes=1,
                          eps=1e-6, base=1e4, positions=4096)
    a.q.heads, a.q.weight_dtype = 2, _lib.MURM_F16
    for k, v in kw.items():
        setattr(a.q if k.startswith("weight") else a, k, v)
    if "freqs" in kw:
        a.freqs = kw["freqs"]
    assert _lib.load_library().murm_norm_rope_fwd(ctypes.byref(a), None) == status


@pytest.mark.parametrize("big", [1 << 31, (1 << 32) + 8])
def test_sizes_past_32_bits_are_refused(fake, big):
    """They were cut to 32 bits: 2^32 + 8 features computed with 8."""
    binding = _native.binding()
    pos = fake(4, dtype=torch.int64)
    for x, w in (((4, big), (3, big)), ((4, 8), (big, 8))):
        with pytest.raises(RuntimeError, match="2\\^31"):
            binding.fused_linear(fake(*x), fake(*w), None, "none", None)
        with pytest.raises(RuntimeError, match="2\\^31"):
            binding.linear_fwd(fake(*x), fake(*w), None, "none", None)
    for shape in ((big, 1, 4, 2), (1, big, 4, 2), (1, 1, big, 2), (1, 1, 4, big)):
        rest = (1e4, None, False, None, "shared", None)
        p = pos if shape[2] == 4 else fake(shape[2], dtype=torch.int64)
        with pytest.raises(RuntimeError, match="2\\^31"):
            binding.rotary(fake(*shape), p, *rest, False)
        with pytest.raises(RuntimeError, match="2\\^31"):
            binding.qk_norm_rope(fake(*shape), None, p, None, None, 1e-6, *rest)


@pytest.mark.parametrize("rows,n", [(8, 1 << 24), (300, 1 << 20), (8, (1 << 31) - 1032), (20000, 64), (5000, 100000)])
@pytest.mark.parametrize("act", [0, 1])
def test_bias_gradient_needs_no_more_than_its_chunks(rows, n, act):
    """The partial sums of db alone: at most one row of them per 24 rows of dz, none where one block sums a
    column (512 rows of them whatever the sizes took 34 GB beside 2^24 outputs)."""
    a = _lib.LinearBwdArgs(rows=rows, in_features=64, out_features=n, dtype=_lib.MURM_BF16, activation=act, slope=4096,
                           grad_out=8192, go_stride=n, grad_bias=16384)
    need = ctypes.c_size_t(0)
    assert _lib.load_library().murm_linear_bwd_workspace(ctypes.byref(a), ctypes.byref(need)) == 0
    assert need.value <= (rows // 24 + 1) * n * 4 * (rows > 16) + 256


def test_public_functions_take_fake_tensors(fake):
    """Under a fake mode the functions give fakes of their results, and refuse what does not fit."""
    x, w = fake(2, 3, 64), fake(32, 64)
    assert fused_linear(x, w, fake(32), activation="silu").shape == (2, 3, 32)
    with pytest.raises(RuntimeError):
        fused_linear(x, fake(32, 65))
    q = fake(2, 5, 4, 64).transpose(1, 2)
    pos = fake(5, dtype=torch.int64)
    assert rotary(q, pos).stride() == q.stride()
    oq, ok = qk_norm_rope(q, q[:, :2], pos)
    assert oq.shape == q.shape and ok.shape == (2, 2, 5, 64)
