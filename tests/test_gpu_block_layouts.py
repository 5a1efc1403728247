"""Rows of the rotation's operators that share memory: windows that slide over a sequence, one row for all
tokens. Results, gradients and the registered operators' fakes against the same call on a copy."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from murmurative_attention_b200 import qk_norm_rope, rotary, torch_ops
from test_gpu_block_large import rope_reference
from test_gpu_rope import close_rows


def layouts(base):
    """Views [2, 3, N, 16] of base [2, 3, 40] whose rows overlap."""
    return [base[..., :20].unfold(2, 16, 1), base.unfold(2, 16, 1), base[..., :16].unsqueeze(2).expand(2, 3, 5, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_overlapping_rows(which, dtype):
    """The rotation bit for bit as on a copy (it sums nothing); the norm, whose sum over a row goes by
    the width of its loads, against the definition within its bounds."""
    g = torch.Generator().manual_seed(1)
    x = layouts(torch.randn(2, 3, 40, generator=g).to(dtype).cuda())[which]
    pos = torch.randint(0, 5000, (2, x.shape[2]), generator=g).cuda()
    go = torch.randn(x.shape, generator=g).to(dtype).cuda()
    w = torch.randn(16, generator=g).to(dtype).cuda()
    res = []
    for t in (x, x.contiguous()):
        t = t.detach().requires_grad_(True)
        out = rotary(t, pos)
        res.append((out.detach(),) + torch.autograd.grad(out, t, go))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    want, wdx, scale, _ = rope_reference(x, w, go, pos, 1e-6)
    for f in (lambda t: qk_norm_rope(t, None, pos, w)[0], lambda t: qk_norm_rope(go, t, pos, w, w)[1]):
        t = x.detach().requires_grad_(True)
        out = f(t)
        close_rows(out.detach(), want, dtype)
        close_rows(torch.autograd.grad(out, t, go)[0], wdx, dtype, scale)


@pytest.mark.parametrize("which", range(3))
def test_fakes_keep_rows_together(which):
    with FakeTensorMode():
        x = layouts(torch.empty(2, 3, 40, device="cuda"))[which]
        assert torch_ops._unit_layout(x).stride(3) == 1
