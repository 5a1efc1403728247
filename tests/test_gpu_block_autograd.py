"""What autograd asks of the block operators beyond a plain backward."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from murmurative_attention_b200 import fused_linear, qk_norm_rope, rotary

pytestmark = pytest.mark.gpu


def rand(*shape):
    return torch.randn(*shape, device="cuda")


def calls():
    """name -> (function of its differentiable inputs, those inputs)"""
    pos = torch.arange(5, device="cuda")
    return {
        "linear": (lambda x, w, b, r: fused_linear(x, w, b, activation="silu", residual=r),
                   [rand(5, 16), rand(8, 16), rand(8), rand(5, 8)]),
        "qk": (lambda q, k, a, b: qk_norm_rope(q, k, pos, a, b)[0],
               [rand(1, 2, 5, 16), rand(1, 1, 5, 16), rand(16), rand(16)]),
        "rotary": (lambda x: rotary(x, pos), [rand(1, 2, 5, 16)]),
    }


@pytest.mark.parametrize("name", ["linear", "qk", "rotary"])
def test_forward_mode_raises(name):
    """No tangent is dropped in silence, whichever input has it."""
    f, inputs = calls()[name]
    for i in range(len(inputs)):
        with fwd.dual_level():
            ts = list(inputs)
            ts[i] = fwd.make_dual(ts[i], torch.ones_like(ts[i]))
            with pytest.raises(NotImplementedError):
                f(*ts)
    f(*inputs)  # and outside of it the call is as before


@pytest.mark.parametrize("name", ["linear", "qk", "rotary"])
def test_jit_trace_raises(name):
    f, inputs = calls()[name]
    with pytest.raises(RuntimeError, match="torch.jit.trace"):
        torch.jit.trace(f, tuple(inputs), check_trace=False)


@pytest.mark.parametrize("name", ["linear", "qk", "rotary"])
def test_dispatch_modes_see_the_operators(name):
    """make_fx's graph gives the call's results on other inputs; a mode that records calls finds the operator."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    class Record(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    f, inputs = calls()[name]
    graph = make_fx(f)(*inputs)
    others = [t + 0.25 for t in inputs]
    torch.testing.assert_close(graph(*others), f(*others))
    seen = []
    with Record():
        out = f(*inputs)
    assert any("murmurative_attention" in s for s in seen) and torch.equal(out, f(*inputs))
    leaves = [t.clone().requires_grad_(True) for t in inputs]
    want = torch.autograd.grad(f(*leaves).square().sum(), leaves, allow_unused=True)
    with Record():
        loss = f(*leaves).square().sum()
    for a, b in zip(torch.autograd.grad(loss, leaves, allow_unused=True), want):
        assert (a is None or not bool(a.any())) if b is None else torch.equal(a, b)
