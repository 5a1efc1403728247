"""The block operators do what a call's gradients need and no more: slopes are saved, gradients formed and
kernels launched for wanted gradients only, in eager calls and under torch.compile alike."""
import pytest
import torch

from murmurative_attention_b200 import _lib, fused_linear, qk_norm_rope

pytestmark = pytest.mark.gpu


def launches(f):
    lib = _lib.load_library()
    f()
    before = lib.murm_kernel_launches()
    out = f()
    return lib.murm_kernel_launches() - before, out


def linear_inputs(m=300, k=64, n=128):
    g = torch.Generator().manual_seed(61)
    return [torch.randn(s, generator=g).cuda() for s in ((m, k), (n, k), (n,), (m, n))]


def compiled(f):
    """f under torch.compile (eager kernels) and the traced calls' arguments by operator."""
    calls = {}

    def backend(gm, _):
        for node in gm.graph.nodes:
            if node.op == "call_function":
                calls.setdefault(str(node.target), []).append(node.args)
        return gm.forward

    torch._dynamo.reset()
    return torch.compile(f, fullgraph=True, backend=backend), calls


@pytest.mark.parametrize("grad", [False, True])
def test_compiled_inference_saves_no_slopes(grad):
    x, w, b, r = linear_inputs()
    w.requires_grad_(True)
    f, calls = compiled(lambda x, r: fused_linear(x, w, b, activation="gelu", residual=r))
    with torch.set_grad_enabled(grad):
        got = f(x, r)
        want = fused_linear(x, w, b, activation="gelu", residual=r)
    assert torch.equal(got, want)
    (args,) = [a for name, c in calls.items() if "fused_linear_fwd" in name for a in c]
    assert args[5] is grad


def test_slopes_only_where_they_are_read():
    x, w, b, r = linear_inputs()
    op = torch.ops.murmurative_attention
    assert op.fused_linear_fwd(x, w, b, "gelu", r, False)[1].numel() == 0
    assert op.fused_linear_fwd(x, w, b, "gelu", r)[1].shape == r.shape
    rr = r.clone().requires_grad_(True)  # the residual's gradient is the upstream one
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = fused_linear(x, w, b, activation="gelu", residual=rr)
    held = torch.cuda.memory_allocated() - before
    assert held <= out.numel() * 4 + 512
    go = torch.randn_like(out)
    assert torch.equal(torch.autograd.grad(out, rr, go)[0], go)
    f, _ = compiled(lambda r: fused_linear(x, w, b, activation="gelu", residual=r))
    assert torch.equal(torch.autograd.grad(f(rr), rr, go)[0], go)


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 1), (1, 2), (0, 1, 2), (3,)])
def test_wanted_gradients_alone(wanted):
    """Eager and compiled: the same gradients by the same number of launches."""
    ts = linear_inputs()
    go = torch.randn_like(ts[3])
    res = []
    for compile_it in (False, True):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(ts)]
        f = lambda x, w, b, r: fused_linear(x, w, b, activation="silu", residual=r)
        if compile_it:
            torch._dynamo.reset()
            f = torch.compile(f, fullgraph=True, backend="aot_eager")
        out = f(*leaves)
        res.append(launches(lambda: torch.autograd.grad(out, [leaves[i] for i in wanted], go, retain_graph=True)))
    assert res[0][0] == res[1][0]
    assert all(torch.equal(a, b) for a, b in zip(res[0][1], res[1][1]))


def test_frozen_gain_costs_no_sum():
    """The sum over the blocks' parts of a gain's gradient is a launch of its own."""
    g = torch.Generator().manual_seed(62)
    q, k = (torch.randn(2, h, 50, 64, generator=g).cuda() for h in (4, 2))
    gains = [torch.randn(64, generator=g).cuda() for _ in range(2)]
    pos = torch.arange(50).cuda()
    res = {}
    for trained in ((), (0,), (0, 1)):
        ws = [w.clone().requires_grad_(i in trained) for i, w in enumerate(gains)]
        qs, ks = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        out = qk_norm_rope(qs, ks, pos, *ws)
        go = [torch.ones_like(o) for o in out]
        want = [qs, ks] + [ws[i] for i in trained]
        res[trained] = launches(lambda: torch.autograd.grad(out, want, go, retain_graph=True))
    assert res[()][0] == 1 and res[(0,)][0] == res[(0, 1)][0] == 2
    for r in res.values():
        assert all(torch.equal(a, b) for a, b in zip(r[1], res[(0, 1)][1]))


@pytest.mark.parametrize("wanted", [(0,), (1,), (0, 1), (2,), (3,), (0, 3), (1, 2), (0, 1, 2, 3)])
def test_wanted_norm_gradients_alone(wanted):
    g = torch.Generator().manual_seed(63)
    ts = [torch.randn(2, h, 50, 64, generator=g).cuda() for h in (4, 2)] + [torch.randn(64, generator=g).cuda() for _ in range(2)]
    pos = torch.arange(50).cuda()
    res = []
    for compile_it in (False, True):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate(ts)]
        f = lambda q, k, a, b: qk_norm_rope(q, k, pos, a, b)
        if compile_it:
            torch._dynamo.reset()
            f = torch.compile(f, fullgraph=True, backend="aot_eager")
        out = f(*leaves)
        loss = sum((o * torch.linspace(1, 2, o.numel(), device="cuda").view_as(o)).sum() for o in out)
        res.append(launches(lambda: torch.autograd.grad(loss, [leaves[i] for i in wanted], retain_graph=True)))
    assert res[0][0] == res[1][0] == 1 + any(i > 1 for i in wanted)
    assert all(torch.equal(a, b) for a, b in zip(res[0][1], res[1][1]))
