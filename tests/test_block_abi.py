"""The block operators' C ABI without a GPU: struct layouts against the header, argument checks and
their status codes, workspace sizes."""
import ctypes
import os
import shutil
import subprocess

import pytest

from murmurative_attention_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts_match_header(tmp_path):
    structs = [("murm_head_rows", _lib.HeadRows), ("murm_norm_rope_args", _lib.NormRopeArgs),
               ("murm_linear_args", _lib.LinearArgs), ("murm_linear_bwd_args", _lib.LinearBwdArgs)]
    body, want = "", []
    for name, st in structs:
        body += f'printf("%zu ", sizeof({name}));'
        want.append(ctypes.sizeof(st))
        for field, _ in st._fields_:
            body += f'printf("%zu ", offsetof({name}, {field}));'
            want.append(getattr(st, field).offset)
    src = tmp_path / "block.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "murm.h"\nint main(void){' + body + "return 0;}\n")
    exe = tmp_path / "block"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def _linear(**kw):
    a = _lib.LinearArgs(8, 64, 32, _lib.MURM_F16, 0, 4096, 64, 8192, 64, None, None, 0, 16384, 32)
    for k, v in kw.items():
        setattr(a, k, v)
    n = ctypes.c_size_t(0)
    return _lib.load_library().murm_linear_workspace(ctypes.byref(a), ctypes.byref(n)), n.value


@pytest.mark.parametrize("kw,status", [
    (dict(), 0), (dict(rows=0), 0), (dict(rows=-1), 1), (dict(in_features=0), 1), (dict(out_features=0), 1),
    (dict(dtype=5), 3), (dict(activation=9), 1), (dict(x=None), 1), (dict(weight=None), 1), (dict(out=None), 1),
    (dict(x=4097), 1), (dict(x_stride=63), 1), (dict(w_stride=10), 1), (dict(out_stride=31), 1),
    (dict(residual=4096, r_stride=31), 1), (dict(rows=1 << 40), 2),
])
def test_linear_argument_checks(kw, status):
    got, _ = _linear(**kw)
    assert got == status
    if status:
        assert _lib.load_library().murm_last_error_message()


def test_linear_workspaces():
    lib = _lib.load_library()
    assert _linear()[1] == 0                                     # few rows, read in place
    assert _linear(x=4098, rows=30000)[1] >= 30000 * 64 * 2      # a copy TMA can address
    assert _linear(dtype=_lib.MURM_F32, rows=30000)[1] >= 3 * 2 * (30000 + 32) * 64  # three planes of both operands
    b = _lib.LinearBwdArgs(300, 64, 32, _lib.MURM_F16, 1, 4096, 64, 8192, 64, 16384, 32768, 32, 65536, 64, 131072, 64,
                           262144)
    n = ctypes.c_size_t(0)
    assert lib.murm_linear_bwd_workspace(ctypes.byref(b), ctypes.byref(n)) == 0
    assert n.value >= 300 * 32 * 2                               # dz
    b.slope = None
    assert lib.murm_linear_bwd_workspace(ctypes.byref(b), ctypes.byref(n)) == 1  # the activation's slopes are needed
    b.activation = 0
    assert lib.murm_linear_bwd_workspace(ctypes.byref(b), ctypes.byref(n)) == 0
    for fn in (lib.murm_linear_fwd, lib.murm_linear_bwd, lib.murm_norm_rope_fwd, lib.murm_norm_rope_bwd):
        assert fn(None, None) == 1


def _rope(**kw):
    a = _lib.NormRopeArgs(batch=0, tokens=4, head_dim=64, rotary_dim=64, dtype=_lib.MURM_F16, normalize=1, axes=1,
                          eps=1e-6, base=1e4)  # no batch: a call that passes the checks launches nothing
    a.q.heads = 2
    for k, v in kw.items():
        if k == "sections":
            a.sections[:len(v)] = v
        else:
            setattr(a, k, v)
    return _lib.load_library().murm_norm_rope_fwd(ctypes.byref(a), None)


@pytest.mark.parametrize("kw,status", [
    (dict(), 0), (dict(batch=-1), 1), (dict(head_dim=63), 2), (dict(head_dim=258), 2), (dict(rotary_dim=65), 1),
    (dict(rotary_dim=66), 1), (dict(rotary_dim=0), 0), (dict(dtype=4), 3), (dict(axes=0), 1), (dict(axes=5), 1),
    (dict(axes=2, sections=(16, 16)), 0), (dict(axes=2, sections=(16, 15)), 1), (dict(axes=2, sections=(33, -1)), 1),
    (dict(position_type=3), 3), (dict(base=0.0), 1), (dict(base=float("inf")), 1), (dict(eps=-1.0), 1),
    (dict(eps=float("nan")), 1),
])
def test_norm_rope_argument_checks(kw, status):
    assert _rope(**kw) == status
    if status:
        assert _lib.load_library().murm_last_error_message()


def test_norm_rope_backward_checks():
    lib = _lib.load_library()
    assert lib.murm_norm_rope_workspace() > 0
    a = _lib.NormRopeArgs(batch=1, tokens=4, head_dim=64, rotary_dim=64, dtype=_lib.MURM_F16, normalize=0, axes=1,
                          eps=1e-6, base=1e4, positions=4096)
    assert lib.murm_norm_rope_bwd(ctypes.byref(a), None) == 1    # the rotation's backward is the forward, inverse
    a.normalize = 1
    a.q.heads, a.q.x, a.q.out = 1, 4096, 8192
    assert lib.murm_norm_rope_bwd(ctypes.byref(a), None) == 1    # no gradient
    a.q.grad, a.q.grad_weight, a.q.weight_dtype = 4096, 4096, _lib.MURM_F16
    for i, s in enumerate((256, 256, 64)):
        a.q.x_stride[i] = a.q.out_stride[i] = a.q.grad_stride[i] = s
    assert lib.murm_norm_rope_bwd(ctypes.byref(a), None) == 4    # a gain gradient needs the workspace
