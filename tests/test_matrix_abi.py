"""The matrix operators' C ABI and Python checks on the CPU: exported symbols,
struct layouts, and refusals that never reach a GPU."""
import ctypes
import os
import re
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "turboadam_b200_matrix.h")

INVALID, ALIGN, UNSUPPORTED, WORKSPACE = 1, 2, 3, 4


@pytest.fixture(scope="module")
def lib():
    from turboadam_b200 import _lib
    from turboadam_b200.csrc import build

    build.build(quiet=True)
    return _lib.load()


def test_header_symbols_exported(lib):
    from turboadam_b200 import _lib

    src = open(HEADER).read()
    names = sorted(set(re.findall(r"TA_API\s+[\w\s\*]+?\b(ta_\w+)\s*\(", src)))
    assert sorted(_lib.MATRIX_EXPORTED) == names
    for n in names:
        assert hasattr(lib, n), n


def test_struct_layout_matches_header():
    from turboadam_b200 import _lib

    structs = {"ta_ortho_tensor": _lib.TaOrthoTensor, "ta_ortho_options": _lib.TaOrthoOptions,
               "ta_linear": _lib.TaLinear, "ta_linear_grad": _lib.TaLinearGrad}
    body, want = [], []
    for name, cls in structs.items():
        body.append(f'printf("%zu ", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f in cls._fields_:
            body.append(f'printf("%zu ", offsetof({name}, {f[0]}));')
            want.append(getattr(cls, f[0]).offset)
    prog = ("#include <stdio.h>\n#include <stddef.h>\n#include \"turboadam_b200_matrix.h\"\n"
            "int main(void) { " + "\n".join(body) + " return 0; }\n")
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        with open(c, "w") as f:
            f.write(prog)
        subprocess.check_call(["gcc", "-I", os.path.dirname(HEADER), c, "-o", exe])
        got = [int(v) for v in subprocess.check_output([exe]).split()]
    assert got == want


# ---------------------------------------------------------------------------
def _ortho(**over):
    from turboadam_b200 import _lib

    t = (_lib.TaOrthoTensor * 1)()
    t[0].in_dev, t[0].out_dev = 4096, 8192
    t[0].batch, t[0].rows, t[0].cols = 2, 96, 70
    t[0].in_dtype, t[0].out_dtype = _lib.TA_F32, _lib.TA_BF16
    arr = (ctypes.c_double * 15)(*([3.4445, -4.775, 2.0315] * 5))
    o = _lib.TaOrthoOptions(ctypes.cast(arr, ctypes.c_void_p), 5, 0, 1e-7, 0.0)
    o._keep = arr
    for k, v in over.items():
        setattr(o if hasattr(o, k) else t[0], k, v)
    return t, o


@pytest.mark.parametrize("over,code", [
    ({"in_dtype": 7}, INVALID),
    ({"out_dtype": 3}, INVALID),
    ({"momentum_dev": 16384, "momentum_dtype": 9}, INVALID),
    ({"rows": -1}, INVALID),
    ({"in_dev": 0}, INVALID),
    ({"out_dev": None}, INVALID),
    ({"in_dev": 4098}, ALIGN),
    ({"out_dev": 8193}, ALIGN),
    ({"rows": 1 << 31}, UNSUPPORTED),
    ({"steps": 0}, INVALID),
    ({"steps": 33}, INVALID),
    ({"eps": -1.0}, INVALID),
    ({"eps": float("nan")}, INVALID),
    ({"coefficients": None}, INVALID),
])
def test_ortho_refusals(lib, over, code):
    t, o = _ortho(**over)
    assert lib.ta_ortho_workspace_size(t, 1, ctypes.byref(o)) == 0
    assert lib.ta_last_error()
    rc = lib.ta_orthogonalize(t, 1, ctypes.byref(o), 1 << 20, 1 << 40, 1 << 10, None)
    assert rc == code, lib.ta_last_error()
    assert lib.ta_last_error()


def test_ortho_workspace_refusals(lib):
    t, o = _ortho()
    need = lib.ta_ortho_workspace_size(t, 1, ctypes.byref(o))
    # two scaled copies and three square matrices of each
    assert need > 2 * (2 * 96 * 72 + 3 * 70 * 72) * 2
    call = lib.ta_orthogonalize
    assert call(t, 1, ctypes.byref(o), 1 << 20, need - 1, 1 << 10, None) == WORKSPACE
    assert call(t, 1, ctypes.byref(o), None, need, 1 << 10, None) == INVALID
    assert call(t, 1, ctypes.byref(o), (1 << 20) + 16, need, 1 << 10, None) == ALIGN
    assert call(t, 1, ctypes.byref(o), 1 << 20, need, None, None) == INVALID


def test_ortho_empty_lists_do_nothing(lib):
    for over in ({"batch": 0}, {"rows": 0}, {"cols": 0}):
        t, o = _ortho(**over)
        assert lib.ta_orthogonalize(t, 1, ctypes.byref(o), None, 0, None, None) == 0
    t, o = _ortho()
    assert lib.ta_orthogonalize(None, 0, ctypes.byref(o), None, 0, None, None) == 0


def _linear(**over):
    from turboadam_b200 import _lib

    op = _lib.TaLinear()
    op.x_dev, op.w_dev, op.y_dev = 1 << 20, 1 << 21, 1 << 22
    op.tokens, op.fan_in, op.fan_out = 8, 32, 16
    op.x_strides, op.w_strides = (ctypes.c_int64 * 2)(32, 1), (ctypes.c_int64 * 2)(32, 1)
    op.y_stride, op.residual_stride = 16, 16
    op.dtype = _lib.TA_BF16
    for k, v in over.items():
        setattr(op, k, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
    return op


@pytest.mark.parametrize("over,code", [
    ({"dtype": 0}, INVALID),
    ({"activation": 5}, INVALID),
    ({"activation": -1}, INVALID),
    ({"bias_dev": 4096, "bias_dtype": 4}, INVALID),
    ({"tokens": -1}, INVALID),
    ({"fan_in": 1 << 31}, UNSUPPORTED),
    ({"x_strides": (64, 2)}, INVALID),
    ({"w_strides": (31, 1)}, INVALID),
    ({"x_dev": None}, INVALID),
    ({"y_dev": None}, INVALID),
    ({"y_stride": 15}, INVALID),
    ({"y_stride": 1 << 31}, UNSUPPORTED),
    ({"deriv_dev": 4098}, ALIGN),
])
def test_linear_refusals(lib, over, code):
    op = _linear(**over)
    rc = lib.ta_linear_forward(ctypes.byref(op), 1 << 23, 1 << 40, 1 << 10, None)
    assert rc == code, lib.ta_last_error()
    assert lib.ta_last_error()


def test_linear_workspace_refusals(lib):
    op = _linear()
    need = lib.ta_linear_workspace_size(ctypes.byref(op))
    # rows that do not start on 16 bytes are copied
    odd = _linear(fan_in=33, x_strides=(33, 1), w_strides=(33, 1))
    assert lib.ta_linear_workspace_size(ctypes.byref(odd)) > need
    call = lib.ta_linear_forward
    if need:
        assert call(ctypes.byref(op), 1 << 23, need - 1, 1 << 10, None) == WORKSPACE
    need = lib.ta_linear_workspace_size(ctypes.byref(odd))
    assert call(ctypes.byref(odd), 1 << 23, need - 1, 1 << 10, None) == WORKSPACE
    assert call(ctypes.byref(odd), 1 << 23, need, None, None) == INVALID


def _grad(**over):
    from turboadam_b200 import _lib

    op = _lib.TaLinearGrad()
    op.dy_dev, op.x_dev, op.w_dev = 1 << 20, 1 << 21, 1 << 22
    op.dx_dev, op.dw_dev = 1 << 23, 1 << 24
    op.tokens, op.fan_in, op.fan_out, op.dy_stride = 8, 32, 16, 16
    for k in ("x_strides", "w_strides", "dw_strides"):
        setattr(op, k, (ctypes.c_int64 * 2)(32, 1))
    op.dtype = _lib.TA_F16
    for k, v in over.items():
        setattr(op, k, (ctypes.c_int64 * 2)(*v) if isinstance(v, tuple) else v)
    return op


@pytest.mark.parametrize("over,code", [
    ({"dtype": 0}, INVALID),
    ({"db_dev": 4096, "bias_dtype": -1}, INVALID),
    ({"dy_dev": None}, INVALID),
    ({"dy_stride": 15}, INVALID),
    ({"w_dev": None}, INVALID),
    ({"x_dev": None}, INVALID),
    ({"x_strides": (64, 2)}, INVALID),
    ({"dw_strides": (16, 1)}, INVALID),
    ({"deriv_dev": 4100}, ALIGN),
    ({"tokens": -2}, INVALID),
])
def test_linear_backward_refusals(lib, over, code):
    op = _grad(**over)
    rc = lib.ta_linear_backward(ctypes.byref(op), 1 << 25, 1 << 40, 1 << 10, None)
    assert rc == code, lib.ta_last_error()


def test_null_operators(lib):
    assert lib.ta_linear_forward(None, None, 0, None, None) == INVALID
    assert lib.ta_linear_backward(None, None, 0, None, None) == INVALID
    assert lib.ta_orthogonalize(None, 1, None, None, 0, None, None) == INVALID


# ---------------------------------------------------------------------------
def test_cpu_tensors_fail_loudly():
    from turboadam_b200 import Muon, linear_act, orthogonalize
    from turboadam_b200._lib import TurboAdamBackendError

    with pytest.raises(TurboAdamBackendError):
        orthogonalize(torch.randn(4, 4))
    with pytest.raises(TurboAdamBackendError):
        linear_act(torch.randn(4, 4).bfloat16(), torch.randn(4, 4).bfloat16())
    p = torch.nn.Parameter(torch.randn(4, 4))
    p.grad = torch.randn(4, 4)
    with pytest.raises(TurboAdamBackendError):
        Muon([p]).step()


def test_muon_constructor():
    from turboadam_b200 import Muon

    p = [torch.nn.Parameter(torch.randn(4, 4))]
    d = Muon(p).defaults
    assert (d["lr"], d["weight_decay"], d["momentum"], d["nesterov"], d["eps"], d["ns_steps"],
            d["ns_coefficients"]) == (1e-3, 0.1, 0.95, True, 1e-7, 5, (3.4445, -4.775, 2.0315))
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(ns_steps=0),
               dict(ns_coefficients=(1.0, 2.0)), dict(adjust_lr_fn="none"), dict(eps=-1.0),
               dict(ns_coefficients=[(1.0, 2.0, 3.0)] * 4), dict(momentum_dtype=torch.int8)):
        with pytest.raises(ValueError):
            Muon(p, **kw)
    with pytest.raises(ValueError, match="TurboAdam"):
        Muon([torch.nn.Parameter(torch.randn(4))])


def test_coefficients_per_step():
    from turboadam_b200.matrix import check_coefficients

    assert check_coefficients((1, 2, 3), 2) == [1.0, 2.0, 3.0] * 2
    assert check_coefficients([(1, 2, 3), (4, 5, 6)], 2) == [1.0, 2.0, 3.0, 4.0, 5.0, 6.0]
    assert check_coefficients([(1, 2, 3)] * 3, 3) == [1.0, 2.0, 3.0] * 3
    for bad in ((1, 2), [(1, 2, 3)], [(1, 2)] * 3):
        with pytest.raises(ValueError):
            check_coefficients(bad, 3)
    for steps in (0, 33, 2.5, True):
        with pytest.raises(ValueError):
            check_coefficients((1, 2, 3), steps)


# ---------------------------------------------------------------------------
# addresses that no kernel could load from: elements at their type's alignment
@pytest.mark.parametrize("over", [
    {"x_dev": (1 << 20) + 1}, {"w_dev": (1 << 21) + 1}, {"y_dev": (1 << 22) + 1},
    {"residual_dev": 4097}, {"bias_dev": 4097, "bias_dtype": 1},
    {"bias_dev": 4098, "bias_dtype": 0},
])
def test_linear_refuses_misaligned_elements(lib, over):
    op = _linear(**over)
    rc = lib.ta_linear_forward(ctypes.byref(op), 1 << 23, 1 << 40, 1 << 10, None)
    assert rc == ALIGN, lib.ta_last_error()
    assert lib.ta_last_error()


@pytest.mark.parametrize("over", [
    {"dy_dev": (1 << 20) + 1}, {"x_dev": (1 << 21) + 1}, {"w_dev": (1 << 22) + 1},
    {"dx_dev": (1 << 23) + 1}, {"dw_dev": (1 << 24) + 1}, {"db_dev": 4097, "bias_dtype": 2},
    {"db_dev": 4098, "bias_dtype": 0},
])
def test_linear_backward_refuses_misaligned_elements(lib, over):
    op = _grad(**over)
    rc = lib.ta_linear_backward(ctypes.byref(op), 1 << 25, 1 << 40, 1 << 10, None)
    assert rc == ALIGN, lib.ta_last_error()


def test_misaligned_status_word(lib):
    op, grad = _linear(), _grad()
    t, o = _ortho()
    for status in ((1 << 10) + 1, (1 << 10) + 2):
        assert lib.ta_linear_forward(ctypes.byref(op), 1 << 23, 1 << 40, status, None) == ALIGN
        assert lib.ta_linear_backward(ctypes.byref(grad), 1 << 25, 1 << 40, status, None) == ALIGN
        assert lib.ta_orthogonalize(t, 1, ctypes.byref(o), 1 << 20, 1 << 40, status,
                                    None) == ALIGN
