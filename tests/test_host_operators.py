"""The operators' C interface without a GPU: the structures as C and Python see them, and what their entry points refuse."""
import ctypes
import os
import subprocess

import pytest

from hccl_amd import _lib, hcclx
from hccl_amd import types as T
from hccl_amd._lib import HcclError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PARA, PTR, NOT_SUPPORT = 1, 2, 5
A = 0x7F0000000000      # an address that nothing dereferences: every call here is refused


def test_structures_are_those_of_the_header(tmp_path):
    names = {"hcclx_rms_norm_t": _lib.RmsNorm, "hcclx_rms_norm_grad_t": _lib.RmsNormGrad, "hcclx_ffn_shape_t": _lib.FfnShape,
             "hcclx_gated_ffn_t": _lib.GatedFfn, "hcclx_gated_ffn_grad_t": _lib.GatedFfnGrad, "hcclx_adamw_tensor_t": _lib.AdamWTensor,
             "hcclx_adamw_step_t": _lib.AdamWStep}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("{c} %zu", sizeof({c}));')
        lines += [f'printf(" %zu", offsetof({c}, {f[0]}));' for f in py._fields_]
        lines.append('printf("\\n");')
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"hcclx_ops.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Wextra", "-pedantic", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, *numbers = line.split()
        py = names[name]
        assert [int(k) for k in numbers] == [ctypes.sizeof(py)] + [getattr(py, f[0]).offset for f in py._fields_], name


def refused(code, make, *words):
    with pytest.raises(HcclError) as e:
        make()
    assert e.value.code == code, str(e.value)
    for w in words:
        assert w in str(e.value)


NORM = dict(x=[A], weight=[A], out=[A], rows=4, row_elems=64, dtype=T.BFP16)


@pytest.mark.parametrize("change,code", [
    (dict(row_elems=0), PARA), (dict(row_elems=16385), PARA), (dict(dtype=T.INT32), NOT_SUPPORT), (dict(dtype=T.FP64), NOT_SUPPORT),
    (dict(out_dtype=T.FP32), NOT_SUPPORT), (dict(out_dtype=T.FP8E4M3, row_elems=72), PARA), (dict(out_dtype=T.FP8E4M3, out=[A + 8]), PARA),
    (dict(x=[A + 1]), PARA), (dict(x=[0]), PTR), (dict(weight=None), PTR), (dict(out=None), PTR), (dict(total=[0]), PTR),
    (dict(residual=[A + 1]), PARA), (dict(x=[], weight=[], out=[]), PARA), (dict(x=[A] * 65, weight=[A] * 65, out=[A] * 65), PARA)])
def test_norm_refuses(change, code):
    refused(code, lambda: hcclx.RmsNormPlan(**{**NORM, **change}))


@pytest.mark.parametrize("change,code", [
    (dict(row_elems=0), PARA), (dict(dtype=T.INT8), NOT_SUPPORT), (dict(dy=[0]), PTR), (dict(total=None), PTR), (dict(dx=[A + 1]), PARA),
    (dict(dweight=[0]), PTR), (dict(dtotal=[A + 1]), PARA)])
def test_norm_gradient_refuses(change, code):
    base = dict(dy=[A], total=[A], weight=[A], dx=[A], dweight=[A], rows=4, row_elems=64, dtype=T.FP16)
    refused(code, lambda: hcclx.RmsNormGradPlan(**{**base, **change}))


FFN = dict(x=[A], w_gate=[A], w_up=[A], w_down=[A], out=[A], capacity=8, dim=64, hidden=32, dtype=T.BFP16)
BAD_SHAPES = [
    (dict(dim=0), PARA), (dict(dim=60), PARA), (dict(hidden=12), PARA), (dict(hidden=262152), PARA), (dict(dtype=T.FP32), NOT_SUPPORT),
    (dict(activation=2), NOT_SUPPORT), (dict(counts=A, counts_per_rank=0), PARA), (dict(counts=A, counts_per_rank=65), PARA),
    (dict(counts=A, count_unit=0), PARA), (dict(counts=A + 4), PARA), (dict(capacity=0x80000000), PARA), (dict(w_gate=None), PTR),
    (dict(w_up=[0]), PTR), (dict(w_down=[A + 8]), PARA), (dict(x=[A + 2]), PARA)]


@pytest.mark.parametrize("change,code", BAD_SHAPES + [
    (dict(out=[0]), PTR), (dict(saved=A + 4), PARA), (dict(x_dtype=T.FP16), NOT_SUPPORT), (dict(x_dtype=T.FP8E4M3, dim=72), PARA),
    (dict(x_dtype=T.FP8E4M3, saved=A), NOT_SUPPORT)])
def test_ffn_refuses(change, code):
    refused(code, lambda: hcclx.GatedFfnPlan(**{**FFN, **change}))


@pytest.mark.parametrize("change,code", BAD_SHAPES + [(dict(saved=0), PTR), (dict(saved=A + 8), PARA), (dict(dx=None), PTR), (dict(dw_down=[A + 2]), PARA)])
def test_ffn_gradient_refuses(change, code):
    base = {k: v for k, v in FFN.items() if k != "out"}
    base.update(dy=[A], saved=A, dx=[A], dw_gate=[A], dw_up=[A], dw_down=[A])
    refused(code, lambda: hcclx.GatedFfnGradPlan(**{**base, **change}))


ONE = dict(count=5, param=A, grad=A, m=A, v=A, m_scale=A, v_scale=A, copy=A)


@pytest.mark.parametrize("change,types,code", [
    (dict(param=0), (T.FP32, T.FP32, T.BFP16), PTR), (dict(grad=A + 2), (T.FP32, T.FP32, T.BFP16), PARA), (dict(grad=A + 1), (T.FP16, T.FP32, T.BFP16), PARA),
    (dict(m=A + 1), (T.FP16, T.FP32, T.BFP16), PARA), (dict(v=0), (T.FP16, T.FP32, T.BFP16), PTR), (dict(m_scale=0), (T.FP16, T.FP8E4M3, T.BFP16), PTR),
    (dict(v_scale=A + 1), (T.FP16, T.FP8E4M3, T.BFP16), PARA), (dict(copy=A + 1), (T.FP16, T.FP32, T.BFP16), PARA),
    ({}, (T.INT8, T.FP32, T.BFP16), NOT_SUPPORT), ({}, (T.FP16, T.FP16, T.BFP16), NOT_SUPPORT), ({}, (T.FP16, T.FP32, T.FP32), NOT_SUPPORT),
    (dict(count=1 << 50), (T.FP16, T.FP32, T.BFP16), PARA)])
def test_adamw_refuses(change, types, code):
    refused(code, lambda: hcclx.AdamWPlan([{**ONE, **change}], *types))


def test_adamw_refuses_a_copy_of_some_tensors():
    refused(PTR, lambda: hcclx.AdamWPlan([ONE, {**ONE, "copy": 0}], T.FP16, T.FP32, T.BFP16), "all tensors")


def test_null_structures_and_lists_of_another_length():
    lib = _lib.load()
    h = ctypes.c_void_p(1)
    for name in ("rms_norm", "rms_norm_grad", "gated_ffn", "gated_ffn_grad"):
        fn = getattr(lib, f"hcclx_{name}_plan_create")
        assert fn(None, ctypes.byref(h)) == PTR and h.value is None
        assert fn(None, None) == PTR
    assert lib.hcclx_adamw_plan_create(None, 1, T.FP32, T.FP32, T.FP32, ctypes.byref(h)) == PTR
    assert lib.hcclx_adamw_plan_create(None, 1, T.FP32, T.FP32, T.FP32, None) == PTR
    assert lib.hcclx_adamw_step(None, None, None) == PTR
    with pytest.raises(ValueError):
        hcclx.RmsNormPlan([A, A], [A], [A, A], 1, 8, T.FP32)
    assert hcclx.gated_ffn_saved_bytes(10, 16) == 10 * 16 * 8


def test_without_a_gpu_the_operators_raise():
    import torch
    if torch.cuda.is_available():
        return
    for make in (lambda: hcclx.RmsNormPlan(**NORM), lambda: hcclx.GatedFfnPlan(**FFN), lambda: hcclx.AdamWPlan([ONE], T.FP16, T.FP32, T.BFP16)):
        with pytest.raises(HcclError) as e:
            make()
        assert e.value.code == T.Result.E_RUNTIME
