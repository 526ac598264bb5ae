"""The output layer's C interface without a GPU: the structures as C and Python see them, and what the entry points refuse."""
import ctypes
import os
import subprocess

import pytest

from hccl_amd import _lib, hcclx
from hccl_amd import types as T
from hccl_amd._lib import HcclError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PARA, PTR, NOT_SUPPORT = 1, 2, 5
A = 0x7F0000000000      # addresses that nothing dereferences: every call here is refused, or ends where a GPU is asked for
B, C, D, F, G = (A + (k << 36) for k in range(1, 6))


def test_structures_are_those_of_the_header(tmp_path):
    names = {"hcclx_logits_t": _lib.Logits, "hcclx_top_logits_t": _lib.TopLogits, "hcclx_teacher_t": _lib.Teacher, "hcclx_distill_t": _lib.Distill,
             "hcclx_distill_grad_t": _lib.DistillGrad, "hcclx_sample_t": _lib.Sample}
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


def taken(make):
    """All checks are passed: a plan, or no GPU."""
    try:
        make()
    except HcclError as e:
        assert e.code == T.Result.E_RUNTIME, str(e)


LOGITS = dict(logits=[A, B], columns=[100, 60], rows=4, dtype=T.BFP16)
TOP = dict(LOGITS, k=5, values=C, indices=D)
TEACHER = dict(LOGITS, k=5, teacher=C, indices=D)
LOSS = dict(TEACHER, loss=F)
GRAD = dict(TEACHER, stats=F, dlogits=[G, G + (1 << 33)])
SAMPLE = dict(LOGITS, random=C, tokens=D)
ALL = [(hcclx.TopLogitsPlan, TOP), (hcclx.DistillPlan, LOSS), (hcclx.DistillGradPlan, GRAD), (hcclx.SamplePlan, SAMPLE)]


@pytest.mark.parametrize("plan,base", ALL)
@pytest.mark.parametrize("change,code", [
    (dict(dtype=T.INT32), NOT_SUPPORT), (dict(dtype=T.FP64), NOT_SUPPORT), (dict(logits=[A + 1, B]), PARA), (dict(logits=[A, 0]), PTR),
    (dict(columns=[0, 0]), PARA), (dict(columns=[1 << 24, 1]), PARA), (dict(columns=[0xFFFFFFFF, 0xFFFFFFFF]), PARA), (dict(rows=1 << 22), PARA),
    (dict(strides=[99, 60]), PARA), (dict(strides=[100, 1 << 32]), PARA)])
def test_logits_refused(plan, base, change, code):
    refused(code, lambda: plan(**{**base, **change}))


@pytest.mark.parametrize("plan,base", ALL)
def test_numbers_of_ranks(plan, base):
    for n in (0, 65):
        many = {k: [A + (i << 24) for i in range(n)] for k in ("logits", "dlogits") if k in base}
        refused(PARA, lambda: plan(**{**base, **many, "columns": [1] * n}), "rank count")
    with pytest.raises(ValueError):
        plan(**{**base, "columns": [100]})
    with pytest.raises(ValueError):
        plan(**{**base, "strides": [100, 60, 1]})


@pytest.mark.parametrize("plan,base", ALL)
@pytest.mark.parametrize("change", [{}, dict(columns=[0, 160], logits=[0, B]), dict(strides=[100, 333]), dict(rows=1, strides=[0, 0]),
                                    dict(logits=[A, A + 200], strides=[160, 160]), dict(rows=(1 << 22) - 1, dtype=T.FP32)])
def test_logits_taken(plan, base, change):
    taken(lambda: plan(**{**base, **change}))


@pytest.mark.parametrize("change,code", [
    (dict(k=0), PARA), (dict(k=161), PARA), (dict(k=1025, columns=[5000, 0]), PARA), (dict(values=0), PTR), (dict(indices=0), PTR), (dict(values=C + 1), PARA),
    (dict(indices=D + 2), PARA), (dict(lse=F + 2), PARA), (dict(values=A + 700), PARA), (dict(indices=B - 4), PARA), (dict(indices=C), PARA),
    (dict(lse=D + 76), PARA), (dict(lse=B + 400), PARA)])
def test_top_logits_refuses(change, code):
    refused(code, lambda: hcclx.TopLogitsPlan(**{**TOP, **change}))


@pytest.mark.parametrize("plan,base", ALL[1:3])
@pytest.mark.parametrize("change,code", [
    (dict(k=0), PARA), (dict(k=1025), PARA), (dict(teacher=0), PTR), (dict(indices=0), PTR), (dict(teacher=C + 1), PARA), (dict(indices=D + 2), PARA),
    (dict(weight=F + 1), PARA), (dict(teacher_dtype=T.INT8), NOT_SUPPORT), (dict(temperature=0.0), PARA), (dict(temperature=-1.0), PARA),
    (dict(temperature=float("nan")), PARA), (dict(temperature=float("inf")), PARA), (dict(dlogits=[G, 0]), PTR), (dict(dlogits=[G + 1, F]), PARA),
    (dict(dlogits=[A + 2, G]), PARA), (dict(dlogits=[B, A]), PARA), (dict(dlogits=[G, G + 700]), PARA), (dict(dlogits=[G, C - 100]), PARA),
    (dict(dlogits=[D + 10, G]), PARA), (dict(dlogits=[F - 2, G], weight=F), PARA), (dict(dlogits=[G, F]), PARA), (dict(stats=F + 4), PARA)])
def test_distillation_refuses(plan, base, change, code):
    refused(code, lambda: plan(**{**base, **change}))


@pytest.mark.parametrize("change,code", [(dict(loss=F + 1), PARA), (dict(loss=A), PARA), (dict(loss=G + 8, dlogits=[G, F]), PARA), (dict(loss=C + 32), PARA),
                                         (dict(loss=D), PARA), (dict(weight=F), PARA), (dict(stats=F + 8), PARA), (dict(stats=B + 8), PARA)])
def test_distillation_loss_refuses(change, code):
    refused(code, lambda: hcclx.DistillPlan(**{**LOSS, **change}))


def test_distillation_gradient_needs_places():
    refused(PTR, lambda: hcclx.DistillGradPlan(**{**GRAD, "stats": 0}), "stats")
    refused(PTR, lambda: hcclx.DistillGradPlan(**{**GRAD, "dlogits": None}), "dlogits")


@pytest.mark.parametrize("plan,base", ALL[1:3])
@pytest.mark.parametrize("change", [dict(dlogits=[A, B]), dict(dlogits=[A, G]), dict(logits=[A, A + 200], strides=[160, 160], dlogits=[A, A + 200]),
                                    dict(logits=[A, A + 200], strides=[160, 160], dlogits=[G, G + 200]), dict(k=1024), dict(temperature=0.01, weight=G + (1 << 30))])
def test_distillation_takes(plan, base, change):
    taken(lambda: plan(**{**base, **change}))


def test_distillation_refuses_columns_that_interleave_wrongly():
    """Ranks that hold columns of one matrix: gradients that lie a column, or a row, off."""
    one = dict(LOSS, logits=[A, A + 200], strides=[160, 160])
    for dlogits in ([A + 2, A + 200], [A, A + 198], [A + 200, A], [A + 320, A + 200], [G, G + 198]):
        refused(PARA, lambda: hcclx.DistillPlan(**{**one, "dlogits": dlogits}), "overlaps")


@pytest.mark.parametrize("change,code", [
    (dict(random=0), PTR), (dict(tokens=0), PTR), (dict(random=C + 1), PARA), (dict(tokens=D + 2), PARA), (dict(temperature=F + 1), PARA), (dict(top_k=F + 2), PARA),
    (dict(top_p=F + 3), PARA), (dict(min_p=F + 1), PARA), (dict(logprob=F + 2), PARA), (dict(tokens=A), PARA), (dict(tokens=C + 12), PARA), (dict(logprob=D), PARA),
    (dict(top_k=D), PARA), (dict(logprob=F, min_p=F), PARA), (dict(logprob=B + 476), PARA)])
def test_sampling_refuses(change, code):
    refused(code, lambda: hcclx.SamplePlan(**{**SAMPLE, **change}))


def test_null_structures():
    lib = _lib.load()
    h = ctypes.c_void_p(1)
    for name, kind in (("top_logits", _lib.TopLogits), ("distill", _lib.Distill), ("distill_grad", _lib.DistillGrad), ("sample", _lib.Sample)):
        fn = getattr(lib, f"hcclx_{name}_plan_create")
        assert fn(None, ctypes.byref(h)) == PTR and h.value is None
        assert fn(None, None) == PTR
        empty = kind()
        empty.logits.n = 1
        empty.logits.dtype = T.FP32
        assert fn(ctypes.byref(empty), ctypes.byref(h)) == PTR          # columns
        columns = (ctypes.c_uint32 * 1)(5)
        empty.logits.columns = columns
        assert fn(ctypes.byref(empty), ctypes.byref(h)) == PTR          # logits


@pytest.mark.parametrize("plan,base", ALL)
def test_without_a_gpu_the_operators_raise(plan, base):
    import torch
    if torch.cuda.is_available():
        return
    refused(T.Result.E_RUNTIME, lambda: plan(**base))
