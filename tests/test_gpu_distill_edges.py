"""The distillation loss and its gradients where a student's row holds +infinity, NaN or nothing but -infinity, by every route that a row takes:
a workgroup to a row, smaller ones for short rows, rows in registers, several workgroups to a row, gradients from saved sums."""
import math

import pytest
import torch

import logits_oracle as L
import ops_oracle as O
from hccl_amd import hcclx
from hccl_amd import types as T
from test_gpu_output_layer import DEV, TD, Split, check_distill, contents, entries, gen, shares

pytestmark = pytest.mark.gpu
INF = math.inf

# rows and columns: several workgroups to a row; rows in registers (16 bits; 32 bits); a workgroup to a row; small workgroups
ROUTES = [(7, 50021), (7, 20011), (7, 12011), (600, 33003), (600, 3001)]


def run(s, values, at, k, weight, in_place):
    """Loss, gradients with it, loss alone, gradients from saved sums."""
    rows = s.rows
    held = dict(s.where, teacher=values.data_ptr(), indices=at.data_ptr(), k=k, teacher_dtype=T.FP32, temperature=1.5, weight=weight.data_ptr())
    loss, alone = torch.full((rows,), 77.0, device=DEV), torch.full((rows,), 77.0, device=DEV)
    stats = torch.full((rows, 2), 77.0, device=DEV)
    blank = torch.zeros_like(s.whole())
    once, later = Split(blank, s.columns, s.dtype, 3), Split(blank, s.columns, s.dtype, 3)
    hcclx.DistillPlan(s.ptrs, loss=alone.data_ptr(), stats=stats.data_ptr(), **held).launch()
    hcclx.DistillGradPlan(s.ptrs, stats=stats.data_ptr(), dlogits=later.ptrs, **held).launch()
    torch.cuda.synchronize()
    to = s if in_place else once
    hcclx.DistillPlan(s.ptrs, loss=loss.data_ptr(), dlogits=to.ptrs, **held).launch()
    torch.cuda.synchronize()
    return loss, to.whole(), alone, later.whole()


def check_rows(whole, values, at, weight, out, nan_rows):
    for r in range(whole.shape[0]):
        for loss, d in (out[:2], out[2:]):
            if r in nan_rows:
                assert math.isnan(float(loss[r])) and bool(d[r].isnan().all()), r
                continue
            want, grad, bound, grad_bound = L.distill(whole[r].double(), values[r].double(), at[r], 1.5, float(weight[r]))
            got = float(loss[r])
            assert got == want or abs(got - want) <= bound + O.E * abs(want), (r, got, want)
            O.assert_close(d[r], grad, grad_bound, f"row {r}")


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,vocab", ROUTES)
@pytest.mark.parametrize("in_place", [False, True])
def test_infinity_in_a_row_makes_it_nan_and_no_other(rows, vocab, in_place, dtype):
    """+infinity or NaN: at the row's ends, at an entry of the teacher's, many of them, next to nothing but -infinity; a masked row of them is 0."""
    k, g = 20, gen(rows + vocab)
    x = torch.randn((rows, vocab), device=DEV, generator=g) * 3
    values, at = entries(x.to(TD[dtype]), k, "plain", g)
    values = values.contiguous()
    weight = torch.rand(rows, device=DEV, generator=g) + 0.1
    x[0, vocab - 1] = INF
    x[1, int(at[1, 3])] = INF
    x[2, ::3] = INF
    x[3] = -INF
    x[3, vocab // 2] = INF
    x[4, 0] = math.nan
    x[5] = INF
    weight[5] = 0
    if rows > 7:
        x[rows - 1, 0] = INF
        x[rows - 2, [5, 2000]] = torch.tensor([INF, math.nan], device=DEV)
    s = Split(x.to(TD[dtype]), shares(vocab, 2), dtype, 3)
    whole = s.whole().clone()
    out = run(s, values, at, k, weight, in_place)
    check_rows(whole, values, at, weight, out, {0, 1, 2, 3, 4} | ({rows - 1, rows - 2} if rows > 7 else set()))
    assert float(out[0][5]) == 0 and not bool(out[1][5].any()) and float(out[2][5]) == 0 and not bool(out[3][5].any())


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("rows,vocab", ROUTES)
def test_a_student_that_rules_entries_or_everything_out(rows, vocab, dtype):
    """-infinity at a teacher's entry: an infinite loss, and q = 0 there. Nothing but -infinity: q = 0 everywhere."""
    k, g = 9, gen(rows + vocab + 1)
    x = torch.randn((rows, vocab), device=DEV, generator=g)
    values, at = entries(x.to(TD[dtype]), k, "plain", g)
    values = values.contiguous()
    weight = torch.rand(rows, device=DEV, generator=g) + 0.1
    x[0, int(at[0, 2])] = -INF
    x[1] = -INF
    x[rows - 1] = -INF
    s = Split(x.to(TD[dtype]), shares(vocab, 3), dtype, 3)
    whole = s.whole().clone()
    out = run(s, values, at, k, weight, False)
    for r in (0, 1, rows - 1):
        assert float(out[0][r]) == INF and float(out[2][r]) == INF
    check_rows(whole, values, at, weight, out, set())


@pytest.mark.parametrize("dtype,chunk", [(T.FP32, 256), (T.BFP16, 512)])
@pytest.mark.parametrize("rows", [5, 520])
@pytest.mark.parametrize("chunks", [16, 24, 32, 64, 128])
def test_lengths_on_both_sides_of_where_a_route_ends(chunks, rows, dtype, chunk):
    for vocab in (chunks * chunk, chunks * chunk + 1):
        check_distill(contents("steep", rows, vocab, gen(vocab)), [vocab], dtype, 30, 1.5, in_place=rows == 5)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("rows,vocab", ROUTES)
def test_improbable_entries_keep_their_gradients(rows, vocab, dtype):
    """A teacher's entries of 1 to 2^-90, a student who finds them as improbable or more: the gradients there are as good as their own size asks for.
    Where two entries name a column, as 2^-61 asks for."""
    k, T_, g = 40, 0.25, gen(rows + vocab + 2)
    x = torch.randn((rows, vocab), device=DEV, generator=g) - 16
    values = -torch.arange(k, device=DEV).float()[None].repeat(rows, 1) * 0.4
    at = torch.stack([torch.randperm(vocab, device=DEV, generator=g)[:k] for _ in range(rows)]).to(torch.int32)
    x[torch.arange(rows, device=DEV)[:, None], at.long()] = values - 3 * torch.rand((rows, k), device=DEV, generator=g)
    at[:, -1] = at[:, -2]
    s = Split(x.to(TD[dtype]), shares(vocab, 2), dtype, 3)
    whole, d = s.whole(), Split(torch.zeros_like(s.whole()), s.columns, dtype, 3)
    later = Split(torch.zeros_like(whole), s.columns, dtype, 3)
    stats = torch.zeros((rows, 2), device=DEV)
    held = dict(s.where, teacher=values.data_ptr(), indices=at.data_ptr(), k=k, teacher_dtype=T.FP32, temperature=T_)
    hcclx.DistillPlan(s.ptrs, stats=stats.data_ptr(), dlogits=d.ptrs, **held).launch()
    hcclx.DistillGradPlan(s.ptrs, stats=stats.data_ptr(), dlogits=later.ptrs, **held).launch()
    torch.cuda.synchronize()
    for r in [*range(min(rows, 7)), rows - 1]:
        _, grad, _, bound = L.distill(whole[r].double(), values[r].double(), at[r], T_, 1.0)
        named = at[r].long()
        bound[named[-1]] += T_ * 2.0 ** -61
        for got in (d, later):
            O.assert_close(got.whole()[r][named], grad[named], bound[named], f"row {r}")
