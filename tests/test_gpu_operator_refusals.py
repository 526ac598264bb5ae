"""What the operators' entry points refuse because a launch could not give the right answer: results on top of what is still to
be read, sizes that no launch holds.  Plans are made and never launched, from addresses that nothing dereferences."""
import pytest
import torch

from hccl_amd import hcclx
from hccl_amd import types as T
from hccl_amd._lib import HcclError

pytestmark = pytest.mark.gpu   # (the checks of addresses come behind the one for a GPU)
PARA = 1
A, B, C, D, W = (0x7F0000000000 + (k << 32) for k in range(5))


def refused(make, *words):
    with pytest.raises(HcclError) as e:
        make()
    assert e.value.code == PARA, str(e.value)
    for w in words:
        assert w in str(e.value)


def norm(rows=4, elems=64, dtype=T.BFP16, **more):
    args = dict(x=[A], weight=[W], out=[B], rows=rows, row_elems=elems, dtype=dtype)
    args.update(more)
    return lambda: hcclx.RmsNormPlan(**args)


ROW = 64 * 2   # bytes of a row of norm()


@pytest.mark.parametrize("change,words", [
    (dict(out=[A], out_dtype=T.FP8E4M3), ("out[0]", "x[0]")),                       # rows of another length than x's
    (dict(out=[C], residual=[C], out_dtype=T.FP8E4M3), ("out[0]", "residual[0]")),
    (dict(out=[C], total=[C], out_dtype=T.FP8E4M3), ("out[0]", "total[0]")),
    (dict(out=[A], out_dtype=T.FP8E4M3, dtype=T.FP32), ("out[0]", "x[0]")),
    (dict(out=[A + 3 * ROW + 112], out_dtype=T.FP8E4M3), ("out[0]", "x[0]")),       # the last 16 bytes of x
    (dict(out=[A - 4 * 80 + 16], out_dtype=T.FP8E4M3), ("out[0]", "x[0]")),         # and the first
    (dict(out=[W]), ("out[0]", "weight[0]")),                                       # other rows read it
    (dict(out=[W - 4 * ROW + 2]), ("out[0]", "weight[0]")),
    (dict(total=[W]), ("total[0]", "weight[0]")),
    (dict(out=[A + ROW]), ("out[0]", "x[0]")),                                      # a row off
    (dict(total=[A - 2]), ("total[0]", "x[0]")),
    (dict(total=[A + 2], rows=1), ("total[0]", "x[0]")),
    (dict(x=[A, A], weight=[W, W], out=[A, B]), ("out[0]", "x[1]")),                # another rank's
    (dict(x=[A, C], weight=[W, W], out=[C, B]), ("out[0]", "x[1]")),
    (dict(x=[A, A], weight=[W, W], out=[B, D], total=[C, A]), ("total[1]", "x[0]")),
    (dict(x=[A, B], weight=[W, W], out=[W, C], rows=1), ("out[0]", "weight[1]")),
    (dict(x=[A, B], weight=[W, W], out=[C, D], residual=[C, C]), ("out[0]", "residual[1]")),
])
def test_norm_refuses_results_on_what_is_still_read(change, words):
    refused(norm(**change), *words)


@pytest.mark.parametrize("change", [
    {}, dict(out=[A]), dict(total=[A]), dict(residual=[C], total=[C], out=[A]), dict(residual=[C], total=[A], out=[C]),
    dict(residual=[A]), dict(out=[A], total=[A]),
    dict(out_dtype=T.FP8E4M3), dict(out=[A + 4 * ROW], out_dtype=T.FP8E4M3), dict(out=[A - 4 * 80], out_dtype=T.FP8E4M3),   # next to x
    dict(out=[A], out_dtype=T.FP8E4M3, rows=1), dict(out=[W], rows=1),              # one row: all is read before it is written
    dict(out=[A], out_dtype=T.FP8E4M3, rows=0),
    dict(x=[A, A], weight=[W, W], out=[B, C]), dict(x=[A, B], weight=[W, W], out=[A, B]),
    dict(x=[A, B], weight=[W, W], out=[C, D], residual=[B, A], total=[C, D]),
])
def test_norm_takes_results_in_place_of_what_only_their_row_reads(change):
    norm(**change)()


def norm_grad(rows=4, **more):
    args = dict(dy=[A], total=[B], weight=[W], dx=[C], dweight=[D], rows=rows, row_elems=64, dtype=T.BFP16)
    args.update(more)
    return lambda: hcclx.RmsNormGradPlan(**args)


@pytest.mark.parametrize("change,words", [
    (dict(dx=[W]), ("dx[0]", "weight[0]")), (dict(dx=[W - 3 * ROW]), ("dx[0]", "weight[0]")), (dict(dx=[A + ROW]), ("dx[0]", "dy[0]")),
    (dict(dx=[B - 2]), ("dx[0]", "total[0]")), (dict(dx=[D + 2 * ROW], dtotal=[D], dweight=None), ("dx[0]", "dtotal[0]")),
    (dict(dy=[A, A], total=[B, B], weight=[W, W], dx=[A, C], dweight=[D, D + ROW]), ("dx[0]", "dy[1]")),
    (dict(dy=[A, B], total=[C, C], weight=[W, W], dx=[D, C], dweight=None), ("dx[1]", "total[0]")),
    (dict(dy=[A, B], total=[C, D], weight=[W, W], dx=[B, A], dweight=None), ("dx[0]", "dy[1]")),
])
def test_norm_gradient_refuses_results_on_what_is_still_read(change, words):
    refused(norm_grad(**change), *words)


@pytest.mark.parametrize("change", [{}, dict(dx=[A]), dict(dx=[B]), dict(dtotal=[C]), dict(dtotal=[A]), dict(dx=[W], rows=1), dict(dx=[W], rows=0),
                                    dict(dweight=[W]), dict(dx=[A + 4 * ROW]), dict(dx=[W + ROW]),
                                    dict(dy=[A, B], total=[C, D], weight=[W, W], dx=[A, B], dweight=None)])
def test_norm_gradient_takes_results_in_place_of_what_only_their_row_reads(change):
    norm_grad(**change)()


def ffn_grad():
    names = ("dy", "x", "w_gate", "w_up", "w_down", "dx", "dw_gate", "dw_up", "dw_down")
    return dict({k: [A + (i << 32), A + (i << 32) + (1 << 20)] for i, k in enumerate(names)}, saved=A + (1 << 40), capacity=8, dim=64, hidden=32,
                dtype=T.BFP16)


@pytest.mark.parametrize("dx", ["dy", "x"])
@pytest.mark.parametrize("dw", ["dw_gate", "dw_up"])
@pytest.mark.parametrize("weight", ["w_gate", "w_up"])
def test_ffn_gradient_refuses_dx_and_dw_in_place_at_once(dx, dw, weight):
    args = ffn_grad()
    args["dx"] = args[dx]
    hcclx.GatedFfnGradPlan(**args)
    hcclx.GatedFfnGradPlan(**{**args, "dw_down": args["w_down"]})
    refused(lambda: hcclx.GatedFfnGradPlan(**{**args, dw: args[weight]}), "at once")
    refused(lambda: hcclx.GatedFfnGradPlan(**{**args, dw: [args[dw][0], args[weight][0]]}), "at once")


@pytest.mark.parametrize("result,on", [("dx", "w_gate"), ("dx", "w_up")] + [(r, k) for r in ("dw_gate", "dw_up", "dw_down") for k in ("x", "dy")])
def test_ffn_gradient_refuses_results_on_what_their_product_reads(result, on):
    args = ffn_grad()
    refused(lambda: hcclx.GatedFfnGradPlan(**{**args, result: args[on]}), result[:1])
    refused(lambda: hcclx.GatedFfnGradPlan(**{**args, result: args[on][::-1]}), " on ")
    hcclx.GatedFfnGradPlan(**{**args, result: args[on], "capacity": 0})
    # a rank without rows, whose buffer begins where those of the others end
    hcclx.GatedFfnGradPlan(**{**args, result: [args[result][0], args[on][0]]})


@pytest.mark.parametrize("n,elems", [(1, 8), (64, 8), (1, 16384)])
def test_norm_gradient_refuses_rows_whose_numbers_wrap(n, elems):
    def make(rows):
        return lambda: hcclx.RmsNormGradPlan(*([at << 50] * n for at in (1, 2, 3, 4)), [5 << 50] * n, rows, elems, T.BFP16)
    make(0xFFFF0000)()
    for rows in (0xFFFFFFFF, 0xFFFFFFFE, 0xFFFFFFFC):
        refused(make(rows), "rows")


def test_norm_of_as_many_rows_as_a_launch_holds():
    """The limit is the launch's: one row less is normed."""
    rows = (1 << 28) - 4
    x = torch.randint(1, 100, (rows,), device="cuda:0", dtype=torch.bfloat16)
    w, out = torch.full((1,), 3, device="cuda:0", dtype=torch.bfloat16), torch.zeros_like(x)
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], [out.data_ptr()], rows, 1, T.BFP16).launch()
    torch.cuda.synchronize()
    assert bool((out == 3).all())                                  # x * 3 / sqrt(x^2 + 1e-6): 3 but for 2^-21 of it
