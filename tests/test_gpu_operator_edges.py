"""The operators where a launch's buffers are one another's, where values leave the range of ordinary ones, and where one plan meets
different contents from launch to launch: against ops_oracle.py's 64 bits, or bit for bit against what has been compared with those."""
import pytest
import torch

import ops_oracle as O
from hccl_amd import hcclx
from hccl_amd import types as T
from test_gpu_operators import DEV, TD, Ffn, Guarded, gen, normal, ptrs

pytestmark = pytest.mark.gpu


# ---- the norm's gradient on top of its inputs -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("n,rows,elems", [(2, 1, 24), (3, 37, 300), (1, 2100, 136), (2, 9, 8200), (1, 6, 16384)])
@pytest.mark.parametrize("on", ["dy", "total", "dtotal"])
def test_norm_gradient_in_place(n, rows, elems, dtype, on):
    g, td = gen(rows), TD[dtype]
    src = {k: [normal((rows, elems), td, g) for _ in range(n)] for k in ("dy", "total", "dtotal")}
    w = [normal((elems,), td, g) for _ in range(n)]
    dx, dw = [torch.empty_like(t) for t in src["dy"]], [torch.empty_like(t) for t in w]

    def launch(to, to_w):
        hcclx.RmsNormGradPlan(ptrs(src["dy"]), ptrs(src["total"]), ptrs(w), ptrs(to), ptrs(to_w), rows, elems, dtype,
                              dtotal=ptrs(src["dtotal"])).launch()
        torch.cuda.synchronize()
    launch(dx, dw)
    for i in range(n):
        wdx, bdx, wdw, bdw = O.norm_grad(src["dy"][i], src["total"][i], w[i], src["dtotal"][i], 1e-6)
        O.assert_close(dx[i], wdx, bdx)
        O.assert_close(dw[i], wdw, bdw)
    launch(src[on], w)
    assert all(torch.equal(a, b) for a, b in zip(src[on] + w, dx + dw))


# ---- the experts' gradient on top of its inputs ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,dim,hidden", [([3, 0, 2], 72, 40), ([130, 1, 129], 136, 264), ([700, 300], 264, 520)])
@pytest.mark.parametrize("on", ["dx on dy", "dx on x", "dx on dy of another rank", "dw on the weights"])
def test_ffn_gradient_in_place(rows, dim, hidden, dtype, on):
    f = Ffn(rows, max(rows), dim, hidden, dtype, dim)
    f.run()
    f.check()
    n, shape = len(rows), {**f.shape, "rows": f.total}
    want = [f.dx[i][:r * dim].clone() for i, r in enumerate(rows)] + [d[i].clone() for d in f.dw for i in range(n)]
    at = [k.ptrs for k in (f.dw[0], f.dw[1], f.dw[2])]
    if on == "dx on dy":
        dx, dw = f.dy, f.dw
    elif on == "dx on x":
        dx, dw = f.x, f.dw
    elif on == "dx on dy of another rank":
        dx, dw = f.dy, f.dw
    else:
        dx, dw = f.dx, f.w
        at = [ptrs(k) for k in f.w]
    turn = 1 if on == "dx on dy of another rank" else 0
    place = [(i + turn) % n for i in range(n)]
    for k in (f.dx, *f.dw):
        if k is not dx:
            k.raw.fill_(0xFF)
    hcclx.GatedFfnGradPlan(f.dy.ptrs, f.x.ptrs, *[ptrs(k) for k in f.w], f.saved.data_ptr(), [dx.ptrs[p] for p in place], *at, **shape).launch()
    torch.cuda.synchronize()
    got = [dx[p][:r * dim] for p, r in zip(place, rows)] + [d[i].view(-1) for d in dw for i in range(n)]
    for k, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), k


# ---- gates far out ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("rows", [1, 100, 300])
def test_ffn_gates_to_the_end_of_the_range(rows, act):
    """Gates of +-2^43 .. 2^123, whose cube passes the range of 32 bits: the activation and its derivative are 0 and 0, or the gate
    and 1.  Every number is a power of two or a small multiple of one, so that results are exact."""
    dim, hidden, powers = 64, 168, torch.arange(20, 101, device=DEV)
    e = torch.cat([powers, powers, powers[:6]]).double()
    sign = torch.ones(hidden, device=DEV, dtype=torch.float64)
    sign[81:162] = -1
    f = Ffn([rows], rows, dim, hidden, T.BFP16, 1)
    x, dy = torch.zeros((rows, dim), device=DEV, dtype=torch.bfloat16), torch.zeros((rows, dim), device=DEV, dtype=torch.bfloat16)
    x[:, 0], dy[:, 0] = 2.0 ** 23, 1
    f.x[0].copy_(x.view(-1)), f.dy[0].copy_(dy.view(-1))
    for w in f.w:
        w[0].zero_()
    f.w[0][0][:, 0] = sign * 2.0 ** e          # gate +-2^(e + 23)
    f.w[1][0][:, 0] = 2.0 ** -23               # up 1
    f.w[2][0][0] = 2.0 ** -(e + 23)
    f.run(act)
    got = [f.out[0].view(rows, dim), f.dx[0].view(rows, dim)] + [d[0].view(w[0].shape) for d, w in zip(f.dw, f.w)]
    for a, (b, _) in zip(got, O.ffn(x, f.w[0][0], f.w[1][0], f.w[2][0], act, torch.bfloat16, dy)):
        assert bool(b.isfinite().all()) and torch.equal(a, b.to(torch.bfloat16))   # (some sums round to infinity)


# ---- one plan, launch after launch -----------------------------------------------------------------------------------------

def taken(rows, capacity, bound):
    """The rows that a plan takes of each rank: up to capacity, and up to the bound on all of them."""
    out = []
    for r in rows:
        out.append(min(r, capacity, bound - sum(out)))
    return out


def counted(f, rows):
    """The counts that stand for `rows`, in three parts each, some of them empty."""
    parts = torch.zeros_like(f.counts)
    for i, r in enumerate(rows):
        parts[i, i % 3], parts[i, (i + 1) % 3] = r // 3, r - r // 3
    return parts


def captured(launch):
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        launch(torch.cuda.current_stream().cuda_stream)
    return graph


# few rows (thin kernels), up to 64 and up to 128 (small tiles), many (whole tiles)
HELD = [(9, 64, 48, 20), (64, 520, 136, 0), (120, 1032, 264, 0), (400, 264, 136, 1000)]


@pytest.mark.parametrize("capacity,dim,hidden,bound", HELD)
def test_one_ffn_plan_with_other_rows_at_every_launch(capacity, dim, hidden, bound):
    """Forward and gradient plans made once, launched by themselves and from a graph: each time with other counts and other rows, and
    with NaN where results belong.  What an earlier launch left in the plans' own memory would show."""
    f = Ffn([1, capacity, 2], capacity, dim, hidden, T.BFP16, capacity, per_rank=3)
    f.run(bound=bound)
    f.check(rows=taken(f.rows, capacity, bound or 3 * capacity))

    def launch(stream):
        f.plan.launch(stream)
        f.grad_plan.launch(stream)
    graph = captured(launch)
    half = capacity // 2
    for k, rows in enumerate(([capacity] * 3, [0, 1, half], [0, 0, 0], [half, 0, 2 * capacity], [3, capacity, 0], [1 << 40, 1, 1 << 33], [1, 0, 0])):
        want = taken(rows, capacity, bound or 3 * capacity)
        f.counts.copy_(counted(f, rows) * dim)
        for j, go in enumerate((lambda: launch(0), graph.replay)):
            g = gen(2 * k + j)
            for b in (f.x, f.dy, f.out, f.dx, *f.dw):
                b.raw.fill_(0xFF)
            f.saved.fill_(0xFF)
            for b in (f.x, f.dy):
                for i, r in enumerate(want):
                    b[i][:r * dim] = normal((r * dim,), torch.bfloat16, g)
            go()
            torch.cuda.synchronize()
            f.check(rows=want)


@pytest.mark.parametrize("capacity,dim,hidden", [(9, 64, 48), (100, 1040, 136), (300, 272, 136)])
def test_one_ffn_plan_of_8_bit_rows_with_other_rows_at_every_launch(capacity, dim, hidden):
    n, wide, w = 3, dim + hcclx.ROW8_TAIL, torch.ones(dim, device=DEV)
    f = Ffn([0, 0, 0], capacity, dim, hidden, T.BFP16, capacity, per_rank=3, unit=wide)
    x8 = torch.empty((n, capacity, wide), device=DEV, dtype=torch.uint8)
    f.out = Guarded(n, capacity * dim, torch.bfloat16)
    plan = hcclx.GatedFfnPlan(ptrs(x8), *[ptrs(k) for k in f.w], f.out.ptrs, x_dtype=T.FP8E4M3, **f.shape)
    graph = captured(plan.launch)
    for k, rows in enumerate(([capacity] * 3, [0, 2, 1], [0, 0, 0], [1, capacity, 0])):
        f.counts.copy_(counted(f, rows) * wide)
        for j, go in enumerate((lambda: plan.launch(0), graph.replay)):
            x = [normal((capacity, dim), torch.float32, gen(10 * k + 2 * i + j), 4.0) for i in range(n)]
            hcclx.RmsNormPlan(ptrs(x), [w.data_ptr()] * n, ptrs(x8), capacity, dim, T.FP32, out_dtype=T.FP8E4M3).launch()
            for i, r in enumerate(rows):
                x8[i, r:] = 0xFF
            f.out.raw.fill_(0xFF)
            go()
            torch.cuda.synchronize()
            for i, r in enumerate(rows):
                b = x8[i, :r]
                values = b[:, :dim].contiguous().view(torch.float8_e4m3fn).double() * b[:, dim:dim + 4].contiguous().view(torch.float32).double()
                want = O.ffn(values, f.w[0][i], f.w[1][i], f.w[2][i], 0, torch.bfloat16)
                O.assert_close(f.out[i][:r * dim].view(r, dim), *want[0], f"out of rank {i}")
            assert f.out.untouched([r * dim for r in rows])
