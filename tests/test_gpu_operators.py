"""The operators of include/hcclx_ops.h on the GPU against their definitions in 64 bits (ops_oracle.py), at the sizes, types,
alignments and contents where they can go wrong."""
import numpy as np
import pytest
import torch

import ops_oracle as O
from hccl_amd import hcclx
from hccl_amd import types as T
from hccl_amd._lib import HcclError

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {T.FP32: torch.float32, T.FP16: torch.float16, T.BFP16: torch.bfloat16}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, device=DEV, generator=g) * scale).to(dtype)


class Guarded:
    """n buffers of `count` elements in one allocation, `skew` elements off an aligned address, 64 elements of guard either side;
    filled with NaN (0xFF bytes)."""

    def __init__(self, n, count, dtype, skew=0):
        self.count, self.first, self.step = count, 64 + skew, (count + 128 + 15) // 16 * 16 + 16
        size = torch.empty(0, dtype=dtype).element_size()
        self.raw = torch.full((n * self.step * size + 256,), 0xFF, device=DEV, dtype=torch.uint8)
        self.all = self.raw[:n * self.step * size].view(dtype)
        self.n = n

    def __getitem__(self, i):
        at = i * self.step + self.first
        return self.all[at:at + self.count]

    @property
    def ptrs(self):
        return [self[i].data_ptr() for i in range(self.n)] if self.count else [self.all.data_ptr() + self.first] * self.n

    def untouched(self, counts=None):
        """Nothing but the first counts[i] elements of each buffer was written."""
        mask = torch.ones(self.all.numel(), dtype=torch.bool, device=DEV)
        for i in range(self.n):
            at = i * self.step + self.first
            mask[at:at + (self.count if counts is None else counts[i])] = False
        size = self.all.element_size()
        return bool((self.raw[:self.all.numel() * size].view(-1, size)[mask] == 0xFF).all())


def ptrs(ts):
    return [t.data_ptr() for t in ts]


# ---- norm ----------------------------------------------------------------------------------------------------------------

NORM_SIZES = [(1, 1, 1), (2, 3, 7), (1, 5, 8), (3, 2, 100), (2, 4, 511), (1, 9, 512), (2, 3, 1001), (1, 3, 2056), (8, 2, 4096),
              (1, 2, 7168), (1, 3, 16384), (64, 1, 24)]


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("n,rows,elems", NORM_SIZES)
@pytest.mark.parametrize("skew", [0, 1])
def test_norm_and_its_gradient(n, rows, elems, dtype, skew):
    check_norm(n, rows, elems, dtype, skew)


def check_norm(n, rows, elems, dtype, skew):
    g, td, eps = gen(n * 7 + elems), TD[dtype], 1e-6
    x = [normal((rows, elems), td, g) for _ in range(n)]
    res = [normal((rows, elems), td, g, 3.0) for _ in range(n)]
    w = [normal((elems,), td, g) for _ in range(n)]
    bx, br, bw = Guarded(n, rows * elems, td, skew), Guarded(n, rows * elems, td, skew), Guarded(n, elems, td, skew)
    for i in range(n):
        bx[i].copy_(x[i].view(-1)), br[i].copy_(res[i].view(-1)), bw[i].copy_(w[i])
    total, out = Guarded(n, rows * elems, td, skew), Guarded(n, rows * elems, td, skew)
    hcclx.RmsNormPlan(bx.ptrs, bw.ptrs, out.ptrs, rows, elems, dtype, residual=br.ptrs, total=total.ptrs, eps=eps).launch()
    dy = [normal((rows, elems), td, g) for _ in range(n)]
    ds = [normal((rows, elems), td, g) for _ in range(n)]
    dx, dw = Guarded(n, rows * elems, td, skew), Guarded(n, elems, td, skew)
    hcclx.RmsNormGradPlan(ptrs(dy), total.ptrs, bw.ptrs, dx.ptrs, dw.ptrs, rows, elems, dtype, dtotal=ptrs(ds), eps=eps).launch()
    torch.cuda.synchronize()
    for i in range(n):
        want = (x[i].double() + res[i].double()).to(td)
        s = total[i].view(rows, elems)
        if dtype == T.FP32:
            want = x[i] + res[i]
        assert torch.equal(s, want), i
        O.assert_close(out[i].view(rows, elems), *O.norm(s, w[i], eps), f"out of rank {i}")
        wdx, bdx, wdw, bdw = O.norm_grad(dy[i], s, w[i], ds[i], eps)
        O.assert_close(dx[i].view(rows, elems), wdx, bdx, f"dx of rank {i}")
        O.assert_close(dw[i], wdw, bdw, f"dw of rank {i}")
    for b in (total, out, dx, dw):
        assert b.untouched()


@pytest.mark.parametrize("rows", [1000, 4099])
def test_norm_gradient_of_many_rows_per_workgroup(rows):
    """More rows than workgroups: each adds up several, and the parts are joined."""
    g, elems, n = gen(rows), 136, 2
    t = [normal((rows, elems), torch.bfloat16, g, 2.0) for _ in range(n)]
    dy = [normal((rows, elems), torch.bfloat16, g) for _ in range(n)]
    w = [normal((elems,), torch.bfloat16, g) for _ in range(n)]
    dx, dw = [torch.empty_like(x) for x in t], [torch.empty_like(x) for x in w]
    plan = hcclx.RmsNormGradPlan(ptrs(dy), ptrs(t), ptrs(w), ptrs(dx), ptrs(dw), rows, elems, T.BFP16, eps=1e-5)
    plan.launch()
    torch.cuda.synchronize()
    first = [x.clone() for x in dw]
    for i in range(n):
        wdx, bdx, wdw, bdw = O.norm_grad(dy[i], t[i], w[i], None, 1e-5)
        O.assert_close(dx[i], wdx, bdx)
        O.assert_close(dw[i], wdw, bdw)
    for _ in range(3):
        plan.launch()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, dw))       # the order of the additions is fixed
    hcclx.RmsNormGradPlan(ptrs(dy), ptrs(t), ptrs(w), ptrs(dy), None, rows, elems, T.BFP16, eps=1e-5).launch()   # dx on top of dy
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(dx, dy))


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("n,rows,elems", [(64, 9, 40), (2, 37, 300), (1, 5, 6000), (3, 6, 8200), (1, 3, 12300), (2, 4, 16384)])
def test_norm_gradient_of_every_workgroup_shape(n, rows, elems, dtype):
    """One to four wavefronts per row, several rows per workgroup, eight, twelve and sixteen wavefronts."""
    check_norm(n, rows, elems, dtype, 0)


def test_norm_gradient_against_differences():
    """The gradients, times a direction, against the 64-bit norm's difference along it."""
    g, rows, elems = gen(3), 6, 264
    t, w = normal((rows, elems), torch.float32, g), normal((elems,), torch.float32, g)
    dy = normal((rows, elems), torch.float32, g)
    dx, dw = torch.empty_like(t), torch.empty_like(w)
    hcclx.RmsNormGradPlan([dy.data_ptr()], [t.data_ptr()], [w.data_ptr()], [dx.data_ptr()], [dw.data_ptr()], rows, elems, T.FP32).launch()
    torch.cuda.synchronize()
    along_t, along_w, h = normal((rows, elems), torch.float64, g), normal((elems,), torch.float64, g), 1e-6

    def loss(k):
        return float((O.norm(t.double() + k * along_t, w.double() + k * along_w, 1e-6)[0] * dy.double()).sum())
    want = (loss(h) - loss(-h)) / (2 * h)
    got = float((dx.double() * along_t).sum() + (dw.double() * along_w).sum())
    size = float((dx.double() * along_t).abs().sum() + (dw.double() * along_w).abs().sum())
    assert abs(got - want) <= 1e-6 * size      # 32-bit gradients: 100 E of each term; the difference: h^2 and 1e-16 / h of them


@pytest.mark.parametrize("in_place", ["total is x", "total is residual", "out is x"])
def test_norm_in_place(in_place):
    g, rows, elems = gen(1), 33, 1032
    x, r = normal((rows, elems), torch.bfloat16, g), normal((rows, elems), torch.bfloat16, g)
    w = normal((elems,), torch.bfloat16, g)
    total, out = torch.empty_like(x), torch.empty_like(x)
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], [out.data_ptr()], rows, elems, T.BFP16, residual=[r.data_ptr()],
                      total=[total.data_ptr()]).launch()
    torch.cuda.synchronize()
    to_total = x if in_place == "total is x" else r if in_place == "total is residual" else torch.empty_like(x)
    to_out = x if in_place == "out is x" else torch.empty_like(x)
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], [to_out.data_ptr()], rows, elems, T.BFP16, residual=[r.data_ptr()],
                      total=[to_total.data_ptr()]).launch()
    torch.cuda.synchronize()
    assert torch.equal(to_total, total) and torch.equal(to_out, out)


def test_norm_without_residual_and_of_no_rows():
    g, rows, elems = gen(2), 4, 40
    x, w = normal((rows, elems), torch.float16, g), normal((elems,), torch.float16, g)
    x[1] = 0                                                       # 1 / sqrt(eps) times nothing
    out = Guarded(1, rows * elems, torch.float16)
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], out.ptrs, 0, elems, T.FP16).launch()
    dw = torch.full_like(w, 7)
    hcclx.RmsNormGradPlan([x.data_ptr()], [x.data_ptr()], [w.data_ptr()], [x.data_ptr()], [dw.data_ptr()], 0, elems, T.FP16).launch()
    torch.cuda.synchronize()
    assert out.untouched([0]) and bool((dw == 0).all())
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], out.ptrs, rows, elems, T.FP16).launch()
    torch.cuda.synchronize()
    O.assert_close(out[0].view(rows, elems), *O.norm(x, w, 1e-6))
    assert out.untouched()


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("n,rows,elems", [(1, 1, 16), (2, 5, 48), (3, 4, 1040), (2, 3, 7168), (1, 2, 16384)])
def test_norm_to_8_bits(n, rows, elems, dtype):
    g, td = gen(elems), TD[dtype]
    x = [normal((rows, elems), td, g) for _ in range(n)]
    r = [normal((rows, elems), td, g) for _ in range(n)]
    w = [normal((elems,), td, g) for _ in range(n)]
    x[0][0], r[0][0] = 0, 0                                        # a row of zeros
    if rows > 1 and dtype != T.FP16:
        for i in range(n):
            w[i] *= 1e-30                                          # results whose scale's inverse is near the end of the range
    total, width = [torch.empty_like(t) for t in x], elems + hcclx.ROW8_TAIL
    out = Guarded(n, rows * width, torch.uint8)
    hcclx.RmsNormPlan(ptrs(x), ptrs(w), out.ptrs, rows, elems, dtype, residual=ptrs(r), total=ptrs(total), out_dtype=T.FP8E4M3).launch()
    torch.cuda.synchronize()
    assert out.untouched()
    for i in range(n):
        b = out[i].view(rows, width)
        codes = b[:, :elems].contiguous().view(torch.float8_e4m3fn).double()
        scale = b[:, elems:elems + 4].contiguous().view(torch.float32).double()
        assert bool((b[:, elems + 4:] == 0).all())
        y, off = O.norm(total[i], w[i], 1e-6)
        want = y.abs().amax(1, keepdim=True) / 448
        assert bool(((scale - want).abs() <= 42 * O.E * want + 2.0 ** -149).all())
        a = (codes.abs() * scale)
        half = O.e4m3_gap(torch.where(scale > 0, y.abs() / scale.clamp(min=1e-300), 0)) * scale / 2
        assert bool(((a - y.abs()).abs() <= half * (1 + 1e-4) + off + 4 * O.E * y.abs()).all())
        assert bool((torch.sign(codes) * torch.sign(y) >= 0).all())
        assert bool((codes[(y == 0)] == 0).all())


def test_norm_keeps_what_is_not_finite_in_its_row():
    g, rows, elems = gen(9), 4, 64
    x, w = normal((rows, elems), torch.bfloat16, g), torch.ones(elems, device=DEV, dtype=torch.bfloat16)
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    out, out8 = torch.empty_like(x), torch.empty((rows, elems + 16), device=DEV, dtype=torch.uint8)
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], [out.data_ptr()], rows, elems, T.BFP16).launch()
    hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], [out8.data_ptr()], rows, elems, T.BFP16, out_dtype=T.FP8E4M3).launch()
    torch.cuda.synchronize()
    codes = out8[:, :elems].contiguous().view(torch.float8_e4m3fn).float()
    assert bool(out[1].isnan().all()) and bool(out[2, 7].isnan()) and bool((out[2, :7] == 0).all())
    assert bool(codes[1].isnan().all()) and bool(codes[2, 7].isnan())
    for r in (0, 3):
        assert bool(out[r].isfinite().all()) and bool(codes[r].isfinite().all())


# ---- AdamW ---------------------------------------------------------------------------------------------------------------

COUNTS = [1, 3, 255, 256, 257, 0, 1024, 2047, 2048, 2049, 5000, 70001]


def adam_tensors(counts, grad, g, pad=0):
    """Flat buffers of all tensors back to back (pad elements between them) and each tensor's place."""
    starts = np.concatenate([[0], np.cumsum([c + pad for c in counts])]).astype(int)
    total = int(starts[-1])
    level = torch.exp(torch.randn(total, device=DEV, generator=g)) * 1e-2
    flat = dict(param=normal((total,), torch.float32, g, 0.5), grad=(torch.randn(total, device=DEV, generator=g) * level).to(grad),
                m=torch.randn(total, device=DEV, generator=g) * level * 0.3, v=(torch.rand(total, device=DEV, generator=g) * level) ** 2)
    return flat, starts[:-1], total


@pytest.mark.parametrize("grad", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("copy", [None, T.BFP16, T.FP16])
def test_adamw_with_32_bit_states(grad, copy):
    """Three steps over tensors of all lengths, back to back (most of them at addresses aligned to an element only)."""
    g = gen(grad)
    flat, starts, total = adam_tensors(COUNTS, TD[grad], g)
    c16 = torch.full((total,), float("nan"), device=DEV, dtype=TD[copy] if copy else torch.float16)
    factor = torch.tensor([0.25], device=DEV)
    decay = [0.1 * (k % 3) for k in range(len(COUNTS))]
    tensors = [dict(count=c, param=flat["param"].data_ptr() + 4 * int(s), m=flat["m"].data_ptr() + 4 * int(s), v=flat["v"].data_ptr() + 4 * int(s),
                    grad=flat["grad"].data_ptr() + flat["grad"].element_size() * int(s), weight_decay=d,
                    copy=c16.data_ptr() + 2 * int(s) if copy else 0) for c, s, d in zip(COUNTS, starts, decay)]
    plan = hcclx.AdamWPlan(tensors, grad, T.FP32, copy)
    wd = torch.cat([torch.full((c,), d, dtype=torch.float64, device=DEV) for c, d in zip(COUNTS, decay)])
    for step in (1, 2, 1000):
        before = {k: v.clone() for k, v in flat.items()}
        lr, b1, b2, eps = 0.01, 0.9, 0.95, 1e-8
        plan.step(step, lr=lr, beta1=b1, beta2=b2, eps=eps, grad_scale=factor.data_ptr() if step == 2 else 0)
        torch.cuda.synchronize()
        x = before["grad"].double() * (0.25 if step == 2 else 1.0)
        p, m, v, update = O.adamw(x, before["param"], before["m"], before["v"], step, lr, b1, b2, eps, wd)
        # betas, their complements and products: a few roundings of each term; the update divides two of them
        big_m = (b1 * before["m"].double()).abs() + ((1 - b1) * x).abs()
        O.assert_close(flat["m"], m, 6 * O.E * big_m, "m")
        O.assert_close(flat["v"], v, 6 * O.E * v, "v")
        big = big_m / m.abs().clamp(min=1e-300) * update.abs()
        O.assert_close(flat["param"], p, lr * 16 * O.E * big + 4 * O.E * (1 + lr * wd) * before["param"].double().abs(), "param")
        if copy:
            assert torch.equal(c16, flat["param"].to(TD[copy]))


def states8(flat, counts, starts, codes_at):
    """8-bit states of m and sqrt(v), nearest codes."""
    total = flat["m"].numel()
    blocks = [(c + 255) // 256 for c in counts]
    at = np.concatenate([[0], np.cumsum(blocks)]).astype(int)
    out = {}
    for name, x in (("m", flat["m"]), ("v", flat["v"].sqrt())):
        codes = torch.full((total + codes_at,), 0xFF, device=DEV, dtype=torch.uint8)
        scales = torch.zeros(int(at[-1]) + 1, device=DEV)
        for c, s, b, nb in zip(counts, starts, at, blocks):
            if c == 0:
                continue
            y = torch.nn.functional.pad(x[s:s + c], (0, nb * 256 - c)).view(nb, 256)
            scale = y.abs().amax(1) / 448
            scales[b:b + nb] = scale
            q = (y / scale.clamp(min=1e-30)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).view(-1)[:c]
            codes[codes_at + s:codes_at + s + c] = q
        out[name], out[name + "_scale"] = codes, scales
    return out, at[:-1], blocks


def tensors8(flat, st, counts, starts, at, codes_at, c16=None, decay=0.0):
    return [dict(count=c, param=flat["param"].data_ptr() + 4 * int(s), grad=flat["grad"].data_ptr() + flat["grad"].element_size() * int(s),
                 m=st["m"].data_ptr() + codes_at + int(s), v=st["v"].data_ptr() + codes_at + int(s), m_scale=st["m_scale"].data_ptr() + 4 * int(b),
                 v_scale=st["v_scale"].data_ptr() + 4 * int(b), copy=c16.data_ptr() + 2 * int(s) if c16 is not None else 0, weight_decay=decay)
            for c, s, b in zip(counts, starts, at)]


@pytest.mark.parametrize("grad", [T.FP32, T.FP16, T.BFP16])
def test_adamw_with_8_bit_states(grad):
    counts, codes_at, seed, step = COUNTS, 3, 0xDEADBEEF, 7
    lr, b1, b2, eps, decay = 0.01, 0.9, 0.999, 1e-8, 0.05
    flat, starts, total = adam_tensors(counts, TD[grad], gen(grad + 50))
    flat["grad"][int(starts[6]):int(starts[6]) + 256] = 0          # a block whose gradients and states are zero
    flat["m"][int(starts[6]):int(starts[6]) + 256] = 0
    flat["v"][int(starts[6]):int(starts[6]) + 256] = 0
    st, at, blocks = states8(flat, counts, starts, codes_at)
    c16 = torch.empty(total, device=DEV, dtype=torch.bfloat16)
    before = {k: v.clone() for k, v in {**flat, **st}.items()}
    flat["m"] = flat["v"] = None
    plan = hcclx.AdamWPlan(tensors8(flat, st, counts, starts, at, codes_at, c16, decay), grad, T.FP8E4M3, T.BFP16)
    plan.step(step, lr=lr, beta1=b1, beta2=b2, eps=eps, seed=seed)
    torch.cuda.synchronize()
    assert torch.equal(c16, flat["param"].to(torch.bfloat16))
    assert bool((st["m"][:codes_at] == 0xFF).all()) and bool((st["v"][:codes_at] == 0xFF).all())
    for k, (c, s, b, nb) in enumerate(zip(counts, starts, at, blocks)):
        if c == 0:
            continue
        s, b = int(s), int(b)

        def old(name):
            codes = before[name][codes_at + s:codes_at + s + c].view(torch.float8_e4m3fn).double()
            return codes * before[name + "_scale"][b:b + nb].double().repeat_interleave(256)[:c]
        g = before["grad"][s:s + c].double()
        m0, v0 = old("m"), old("v") ** 2
        p, m, v, update = O.adamw(g, before["param"][s:s + c], m0, v0, step, lr, b1, b2, eps, decay)
        big_m = (b1 * m0).abs() + ((1 - b1) * g).abs()
        big = big_m / m.abs().clamp(min=1e-300) * update.abs()
        O.assert_close(flat["param"][s:s + c], p, lr * 24 * O.E * big + 4 * O.E * before["param"][s:s + c].double().abs(), f"param of {k}")
        us = O.draws(seed, k, c)
        for name, x, u, loose in (("m", m, us[0], 8 * O.E * big_m), ("v", v.sqrt(), us[1], 8 * O.E * v.sqrt())):
            scale = torch.nn.functional.pad(x, (0, nb * 256 - c)).view(nb, 256).abs().amax(1) / 448
            got_scale = st[name + "_scale"][b:b + nb].double()
            worst = torch.nn.functional.pad(loose, (0, nb * 256 - c)).view(nb, 256).amax(1) / 448
            assert bool(((got_scale - scale).abs() <= worst + 2 * O.E * scale).all()), (k, name)
            each = got_scale.repeat_interleave(256)[:c]
            q = st[name][codes_at + s:codes_at + s + c].view(torch.float8_e4m3fn).double()
            a = torch.where(each > 0, x.abs() / each.clamp(min=1e-300), 0).clamp(max=448)
            slack = torch.where(each > 0, loose / each.clamp(min=1e-300), 0) + 4 * O.E * a
            # a magnitude that rounds to the next power of two in 32 bits has that one's gap
            gap = O.e4m3_gap(a)
            place = a / gap
            frac = place - torch.floor(place) + u.to(DEV)
            want = (torch.floor(place) + (frac >= 1).double()) * gap
            unsure = ((frac - 1).abs() <= slack / gap + 2.0 ** -22) | ((place - torch.round(place)).abs() <= slack / gap + 2.0 ** -22)
            unsure &= x != 0                                       # a zero is a zero
            off = (q.abs() - want).abs()
            assert bool((off[~unsure] == 0).all()), (k, name, int((off[~unsure] != 0).sum()))
            assert bool((off <= gap * (1 + 1e-9)).all())
            assert bool((torch.sign(q) * torch.sign(x) >= 0).all())
            assert float(unsure.double().mean()) < 0.05 or c < 100


def test_adamw_8_bit_moving_average_moves():
    """v, whose change of a step is far below half a code, reaches the gradients' mean square all the same."""
    n = 256 * 64
    g = torch.full((n,), 0.01, device=DEV)
    g[::256] = 1.0                                                 # every block's scale is another element's
    p = torch.zeros(n, device=DEV)
    codes = [torch.zeros(n, device=DEV, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.zeros(n // 256, device=DEV) for _ in range(2)]
    plan = hcclx.AdamWPlan([dict(count=n, param=p.data_ptr(), grad=g.data_ptr(), m=codes[0].data_ptr(), v=codes[1].data_ptr(),
                                 m_scale=scales[0].data_ptr(), v_scale=scales[1].data_ptr())], T.FP32, T.FP8E4M3)
    b2, steps = 0.99, 600
    for k in range(steps):
        plan.step(k + 1, lr=0.0, beta2=b2, seed=k)
    torch.cuda.synchronize()
    v = (codes[1].view(torch.float8_e4m3fn).double() * scales[1].double().repeat_interleave(256)) ** 2
    small = torch.ones(n, dtype=torch.bool, device=DEV)
    small[::256] = False
    want = 1e-4 * (1 - b2 ** steps)
    # a step moves sqrt(v) by (1 - b2) / 2 of its distance and adds noise of at most gap^2 / 4 (gap: 1/8): what stays of the noise
    # is a few percent of each element, and over 16320 elements a fraction of a percent of the mean of sqrt(v)
    assert abs(float(v[small].sqrt().mean()) / want ** 0.5 - 1) < 0.02


def test_adamw_what_is_not_finite_stays_in_its_block():
    n = 1024
    for small in (False, True):
        g = torch.full((n,), 0.1, device=DEV)
        g[3], g[300] = float("nan"), float("inf")
        p = torch.ones(n, device=DEV)
        m, v = (torch.zeros(n, device=DEV, dtype=torch.uint8 if small else torch.float32) for _ in range(2))
        ms, vs = (torch.zeros(4, device=DEV) for _ in range(2))
        hcclx.AdamWPlan([dict(count=n, param=p.data_ptr(), grad=g.data_ptr(), m=m.data_ptr(), v=v.data_ptr(), m_scale=ms.data_ptr(),
                              v_scale=vs.data_ptr())], T.FP32, T.FP8E4M3 if small else T.FP32).step(1, lr=0.1)
        torch.cuda.synchronize()
        assert bool(p[3].isnan()) and bool(p[300].isnan())
        ok = torch.ones(n, dtype=torch.bool, device=DEV)
        ok[3], ok[300] = False, False
        assert torch.allclose(p[ok], torch.full_like(p[ok], 0.9), rtol=1e-6)
        if small:
            f = m.view(torch.float8_e4m3fn).float()
            assert bool(f[3].isnan()) and bool(f[512:].isfinite().all()) and bool((f[512:] == 448).all())


# ---- the experts' block --------------------------------------------------------------------------------------------------

class Ffn:
    """Inputs of an experts' block with `rows` rows per rank in buffers of `capacity`, NaN behind them."""

    def __init__(self, rows, capacity, dim, hidden, dtype, seed, per_rank=1, unit=None, scale=1.0):
        g, td, n = gen(seed), TD[dtype], len(rows)
        self.rows, self.capacity, self.dim, self.hidden, self.dtype, self.n = rows, capacity, dim, hidden, dtype, n
        self.x, self.dy = Guarded(n, capacity * dim, td), Guarded(n, capacity * dim, td)
        for i, r in enumerate(rows):
            self.x[i][:r * dim] = normal((r * dim,), td, g, scale)
            self.dy[i][:r * dim] = normal((r * dim,), td, g)
        self.w = [[normal((hidden, dim), td, g, dim ** -0.5) for _ in range(n)], [normal((hidden, dim), td, g, dim ** -0.5) for _ in range(n)],
                  [normal((dim, hidden), td, g, hidden ** -0.5) for _ in range(n)]]
        unit = unit or dim
        parts = torch.zeros((n, per_rank), dtype=torch.int64)
        for i, r in enumerate(rows):
            for k in range(r):
                parts[i, (k * k + i) % per_rank] += 1
        self.counts = (parts * unit).to(DEV)
        self.shape = dict(capacity=capacity, dim=dim, hidden=hidden, dtype=dtype, counts=self.counts.data_ptr(), counts_per_rank=per_rank, count_unit=unit)
        self.total = sum(rows)

    def run(self, act=0, bound=None, grad=True, **more):
        shape = {**self.shape, "rows": self.total if bound is None else bound, "activation": act, **more}
        room = shape["rows"] or self.n * self.capacity
        td = TD[self.dtype]
        self.saved = torch.full((hcclx.gated_ffn_saved_bytes(room, self.hidden) + 256,), 0xFF, device=DEV, dtype=torch.uint8)
        self.out, self.dx = Guarded(self.n, self.capacity * self.dim, td), Guarded(self.n, self.capacity * self.dim, td)
        self.dw = [Guarded(self.n, self.hidden * self.dim, td) for _ in range(3)]
        w = [ptrs(k) for k in self.w]
        self.plan = hcclx.GatedFfnPlan(self.x.ptrs, *w, self.out.ptrs, saved=self.saved.data_ptr() if grad else 0, **shape)
        self.plan.launch()
        if grad:
            self.grad_plan = hcclx.GatedFfnGradPlan(self.dy.ptrs, self.x.ptrs, *w, self.saved.data_ptr(), self.dx.ptrs,
                                                    *[k.ptrs for k in self.dw], **shape)
            self.grad_plan.launch()
        torch.cuda.synchronize()

    def check(self, act=0, grad=True, rows=None):
        rows = rows or self.rows
        for i, r in enumerate(rows):
            view = lambda b: b[i][:r * self.dim].view(r, self.dim)
            want = O.ffn(view(self.x), self.w[0][i], self.w[1][i], self.w[2][i], act, TD[self.dtype], view(self.dy) if grad else None)
            O.assert_close(view(self.out), *want[0], f"out of rank {i}")
            if grad:
                O.assert_close(view(self.dx), *want[1], f"dx of rank {i}")
                for k, name in enumerate(("dw_gate", "dw_up", "dw_down")):
                    shape = (self.dim, self.hidden) if k == 2 else (self.hidden, self.dim)
                    O.assert_close(self.dw[k][i].view(shape), *want[2 + k], f"{name} of rank {i}")
        counts = [r * self.dim for r in rows]
        assert self.out.untouched(counts)
        if grad:
            assert self.dx.untouched(counts) and all(d.untouched() for d in self.dw)
            assert bool((self.saved[hcclx.gated_ffn_saved_bytes(sum(rows), self.hidden):] == 0xFF).all())


FFN_CASES = [([1], 1, 8, 8), ([3], 3, 16, 24), ([0, 5, 1], 6, 72, 40), ([17, 0, 0, 2], 20, 64, 64), ([130, 1, 129], 131, 136, 264),
             ([64, 200], 200, 520, 136), ([2, 33], 40, 1032, 520), ([1] * 16, 2, 256, 128), ([0, 0], 3, 32, 32), ([300], 300, 328, 72)]


@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,capacity,dim,hidden", FFN_CASES)
@pytest.mark.parametrize("act", [0, 1])
def test_ffn_forward_and_backward(rows, capacity, dim, hidden, dtype, act):
    f = Ffn(rows, capacity, dim, hidden, dtype, dim + hidden, per_rank=1 + dim % 5, scale=2.0)
    f.run(act)
    f.check(act)


@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,dim,hidden", [([1], 4096, 2048), ([5, 0, 16, 2], 2880, 1432), ([16, 17], 1024, 4096), ([40, 64, 7, 1], 1536, 768)])
def test_ffn_of_few_rows(rows, dim, hidden, dtype):
    f = Ffn(rows, max(rows), dim, hidden, dtype, dim)
    f.run(grad=False)
    f.check(grad=False)


@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,dim,hidden", [([2100, 3900, 0, 1001], 2064, 2312), ([4096], 4104, 4096)])
def test_ffn_of_many_rows(rows, dim, hidden, dtype):
    """Tiles of the largest products, with ragged edges in every direction."""
    f = Ffn(rows, max(rows), dim, hidden, dtype, 5)
    f.run()
    f.check()


# On both sides of where another kernel, tile or split of what is left of a round takes over (256 CUs).
FFN_EDGES = [([16], 16, 264, 520), ([17], 17, 264, 520), ([32], 32, 520, 264), ([33], 33, 520, 264), ([64], 64, 1032, 136), ([65], 65, 1032, 136),
             ([128, 128], 128, 264, 136), ([128, 129], 129, 264, 136), ([100, 0, 20, 128], 128, 1032, 520), ([0, 0], 400, 264, 136),
             ([0, 700, 0], 700, 136, 264), ([2000], 2000, 648, 1272), ([3900], 3900, 1288, 1272), ([1], 700, 520, 264),
             ([90, 0, 128, 33, 70, 1, 65, 120], 128, 5128, 2120), ([100, 3] * 16, 100, 1288, 1096)]


@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,capacity,dim,hidden", FFN_EDGES)
def test_ffn_at_the_edges_of_its_kernels(rows, capacity, dim, hidden, dtype):
    f = Ffn(rows, capacity, dim, hidden, dtype, 3 * dim + hidden)
    f.run()
    f.check()
    if capacity > max(rows):                                       # the same rows in plans made for capacity
        f.run(bound=0)
        f.check()


@pytest.mark.parametrize("capacity", [4, 100, 300])
def test_ffn_of_64_ranks(capacity):
    """As many ranks as there are, some without rows, in plans for few rows, small tiles and whole ones."""
    f = Ffn([k * 7 % 5 for k in range(64)], capacity, 72, 136, T.BFP16, capacity, per_rank=3)
    f.run(bound=0)
    f.check()


def test_ffn_of_rows_from_many_senders():
    f = Ffn([5, 164, 0], 170, 72, 136, T.BFP16, 12, per_rank=63)
    f.run()
    f.check()


def test_ffn_rows_are_counted_on_the_device():
    """One plan, launched after the counts change; rows beyond capacity, and beyond the bound on all rows, are left alone."""
    f = Ffn([9, 4, 7], 9, 64, 48, T.BFP16, 4, per_rank=3)
    f.run(bound=20)
    f.check()
    g = torch.zeros_like(f.counts)
    for rows, bound, want in (([2, 9, 0], 20, [2, 9, 0]), ([12, 3, 1], 20, [9, 3, 1]), ([9, 9, 9], 20, [9, 9, 2]), ([30, 30, 30], 5, [5, 0, 0])):
        f.x, f.dy = Guarded(3, 9 * 64, torch.bfloat16), Guarded(3, 9 * 64, torch.bfloat16)
        gg = gen(sum(rows))
        for i, r in enumerate(want):
            f.x[i][:r * 64] = normal((r * 64,), torch.bfloat16, gg)
            f.dy[i][:r * 64] = normal((r * 64,), torch.bfloat16, gg)
        g[:, 1] = torch.tensor(rows, device=DEV) * 64
        f.counts.copy_(g)
        f.run(bound=bound)
        f.check(rows=want)
    f.counts.fill_(1 << 40)                                        # nonsense counts: capacity rows, as far as the bound goes
    f.x, f.dy = Guarded(3, 9 * 64, torch.bfloat16), Guarded(3, 9 * 64, torch.bfloat16)
    for i in range(3):
        f.x[i].copy_(normal((9 * 64,), torch.bfloat16, gen(i)))
        f.dy[i].copy_(normal((9 * 64,), torch.bfloat16, gen(9 + i)))
    f.run(bound=0)
    f.check(rows=[9, 9, 9])
    f.run(bound=0, counts=0)
    f.check(rows=[9, 9, 9])


def test_ffn_gradient_against_differences():
    """The gradients, times a direction, against the 64-bit block's difference along it."""
    f = Ffn([13, 6], 13, 72, 56, T.FP16, 8)
    f.run()
    g = gen(77)
    got = size = 0.0
    dirs = []
    for i, r in enumerate(f.rows):
        d = [normal((r, 72), torch.float64, g)] + [normal(tuple(w[i].shape), torch.float64, g, 0.1) for w in f.w]
        dirs.append(d)
        for t, grad in zip(d, [f.dx[i][:r * 72].view(r, 72)] + [k[i].view(w[i].shape) for k, w in zip(f.dw, f.w)]):
            got += float((grad.double() * t).sum())
            size += float((grad.double() * t).abs().sum())

    def loss(h):
        total = 0.0
        for i, r in enumerate(f.rows):
            x, wg, wu, wd = (t.double() + h * d for t, d in zip([f.x[i][:r * 72].view(r, 72)] + [w[i] for w in f.w], dirs[i]))
            a, _ = O.act(x @ wg.T, 0)
            total += float((((a * (x @ wu.T)) @ wd.T) * f.dy[i][:r * 72].view(r, 72).double()).sum())
        return total
    h = 1e-5
    want = (loss(h) - loss(-h)) / (2 * h)
    assert abs(got - want) <= 4 * O.U[torch.float16] * size        # each gradient: its own rounding and its operands'


@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,dim,hidden", [([1], 16, 8), ([3, 0, 70], 1040, 136), ([2, 2], 2048, 512), ([600, 900], 528, 264)])
def test_ffn_of_8_bit_rows(rows, dim, hidden, dtype):
    """Rows as the norm writes them: codes and a scale each; counts in elements of those rows."""
    check_8_bit_rows(rows, dim, hidden, dtype)


@pytest.mark.parametrize("dtype", [T.FP16, T.BFP16])
@pytest.mark.parametrize("rows,dim,hidden", [([16], 272, 136), ([17], 272, 136), ([20, 40, 3], 528, 72), ([64], 1040, 136), ([65], 1040, 136),
                                             ([100, 0, 9, 128], 1040, 264), ([129], 272, 136)])
def test_ffn_of_8_bit_rows_at_the_edges_of_its_kernels(rows, dim, hidden, dtype):
    check_8_bit_rows(rows, dim, hidden, dtype)


def check_8_bit_rows(rows, dim, hidden, dtype):
    n, cap, g, td = len(rows), max(rows), gen(dim), TD[dtype]
    x = [normal((cap, dim), torch.float32, g, 4.0) for _ in range(n)]
    w = torch.ones(dim, device=DEV)
    x8 = torch.empty((n, cap, dim + 16), device=DEV, dtype=torch.uint8)
    hcclx.RmsNormPlan(ptrs(x), [w.data_ptr()] * n, ptrs(x8), cap, dim, T.FP32, out_dtype=T.FP8E4M3).launch()
    f = Ffn(rows, cap, dim, hidden, dtype, 6, unit=dim + 16)
    f.out = Guarded(n, cap * dim, td)
    for i, r in enumerate(rows):
        x8[i, r:] = 0xFF
    hcclx.GatedFfnPlan(ptrs(x8), *[ptrs(k) for k in f.w], f.out.ptrs, rows=sum(rows), x_dtype=T.FP8E4M3, **f.shape).launch()
    torch.cuda.synchronize()
    for i, r in enumerate(rows):
        b = x8[i, :r]
        values = b[:, :dim].contiguous().view(torch.float8_e4m3fn).double() * b[:, dim:dim + 4].contiguous().view(torch.float32).double()
        want = O.ffn(values, f.w[0][i], f.w[1][i], f.w[2][i], 0, td)
        O.assert_close(f.out[i][:r * dim].view(r, dim), *want[0], f"out of rank {i}")
    assert f.out.untouched([r * dim for r in rows])


def test_ffn_saturated_activations():
    """Gates far out on both sides, where exp overflows."""
    f = Ffn([6], 6, 64, 64, T.BFP16, 2, scale=200.0)
    for act in (0, 1):
        f.run(act)
        assert all(bool(t.isfinite().all()) for t in (f.out[0], f.dx[0], f.dw[0][0], f.dw[1][0], f.dw[2][0]))
        f.check(act)


# ---- streams, graphs, refusals ---------------------------------------------------------------------------------------------

def test_operators_in_a_graph_and_on_another_stream():
    """Every plan captured into one graph and replayed between eager work, each replay against eager launches."""
    f = Ffn([20, 3], 20, 136, 72, T.BFP16, 1)
    f.run()
    g = gen(5)
    rows, elems = 10, 136
    x, r, w = normal((rows, elems), torch.bfloat16, g), normal((rows, elems), torch.bfloat16, g), normal((elems,), torch.bfloat16, g)
    total, out, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty_like(w)
    norm = hcclx.RmsNormPlan([x.data_ptr()], [w.data_ptr()], [out.data_ptr()], rows, elems, T.BFP16, residual=[r.data_ptr()],
                             total=[total.data_ptr()])
    norm_grad = hcclx.RmsNormGradPlan([out.data_ptr()], [total.data_ptr()], [w.data_ptr()], [dx.data_ptr()], [dw.data_ptr()], rows, elems, T.BFP16)
    p, m, v = (torch.zeros(5000, device=DEV) for _ in range(3))
    grad = normal((5000,), torch.float32, g)
    adam = hcclx.AdamWPlan([dict(count=5000, param=p.data_ptr(), grad=grad.data_ptr(), m=m.data_ptr(), v=v.data_ptr())], T.FP32, T.FP32)

    def everything(stream):
        norm.launch(stream)
        norm_grad.launch(stream)
        f.plan.launch(stream)
        f.grad_plan.launch(stream)
        adam.step(3, lr=0.1, stream=stream)

    outputs = [total, out, dx, dw, f.out.all, f.dx.all] + [d.all for d in f.dw]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        everything(torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        f.x[0][:20 * 136] = normal((20 * 136,), torch.bfloat16, g)
        x.copy_(normal((rows, elems), torch.bfloat16, g))
        states = [t.clone() for t in (p, m, v)]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            everything(stream.cuda_stream)
        stream.synchronize()
        want = [t.view(torch.uint8).clone() for t in outputs + [p, m, v]]
        for t, s in zip((p, m, v), states):
            t.copy_(s)
        for t in (total, out, dx, dw):
            t.fill_(float(k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outputs + [p, m, v]):
            assert torch.equal(a, b.view(torch.uint8))


def test_a_plan_says_what_it_is():
    f = Ffn([3], 3, 16, 16, T.BFP16, 1)
    f.run()
    assert f.plan.bytes > 0 and f.plan.table_bytes > 0
    p = torch.zeros(8, device=DEV)
    adam = hcclx.AdamWPlan([dict(count=8, param=p.data_ptr(), grad=p.data_ptr(), m=p.data_ptr(), v=p.data_ptr())], T.FP32, T.FP32)
    with pytest.raises(HcclError) as e:
        adam.launch()
    assert e.value.code == 1 and "hcclx_adamw_step" in str(e.value)
    for bad in (dict(step=0, lr=1.0), dict(step=1, lr=1.0, beta1=1.0), dict(step=1, lr=1.0, beta2=-0.1), dict(step=1, lr=1.0, eps=-1.0)):
        with pytest.raises(HcclError):
            adam.step(**bad)
    before = hcclx.kernels_launched()
    hcclx.AdamWPlan([], T.FP32, T.FP32).step(1, lr=1.0)
    assert hcclx.kernels_launched() == before
    f.plan.launch()
    assert hcclx.kernels_launched() >= before + 2
