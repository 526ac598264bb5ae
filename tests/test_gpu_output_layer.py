"""The operators of the output layer on the GPU against their definitions in 64 bits (logits_oracle.py): the largest logits, the
distillation loss and its gradients, and the draw, over types, splits over the ranks, sizes, strides and the contents where they can go
wrong."""
import math

import numpy as np
import pytest
import torch

import logits_oracle as L
import ops_oracle as O
from hccl_amd import hcclx
from hccl_amd import types as T

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {T.FP32: torch.float32, T.FP16: torch.float16, T.BFP16: torch.bfloat16}
INF = math.inf


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


class Split:
    """A matrix of logits whose columns the ranks hold: `pad` elements behind every row and `skew` before the first, all NaN; or (one)
    columns of a single matrix."""

    def __init__(self, whole, columns, dtype, pad=0, skew=0, one=False):
        self.rows, self.columns, self.dtype = whole.shape[0], columns, dtype
        td = TD[dtype]
        self.raw, self.parts, at = [], [], 0
        if one:
            raw = torch.full((skew + self.rows * (sum(columns) + pad),), math.nan, device=DEV, dtype=td)
            m = raw[skew:].view(self.rows, -1)
        for c in columns:
            if not one:
                raw = torch.full((skew + self.rows * (c + pad) + 64,), math.nan, device=DEV, dtype=td)
                self.raw.append(raw)
                m = raw[skew:skew + self.rows * (c + pad)].view(self.rows, c + pad)
            part = m[:, at:at + c] if one else m[:, :c]
            part.copy_(whole[:, at:at + c])
            self.parts.append(part)
            at += c
        if one:
            self.raw.append(raw)
        self.strides = [sum(columns) + pad if one else c + pad for c in columns]
        self.ptrs = [p.data_ptr() for p in self.parts]

    @property
    def where(self):
        return dict(columns=self.columns, rows=self.rows, dtype=self.dtype, strides=self.strides)

    def whole(self):
        return torch.cat(self.parts, 1)

    def untouched(self):
        """What lies between the rows is as it was."""
        for p in self.parts:
            p.zero_()
        return all(bool((r.isnan() | (r == 0)).all()) and int((r == 0).sum()) == sum(p.numel() for p in (self.parts if len(self.raw) == 1 else [q]))
                   for r, q in zip(self.raw, self.parts))


def shares(vocab, n):
    each = -(-vocab // n)
    return [max(0, min(each, vocab - j * each)) for j in range(n)]


def contents(kind, rows, vocab, g):
    """Logits of a kind, in 32 bits."""
    x = torch.randn((rows, vocab), device=DEV, generator=g) * 3
    if kind == "steep":
        x = torch.empty((rows, vocab), device=DEV).exponential_(1.0, generator=g) * 1.6 - 4
    if kind == "equal":
        x = torch.full((rows, vocab), -2.5, device=DEV)
    if kind == "coarse":
        x = torch.round(x)                                          # many equal values, zeros of both signs
        x = torch.where((x == 0) & (torch.rand(x.shape, device=DEV, generator=g) < 0.5), -x, x)
    if kind == "falling":
        x = torch.linspace(9, -9, vocab, device=DEV).expand(rows, -1).contiguous()
    if kind == "rising":
        x = torch.linspace(-9, 9, vocab, device=DEV).expand(rows, -1).contiguous()
    if kind == "masked":
        x[torch.rand(x.shape, device=DEV, generator=g) < 0.9] = -INF
        x[:, vocab // 2] = 1.0
    if kind == "odd":                                               # NaN, infinities, the type's lowest value
        r = torch.rand(x.shape, device=DEV, generator=g)
        x[r < 0.05] = math.nan
        x[(r > 0.1) & (r < 0.3)] = -INF
        x[(r > 0.3) & (r < 0.5)] = -60000.0
    if kind == "nothing":
        x[:] = -INF
        x[:, ::3] = math.nan
    return x


KINDS = ["normal", "steep", "equal", "coarse", "falling", "rising", "masked", "odd", "nothing"]

# ---- the largest logits ----------------------------------------------------------------------------------------------------


def check_top(x, columns, dtype, k, pad=0, skew=0, one=False):
    s = Split(x.to(TD[dtype]), columns, dtype, pad, skew, one)
    rows = s.rows
    values = torch.full((rows, k), 77, device=DEV, dtype=TD[dtype])
    indices = torch.full((rows, k), 77, device=DEV, dtype=torch.int32)
    lse = torch.full((rows,), 77.0, device=DEV)
    hcclx.TopLogitsPlan(s.ptrs, k=k, values=values.data_ptr(), indices=indices.data_ptr(), lse=lse.data_ptr(), **s.where).launch()
    again = torch.empty_like(indices)
    hcclx.TopLogitsPlan(s.ptrs, k=k, values=values.data_ptr(), indices=again.data_ptr(), **s.where).launch()     # without lse
    torch.cuda.synchronize()
    assert torch.equal(again, indices)
    whole = s.whole()
    for r in range(rows):
        l = L.plain(whole[r])
        first = L.order(l)[:k]
        assert torch.equal(indices[r].long(), first), (r, (indices[r].long() != first).nonzero()[:3].flatten().tolist())
        assert torch.equal(values[r].double(), l[first]), r
        want, bound = L.lse(l)
        got = float(lse[r])
        assert got == want or abs(got - want) <= bound + O.E * abs(want), (r, got, want, bound)


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab,n,k", [(1, 1, 1), (7, 2, 7), (65, 1, 3), (1000, 3, 1), (2500, 8, 50), (32003, 4, 700)])
def test_top_logits(vocab, n, k, kind, dtype):
    x = contents(kind, 3, vocab, gen(vocab + k))
    check_top(x, shares(vocab, n), dtype, k, pad=5, skew=1)


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("kind", ["normal", "steep", "equal", "coarse", "falling", "masked"])
@pytest.mark.parametrize("k", [1, 33, 256, 1024])
def test_top_logits_of_many_columns(k, kind, dtype):
    x = contents(kind, 2, 131072 + 77, gen(k))
    check_top(x, [40000, 0, 1, 70000, 131072 + 77 - 110001], dtype, k)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("rows", [1, 300, 1500])
def test_top_logits_of_many_rows(rows, dtype):
    """More rows: more chunks to a wavefront; columns of one matrix."""
    check_top(contents("steep", rows, 5000, gen(rows)), shares(5000, 3), dtype, 20, one=True)


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("kind", KINDS)
def test_top_logits_of_rows_that_fill_the_device(kind, dtype):
    """Small workgroups, whose lists are shorter: up to 256 entries, rows where more than a list holds reaches the k-th."""
    check_top(contents(kind, 800, 1201, gen(62)), shares(1201, 3), dtype, 256, pad=1)
    check_top(contents(kind, 780, 30011, gen(63)), shares(30011, 2), dtype, 100)


def test_top_logits_of_64_ranks_and_a_million_columns():
    check_top(contents("normal", 2, 1 << 20, gen(1)), shares(1 << 20, 64), T.BFP16, 100)
    check_top(contents("coarse", 2, 650, gen(2)), shares(650, 64), T.FP32, 650)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_top_logits_of_any_magnitude(dtype):
    x = contents("normal", 8, 9001, gen(61))
    for r, scale in enumerate((1e30, -1e30, 1e-30, 1e3, 1e6, 1e7, 3e37, 1.0)):
        x[r] *= scale
    x[7, ::2] = torch.finfo(TD[dtype]).min
    check_top(x, shares(9001, 3), dtype, 30)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("each,k", [(3, 100), (3, 192), (10, 70), (40, 300), (40, 900)])
def test_top_logits_of_more_than_there_are_groups(each, k, dtype):
    """Many ranks of few columns: fewer groups of neighbouring columns hold anything than entries are asked for."""
    check_top(contents("normal", 2, 64 * each, gen(k)), [each] * 64, dtype, k)


# ---- distillation ------------------------------------------------------------------------------------------------------------


def entries(whole, k, kind, g):
    """A teacher's list for every row."""
    rows, vocab = whole.shape
    t = torch.nan_to_num(whole.float(), nan=-5.0, neginf=-5.0, posinf=5.0).clamp(-20, 20) + torch.randn(whole.shape, device=DEV, generator=g)
    values, at = t.topk(min(k, vocab), dim=1)
    if k > vocab:
        values, at = torch.nn.functional.pad(values, (0, k - vocab)), torch.nn.functional.pad(at, (0, k - vocab), value=-1)
    at = at.to(torch.int32)
    if kind == "holes":                                             # no entry, none that is a column's, no weight
        at[:, ::3] = -1
        at[:, 1::7] = vocab + 5
        at[:, 2::11] = 0x7FFFFFFF
        values[:, 4::5] = -INF
        at[0] = -1
        if rows > 1:
            values[1] = -INF
    if kind == "twice":
        at[:, k // 2:] = at[:, :k - k // 2].clone()
        at[0] = int(at[0, 0])
    return values, at


def check_distill(x, columns, dtype, k, temperature, kind="plain", pad=0, skew=0, one=False, weights=True, teacher_dtype=None, seed=0, in_place=False):
    g = gen(seed + k)
    s = Split(x.to(TD[dtype]), columns, dtype, pad, skew, one)
    rows, whole = s.rows, s.whole().clone()
    teacher_dtype = dtype if teacher_dtype is None else teacher_dtype
    values, at = entries(whole, k, kind, g)
    values = values.to(TD[teacher_dtype]).contiguous()
    weight = torch.rand(rows, device=DEV, generator=g) + 0.1
    weight[2::4] = 0
    held = dict(s.where, teacher=values.data_ptr(), indices=at.data_ptr(), k=k, teacher_dtype=teacher_dtype, temperature=temperature,
                weight=weight.data_ptr() if weights else 0)
    blank = torch.full_like(whole, math.nan)
    once, apart = Split(blank, columns, dtype, pad, skew, one), Split(blank, columns, dtype, pad, skew, one)
    loss, alone = torch.full((rows,), 77.0, device=DEV), torch.full((rows,), 77.0, device=DEV)
    stats = torch.full((rows, 2), 77.0, device=DEV)
    hcclx.DistillPlan(s.ptrs, loss=alone.data_ptr(), stats=stats.data_ptr(), **held).launch()
    hcclx.DistillGradPlan(s.ptrs, stats=stats.data_ptr(), dlogits=apart.ptrs, **held).launch()
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(s.whole().float()), torch.nan_to_num(whole.float()))
    if in_place:
        hcclx.DistillPlan(s.ptrs, loss=loss.data_ptr(), dlogits=s.ptrs, **held).launch()
        once = s
    else:
        hcclx.DistillPlan(s.ptrs, loss=loss.data_ptr(), dlogits=once.ptrs, **held).launch()
    torch.cuda.synchronize()
    a, b = once.whole(), apart.whole()
    for r in range(rows):
        w = float(weight[r]) if weights else 1.0
        l = whole[r].double()
        if w != 0 and (bool(l.isnan().any()) or bool((l == INF).any())) and float(loss[r]) != 0:
            assert math.isnan(float(loss[r])) and math.isnan(float(alone[r])) and bool(a[r].isnan().all()) and bool(b[r].isnan().all())
            continue
        want, grad, bound, grad_bound = L.distill(l, values[r].double(), at[r], temperature, w)
        for got in (float(loss[r]), float(alone[r])):
            assert got == want or abs(got - want) <= bound + O.E * abs(want), (r, got, want, bound)
        O.assert_close(a[r], grad, grad_bound, f"row {r}, with the loss")
        O.assert_close(b[r], grad, grad_bound, f"row {r}, from stats")
        if want == 0 and w == 0:
            assert not bool(a[r].any()) and not bool(b[r].any())
    assert once.untouched() and apart.untouched()


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("kind", ["plain", "holes", "twice"])
@pytest.mark.parametrize("vocab,n,k,temperature", [(1, 1, 1, 1.0), (9, 2, 4, 0.5), (70, 1, 70, 1.0), (1000, 3, 33, 2.0), (4099, 8, 64, 1.5), (20001, 2, 1000, 1.0)])
def test_distillation(vocab, n, k, temperature, kind, dtype):
    """Five rows: workgroups of several to a row where it is long."""
    check_distill(contents("steep", 5, vocab, gen(vocab)), shares(vocab, n), dtype, k, temperature, kind, pad=3, skew=1)


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("in_place", [False, True])
def test_distillation_of_few_and_many_rows(rows, dtype, in_place):
    check_distill(contents("steep", rows, 30011, gen(rows)), shares(30011, 4), dtype, 40, 2.0, one=True, weights=rows > 1, in_place=in_place)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("kind", ["holes", "twice"])
@pytest.mark.parametrize("rows,vocab,k", [(5, 3000, 1024), (600, 20001, 300), (513, 700, 64), (40, 24000, 1024)])
def test_distillation_of_short_rows_and_long_lists(rows, vocab, k, kind, dtype):
    """Small workgroups, several entries to a thread; rows that stay in registers."""
    check_distill(contents("steep", rows, vocab, gen(81)), shares(vocab, 2), dtype, k, 1.0, kind, pad=1)


@pytest.mark.parametrize("rows", [4, 270])
@pytest.mark.parametrize("kind", ["normal", "equal", "falling", "masked", "odd", "nothing"])
@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_distillation_of_unusual_logits(kind, dtype, rows):
    check_distill(contents(kind, rows, 9000, gen(5)), shares(9000, 3), dtype, 24, 1.0, "holes", skew=1)


@pytest.mark.parametrize("teacher_dtype", [T.FP32, T.FP16, T.BFP16])
def test_distillation_from_a_teacher_of_another_type(teacher_dtype):
    check_distill(contents("steep", 3, 3001, gen(6)), shares(3001, 2), T.BFP16, 17, 1.0, teacher_dtype=teacher_dtype)


def test_distillation_of_masked_rows_of_nan():
    """Rows of weight 0 are not read, whatever they hold."""
    x = contents("steep", 8, 2000, gen(7))
    x[2::4] = math.nan
    check_distill(x, shares(2000, 2), T.FP16, 10, 1.0)


def test_distillation_of_many_columns_and_a_long_list():
    check_distill(contents("steep", 2, 300007, gen(8)), shares(300007, 64), T.BFP16, 1024, 1.0, weights=False)
    check_distill(contents("steep", 257, 131072, gen(9)), shares(131072, 8), T.BFP16, 64, 2.0)


@pytest.mark.parametrize("rows", [6, 300])
@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_distillation_of_a_teacher_that_is_no_number(dtype, rows):
    """NaN or +infinity among a row's entries make its loss and all its gradients NaN, and no other row's."""
    vocab, k = 6000, 12
    g = gen(51)
    s = Split(contents("steep", rows, vocab, g).to(TD[dtype]), shares(vocab, 2), dtype)
    values, at = entries(s.whole(), k, "plain", g)
    values[1, 3], values[2, 0], values[5, k - 1] = math.nan, INF, math.nan
    at[5, k - 1] = -1                                                # (an entry that names no column does not count)
    for p in s.parts:
        p[2] = -INF                                                  # with a student who rules everything out
    loss, stats = torch.zeros(rows, device=DEV), torch.zeros((rows, 2), device=DEV)
    d, later = [torch.zeros_like(p) for p in s.parts], [torch.zeros_like(p) for p in s.parts]
    held = dict(s.where, strides=None, teacher=values.data_ptr(), indices=at.data_ptr(), k=k, teacher_dtype=T.FP32)
    hcclx.DistillPlan(s.ptrs, loss=loss.data_ptr(), stats=stats.data_ptr(), dlogits=[t.data_ptr() for t in d], **held).launch()
    hcclx.DistillGradPlan(s.ptrs, stats=stats.data_ptr(), dlogits=[t.data_ptr() for t in later], **held).launch()
    torch.cuda.synchronize()
    none = torch.zeros(rows, dtype=torch.bool, device=DEV)
    none[1] = none[2] = True
    assert torch.equal(loss.isnan(), none)
    for t in d + later:
        assert torch.equal(t.isnan(), none[:, None].expand_as(t))


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("rows", [3, 280])
def test_distillation_of_logits_of_any_magnitude(rows, dtype):
    """Logits around 1e30, masks of the type's lowest value, temperatures from end to end."""
    g = gen(52)
    x = contents("normal", rows, 5000, g)
    x[0] *= 1e30
    x[1] = x[1] * 1e-30
    x[2, ::2] = torch.finfo(TD[dtype]).min
    check_distill(x, shares(5000, 2), dtype, 20, 1.0, weights=False)
    check_distill(x, shares(5000, 2), dtype, 20, 1e6, weights=False)
    check_distill(contents("normal", rows, 5000, g) * 1000, shares(5000, 2), dtype, 20, 1e-6, weights=False)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_gradients_from_stats_on_the_logits(rows, dtype):
    """The gradient of the saved sums may lie on the logits as well, by several workgroups to a row."""
    vocab, k = 50021, 100
    g = gen(53)
    s = Split(contents("steep", rows, vocab, g).to(TD[dtype]), shares(vocab, 3), dtype, pad=2, skew=1)
    values, at = entries(s.whole(), k, "twice", g)
    weight = torch.rand(rows, device=DEV, generator=g)
    weight[1::3] = 0
    stats = torch.zeros((rows, 2), device=DEV)
    held = dict(s.where, teacher=values.data_ptr(), indices=at.data_ptr(), k=k, teacher_dtype=T.FP32, weight=weight.data_ptr())
    hcclx.DistillPlan(s.ptrs, stats=stats.data_ptr(), **held).launch()
    apart = Split(torch.zeros_like(s.whole()), shares(vocab, 3), dtype, pad=2, skew=1)
    hcclx.DistillGradPlan(s.ptrs, stats=stats.data_ptr(), dlogits=apart.ptrs, **held).launch()
    hcclx.DistillGradPlan(s.ptrs, stats=stats.data_ptr(), dlogits=s.ptrs, **held).launch()
    torch.cuda.synchronize()
    assert bool(apart.whole().any()) and torch.equal(s.whole(), apart.whole())
    assert s.untouched()


def test_the_most_columns():
    """2^24 of them: rows of 65536 chunks of 32-bit logits."""
    vocab = 1 << 24
    row = contents("steep", 1, vocab, gen(54))
    check_top(row, shares(vocab, 3), T.FP32, 1024)
    check_top(row, shares(vocab, 64), T.BFP16, 40)
    check_distill(row, shares(vocab, 3), T.BFP16, 30, 1.5, weights=False)
    for settings in (dict(), dict(top_k=50), dict(top_p=0.9), dict(T_=0.8, top_p=0.95), dict(top_k=100000), dict(min_p=0.0001)):
        check_draws(row[0], shares(vocab, 3), T.FP32, most=3, **settings)


def test_gradient_against_differences():
    """Central differences of the loss, h = 1/32: their error is h^2 / 6 of the third derivative, of which q's third cumulant, at most
    0.0963, is all (T = 1), and the loss's own error, as the oracle bounds it, over h."""
    vocab, k, h = 40, 6, 1 / 32
    g = gen(10)
    base = torch.randn(vocab, device=DEV, generator=g).mul(64).round() / 64            # (sums with h are exact)
    x = base.repeat(2 * vocab, 1)
    x[torch.arange(vocab), torch.arange(vocab)] += h
    x[vocab + torch.arange(vocab), torch.arange(vocab)] -= h
    x = torch.cat([x, base[None]])
    values = torch.randn(k, device=DEV, generator=g).repeat(len(x), 1)
    at = torch.randperm(vocab, device=DEV, generator=g)[:k].to(torch.int32).repeat(len(x), 1)
    loss, d = torch.empty(len(x), device=DEV), torch.empty_like(x)
    hcclx.DistillPlan([x.data_ptr()], [vocab], len(x), values.data_ptr(), at.data_ptr(), k, T.FP32, loss=loss.data_ptr(), dlogits=[d.data_ptr()]).launch()
    torch.cuda.synchronize()
    _, grad, bound, grad_bound = L.distill(base.double(), values[0].double(), at[0], 1.0, 1.0)
    difference = (loss[:vocab].double() - loss[vocab:2 * vocab].double()) / (2 * h)
    off = h * h / 6 * 0.0963 + 1.5 * (bound + O.E * float(loss.max())) / h
    assert off < 1e-3                                                # (gradients are up to 0.5)
    assert bool(((d[-1].double() - difference).abs() <= off + grad_bound).all())


# ---- sampling ----------------------------------------------------------------------------------------------------------------


def draw(s, settings, u):
    """Tokens and logprobs of a plan; settings: dict of lists (or absent), one number per row."""
    rows = s.rows
    tensors = {k: torch.tensor(v, device=DEV, dtype=torch.int32 if k == "top_k" else torch.float32) for k, v in settings.items()}
    random = torch.tensor(u, device=DEV, dtype=torch.float32)
    tokens, logprob = torch.full((rows,), -77, device=DEV, dtype=torch.int32), torch.full((rows,), 77.0, device=DEV)
    plan = hcclx.SamplePlan(s.ptrs, random=random.data_ptr(), tokens=tokens.data_ptr(), logprob=logprob.data_ptr(),
                            **{k: t.data_ptr() for k, t in tensors.items()}, **s.where)
    plan.launch()
    torch.cuda.synchronize()
    return tokens.tolist(), logprob.tolist()


def check_draws(row, columns, dtype, T_=1.0, top_k=0, top_p=1.0, min_p=0.0, most=24, pad=0, one=False):
    """Draws in the middle of every token's share of [0, 1), and at its ends, give that token and its probability."""
    l = L.plain(row.to(TD[dtype]))
    as32 = lambda v: float(np.float32(v))  # noqa: E731
    T_, top_p, min_p = as32(T_), as32(top_p), as32(min_p)
    u, tokens = L.middles(l, T_, top_k, top_p, min_p, most)
    assert len(u) != 0
    s = Split(row.to(TD[dtype])[None].repeat(len(u), 1), columns, dtype, pad, 1, one)
    got, logprob = draw(s, dict(temperature=[T_] * len(u), top_k=[top_k] * len(u), top_p=[top_p] * len(u), min_p=[min_p] * len(u)), u.tolist())
    assert got == tokens.tolist(), [(i, a, b) for i, (a, b) in enumerate(zip(got, tokens.tolist())) if a != b][:3]
    for x, token, p in zip(u.tolist(), tokens.tolist(), logprob):
        want = L.sample(l, T_, top_k, top_p, min_p, x)
        assert want[0] == token
        assert abs(p - want[1]) <= 1e-9 + 2 * O.E * abs(want[1]), (token, p, want[1])


SETTINGS = [dict(), dict(T_=0.5), dict(T_=3.0), dict(top_k=1), dict(top_k=7), dict(top_k=40, T_=0.7), dict(top_p=0.5), dict(top_p=0.93), dict(min_p=0.05),
            dict(min_p=0.9), dict(top_k=20, top_p=0.8, min_p=0.02, T_=1.3), dict(top_k=900, top_p=0.99), dict(top_p=0.7, min_p=0.01), dict(top_p=0.0),
            dict(min_p=2.0), dict(T_=0.0), dict(T_=-1.0), dict(T_=math.nan), dict(top_p=math.nan, min_p=math.nan), dict(top_k=-3), dict(T_=1e-30), dict(T_=INF)]


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("vocab,n,kind", [(1, 1, "normal"), (5, 2, "normal"), (1000, 3, "steep"), (777, 8, "coarse"), (2049, 1, "masked"), (3000, 4, "odd"), (20000, 2, "steep")])
def test_sampling(vocab, n, kind, dtype):
    row = contents(kind, 1, vocab, gen(vocab))[0]
    for settings in SETTINGS:
        check_draws(row, shares(vocab, n), dtype, pad=3, **settings)


WIDE = [dict(T_=5.0), dict(top_k=5000), dict(top_k=30000, T_=5.0, top_p=0.9), dict(top_p=0.95, T_=5.0), dict(top_k=1500, min_p=0.3, T_=5.0), dict(min_p=0.001, T_=4.0),
        dict(top_k=1025, top_p=0.2, T_=5.0), dict(top_p=0.6, T_=INF), dict(top_k=2000, T_=INF), dict(top_k=49999), dict(top_k=3000, top_p=0.0), dict(top_k=3000, min_p=3.0)]


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
@pytest.mark.parametrize("kind", ["normal", "equal", "coarse", "falling", "steep"])
def test_sampling_from_more_than_a_list_holds(kind, dtype):
    row = contents(kind, 1, 50000, gen(11))[0]
    for settings in WIDE:
        check_draws(row, [10000, 25001, 14999], dtype, most=12, **settings)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_sampling_from_many_columns(dtype):
    row = contents("steep", 1, 600001, gen(12))[0]
    for settings in (dict(), dict(top_k=50), dict(top_p=0.9), dict(T_=2.0, top_p=0.97), dict(top_k=100000)):
        check_draws(row, shares(600001, 5), dtype, most=6, **settings)


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
def test_ends_of_the_random_numbers_and_unusual_rows(dtype):
    vocab = 300
    x = contents("normal", 12, vocab, gen(13))
    x[8] = -INF                                                      # nothing to draw
    x[9] = math.nan
    x[10] = -INF
    x[10, 123] = -7.0                                                # one token
    x[11, [5, 50, 250]] = INF
    s = Split(x.to(TD[dtype]), shares(vocab, 3), dtype)
    for settings in (dict(), dict(top_k=[9] * 12), dict(top_p=[0.5] * 12), dict(temperature=[2.0] * 12, min_p=[0.1] * 12)):
        for u in (0.0, -1.0, math.nan, 1.0, 7.0, 0.5):
            got, logprob = draw(s, settings, [u] * 12)
            for r in range(12):
                l = L.plain(s.whole()[r])
                want = L.sample(l, settings.get("temperature", [1.0])[0], settings.get("top_k", [0])[0], settings.get("top_p", [1.0])[0],
                                float(np.float32(settings.get("min_p", [0.0])[0])), u)
                assert got[r] == want[0], (r, u, settings, got[r], want)
                assert logprob[r] == want[1] or abs(logprob[r] - want[1]) <= 1e-9 + 2 * O.E * abs(want[1])


def test_rows_of_one_launch_have_settings_of_their_own():
    """All settings in all combinations, a row each, with the same logits."""
    vocab, g = 40000, gen(14)
    one = contents("steep", 1, vocab, g)[0].bfloat16()
    table = [(t, k, p, m) for t in (0.0, 0.7, 1.0, 4.0) for k in (0, 1, 30, 5000) for p in (1.0, 0.9, 0.3) for m in (0.0, 0.05)]
    s = Split(one.repeat(len(table), 1), shares(vocab, 8), T.BFP16)
    l = L.plain(one)
    u = [float(np.float32(x)) for x in np.random.default_rng(3).random(len(table))]
    names = ("temperature", "top_k", "top_p", "min_p")
    got, _ = draw(s, {name: [row[i] for row in table] for i, name in enumerate(names)}, u)
    want = [L.sample(l, float(np.float32(t)), k, float(np.float32(p)), float(np.float32(m)), x)[0] for (t, k, p, m), x in zip(table, u)]
    assert got == want


# ---- launches ----------------------------------------------------------------------------------------------------------------


def plans(rows=6, vocab=20011, n=3, k=16, dtype=T.BFP16, seed=20):
    """All plans over the same logits, and what they write."""
    g = gen(seed)
    s = Split(contents("steep", rows, vocab, g).to(TD[dtype]), shares(vocab, n), dtype)
    out = dict(values=torch.zeros((rows, k), device=DEV, dtype=TD[dtype]), indices=torch.zeros((rows, k), device=DEV, dtype=torch.int32),
               lse=torch.zeros(rows, device=DEV), loss=torch.zeros(rows, device=DEV), stats=torch.zeros((rows, 2), device=DEV),
               tokens=torch.zeros(rows, device=DEV, dtype=torch.int32), logprob=torch.zeros(rows, device=DEV),
               dlogits=[torch.zeros_like(p) for p in s.parts], later=[torch.zeros_like(p) for p in s.parts])
    random, top_p = torch.rand(rows, device=DEV, generator=g), torch.full((rows,), 0.95, device=DEV)
    p = {k: v.data_ptr() for k, v in out.items() if not isinstance(v, list)}
    teacher = dict(teacher=p["values"], indices=p["indices"], k=k, temperature=2.0)
    made = [hcclx.TopLogitsPlan(s.ptrs, k=k, values=p["values"], indices=p["indices"], lse=p["lse"], **s.where),
            hcclx.DistillPlan(s.ptrs, loss=p["loss"], stats=p["stats"], dlogits=[t.data_ptr() for t in out["dlogits"]], **teacher, **dict(s.where, strides=None)),
            hcclx.DistillGradPlan(s.ptrs, stats=p["stats"], dlogits=[t.data_ptr() for t in out["later"]], **teacher, **dict(s.where, strides=None)),
            hcclx.SamplePlan(s.ptrs, random=random.data_ptr(), tokens=p["tokens"], logprob=p["logprob"], top_p=top_p.data_ptr(), **s.where)]
    return s, out, made, (random, top_p)


def copied(out):
    return {k: [t.clone() for t in v] if isinstance(v, list) else v.clone() for k, v in out.items()}


def same(a, b):
    return all(torch.equal(x, y) for k in a for x, y in zip(*((v[k] if isinstance(v[k], list) else [v[k]]) for v in (a, b))))


@pytest.mark.parametrize("rows", [2, 300])
def test_a_captured_step_replays_with_other_logits(rows):
    s, out, made, (random, _) = plans(rows)
    stream = torch.cuda.Stream()
    g = gen(21)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for plan in made:
            plan.launch(torch.cuda.current_stream().cuda_stream)
    for turn in range(4):
        for p in s.parts:
            p.copy_(torch.randn(p.shape, device=DEV, generator=g) * 4)
        random.copy_(torch.rand(rows, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = copied(out)
        for v in out.values():
            for t in v if isinstance(v, list) else [v]:
                t.zero_()
        for plan in made:
            plan.launch(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert same(got, out), turn


def test_plans_on_two_streams_at_once():
    """Plans of their own do not share memory."""
    one, two = plans(rows=40, seed=22), plans(rows=50, seed=23)
    want = []
    for _, out, made, _ in (one, two):
        for plan in made:
            plan.launch()
        torch.cuda.synchronize()
        want.append(copied(out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (_, _, made, _), stream in zip((one, two), streams):
            for plan in made:
                plan.launch(stream.cuda_stream)
    torch.cuda.synchronize()
    assert same(one[1], want[0]) and same(two[1], want[1])


def test_a_teacher_a_student_and_an_answer():
    """All of them one behind the other, as a step that distils and then answers uses them: a teacher's list of 32-bit logits, the loss and the
    gradients of a student whose columns are shared differently, logits that follow the gradients, their list and a draw."""
    rows, vocab, k, temperature, g = 40, 12001, 48, 2.0, gen(71)
    teacher = Split(contents("steep", rows, vocab, g), shares(vocab, 2), T.FP32, pad=1)
    student = Split((teacher.whole() * 0.5 + torch.randn((rows, vocab), device=DEV, generator=g)).bfloat16(), shares(vocab, 8), T.BFP16)
    values, indices = torch.empty((rows, k), device=DEV), torch.empty((rows, k), device=DEV, dtype=torch.int32)
    weight = torch.rand(rows, device=DEV, generator=g)
    weight[::10] = 0
    loss, d = torch.empty(rows, device=DEV), [torch.zeros_like(p) for p in student.parts]
    best, numbers = torch.empty((rows, 5), device=DEV, dtype=torch.bfloat16), torch.empty((rows, 5), device=DEV, dtype=torch.int32)
    random, top_p = torch.rand(rows, device=DEV, generator=g), torch.full((rows,), 0.9, device=DEV)
    tokens, lse = torch.empty(rows, device=DEV, dtype=torch.int32), torch.empty(rows, device=DEV)
    before = student.whole().clone()
    where = dict(student.where, strides=None)
    plans = [hcclx.TopLogitsPlan(teacher.ptrs, k=k, values=values.data_ptr(), indices=indices.data_ptr(), **teacher.where),
             hcclx.DistillPlan(student.ptrs, teacher=values.data_ptr(), indices=indices.data_ptr(), k=k, teacher_dtype=T.FP32, temperature=temperature,
                               weight=weight.data_ptr(), loss=loss.data_ptr(), dlogits=[t.data_ptr() for t in d], **where),
             hcclx.TopLogitsPlan(student.ptrs, k=5, values=best.data_ptr(), indices=numbers.data_ptr(), lse=lse.data_ptr(), **where),
             hcclx.SamplePlan(student.ptrs, random=random.data_ptr(), tokens=tokens.data_ptr(), top_p=top_p.data_ptr(), **where)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for i, plan in enumerate(plans):
            plan.launch(stream.cuda_stream)
            if i == 1:
                for p, t in zip(student.parts, d):
                    p.sub_(t, alpha=10.0)
    stream.synchronize()
    gradient, after = torch.cat(d, 1), student.whole()
    for r in range(rows):
        l = L.plain(teacher.whole()[r])
        assert torch.equal(indices[r].long(), L.order(l)[:k])
        want, grad, bound, grad_bound = L.distill(before[r].double(), values[r].double(), indices[r], temperature, float(weight[r]))
        assert abs(float(loss[r]) - want) <= bound + O.E * abs(want)
        O.assert_close(gradient[r], grad, grad_bound, f"row {r}")
        l = L.plain(after[r])
        first = L.order(l)[:5]
        assert torch.equal(numbers[r].long(), first) and torch.equal(best[r].double(), l[first])
        want, bound = L.lse(l)
        assert abs(float(lse[r]) - want) <= bound + O.E * abs(want)
        assert int(tokens[r]) == L.sample(l, 1.0, 0, float(np.float32(0.9)), 0.0, float(random[r]))[0]


def test_no_rows():
    s = Split(torch.zeros((0, 100), device=DEV, dtype=torch.bfloat16), [60, 40], T.BFP16)
    hcclx.TopLogitsPlan([1 << 40] * 2, k=3, values=0, indices=0, **dict(s.where, strides=None)).launch()
    hcclx.DistillPlan([1 << 40] * 2, teacher=0, indices=0, k=3, **dict(s.where, strides=None)).launch()
    hcclx.DistillGradPlan([1 << 40] * 2, teacher=0, indices=0, k=3, stats=0, dlogits=[1 << 41] * 2, **dict(s.where, strides=None)).launch()
    hcclx.SamplePlan([1 << 40] * 2, random=0, tokens=0, **dict(s.where, strides=None)).launch()
    torch.cuda.synchronize()


def test_rows_behind_4_gib():
    """Offsets that pass 32 bits: the last rows of a matrix of 4.6 GB."""
    rows, vocab = 17600, 131072
    whole = torch.zeros((rows, vocab), device=DEV, dtype=torch.bfloat16)
    whole[:, 1000] = 1.0
    whole[-1, 130000] = 9.0
    where = dict(columns=[vocab], rows=rows, dtype=T.BFP16)
    values, indices = torch.empty((rows, 2), device=DEV, dtype=torch.bfloat16), torch.empty((rows, 2), device=DEV, dtype=torch.int32)
    hcclx.TopLogitsPlan([whole.data_ptr()], k=2, values=values.data_ptr(), indices=indices.data_ptr(), **where).launch()
    loss = torch.empty(rows, device=DEV)
    hcclx.DistillPlan([whole.data_ptr()], teacher=values.data_ptr(), indices=indices.data_ptr(), k=2, loss=loss.data_ptr(), dlogits=[whole.data_ptr()],
                      **where).launch()
    torch.cuda.synchronize()
    assert indices[-1].tolist() == [130000, 1000] and indices[-2].tolist() == [1000, 0] and values[-1].tolist() == [9.0, 1.0]
    last = torch.zeros(vocab, dtype=torch.float64, device=DEV)
    last[1000], last[130000] = 1.0, 9.0
    want, grad, bound, grad_bound = L.distill(last, values[-1].double(), indices[-1], 1.0, 1.0)
    assert abs(float(loss[-1]) - want) <= bound + O.E * abs(want)
    O.assert_close(whole[-1], grad, grad_bound)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_sampling_of_many_infinities(dtype):
    row = contents("normal", 1, 30000, gen(55))[0]
    row[7::97] = INF
    row[11::13] = math.nan
    for settings in (dict(), dict(top_p=0.9), dict(top_p=0.5, T_=0.3), dict(min_p=0.2), dict(top_k=200), dict(top_k=5000, top_p=0.8), dict(top_k=5000), dict(T_=0.0)):
        check_draws(row, shares(30000, 4), dtype, most=12, **settings)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_sampling_from_ranks_of_few_columns(dtype):
    for each in (3, 40):
        row = contents("normal", 1, 64 * each, gen(each))[0]
        for settings in (dict(top_k=100), dict(top_p=0.95), dict(top_p=0.5), dict(T_=3.0, min_p=0.01), dict(T_=9.0, top_k=700, top_p=0.9)):
            check_draws(row, [each] * 64, dtype, most=12, **settings)


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16, T.BFP16])
def test_sampling_where_two_filters_cut_nearly_the_same(dtype):
    """min_p between, at and next to the values around which top_p or top_k cut."""
    row = contents("steep", 1, 30000, gen(31))[0].to(TD[dtype]).float()
    l = row.double()
    order = L.order(l)
    w = torch.exp((l - l.max()) / 4.0)[order]
    c = w.cumsum(0) / w.sum()
    for place in (700, 5000, 20000):
        for min_p in (float(w[place]), float(w[place]) * 1.0000005, float(w[place]) * 0.9999995, float(w[place + 3]), float(w[place - 2]), float(w[place + 400])):
            check_draws(row, shares(30000, 3), dtype, T_=4.0, min_p=min_p, top_p=float(c[place]) + 1e-6, most=8)
            check_draws(row, shares(30000, 3), dtype, T_=4.0, min_p=min_p, top_k=place + 400, most=8)


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_sampling_from_improbable_tokens_and_dense_ones(dtype):
    """A top_k that reaches tokens of 2^-40 of the first's weight and less; a cut among thousands of tokens of nearly the same weight."""
    steep = contents("steep", 1, 40000, gen(41))[0] * 2
    for settings in (dict(top_k=3000), dict(top_k=39999, T_=0.4), dict(top_k=20000, T_=0.15), dict(top_p=0.9999999, T_=0.5), dict(min_p=1e-12)):
        check_draws(steep, shares(40000, 3), dtype, most=8, **settings)
    flat = contents("normal", 1, 300000, gen(42))[0] * 0.25
    for settings in (dict(top_k=150000), dict(top_p=0.5), dict(top_p=0.5, min_p=0.4), dict(top_k=150000, top_p=0.7)):
        check_draws(flat, shares(300000, 2), dtype, most=8, **settings)


@pytest.mark.parametrize("rows,vocab", [(1, 20011), (150, 20011), (1100, 20011), (4200, 1501)])
def test_many_rows_of_wide_draws(rows, vocab):
    """Rows whose list is too short among others, more and fewer workgroups to a row."""
    g = gen(rows)
    x = contents("steep", rows, vocab, g)
    s = Split(x.bfloat16(), shares(vocab, 3), T.BFP16)
    pick = lambda *v: [v[i % len(v)] for i in range(rows)]  # noqa: E731
    settings = dict(temperature=pick(3.0, 1.0, 2.5, 3.0, 4.0), top_p=pick(0.95, 0.9, 1.0, 0.6, 1.0), top_k=pick(0, 0, 5000, 0, 0), min_p=pick(0.0, 0.0, 0.0, 0.001, 0.002))
    u = torch.rand(rows, device=DEV, generator=g).tolist()
    got, logprob = draw(s, settings, u)
    whole = s.whole()
    as32 = lambda v: float(np.float32(v))  # noqa: E731
    for r in [*range(0, rows, 1 if rows < 200 else 7 if rows < 2000 else 61), *range(max(0, rows - 20), rows)]:
        l = L.plain(whole[r])
        want = L.sample(l, settings["temperature"][r], settings["top_k"][r], as32(settings["top_p"][r]), as32(settings["min_p"][r]), u[r])
        assert got[r] == want[0], (r, got[r], want)
        assert abs(logprob[r] - want[1]) <= 1e-9 + 2 * O.E * abs(want[1])


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
def test_top_p_among_groups_that_are_as_large(dtype):
    """More groups of 64 columns reach the same value than are looked at, and most groups hold it more than once: what is listed of
    some groups is not the beginning of the order."""
    vocab = 64 * 700
    row = torch.full((vocab,), -1.0, device=DEV)
    row[::64] = 2.0
    row[5::192] = 2.0
    row[torch.arange(9, vocab, 640)] = 3.0
    for settings in (dict(top_p=0.3), dict(top_p=0.55), dict(top_p=0.6), dict(min_p=0.3), dict(top_k=300), dict(top_k=900)):
        check_draws(row, shares(vocab, 2), dtype, most=40, **settings)
