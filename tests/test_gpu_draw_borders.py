"""Draws whose random number, or whose top_p, lies at or next to a border between two tokens: which side it is on follows from the whole
numbers that the weights are (include/hcclx_ops.h: hcclx_sample_t), and from nothing else."""
import numpy as np
import pytest
import torch

import logits_oracle as L
from hccl_amd import hcclx
from hccl_amd import types as T
from test_gpu_output_layer import DEV, TD, Split, draw, gen, shares

pytestmark = pytest.mark.gpu


def mirrored(half):
    """Rows whose second half repeats the first: half of what stays is reached with the last token of the first half, exactly."""
    return torch.cat([half, half], 1)


def first_of_second_half(row, T_, top_k, min_p):
    """The token at half of the weight of a mirrored row: running sums up to there are not more than half."""
    first, w = L.kept(L.plain(row), T_, top_k, 1.0, min_p)
    at = first[(first >= row.numel() // 2) & (w[first] > 0)]
    assert 2 * at.numel() == int((w[first] > 0).sum())
    return int(at.min())


@pytest.mark.parametrize("dtype,top_k,min_p,spread", [(T.FP32, k, p, d) for k, p, d in (
    (0, 1e-6, 4.0), (2, 0.0, 4.0), (900, 0.0, 4.0), (1500, 0.0, 4.0), (20000, 1e-6, 4.0), (118000, 0.0, 4.0), (5000, 0.0, 0.001))]
    + [(T.BFP16, 0, 1e-6, 4.0), (T.FP16, 0, 1e-6, 4.0)])             # (16 bits: equal values, of which a top_k takes no mirror image)
def test_half_of_a_mirrored_row(dtype, top_k, min_p, spread):
    """random times a whole of more than 53 bits: no bit of the product is lost."""
    rows, vocab = 24, 120000
    half = -torch.arange(vocab // 2, device=DEV) * (spread / (vocab // 2))
    half = torch.stack([half[torch.randperm(vocab // 2, device=DEV, generator=gen(r))] for r in range(rows)])
    s = Split(mirrored(half).to(TD[dtype]), shares(vocab, 3), dtype, skew=1)
    temperature = [float(np.float32(0.5 + 0.1 * r)) for r in range(rows)]
    got, _ = draw(s, dict(temperature=temperature, top_k=[top_k] * rows, min_p=[min_p] * rows), [0.5] * rows)
    want = [first_of_second_half(s.whole()[r], temperature[r], top_k, float(np.float32(min_p))) for r in range(rows)]
    assert got == want, [(r, a, b) for r, (a, b) in enumerate(zip(got, want)) if a != b]


@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("vocab,n", [(131072, 1), (120001, 5), (600000, 2)])
def test_half_of_a_mirrored_row_without_a_filter(vocab, n, dtype):
    """The same rows in plans of few and many rows, whose first launch sums up longer and shorter runs, with settings that filter nothing
    and without any: the same tokens, those of the whole numbers."""
    vocab -= vocab % 2
    half = torch.empty((20, vocab // 2), device=DEV).exponential_(1.0, generator=gen(vocab)) * 1.6 - 4
    rows = mirrored(half).to(TD[dtype])
    for times in (1, 4, 8, 16):
        s = Split(rows.repeat(times, 1), shares(vocab, n), dtype)
        for settings in (dict(), dict(top_k=[0] * s.rows, top_p=[1.0] * s.rows)):
            got, _ = draw(s, settings, [0.5] * s.rows)
            assert got == [vocab // 2] * s.rows, (times, [(r, a) for r, a in enumerate(got) if a != vocab // 2])


@pytest.mark.parametrize("vocab", [65536, 1 << 19])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=1.0), dict(min_p=0.5), dict(T_=0.25, min_p=1.0)])
def test_equal_logits_at_every_border(vocab, settings):
    """Token j takes [j / vocab, (j + 1) / vocab)."""
    places = torch.randint(0, vocab, (60,), device=DEV, generator=gen(3)).tolist() + [0, 1, vocab // 2, vocab - 1]
    rows = 2 * len(places)
    s = Split(torch.full((rows, vocab), 3.5, device=DEV, dtype=torch.bfloat16), shares(vocab, 3), T.BFP16)
    below = np.nextafter(np.array([(j + 1) / vocab for j in places], dtype=np.float32), np.float32(0))
    u = [j / vocab for j in places] + below.tolist()
    got, logprob = draw(s, {("temperature" if k == "T_" else k): [v] * rows for k, v in settings.items()}, u)
    assert got == places * 2
    assert np.allclose(logprob, -np.log(vocab), rtol=1e-7, atol=0)


@pytest.mark.parametrize("vocab,bits", [(131072, 45), (600000, 42)])
@pytest.mark.parametrize("settings", [dict(), dict(top_p=1.0, top_k=0), dict(min_p=1e-30)])
def test_what_is_less_than_half_of_a_part_is_never_drawn(vocab, bits, settings):
    """Weights are whole numbers of 2^-51 of the largest without a filter, otherwise of 2^-45 for 131072 columns and 2^-42 for 600000: a little
    less than half of that is nothing, a little more is one."""
    if "min_p" not in settings:
        bits = 51
    x = torch.zeros((8, vocab), device=DEV)
    for r, (place, more) in enumerate([(vocab - 1, -0.01), (vocab - 1, 0.01), (0, -0.01), (0, 0.01)] * 2):
        x[r] = float((-(bits + 1) + more) * np.log(2))
        x[r, place] = 0.0
    s = Split(x, shares(vocab, 2), T.FP32)
    got, _ = draw(s, {k: [v] * 8 for k, v in settings.items()}, [0.0] * 4 + [1.0] * 4)
    assert got == [vocab - 1, 0, 0, 0, vocab - 1, vocab - 1, 0, vocab - 1]


@pytest.mark.parametrize("dtype", [T.FP32, T.FP16])
def test_ends_of_rows_without_a_filter(dtype):
    """0 draws the first column that has any weight, 1 and more the last."""
    x = torch.randn((6, 40000), device=DEV, generator=gen(9))
    x[:, 0] = x[:, -1] = -float("inf")
    x[1, :30000] = float("nan")
    x[2, 20000:] = -float("inf")
    x[3] = -float("inf")
    x[3, 777] = -3.0
    x[4, [300, 500]] = float("inf")
    s = Split(x.to(TD[dtype]), shares(40000, 3), dtype, pad=1)
    for settings in (dict(), dict(min_p=[0.0] * 6)):
        for T_ in (1.0, 2.5, float("inf")):
            first, _ = draw(s, dict(settings, temperature=[T_] * 6), [0.0] * 6)
            last, _ = draw(s, dict(settings, temperature=[T_] * 6), [1.0] * 3 + [2.0] * 3)
            assert first == [1, 30000, 1, 777, 300, 1] and last == [39998, 39998, 19999, 777, 500, 39998]


@pytest.mark.parametrize("seed,top_p,stay", [(3483, 0.5376677513122559, None), (2737, 0.6722675561904907, 75747), (952, 0.9737805724143982, 125109),
                                             (1731, 0.826088011264801, 98931), (5860, 0.6229817867279053, 68836)])
def test_top_p_next_to_where_a_token_ends(seed, top_p, stay):
    """Descending rows of which the first `stay` tokens reach top_p of the whole by 2^-35 of it, or the one less fails it by that (which of the two,
    the first row does not say: it is nearer than that).  random 1 draws the last that stays.  The same in plans of few and many rows."""
    vocab = 131072
    row = np.sort(np.random.default_rng(seed).standard_normal(vocab).astype(np.float32) * np.float32(0.25))[::-1].copy()
    seen = set()
    for rows in (1, 64, 128, 300):
        s = Split(torch.from_numpy(row).to(DEV)[None].expand(rows, -1), [vocab], T.FP32)
        for settings in (dict(), dict(min_p=[1e-9] * rows)):
            seen |= set(draw(s, dict(settings, top_p=[top_p] * rows), [1.0] * rows)[0])
    assert len(seen) == 1 and (stay is None or seen == {stay - 1}), seen


@pytest.mark.parametrize("later", [3, 4, 5])
def test_top_p_where_min_p_cuts_behind_it(later):
    """A largest token, 2^20 tokens that are less probable than min_p, and 2^21 equal ones, all over min_p, of which top_p cuts off the last `later`.
    That is less of their weight than whole numbers of 2^-40 round them up by (w is two fifths below such a number)."""
    many, few, bits = 1 << 21, 1 << 20, 40
    d = next(x for x in np.arange(1538, 1542, 1 / 512) if 0.55 < np.exp(-float(np.float32(x / 92.332))) * 2.0 ** bits % 1 < 0.65)
    d, d2 = float(np.float32(d / 92.332)), float(np.float32(1556 / 92.332))
    w, w2 = np.exp(-d), np.exp(-d2)
    number = int(np.rint(w * 2.0 ** bits))
    whole = (1 << 51) + many * int(np.rint(w * 2.0 ** 51)) + few * int(np.rint(w2 * 2.0 ** 51))
    # a top_p in the middle of the last token that it leaves, over 2^-26 of itself from that one's ends: half a step of a float
    stay = many - later
    for extra in range(200):                                         # (some more of the improbable ones, until a float lies there)
        total = whole + extra * int(np.rint(w2 * 2.0 ** 51))
        top_p = float(np.float32(((1 << bits) + (stay - 0.5) * number) * 2.0 ** (51 - bits) / total))
        asked = -(-int(top_p * 2 ** 30) * total // 2 ** (30 + 51 - bits))
        if (1 << bits) + (stay - 1) * number + 1000 < asked < (1 << bits) + stay * number - 1000:
            break
    assert int(top_p * 2 ** 30) == top_p * 2 ** 30 and -(-(asked - (1 << bits)) // number) == stay
    vocab = 1 + few + extra + many
    row = torch.full((1, vocab), -d2, device=DEV)
    row[0, 0] = 0.0
    row[0, 1 + few + extra:] = -d
    s = Split(row, shares(vocab, 2), T.FP32)
    got, _ = draw(s, dict(top_p=[top_p], min_p=[2.0 ** (-1546 / 64)]), [1.0])
    assert got == [vocab - 1 - later]


@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("filtered", [False, True])
def test_borders_in_a_graph_that_is_replayed(rows, filtered):
    """Rows over 64 ranks that are weighed again, between others, from a graph with other random numbers at every replay."""
    vocab = 64 * 300
    half = torch.randn((rows, vocab // 2), device=DEV, generator=gen(rows)) * 2
    whole = mirrored(half).half()
    s = Split(whole, [300] * 64, T.FP16, pad=1)
    random, tokens = torch.zeros(rows, device=DEV), torch.zeros(rows, device=DEV, dtype=torch.int32)
    neutral = torch.ones(rows, device=DEV)
    plan = hcclx.SamplePlan(s.ptrs, random=random.data_ptr(), tokens=tokens.data_ptr(), top_p=neutral.data_ptr() if filtered else 0, **s.where)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        plan.launch(torch.cuda.current_stream().cuda_stream)
    l = L.plain(s.whole()[0])
    u, middles = L.middles(l, 1.0, 0, 1.0, 0.0, 5)
    for x, token in [(0.5, vocab // 2), *zip(u.tolist(), middles.tolist()), (1.0, vocab - 1), (0.0, 0), (0.5, vocab // 2)]:
        random.fill_(0.5)
        random[0] = x
        tokens.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        got = tokens.clone()
        plan.launch()
        torch.cuda.synchronize()
        assert got.tolist() == [token] + [vocab // 2] * (rows - 1) and torch.equal(got, tokens), x
