"""Draws whose random number, or whose top_p, lies at or next to a border between two tokens: which side it is on follows from the whole
numbers that the weights are (include/hcclx_ops.h: hcclx_sample_t), and from nothing else."""
import numpy as np
import pytest
import torch

import logits_oracle as L
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
