"""The operators of the output layer (include/hcclx_ops.h: hcclx_logits_t and what takes it) from their definitions, in 64 bits, a
row at a time, with bounds on what 32-bit sums and one rounding may differ by."""
import math

import numpy as np
import torch

from ops_oracle import E

MOST = 1024


def plain(l):
    """A row in 64 bits, NaN as -infinity."""
    l = l.double()
    return torch.where(l.isnan(), torch.full_like(l, -math.inf), l)


def order(l):
    """Columns of a row (64 bits, no NaN), descending, of equal values the first."""
    return torch.sort(l, descending=True, stable=True).indices


def lse(l):
    """log sum exp of a row, and its bound.  Terms: exp2's 2^-22 together with its argument's rounding, |l - most| log2(e) 2^-23 (the
    difference and the product, in powers of two), which for a term of size exp(-d) is d 2^-22 exp(-d), 2^-22 at most against the
    sum, which is 1 at least: n of them share less than sum d exp(-d) / sum exp(-d), the mean of d.  The sum: a chain of at most 64
    elements per lane, six steps in a wavefront."""
    m = float(l.max())
    if m == -math.inf or m == math.inf:
        return m, 0.0
    w = torch.exp(l - m)
    total = float(w.sum())
    mean = float((torch.where(w > 0, w * (m - l), torch.zeros_like(w))).sum()) / total
    return m + math.log(total), (mean + 1) * 2.0 ** -21 + 72 * E


def distill(l, teacher, at, T, weight):
    """loss, gradient of a row and their bounds.  l, teacher: 64 bits; at: columns.  None for a row that holds NaN.

    q: the terms' arguments in powers of two, a = (l - m) log2(e) / T, are off by 2^-23 (|a| + 2) (one operation, with c = log2(e) / T
    itself in two floats), exp2 by 2^-22 of itself; the sum is a chain of at most 72 steps beyond what a thread adds up in blocks of
    32 elements (n / (32 * 512) of them) and six rescalings.  So q is off by a relative D = 2^-22 (|a| + mean |a| + 8) + (120 + n / 16384) E,
    and log q by as much; the loss sums that with weights p, which are good to 2^-48."""
    n = l.numel()
    d = torch.zeros_like(l)
    ok = (at >= 0) & (at < n)
    at, t = at[ok].long(), teacher[ok]
    if weight == 0 or t.numel() == 0 or float(t.max()) == -math.inf:
        return 0.0, d, 0.0, d
    p = torch.softmax(t / T, 0)
    m = float(l.max())
    if m == -math.inf:
        q, logq = torch.zeros_like(l), torch.full_like(l, -math.inf)
        rel = torch.zeros_like(l)
    else:
        x = (l - m) / T
        logq = x - torch.logsumexp(x, 0)
        q = torch.exp(logq)
        a = torch.where(torch.isinf(x), torch.zeros_like(x), x.abs() * 1.4427)
        rel = 2.0 ** -22 * (a + float((q * a).sum()) + 8) + (120 + n / 16384) * E
    used = p > 0
    logp = torch.log_softmax(t / T, 0)
    terms = p[used] * (logp[used] - logq[at[used]])
    loss = weight * T * T * float(terms.sum())
    bound = abs(weight) * T * T * (float((p[used] * rel[at[used]]).sum()) + 1e-12 * float(terms[torch.isfinite(terms)].abs().sum()))
    g = q.clone().index_add_(0, at, -p)
    return loss, weight * T * g, bound, abs(weight) * T * (q * rel + 4 * E * (q + g.abs()))


def kept(l, T, top_k, top_p, min_p):
    """The columns that stay of a row (64 bits, no NaN), as the header says, and w of all."""
    n = l.numel()
    m = float(l.max())
    first = order(l)
    if not T > 0:
        return first[:1], torch.where(l == m, 1.0, 0.0)
    x = torch.where(l == m, torch.zeros_like(l), l - m)
    w = torch.where(l == -math.inf, torch.zeros_like(l), torch.exp(x / T)) if m != math.inf else torch.where(l == m, 1.0, 0.0).double()
    if 0 < top_k < n:
        first = first[:top_k]
    ws = w[first]
    if top_p < 1:
        before = torch.cat([torch.zeros(1, dtype=torch.float64, device=l.device), ws.cumsum(0)])[:-1]
        take = before < top_p * float(ws.sum())
        take[0] = True
        first = first[:int(take.sum())]
        ws = w[first]
    if min_p > 0:
        take = ws >= min(min_p, 1.0)
        first = first[:max(1, int(take.sum()))]
    return first, w


def sample(l, T, top_k, top_p, min_p, u):
    """The token and its logarithm's probability."""
    if float(l.max()) == -math.inf:
        return -1, -math.inf
    first, w = kept(l, T, top_k, top_p, min_p)
    places = first.sort().values
    c = w[places].cumsum(0)
    total = float(c[-1])
    u = 0.0 if math.isnan(u) else u
    k = int(torch.searchsorted(c, torch.tensor(u * total, dtype=torch.float64, device=l.device), right=True))
    alive = (w[places] > 0).nonzero().flatten()
    k = min(max(k, int(alive[0])), int(alive[-1]))
    return int(places[k]), math.log(float(w[places[k]]) / total)


def middles(l, T, top_k, top_p, min_p, most=None):
    """Random numbers in the middle of what every token that stays takes of [0, 1), and those tokens; wide enough ones alone (the
    numbers are floats)."""
    first, w = kept(l, T, top_k, top_p, min_p)
    places = first.sort().values
    c = w[places].cumsum(0).cpu().numpy()
    low = np.concatenate([[0.0], c[:-1]]) / c[-1]
    high = c / c[-1]
    wide = high - low > 2.0 ** -20
    u, tokens = ((low + high) / 2)[wide], places.cpu().numpy()[wide]
    if most is not None and len(u) > most:
        pick = np.linspace(0, len(u) - 1, most).astype(int)
        u, tokens = u[pick], tokens[pick]
    return u.astype(np.float32), tokens
