"""The operators of the output layer, whose vocabulary is split over the ranks: what a teacher or a server lists of a row of
logits, the loss of a student that learns from such a list, and the draw of the next token.

listed() names the cases, draw() makes more of the same kinds; prepare() builds what a program holds before the call, run()
is one pass through an operator and returns its outputs whole.  With own = False run() computes them from elementary torch
operations, with own = True through hccl_amd.hcclx.  exact() gives them from the definitions in 64 bits.

Rank j of n holds columns[j] columns of each of the rows (as many as the others, the last ones fewer where they do not go into
the vocabulary evenly), `pad` elements behind every row belong to nobody.  l: a row over all ranks.

top: the k largest of l in descending order, of equal ones the first, their numbers, and log sum exp(l).

distill: a teacher lists k logits t and their numbers i.  p = softmax(t / T), q = softmax(l / T) over the whole vocabulary;
loss = w T^2 sum over k of p (log p - log q[i]);  its gradient is w T (q - p at i).  w: the weight of the row, 0 for rows that
are masked.  "train": loss and gradient; "apart": the loss first, the gradient in a second call; "loss": no gradient.

sample: of the order of top, the first top_k; of those the shortest beginning that holds top_p of their probability; of those
the ones that are min_p times as probable as the first.  With c the running sum of what is left of exp((l - max l) / T), in
order of the tokens' numbers: the first token whose c is over u times the whole, u from a random generator.  T = 0: the first of
the largest.  And the logarithm of the probability with which the token was drawn."""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda:0"

# what a drawn case costs at most (the largest listed one costs more)
DRAW_BYTES = 9e8


def listed():
    return [
        # a teacher lists its logits for a batch of training sequences
        {"name": "top_teacher", "op": "top", "ranks": 8, "rows": 4096, "vocab": 131072, "k": 64, "dtype": "bf16", "pad": 0},
        # alternatives with their probabilities for four answers that are being written, 32-bit logits
        {"name": "top_alternatives", "op": "top", "ranks": 8, "rows": 4, "vocab": 131072, "k": 20, "dtype": "fp32", "pad": 0},
        # long lists of few columns, odd sizes
        {"name": "top_long_list", "op": "top", "ranks": 3, "rows": 301, "vocab": 32003, "k": 700, "dtype": "fp16", "pad": 5},
        # a training step: loss and gradient together
        {"name": "distill_train", "op": "distill", "kind": "train", "ranks": 8, "rows": 4096, "vocab": 131072, "k": 64, "T": 2.0,
         "dtype": "bf16", "pad": 0},
        # the same where what reaches the loss is known later: 32-bit logits, odd sizes
        {"name": "distill_apart", "op": "distill", "kind": "apart", "ranks": 2, "rows": 1500, "vocab": 100003, "k": 50, "T": 1.5,
         "dtype": "fp32", "pad": 1},
        # an evaluation of the loss alone
        {"name": "distill_loss", "op": "distill", "kind": "loss", "ranks": 4, "rows": 2048, "vocab": 65536, "k": 128, "T": 1.0,
         "dtype": "fp16", "pad": 0},
        # a small batch and a small vocabulary: latency
        {"name": "distill_small", "op": "distill", "kind": "train", "ranks": 1, "rows": 16, "vocab": 32000, "k": 32, "T": 1.0,
         "dtype": "bf16", "pad": 0},
        # the next token of one answer
        {"name": "sample_one", "op": "sample", "ranks": 1, "rows": 1, "vocab": 131072, "dtype": "bf16", "pad": 0},
        # a step of a batch of answers, each with settings of its own
        {"name": "sample_batch", "op": "sample", "ranks": 8, "rows": 64, "vocab": 131072, "dtype": "bf16", "pad": 0},
        # odd sizes, fp16
        {"name": "sample_odd", "op": "sample", "ranks": 3, "rows": 37, "vocab": 50021, "dtype": "fp16", "pad": 3},
        # many short answers at once, 32-bit logits
        {"name": "sample_many", "op": "sample", "ranks": 8, "rows": 1024, "vocab": 131072, "dtype": "fp32", "pad": 0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    c = {"op": rng.choice(["top", "distill", "distill", "sample", "sample"]), "ranks": rng.choice([1, 2, 3, 4, 8, 8, 16]),
         "vocab": _log_int(rng, 1000, 262144), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "pad": rng.choice([0, 0, 1, 3, 8])}
    c["rows"] = _log_int(rng, 1, min(1024 if c["op"] == "sample" else 4096, int(DRAW_BYTES / (8 * c["vocab"]))))
    if c["op"] == "distill":
        c["kind"] = rng.choice(["train", "train", "apart", "loss"])
        c["T"] = rng.choice([1.0, 1.5, 2.0, 4.0])
    if c["op"] != "sample":
        c["k"] = _log_int(rng, 1, 256 if c["op"] == "distill" else 1000)
    return c


# ---- what a case consists of ------------------------------------------------------------------------------------------

def _columns(case):
    share, vocab = -(-case["vocab"] // case["ranks"]), case["vocab"]
    return [max(0, min(share, vocab - j * share)) for j in range(case["ranks"])]


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _logits(case, g):
    """A few tokens are likely and most are not: the r-th most likely token of a row has a probability of about r^-s, with an s for
    each row, which is what exponentially distributed logits have."""
    rows, vocab = case["rows"], case["vocab"]
    s = 1.2 + 0.8 * torch.rand((rows, 1), device=DEV, generator=g)
    whole = torch.empty((rows, vocab), device=DEV).exponential_(1.0, generator=g).mul_(s).sub_(4.0)
    held, at = [], 0
    for c in _columns(case):
        part = torch.zeros((rows, c + case["pad"]), device=DEV, dtype=TYPES[case["dtype"]])
        part[:, :c] = whole[:, at:at + c]
        held.append(part)
        at += c
    return whole, held


def _inputs(case, seed):
    g, rows, vocab = _generator(seed), case["rows"], case["vocab"]
    whole, held = _logits(case, g)
    s = {"case": case, "logits": held, "columns": _columns(case)}
    if case["op"] == "distill":
        # a teacher that mostly agrees
        whole.add_(torch.randn(whole.shape, device=DEV, generator=g))
        values, indices = whole.topk(case["k"], dim=1)
        s["teacher"], s["indices"] = values.to(TYPES[case["dtype"]]), indices.to(torch.int32)
        # every tenth row is masked
        live = (torch.arange(rows, device=DEV) % 10 != 9).float()
        s["weight"] = live * (0.5 + torch.rand(rows, device=DEV, generator=g)) / rows
    if case["op"] == "sample":
        # by row in turn: all three filters; a short list; the probable part; no filter; the largest; what is not too improbable
        kind = torch.arange(rows, device=DEV) % 6
        r = torch.rand((4, rows), device=DEV, generator=g)
        s["temperature"] = torch.where(kind == 4, torch.zeros_like(r[0]), 0.6 + 0.6 * r[0])
        s["top_k"] = torch.where(kind == 0, 50, torch.where(kind == 1, 1 + (39 * r[1]).int(), 0)).to(torch.int32)
        s["top_p"] = torch.where((kind == 0) | (kind == 2), 0.8 + 0.15 * r[2], torch.ones_like(r[2]))
        s["min_p"] = torch.where((kind == 0) | (kind == 5), 0.02 + 0.08 * r[3], torch.zeros_like(r[3]))
        s["random"] = torch.rand(rows, device=DEV, generator=g)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        {"top": _plan_top, "distill": _plan_distill, "sample": _plan_sample}[case["op"]](s)
    return s


def run(state):
    if own:
        return {"top": _own_top, "distill": _own_distill, "sample": _own_sample}[state["case"]["op"]](state)
    return {"top": _plain_top, "distill": _plain_distill, "sample": _plain_sample}[state["case"]["op"]](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "top":
        return {"bytes": rows * (vocab * size + case["k"] * (size + 4) + 4), "flops": 4 * rows * vocab}
    if case["op"] == "sample":
        return {"bytes": rows * (vocab * size + 28), "flops": 4 * rows * vocab}
    live = rows - rows // 10                       # (of masked rows nothing has to be read)
    moved = live * (vocab * size + case["k"] * (size + 4)) + rows * 8
    if case["kind"] == "loss":
        return {"bytes": moved, "flops": 4 * live * vocab}
    return {"bytes": moved + rows * vocab * size, "flops": 8 * live * vocab}


# ---- the operators of this repository -----------------------------------------------------------------------------------

def _dtype(case):
    from hccl_amd import types as T
    return {"bf16": T.BFP16, "fp16": T.FP16, "fp32": T.FP32}[case["dtype"]]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _held(s, parts):
    """What says where the logits, or their gradients, are."""
    return dict(columns=s["columns"], rows=s["case"]["rows"], dtype=_dtype(s["case"]), strides=[t.stride(0) for t in parts])


def _each(parts):
    return [t.data_ptr() for t in parts]


def _plan_top(s):
    from hccl_amd import hcclx
    rows, k = s["case"]["rows"], s["case"]["k"]
    s["values"] = torch.empty((rows, k), device=DEV, dtype=TYPES[s["case"]["dtype"]])
    s["numbers"] = torch.empty((rows, k), device=DEV, dtype=torch.int32)
    s["lse"] = torch.empty(rows, device=DEV)
    s["plan"] = hcclx.TopLogitsPlan(_each(s["logits"]), k=k, values=s["values"].data_ptr(), indices=s["numbers"].data_ptr(),
                                    lse=s["lse"].data_ptr(), **_held(s, s["logits"]))


def _own_top(s):
    s["plan"].launch(_stream())
    return {"values": s["values"], "indices": s["numbers"], "lse": s["lse"]}


def _plan_distill(s):
    from hccl_amd import hcclx
    case = s["case"]
    rows, kind = case["rows"], case["kind"]
    s["loss"] = torch.empty(rows, device=DEV)
    held = dict(_held(s, s["logits"]), k=case["k"], teacher=s["teacher"].data_ptr(), indices=s["indices"].data_ptr(), temperature=case["T"],
                weight=s["weight"].data_ptr())
    if kind != "loss":
        s["dlogits"] = [torch.zeros_like(t) for t in s["logits"]]
    if kind == "train":
        held["dlogits"] = _each(s["dlogits"])
    if kind == "apart":
        s["stats"] = torch.empty((rows, 2), device=DEV)
        s["grad_plan"] = hcclx.DistillGradPlan(_each(s["logits"]), stats=s["stats"].data_ptr(), dlogits=_each(s["dlogits"]), **held)
        held["stats"] = s["stats"].data_ptr()
    s["plan"] = hcclx.DistillPlan(_each(s["logits"]), loss=s["loss"].data_ptr(), **held)


def _own_distill(s):
    stream = _stream()
    s["plan"].launch(stream)
    if s["case"]["kind"] == "loss":
        return {"loss": s["loss"]}
    if s["case"]["kind"] == "apart":
        s["grad_plan"].launch(stream)
    return {"loss": s["loss"], "dlogits": [t[:, :c] for t, c in zip(s["dlogits"], s["columns"])]}


def _plan_sample(s):
    from hccl_amd import hcclx
    rows = s["case"]["rows"]
    s["tokens"] = torch.empty(rows, device=DEV, dtype=torch.int32)
    s["logprob"] = torch.empty(rows, device=DEV)
    s["plan"] = hcclx.SamplePlan(_each(s["logits"]), tokens=s["tokens"].data_ptr(), logprob=s["logprob"].data_ptr(),
                                 **{k: s[k].data_ptr() for k in ("random", "temperature", "top_k", "top_p", "min_p")}, **_held(s, s["logits"]))


def _own_sample(s):
    s["plan"].launch(_stream())
    return {"tokens": s["tokens"], "logprob": s["logprob"]}


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _whole(s):
    return torch.cat([t[:, :c] for t, c in zip(s["logits"], s["columns"])], dim=1)


def _plain_top(s):
    l = _whole(s)
    k = s["case"]["k"]
    order = torch.sort(l, dim=1, descending=True, stable=True)
    f = l.float()
    most = f.amax(dim=1, keepdim=True)
    lse = most[:, 0] + torch.exp(f - most).sum(dim=1).log()
    return {"values": order.values[:, :k], "indices": order.indices[:, :k].to(torch.int32), "lse": lse}


def _plain_distill(s):
    case, w, T = s["case"], s["weight"][:, None], s["case"]["T"]
    f = _whole(s).float() / T
    t, at = s["teacher"].float() / T, s["indices"].long()
    f = f - f.amax(dim=1, keepdim=True)
    logq = f - torch.exp(f).sum(dim=1, keepdim=True).log()
    t = t - t.amax(dim=1, keepdim=True)
    logp = t - torch.exp(t).sum(dim=1, keepdim=True).log()
    p = torch.exp(logp)
    loss = (w * T * T * (p * (logp - logq.gather(1, at))).sum(dim=1, keepdim=True))[:, 0]
    if case["kind"] == "loss":
        return {"loss": loss}
    d = torch.exp(logq).scatter_add_(1, at, -p).mul_(w * T).to(TYPES[case["dtype"]])
    return {"loss": loss, "dlogits": list(d.split(s["columns"], dim=1))}


def _plain_sample(s):
    """In 64 bits: which token the running sum passes u at, and how far a beginning of the order reaches, is decided by values next
    to a border."""
    l = _whole(s)
    vocab = l.shape[1]
    T, top_p, min_p, u = (s[k].double()[:, None] for k in ("temperature", "top_p", "min_p", "random"))
    greedy = T <= 0
    T = torch.where(greedy, torch.ones_like(T), T)
    k = s["top_k"].long()[:, None]
    k = torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, torch.full_like(k, vocab)))
    order = torch.sort(l, dim=1, descending=True, stable=True)
    values = order.values.double()
    x = (values - values[:, :1]) / T
    w = torch.exp(x)
    rank = torch.arange(vocab, device=l.device)
    keep = rank < k
    w = w * keep
    c = w.cumsum(dim=1)
    before = torch.nn.functional.pad(c, (1, 0))[:, :-1]
    keep &= (top_p >= 1) | (rank == 0) | (before < top_p * c[:, -1:])
    keep &= w >= min_p
    w = torch.zeros_like(w).scatter_(1, order.indices, w * keep)
    c = w.cumsum(dim=1)
    token = (c <= u * c[:, -1:]).sum(dim=1, keepdim=True).clamp_(max=vocab - 1)
    logprob = (l.gather(1, token).double() - values[:, :1]) / T - c[:, -1:].log()
    return {"tokens": token[:, 0].to(torch.int32), "logprob": logprob[:, 0].float()}


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    l = torch.cat([t.double()[:, :c] for t, c in zip(s["logits"], s["columns"])], dim=1)
    return {"top": _exact_top, "distill": _exact_distill, "sample": _exact_sample}[case["op"]](s, l)


def _exact_top(s, l):
    first = l.argsort(dim=1, descending=True, stable=True)[:, :s["case"]["k"]]
    return {"values": l.gather(1, first), "indices": first.to(torch.int32), "lse": torch.logsumexp(l, dim=1)}


def _exact_distill(s, l):
    case, T, at = s["case"], s["case"]["T"], s["indices"].long()
    wanted = case["kind"] != "loss"
    l.requires_grad_(wanted)
    p = torch.softmax(s["teacher"].double() / T, dim=1)
    q = torch.log_softmax(l / T, dim=1).gather(1, at)
    loss = T ** 2 * s["weight"].double() * (p * (p.log() - q)).sum(dim=1)
    if not wanted:
        return {"loss": loss}
    return {"loss": loss.detach(), "dlogits": [t.contiguous() for t in torch.autograd.grad(loss.sum(), l)[0].split(s["columns"], dim=1)]}


def _exact_sample(s, l):
    """By the least value that stays instead of by places in the order: of the tokens with that value, the first ones."""
    T = s["temperature"].double()[:, None]
    greedy = (T == 0).squeeze(1)
    e = torch.exp((l - l.amax(dim=1, keepdim=True)) / torch.where(T == 0, torch.ones_like(T), T))
    down, places = (-l).sort(dim=1, stable=True)
    falling = e.gather(1, places)
    many = torch.where(s["top_k"] > 0, s["top_k"].long(), l.shape[1])
    many = torch.where(greedy, 1, many)
    sums = falling.cumsum(dim=1)
    whole = sums.gather(1, many[:, None] - 1)
    p = s["top_p"].double()[:, None]
    reach = torch.searchsorted(sums, p * whole)[:, 0] + 1        # the first place at which top_p is reached
    many = torch.where(p[:, 0] < 1, torch.minimum(many, reach), many)
    probable = (falling >= s["min_p"].double()[:, None]).sum(dim=1)
    many = torch.minimum(many, probable)
    place = torch.empty_like(places).scatter_(1, places, torch.arange(l.shape[1], device=l.device).expand_as(places))
    c = torch.where(place < many[:, None], e, torch.zeros_like(e)).cumsum(dim=1)
    token = torch.searchsorted(c, s["random"].double()[:, None] * c[:, -1:], right=True).clamp(max=l.shape[1] - 1)
    return {"tokens": token[:, 0].to(torch.int32), "logprob": (e.gather(1, token) / c[:, -1:]).log()[:, 0]}
