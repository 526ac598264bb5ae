"""The model-side operators that stand next to the collectives of a training or serving step: the norm in front of an MoE
exchange, the experts behind it, and the optimizer step on the sharded gradients.

listed() names the cases, draw() makes more of the same kinds; prepare() builds what a program holds before the call, run()
is one pass through an operator and returns its outputs whole.  With own = False run() computes them from elementary torch
operations in 32 bits, with own = True through hccl_amd.hcclx.  exact() gives them from the definitions in 64 bits.

rms_norm: n ranks hold `rows` rows of `dim` elements.  s = x + residual, rounded to the rows' type (the residual stream that
the next layer reads); y = s * w / sqrt(mean(s^2) + eps).  "train" cases go on to the gradients: with dy of y and ds of s,
dx = r * (dy * w - s * r^2 * mean(dy * w * s)) + ds,  dw = sum over rows of dy * s * r,  r = 1 / sqrt(mean(s^2) + eps).
"quant" cases write y in 8 bits (e4m3) with a scale max|y| / 448 per row, 0 codes for a row of zeros.

gated_ffn: rank j holds rows_j rows and an expert's three weights; out = (silu(x Wg^T) * (x Wu^T)) Wd^T.  "quant" cases read
rows of e4m3 codes and a scale each, as the norm writes them; "train" cases return the gradients of x and of the weights.

adamw: m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p - lr (wd p + (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)),
on 32-bit parameters, with a 16-bit copy of them for the gather that follows.  With states in 8 bits, m and sqrt(v) are held as
e4m3 codes with a scale max / 448 per 256 elements, rounded stochastically (to nearest, a moving average that changes by less
than half a code per step would stand still): random number k of tensor t in a step with a given seed is
    mix(k + mix(seed + (t + 1) * 0x9E3779B9)),  mix as in _mix below, its low 16 bits for m and its high ones for sqrt(v)."""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda:0"
EPS = 1e-6
E4M3_MOST = 448.0
TAIL = 16            # bytes behind the codes of an 8-bit row: its scale and padding
STEP, LR, BETA1, BETA2, ADAM_EPS = 1000, 1e-4, 0.9, 0.999, 1e-8
BLOCK = 256          # elements that share a scale of the 8-bit states

# what a drawn case costs at most (the largest listed ones cost more)
DRAW_FLOPS = 2.5e12
DRAW_BYTES = 1.5e9


def listed():
    return [
        # one decoding step: few tokens per rank, the stream is added and the rows go into the exchange in 8 bits
        {"name": "norm_quant_decode", "op": "norm", "kind": "quant", "ranks": 8, "rows": 64, "dim": 7168, "dtype": "bf16"},
        # the same in prefill (4096 tokens per rank): all bandwidth
        {"name": "norm_quant_prefill", "op": "norm", "kind": "quant", "ranks": 8, "rows": 4096, "dim": 7168, "dtype": "bf16"},
        # a training step's norm, forward and backward
        {"name": "norm_train", "op": "norm", "kind": "train", "ranks": 8, "rows": 2048, "dim": 4096, "dtype": "bf16"},
        # odd numbers of rows and elements, 32-bit rows
        {"name": "norm_train_odd", "op": "norm", "kind": "train", "ranks": 3, "rows": 777, "dim": 1001, "dtype": "fp32"},
        # one token through one expert: the weights' bandwidth and two launches
        {"name": "ffn_one_token", "op": "ffn", "kind": "serve", "ranks": 1, "tokens": 1, "dim": 4096, "hidden": 2048,
         "dtype": "bf16"},
        # a decoding step of 8 ranks x 64 tokens, ragged over the experts, in the 8-bit rows that the exchange carried
        {"name": "ffn_quant_decode", "op": "ffn", "kind": "quant", "ranks": 8, "tokens": 64, "dim": 7168, "hidden": 2048,
         "dtype": "bf16"},
        # prefill: 8 ranks x 4096 tokens, ragged
        {"name": "ffn_prefill", "op": "ffn", "kind": "serve", "ranks": 8, "tokens": 4096, "dim": 7168, "hidden": 2048,
         "dtype": "bf16"},
        # training, forward and backward
        {"name": "ffn_train", "op": "ffn", "kind": "train", "ranks": 8, "tokens": 2048, "dim": 4096, "hidden": 2048,
         "dtype": "bf16"},
        # training with ragged edges everywhere, fp16
        {"name": "ffn_train_ragged", "op": "ffn", "kind": "train", "ranks": 3, "tokens": 1001, "dim": 2880, "hidden": 1432,
         "dtype": "fp16"},
        # the parameters of a small model or of the norms alone: latency
        {"name": "adamw_small", "op": "adamw", "bits": 32, "tensors": 9, "elements": 40001, "dtype": "fp32"},
        # a rank's shard of a model: bf16 gradients, states in 32 bits
        {"name": "adamw_shard", "op": "adamw", "bits": 32, "tensors": 61, "elements": 100000003, "dtype": "bf16"},
        # the same with states in 8 bits
        {"name": "adamw_shard_8bit", "op": "adamw", "bits": 8, "tensors": 61, "elements": 100000003, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "ffn", "ffn", "adamw"])
    if op == "adamw":
        return {"op": op, "bits": rng.choice([8, 32]), "tensors": _log_int(rng, 1, 120), "elements": _log_int(rng, 2000, int(DRAW_BYTES / 30)),
                "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    c = {"op": op, "ranks": rng.choice([1, 2, 3, 4, 8, 8, 12, 16])}
    if op == "norm":
        c["kind"] = rng.choice(["quant", "train"])
        c["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        c["dim"] = 16 * _log_int(rng, 8, 512) if c["kind"] == "quant" else _log_int(rng, 100, 8192)
        c["rows"] = _log_int(rng, 1, min(4096, int(DRAW_BYTES / (c["ranks"] * c["dim"] * 20))))
        return c
    c["kind"] = rng.choice(["serve", "quant", "train"])
    c["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
    c["dim"] = 16 * _log_int(rng, 16, 448) if c["kind"] == "quant" else 8 * _log_int(rng, 32, 896)
    c["hidden"] = 8 * _log_int(rng, 32, 512)
    flops = 6.0 * c["ranks"] * c["dim"] * c["hidden"] * (3 if c["kind"] == "train" else 1)
    c["tokens"] = _log_int(rng, 1, max(2, min(4096, int(DRAW_FLOPS / flops))))
    return c


# ---- what a case consists of ------------------------------------------------------------------------------------------

def _shares(case):
    """Rows of each rank: ranks x tokens in all, in shares as a router with favourites gives them (rank 0 the most, the last of
    many ranks few or none)."""
    n, total = case["ranks"], case["ranks"] * case["tokens"]
    weights = [1.0 / (k + 1) ** 0.4 for k in range(n)]
    ends = [round(total * sum(weights[:k + 1]) / sum(weights)) for k in range(n)]
    return [b - a for a, b in zip([0] + ends, ends)]


def _sizes(case):
    """Elements of each tensor: as many as there are in all, in sizes that span three orders of magnitude, odd ones among them."""
    r = random.Random(case["tensors"] * 1000003 + case["elements"])
    weights = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    spare = case["elements"] - case["tensors"]
    ends = [round(spare * sum(weights[:k + 1]) / sum(weights)) for k in range(case["tensors"])]
    return [b - a + 1 for a, b in zip([0] + ends, ends)]


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(shape, dtype, g, scale=1.0):
    return torch.randn(shape, device=DEV, generator=g, dtype=torch.float32).mul_(scale).to(dtype)


def _to_rows8(y):
    """Rows of 32-bit floats as the exchange carries them in 8 bits: codes, the scale, padding."""
    scale = y.abs().amax(dim=1, keepdim=True) / E4M3_MOST
    codes = (y / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn)
    rows = torch.zeros((y.shape[0], y.shape[1] + TAIL), device=y.device, dtype=torch.uint8)
    rows[:, :y.shape[1]] = codes.view(torch.uint8)
    rows[:, y.shape[1]:y.shape[1] + 4] = scale.view(torch.uint8)
    return rows


def _inputs_norm(case, seed):
    n, rows, dim, dt, g = case["ranks"], case["rows"], case["dim"], TYPES[case["dtype"]], _generator(seed)
    s = {"x": _normal((n, rows, dim), dt, g), "residual": _normal((n, rows, dim), dt, g, 2.0),
         "weight": (1.0 + 0.1 * torch.randn((n, dim), device=DEV, generator=g)).to(dt)}
    if case["kind"] == "train":
        s["dy"] = _normal((n, rows, dim), dt, g)
        s["ds"] = _normal((n, rows, dim), dt, g)
    return s


def _inputs_ffn(case, seed):
    n, dim, hidden, dt, g = case["ranks"], case["dim"], case["hidden"], TYPES[case["dtype"]], _generator(seed)
    rows = _shares(case)
    s = {"rows": rows, "x": _normal((sum(rows), dim), dt, g), "w_gate": _normal((n, hidden, dim), dt, g, dim ** -0.5),
         "w_up": _normal((n, hidden, dim), dt, g, dim ** -0.5), "w_down": _normal((n, dim, hidden), dt, g, hidden ** -0.5)}
    if case["kind"] == "quant":
        s["x"] = _to_rows8(s["x"].float())
    if case["kind"] == "train":
        s["dy"] = _normal((sum(rows), dim), dt, g)
    return s


def _inputs_adamw(case, seed):
    sizes, g, total = _sizes(case), _generator(seed), case["elements"]
    s = {"sizes": sizes, "param": _normal(total, torch.float32, g, 0.02),
         "copy": torch.zeros(total, device=DEV, dtype=torch.bfloat16),
         "decay": [0.1 if k % 3 else 0.0 for k in range(len(sizes))], "seed": seed & 0xFFFFFFFF}
    # gradients and the states that a thousand of them left, of a size of its own for every stretch of the tensors
    level = torch.exp(torch.randn(total // 1024 + 1, device=DEV, generator=g)).repeat_interleave(1024)[:total] * 1e-3
    s["grad"] = (torch.randn(total, device=DEV, generator=g) * level).to(TYPES[case["dtype"]])
    m = torch.randn(total, device=DEV, generator=g) * level * 0.2
    r = level * (0.5 + torch.rand(total, device=DEV, generator=g))
    if case["bits"] == 32:
        s["m"], s["v"] = m, r * r
        return s
    blocks = [(k + BLOCK - 1) // BLOCK for k in sizes]
    s["m"], s["v"] = (torch.zeros(total, device=DEV, dtype=torch.float8_e4m3fn) for _ in range(2))
    s["m_scale"], s["v_scale"] = (torch.zeros(sum(blocks), device=DEV) for _ in range(2))
    at = block = 0
    for size, nb in zip(sizes, blocks):
        for values, codes, scales in ((m, s["m"], s["m_scale"]), (r, s["v"], s["v_scale"])):
            x = torch.nn.functional.pad(values[at:at + size], (0, nb * BLOCK - size)).view(nb, BLOCK)
            scale = x.abs().amax(dim=1) / E4M3_MOST
            scales[block:block + nb] = scale
            codes[at:at + size] = (x / scale[:, None]).clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn).view(-1)[:size]
        at, block = at + size, block + nb
    return s


def prepare(case, seed):
    s = {"norm": _inputs_norm, "ffn": _inputs_ffn, "adamw": _inputs_adamw}[case["op"]](case, seed)
    s["case"] = case
    if own:
        {"norm": _plan_norm, "ffn": _plan_ffn, "adamw": _plan_adamw}[case["op"]](s)
    return s


def run(state):
    if own:
        return {"norm": _own_norm, "ffn": _own_ffn, "adamw": _own_adamw}[state["case"]["op"]](state)
    return {"norm": _plain_norm, "ffn": _plain_ffn, "adamw": _plain_adamw}[state["case"]["op"]](state)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "norm":
        elements = case["ranks"] * case["rows"] * case["dim"]
        if case["kind"] == "quant":
            return {"bytes": elements * (3 * size + 1), "flops": 6 * elements}
        return {"bytes": elements * 7 * size, "flops": 20 * elements}   # x, residual, dy, ds in; s, y, dx out
    if case["op"] == "ffn":
        rows, weights = case["ranks"] * case["tokens"], 3 * case["ranks"] * case["dim"] * case["hidden"]
        flops = 6 * rows * case["dim"] * case["hidden"]
        if case["kind"] == "train":
            return {"bytes": 2 * (2 * weights + 4 * rows * case["dim"]), "flops": 3 * flops}
        return {"bytes": 2 * weights + rows * case["dim"] * (3 if case["kind"] == "quant" else 4), "flops": flops}
    # parameter, both states, gradient, copy
    return {"bytes": case["elements"] * (8 + (16 if case["bits"] == 32 else 4) + size + 2), "flops": 20 * case["elements"]}


# ---- the operators of this repository -----------------------------------------------------------------------------------

def _stream():
    return torch.cuda.current_stream().cuda_stream


def _each(t):
    """The address of every rank's part of a stacked tensor."""
    step = t.stride(0) * t.element_size()
    return [t.data_ptr() + k * step for k in range(t.shape[0])]


def _ranks_rows(t, rows):
    """The address of every rank's first row in a tensor of all ranks' rows."""
    step, starts = t.stride(0) * t.element_size(), [sum(rows[:k]) for k in range(len(rows))]
    return [t.data_ptr() + k * step for k in starts]


def _dtype(case):
    from hccl_amd import types as T
    return {"bf16": T.BFP16, "fp16": T.FP16, "fp32": T.FP32}[case["dtype"]]


def _plan_norm(s):
    from hccl_amd import hcclx
    from hccl_amd import types as T
    case, dt = s["case"], _dtype(s["case"])
    n, rows, dim = case["ranks"], case["rows"], case["dim"]
    s["sum"] = torch.empty_like(s["x"])
    quant = case["kind"] == "quant"
    s["out"] = torch.empty((n, rows, dim + TAIL), device=DEV, dtype=torch.uint8) if quant else torch.empty_like(s["x"])
    s["plan"] = hcclx.RmsNormPlan(_each(s["x"]), _each(s["weight"]), _each(s["out"]), rows, dim, dt,
                                  residual=_each(s["residual"]), total=_each(s["sum"]),
                                  out_dtype=T.FP8E4M3 if quant else dt, eps=EPS)
    if not quant:
        s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["weight"])
        s["grad_plan"] = hcclx.RmsNormGradPlan(_each(s["dy"]), _each(s["sum"]), _each(s["weight"]), _each(s["dx"]),
                                               _each(s["dw"]), rows, dim, dt, dtotal=_each(s["ds"]), eps=EPS)


def _own_norm(s):
    stream = _stream()
    s["plan"].launch(stream)
    if s["case"]["kind"] == "quant":
        dim = s["case"]["dim"]
        rows = s["out"].view(-1, dim + TAIL)
        return {"sum": s["sum"], "codes": rows[:, :dim].view(torch.float8_e4m3fn), "scale": rows[:, dim:dim + 4].view(torch.float32)}
    s["grad_plan"].launch(stream)
    return {"sum": s["sum"], "out": s["out"], "dx": s["dx"], "dw": s["dw"]}


def _plan_ffn(s):
    from hccl_amd import hcclx
    from hccl_amd import types as T
    case, dt, rows = s["case"], _dtype(s["case"]), s["rows"]
    dim, hidden = case["dim"], case["hidden"]
    total = sum(rows)
    quant = case["kind"] == "quant"
    s["out"] = torch.empty((total, dim), device=DEV, dtype=TYPES[case["dtype"]])
    # the number of rows is known on the device alone, as an exchange leaves it: elements per rank
    s["counts"] = torch.tensor([k * s["x"].shape[1] for k in rows], device=DEV, dtype=torch.int64)
    shape = dict(capacity=total, dim=dim, hidden=hidden, dtype=dt, rows=total, counts=s["counts"].data_ptr(), counts_per_rank=1,
                 count_unit=s["x"].shape[1])
    weights = [_each(s[w]) for w in ("w_gate", "w_up", "w_down")]
    x = _ranks_rows(s["x"], rows)
    if case["kind"] == "train":
        s["saved"] = torch.empty(hcclx.gated_ffn_saved_bytes(total, hidden), device=DEV, dtype=torch.uint8)
        s["dx"] = torch.empty_like(s["x"])
        s["dw_gate"], s["dw_up"], s["dw_down"] = (torch.empty_like(s[w]) for w in ("w_gate", "w_up", "w_down"))
        s["plan"] = hcclx.GatedFfnPlan(x, *weights, _ranks_rows(s["out"], rows), saved=s["saved"].data_ptr(), **shape)
        s["grad_plan"] = hcclx.GatedFfnGradPlan(_ranks_rows(s["dy"], rows), x, *weights, s["saved"].data_ptr(),
                                                _ranks_rows(s["dx"], rows), _each(s["dw_gate"]), _each(s["dw_up"]),
                                                _each(s["dw_down"]), **shape)
    else:
        s["plan"] = hcclx.GatedFfnPlan(x, *weights, _ranks_rows(s["out"], rows), x_dtype=T.FP8E4M3 if quant else dt, **shape)


def _own_ffn(s):
    stream = _stream()
    s["plan"].launch(stream)
    if s["case"]["kind"] != "train":
        return {"out": s["out"]}
    s["grad_plan"].launch(stream)
    return {k: s[k] for k in ("out", "dx", "dw_gate", "dw_up", "dw_down")}


def _plan_adamw(s):
    from hccl_amd import hcclx
    from hccl_amd import types as T
    tensors, at, block = [], 0, 0
    small, size_of = s["case"]["bits"] == 8, s["grad"].element_size()
    for size, decay in zip(s["sizes"], s["decay"]):
        t = dict(count=size, param=s["param"].data_ptr() + 4 * at, grad=s["grad"].data_ptr() + size_of * at,
                 m=s["m"].data_ptr() + (at if small else 4 * at), v=s["v"].data_ptr() + (at if small else 4 * at),
                 copy=s["copy"].data_ptr() + 2 * at, weight_decay=decay)
        if small:
            t.update(m_scale=s["m_scale"].data_ptr() + 4 * block, v_scale=s["v_scale"].data_ptr() + 4 * block)
        tensors.append(t)
        at, block = at + size, block + (size + BLOCK - 1) // BLOCK
    s["plan"] = hcclx.AdamWPlan(tensors, grad_dtype=_dtype(s["case"]), state_dtype=T.FP8E4M3 if small else T.FP32, copy_dtype=T.BFP16)


def _own_adamw(s):
    s["plan"].step(STEP, lr=LR, beta1=BETA1, beta2=BETA2, eps=ADAM_EPS, seed=s["seed"], stream=_stream())
    return _states(s)


def _states(s):
    return {k: s[k] for k in ("param", "copy", "m", "v", "m_scale", "v_scale") if k in s}


# ---- the plain forms ------------------------------------------------------------------------------------------------------

def _plain_norm(s):
    dt = s["x"].dtype
    total = (s["x"].float() + s["residual"].float()).to(dt)
    f, w = total.float(), s["weight"].float()[:, None, :]
    r = torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + EPS)
    y = f * r * w
    if s["case"]["kind"] == "quant":
        y = y.view(-1, y.shape[-1])
        scale = y.abs().amax(dim=1, keepdim=True) / E4M3_MOST
        codes = (y / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn)
        return {"sum": total, "codes": codes, "scale": scale}
    dy = s["dy"].float()
    a = dy * w
    dx = r * (a - f * (r * r) * (a * f).mean(dim=-1, keepdim=True)) + s["ds"].float()
    return {"sum": total, "out": y.to(dt), "dx": dx.to(dt), "dw": (dy * f * r).sum(dim=1).to(dt)}


def _plain_expert(case, x, w_gate, w_up, w_down, dy):
    w_gate, w_up, w_down = w_gate.float(), w_up.float(), w_down.float()
    if case["kind"] == "quant":
        x = x[:, :case["dim"]].view(torch.float8_e4m3fn).float() * x[:, case["dim"]:case["dim"] + 4].contiguous().view(torch.float32)
    x = x.float()
    gate, up = x @ w_gate.T, x @ w_up.T
    sig = torch.sigmoid(gate)
    h = gate * sig * up
    out = (h @ w_down.T,)
    if dy is None:
        return out
    dy = dy.float()
    dh = dy @ w_down
    dgate = dh * up * (sig * (1 + gate * (1 - sig)))
    dup = dh * gate * sig
    return out + (dgate @ w_gate + dup @ w_up, dgate.T @ x, dup.T @ x, dy.T @ h)


def _plain_ffn(s):
    case, dt = s["case"], TYPES[s["case"]["dtype"]]
    dys = s["dy"].split(s["rows"]) if "dy" in s else [None] * len(s["rows"])
    got = [[t.to(dt) for t in _plain_expert(case, *one)] for one in zip(s["x"].split(s["rows"]), s["w_gate"], s["w_up"], s["w_down"], dys)]
    if case["kind"] != "train":
        return {"out": torch.cat([g[0] for g in got])}
    return {"out": torch.cat([g[0] for g in got]), "dx": torch.cat([g[1] for g in got]), "dw_gate": torch.stack([g[2] for g in got]),
            "dw_up": torch.stack([g[3] for g in got]), "dw_down": torch.stack([g[4] for g in got])}


def _mix(x):
    """A bijection of the 32-bit integers (in 64-bit ones) whose every output bit depends on every input bit."""
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _uniforms(seed, tensor, size):
    """The random numbers of a step for the elements of a tensor, in [0, 1): for m and for sqrt(v)."""
    word = _mix(torch.arange(size, device=DEV) + _mix(seed + (tensor + 1) * 0x9E3779B9))
    return (word & 0xFFFF).float() / 65536, (word >> 16).float() / 65536


def _plain_round(x, u):
    """To the e4m3 value below |x| or the one above, the one above with the probability of the distance from the one below."""
    a = x.abs().clamp(max=E4M3_MOST)
    step = torch.ldexp(torch.ones_like(a), torch.frexp(a).exponent.clamp(min=-5) - 4)
    return (torch.floor(a / step + u) * step).copysign(x).to(torch.float8_e4m3fn)


def _plain_adamw(s):
    at, block, small = 0, 0, s["case"]["bits"] == 8
    for k, (size, decay) in enumerate(zip(s["sizes"], s["decay"])):
        here, nb = slice(at, at + size), (size + BLOCK - 1) // BLOCK
        g, p, m, v = (s[x][here].float() for x in ("grad", "param", "m", "v"))
        if small:
            blocks = slice(block, block + nb)
            m = m * s["m_scale"][blocks].repeat_interleave(BLOCK)[:size]
            v = (v * s["v_scale"][blocks].repeat_interleave(BLOCK)[:size]).square()
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        p = p - LR * (decay * p + (m / (1 - BETA1 ** STEP)) / (torch.sqrt(v / (1 - BETA2 ** STEP)) + ADAM_EPS))
        s["param"][here] = p
        s["copy"][here] = p.to(torch.bfloat16)
        if small:
            us = _uniforms(s["seed"], k, size)
            for x, u, codes, scales in ((m, us[0], "m", "m_scale"), (torch.sqrt(v), us[1], "v", "v_scale")):
                x, u = (torch.nn.functional.pad(t, (0, nb * BLOCK - size)).view(nb, BLOCK) for t in (x, u))
                scale = x.abs().amax(dim=1) / E4M3_MOST
                s[scales][blocks] = scale
                q = _plain_round(x / torch.where(scale > 0, scale, torch.ones_like(scale))[:, None], u)
                s[codes][here] = q.view(-1)[:size]
        else:
            s["m"][here], s["v"][here] = m, v
        at, block = at + size, block + nb
    return _states(s)


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    return {"norm": _exact_norm, "ffn": _exact_ffn, "adamw": _exact_adamw}[case["op"]](case, seed)


def _nearest_e4m3(x):
    """The e4m3 value nearest to each element (of two, the one with an even last bit): 2^-9 apart below 2^-6, eight to a power
    of two above."""
    a = x.abs().clamp(min=2.0 ** -6)
    gap = 2.0 ** (torch.floor(torch.log2(a)) - 3)
    return (torch.round(x / gap) * gap).clamp(-E4M3_MOST, E4M3_MOST)


def _exact_norm(case, seed):
    s = _inputs_norm(case, seed)
    stored = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()
    train = case["kind"] == "train"
    stored.requires_grad_(train)
    w = s["weight"].double().requires_grad_(train)
    y = stored / (stored.square().mean(-1, keepdim=True) + EPS).sqrt() * w[:, None, :]
    if train:
        dx, dw = torch.autograd.grad(y, (stored, w), s["dy"].double())
        return {"sum": stored.detach(), "out": y.detach(), "dx": dx + s["ds"].double(), "dw": dw}
    y = y.reshape(-1, case["dim"])
    scale = y.abs().max(dim=1, keepdim=True).values / E4M3_MOST
    return {"sum": stored, "codes": _nearest_e4m3((y / scale).nan_to_num(0.0)), "scale": scale}


def _exact_ffn(case, seed):
    s = _inputs_ffn(case, seed)
    train, got, at = case["kind"] == "train", [], 0
    for j, rows in enumerate(s["rows"]):
        x = s["x"][at:at + rows]
        if case["kind"] == "quant":
            x = x[:, :-TAIL].view(torch.float8_e4m3fn).double() * x[:, -TAIL:-TAIL + 4].contiguous().view(torch.float32).double()
        leaves = [t.double().requires_grad_(train) for t in (x, s["w_gate"][j], s["w_up"][j], s["w_down"][j])]
        gate = torch.nn.functional.silu(torch.matmul(leaves[0], leaves[1].t()))
        out = torch.matmul(gate * torch.matmul(leaves[0], leaves[2].t()), leaves[3].t())
        got.append((out.detach(),) + (torch.autograd.grad(out, leaves, s["dy"][at:at + rows].double()) if train else ()))
        at += rows
    if not train:
        return {"out": torch.cat([g[0] for g in got])}
    names = ("dw_gate", "dw_up", "dw_down")
    return {"out": torch.cat([g[0] for g in got]), "dx": torch.cat([g[1] for g in got]),
            **{w: torch.stack([g[2 + k] for g in got]) for k, w in enumerate(names)}}


def _exact_adamw(case, seed):
    s = _inputs_adamw(case, seed)
    total, small = case["elements"], case["bits"] == 8
    size = torch.tensor(s["sizes"], device=DEV)
    tensor = torch.repeat_interleave(torch.arange(len(s["sizes"]), device=DEV), size)          # of every element
    inside = torch.arange(total, device=DEV) - (size.cumsum(0) - size)[tensor]                # its place in the tensor
    blocks = torch.div(size + BLOCK - 1, BLOCK, rounding_mode="floor")
    block = (blocks.cumsum(0) - blocks)[tensor] + torch.div(inside, BLOCK, rounding_mode="floor")
    g, p, m, v = (s[k].double() for k in ("grad", "param", "m", "v"))
    if small:
        m, v = m * s["m_scale"].double()[block], (v * s["v_scale"].double()[block]) ** 2
    m = m + (1 - BETA1) * (g - m)
    v = v + (1 - BETA2) * (g ** 2 - v)
    decay = torch.tensor(s["decay"], device=DEV, dtype=torch.float64)[tensor]
    p = (1 - LR * decay) * p - LR * m / (1 - BETA1 ** STEP) / ((v / (1 - BETA2 ** STEP)) ** 0.5 + ADAM_EPS)
    if not small:
        return {"param": p, "copy": p, "m": m, "v": v}
    key = _mix(s["seed"] + (torch.arange(len(s["sizes"]), device=DEV) + 1) * 0x9E3779B9)
    word = _mix(inside + key[tensor])
    got = {"param": p, "copy": p}
    for name, x, u in (("m", m, word % 65536), ("v", v.sqrt(), torch.div(word, 65536, rounding_mode="floor"))):
        scale = torch.zeros(int(blocks.sum()), device=DEV, dtype=torch.float64).scatter_reduce(0, block, x.abs(), "amax") / E4M3_MOST
        a = x.abs() / scale[block].clamp(min=1e-300)
        gap = 2.0 ** (torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
        low = torch.floor(a / gap) * gap
        q = torch.where((a - low) / gap + u.double() / 65536 >= 1, low + gap, low)
        got[name], got[name + "_scale"] = q * torch.sign(x), scale
    return got
