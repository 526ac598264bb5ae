"""The operators of include/hcclx_ops.h from their definitions in 64 bits, with bounds on what 32-bit arithmetic and one rounding
to the outputs' type may differ by, element by element."""
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}    # relative error of a rounding
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # absolute, of subnormal results
E = 2.0 ** -24


def norm(total, weight, eps):
    """y, and its bound: the mean square's sum is a chain of at most 32 elements per thread, six steps in a wavefront and 16
    wavefronts, half of whose relative error reaches y; a handful of roundings more."""
    t, w = total.double(), weight.double()
    y = t / (t.square().mean(-1, keepdim=True) + eps).sqrt() * w
    return y, 40 * E * y.abs()


def norm_grad(dy, total, weight, dtotal, eps):
    """dx, dw and their bounds (total's rows along the first axis)."""
    t, w, d = total.double(), weight.double(), dy.double()
    r = 1 / (t.square().mean(-1, keepdim=True) + eps).sqrt()
    a = d * w
    c = (a * t).mean(-1, keepdim=True)
    dx = r * (a - t * r * r * c)
    big = r * (a.abs() + t.abs() * r * r * (a * t).abs().mean(-1, keepdim=True))
    if dtotal is not None:
        dx, big = dx + dtotal.double(), big + dtotal.double().abs()
    each = d * t * r
    return dx, 100 * E * big, each.sum(0), (60 + t.shape[0]) * E * each.abs().sum(0)


def act(a, kind):
    """act, its derivative; kind 0: silu, 1: gelu (tanh form)."""
    if kind == 0:
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    k = (2 / torch.pi) ** 0.5
    t = torch.tanh(k * (a + 0.044715 * a ** 3))
    return 0.5 * a * (1 + t), 0.5 * (1 + t) + 0.5 * a * (1 - t * t) * k * (1 + 3 * 0.044715 * a * a)


def ffn(x, wg, wu, wd, kind, dtype, dy=None):
    """out and, with dy, (dx, dwg, dwu, dwd), each with its bound (without the last rounding).  x as the values it stands for.

    A product's 32-bit sum of K terms is off by at most K E of the sum of their magnitudes; a rounded operand by u of itself;
    |act'| < 1.2, |act''| < 1; exp and the division are good for 2^-20 together."""
    u, least = U[dtype], LEAST[dtype]
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    rows, dim, hidden = x.shape[0], x.shape[1], wg.shape[0]
    g, up = x @ wg.T, x @ wu.T
    eg, eu = (dim + 4) * E * (x.abs() @ wg.abs().T), (dim + 4) * E * (x.abs() @ wu.abs().T)
    f, slope = act(g, kind)
    h = f * up
    eh = 1.2 * eg * up.abs() + f.abs() * eu + 1.2 * eg * eu + 2.0 ** -20 * h.abs()
    eh = eh + u * (h.abs() + eh) + least
    out = h @ wd.T
    got = [(out, eh @ wd.abs().T + (hidden + 4) * E * ((h.abs() + eh) @ wd.abs().T))]
    if dy is None:
        return got
    dy = dy.double()
    dh = dy @ wd
    edh = (dim + 4) * E * (dy.abs() @ wd.abs())
    dg, du = dh * up * slope, dh * f
    edg = edh * up.abs() * 1.2 + (dh.abs() + edh) * (1.2 * eu + (up.abs() + eu) * eg + 2.0 ** -19 * up.abs())
    edg = edg + u * (dg.abs() + edg) + least
    edu = edh * f.abs() + (dh.abs() + edh) * (1.2 * eg + 2.0 ** -20 * f.abs())
    edu = edu + u * (du.abs() + edu) + least
    k = (2 * hidden + 8) * E
    got.append((dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + k * ((dg.abs() + edg) @ wg.abs() + (du.abs() + edu) @ wu.abs())))
    k = (rows + 4) * E
    got.append((dg.T @ x, edg.T @ x.abs() + k * ((dg.abs() + edg).T @ x.abs())))
    got.append((du.T @ x, edu.T @ x.abs() + k * ((du.abs() + edu).T @ x.abs())))
    got.append((dy.T @ h, dy.abs().T @ eh + k * (dy.abs().T @ (h.abs() + eh))))
    return got


def assert_close(got, want, bound, what=""):
    """|got - want| <= bound + the rounding to got's type."""
    u, least = U[got.dtype], LEAST[got.dtype]
    g = got.double()
    limit = bound + u * (want.abs() + bound) + least
    off = (g - want).abs()
    bad = ~(off <= limit)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound, the worst by "
                                 f"{float((off / limit)[bad].max()):.3g} times, first at {bad.nonzero()[0].tolist()}: "
                                 f"got {float(g[bad][0])!r} want {float(want[bad][0])!r} +- {float(limit[bad][0])!r}")


def mix(x):
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def draws(seed, tensor, count):
    """The random numbers of a tensor's elements, for m and for sqrt(v), in [0, 1)."""
    w = mix(torch.arange(count, dtype=torch.int64) + int(mix(torch.tensor(seed + (tensor + 1) * 0x9E3779B9))))
    return (w & 0xFFFF).double() / 65536, (w >> 16).double() / 65536


def e4m3_gap(a):
    """Distance of the e4m3 values around a magnitude: its power of two / 8, by the exponent's bits (pow is not exact on a GPU)."""
    power = a.clamp(min=2.0 ** -6).contiguous().view(torch.int64) >> 52
    return ((power - 3) << 52).view(torch.float64)


def adamw(g, p, m, v, step, lr, beta1, beta2, eps, decay):
    g, p, m, v = (t.double() for t in (g, p, m, v))
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    update = (m / (1 - beta1 ** step)) / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return p - lr * (decay * p + update), m, v, update
