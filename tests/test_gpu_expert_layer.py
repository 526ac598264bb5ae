"""The expert layer of hccl_amd/examples/expert_layer.py against the same layer in 64 bits.

Tolerances: a tensor on the way is rounded to bf16, by 2^-9 of each element at most; its error in norm is at most that part, and
at most doubles on its way through a gated product.  So a result that k rounded tensors lie behind may be off by k * 2^-8."""
import pytest
import torch

from hccl_amd import api, hcclx
from hccl_amd.examples import expert_layer as E

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def close(got, want, roundings, what):
    got, want = got.double(), want.detach().double()
    off = float((got - want).norm() / want.norm())
    assert off <= roundings * U, (what, off)


def filled(world, tokens, topk, dim, hidden, training, seed=5):
    g = torch.Generator(device=E.DEV).manual_seed(seed)
    layer = E.ExpertLayer(world, tokens, topk, dim, hidden, training=training)
    for t in layer.stream_in + layer.added:
        t.copy_(torch.randn(t.shape, device=E.DEV, generator=g))
    for w in layer.weights[0]:
        w.copy_(torch.rand(dim, device=E.DEV, generator=g) + 0.5)
    # (an expert that nobody names, and entries that are dropped)
    dest = [torch.randint(-1, world.n - 1, (tokens * topk,), device=E.DEV, generator=g, dtype=torch.int32) for _ in range(world.n)]
    return layer, dest, g


def experts(layer, rows, dest, weights):
    """The sum over every token's experts of their results for `rows`, in the rows' type."""
    out = []
    for x, d in zip(rows, dest):
        y = torch.zeros((x.shape[0], layer.dim), dtype=x.dtype, device=x.device)
        for k in range(layer.topk):
            for e in range(layer.n):
                at = (d.view(-1, layer.topk)[:, k] == e).nonzero().flatten()
                gate, up = x[at] @ weights[1][e].T, x[at] @ weights[2][e].T
                y = y.index_add(0, at, (gate * torch.sigmoid(gate) * up) @ weights[3][e].T)
        out.append(y)
    return out


@pytest.mark.parametrize("n,tokens,topk,dim,hidden", [(4, 40, 2, 128, 72), (8, 33, 1, 264, 136), (3, 300, 3, 72, 200)])
def test_training_step_against_64_bits(n, tokens, topk, dim, hidden):
    world = api.World(n)
    layer, dest, g = filled(world, tokens, topk, dim, hidden, True)
    layer.forward(dest)
    for d in layer.d_result:
        d.copy_(torch.randn(d.shape, device=E.DEV, generator=g))
    layer.backward()
    torch.cuda.synchronize()
    stream = [(a.double() + b.double()).requires_grad_() for a, b in zip(layer.stream_in, layer.added)]
    weights = [[w.double().requires_grad_() for w in kind] for kind in layer.weights]
    normed = [t * w / (t * t).mean(1, keepdim=True).add(1e-6).sqrt() for t, w in zip(stream, weights[0])]
    want = experts(layer, normed, dest, weights)
    sum(((t + y) * d.double()).sum() for t, y, d in zip(stream, want, layer.d_result)).backward()
    for i in range(n):
        close(layer.result[i], want[i], 5, f"result of rank {i}")              # total, normed, h, expert_out, result
        close(layer.d_stream[i], stream[i].grad, 9, f"d_stream of rank {i}")   # total, normed, h, dproj x 2, d_expert_in, d_normed, d_stream
        close(layer.grads[0][i], weights[0][i].grad, 9, f"gradient of the norm's weight of rank {i}")
        for k in (1, 2, 3):
            grad = weights[k][i].grad
            if bool((torch.cat(dest) == i).any()):
                close(layer.grads[k][i], grad, 6, f"gradient {k} of rank {i}") # total, normed, h or dproj, the gradient
            else:
                assert not bool(layer.grads[k][i].any())
    layer.update(lr=0.01)
    torch.cuda.synchronize()
    summed = sum(g.double() for g in layer.grads[0])
    for j in range(n):
        assert torch.equal(layer.weights[0][j], layer.weights[0][0])
        close(layer.norm_grad_sum[j], summed, n, "AllReduce")                  # a rounding per addition
        first = layer.states[j]                                                # m / sqrt(v) of a first step is the gradient's sign
        moved = first["param"].double() - 1.0
        sure = layer.norm_grad_sum[j].double().abs() > 1e-6
        assert torch.allclose(moved[sure], -0.01 * layer.norm_grad_sum[j].double().sign()[sure], rtol=0.02)
        assert torch.equal(first["copy"], first["param"].bfloat16())
    world.close()


def test_training_lowers_the_loss():
    losses = E.main(4, 128, 256, 128, 6)
    assert all(b < a for a, b in zip(losses, losses[1:])), losses


@pytest.mark.parametrize("n,tokens,topk,dim,hidden", [(8, 1, 2, 256, 128), (4, 40, 2, 128, 72), (2, 130, 1, 272, 136)])
def test_serving_with_8_bit_rows(n, tokens, topk, dim, hidden):
    world = api.World(n)
    layer, dest, _ = filled(world, tokens, topk, dim, hidden, False)
    layer.forward(dest)
    torch.cuda.synchronize()
    rows = [r[:, :dim].contiguous().view(torch.float8_e4m3fn).double() * r[:, dim:dim + 4].contiguous().view(torch.float32).double()
            for r in layer.normed]
    for i in range(n):
        total = layer.stream_in[i].double() + layer.added[i].double()
        normed = total * layer.weights[0][i].double() / (total * total).mean(1, keepdim=True).add(1e-6).sqrt()
        assert float((rows[i] - normed).norm() / normed.norm()) <= 2.0 ** -4 + 2 * U   # e4m3: 2^-4 of an element at most
    want = experts(layer, rows, dest, [[w.double() for w in kind] for kind in layer.weights])
    for i in range(n):
        if bool(want[i].any()):
            close(layer.result[i], want[i], 3, f"result of rank {i}")          # h, expert_out, result
        else:
            assert not bool(layer.result[i].any())
    world.close()
