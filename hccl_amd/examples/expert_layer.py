"""A layer of experts, one per virtual rank, trained and served with the operators next to the collectives.

    python -m hccl_amd.examples.expert_layer [ranks] [tokens per rank] [dim] [hidden] [steps]

Every rank has tokens of the residual stream and one expert.  Forward: add and norm, dispatch of every token to the experts that
`dest` names, the experts' feed-forward block on the rows that arrived, the way back with the sum over a token's experts.  The
loss is half the squared distance of stream + result from a target.  Backward: the transposed ways (the gradient of a combine is
a dispatch and the other way round) around the block's and the norm's gradients.  Step: the norm's weight is the same in every
rank, so its gradient is summed over the ranks by an AllReduce and its AdamW states are floats, with which every rank takes the
same step; the experts' weights are each rank's own, with states of 8 bits.  Either step leaves the bf16 weights that the next
forward pass reads.  A layer that only serves (training=False) sends its rows to the experts in 8 bits."""
import contextlib
import math
import sys

import torch

from hccl_amd import api, hcclx, types as T
from hccl_amd._lib import check

DEV = "cuda:0"


def ptrs(ts):
    return [t.data_ptr() for t in ts]


class Routes:
    """Where the entries (topk for each token) of every rank go, for rows of row_elems elements."""

    def __init__(self, n, entries, row_elems):
        self.entries, self.row_elems = entries, row_elems
        self.send_counts, self.sdispls, self.recv_counts, self.rdispls = (torch.zeros(n * n, dtype=torch.int64, device=DEV) for _ in range(4))
        self.perm = [torch.empty(entries, dtype=torch.int32, device=DEV) for _ in range(n)]
        self.workspace = torch.empty(hcclx.moe_workspace_bytes(n, entries), dtype=torch.uint8, device=DEV)

    def find(self, dest, stream):
        self.dest = ptrs(dest)
        hcclx.moe_route(self.dest, self.entries, self.row_elems, self.send_counts.data_ptr(), self.sdispls.data_ptr(),
                        self.recv_counts.data_ptr(), self.rdispls.data_ptr(), ptrs(self.perm), self.workspace.data_ptr(), stream)

    def there(self, tokens, topk, dtype, recv, stream):
        hcclx.moe_dispatch(ptrs(tokens), self.dest, ptrs(self.perm), self.entries, topk, self.row_elems, dtype, self.sdispls.data_ptr(),
                           self.rdispls.data_ptr(), ptrs(recv), stream)

    def back(self, expert, tokens, topk, out, stream):
        hcclx.moe_gather_combine(ptrs(expert), self.dest, ptrs(self.perm), tokens, topk, self.row_elems, T.BFP16, self.sdispls.data_ptr(),
                                 self.rdispls.data_ptr(), ptrs(out), stream)


class ExpertLayer:
    def __init__(self, world, tokens, topk, dim, hidden, seed=0, training=True):
        n = world.n
        g = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g) / math.sqrt(shape[-1])
        rows = lambda: [torch.empty((tokens, dim), dtype=torch.bfloat16, device=DEV) for _ in range(n)]
        self.stream = torch.cuda.Stream()                          # (the collectives take no default stream)
        self.world, self.n, self.tokens, self.topk, self.dim, self.steps = world, n, tokens, topk, dim, 0
        self.capacity = n * tokens * topk                          # of an expert: every entry of every rank
        arrived = lambda width, dtype: [torch.empty((self.capacity, width), dtype=dtype, device=DEV) for _ in range(n)]
        master = [[torch.ones(dim, device=DEV) for _ in range(n)], [rand(hidden, dim) for _ in range(n)], [rand(hidden, dim) for _ in range(n)],
                  [rand(dim, hidden) for _ in range(n)]]
        self.weights = [[w.bfloat16() for w in kind] for kind in master]
        norm, *experts = (ptrs(kind) for kind in self.weights)
        self.stream_in, self.added, self.total, self.result = rows(), rows(), rows(), rows()
        self.expert_out = arrived(dim, torch.bfloat16)
        if training:
            self.routes = self.way_back = Routes(n, tokens * topk, dim)
            self.normed, self.expert_in = rows(), arrived(dim, torch.bfloat16)
        else:                                                      # rows of 8 bits: codes, and the scale behind them
            wide = dim + hcclx.ROW8_TAIL
            self.routes, self.way_back = Routes(n, tokens * topk, wide), Routes(n, tokens * topk, dim)
            self.normed = [torch.empty((tokens, wide), dtype=torch.uint8, device=DEV) for _ in range(n)]
            self.expert_in = arrived(wide, torch.uint8)
        self.row_dtype = T.BFP16 if training else T.FP8E4M3
        self.norm = hcclx.RmsNormPlan(ptrs(self.stream_in), norm, ptrs(self.normed), tokens, dim, T.BFP16, residual=ptrs(self.added),
                                      total=ptrs(self.total), out_dtype=self.row_dtype)
        shape = dict(capacity=self.capacity, dim=dim, hidden=hidden, dtype=T.BFP16, rows=self.capacity,
                     counts=self.routes.recv_counts.data_ptr(), counts_per_rank=n, count_unit=self.routes.row_elems)
        if not training:
            self.block = hcclx.GatedFfnPlan(ptrs(self.expert_in), *experts, ptrs(self.expert_out), x_dtype=T.FP8E4M3, **shape)
            return
        self.saved = torch.empty(hcclx.gated_ffn_saved_bytes(self.capacity, hidden), dtype=torch.uint8, device=DEV)
        self.block = hcclx.GatedFfnPlan(ptrs(self.expert_in), *experts, ptrs(self.expert_out), saved=self.saved.data_ptr(), **shape)
        self.d_result, self.d_normed, self.d_stream = rows(), rows(), rows()
        self.d_expert_out, self.d_expert_in = arrived(dim, torch.bfloat16), arrived(dim, torch.bfloat16)
        self.grads = [[torch.empty_like(w) for w in kind] for kind in self.weights]
        self.norm_grad_sum = [torch.empty_like(w) for w in self.grads[0]]
        self.block_grad = hcclx.GatedFfnGradPlan(ptrs(self.d_expert_out), ptrs(self.expert_in), *experts, self.saved.data_ptr(),
                                                 ptrs(self.d_expert_in), *(ptrs(kind) for kind in self.grads[1:]), **shape)
        self.norm_grad = hcclx.RmsNormGradPlan(ptrs(self.d_normed), ptrs(self.total), norm, ptrs(self.d_stream), ptrs(self.grads[0]), tokens,
                                               dim, T.BFP16, dtotal=ptrs(self.d_result))
        self.states, self.adamw = [], []
        for kinds, grads, small in ((master[:1], [self.norm_grad_sum], False), (master[1:], self.grads[1:], True)):
            tensors = []
            for kind, w, grad in ((k, w, g) for k, (ws, gs) in enumerate(zip(kinds, grads)) for w, g in zip(ws, gs)):
                count = w.numel()
                blocks = -(-count // hcclx.ADAMW_BLOCK)
                copies = self.weights[kind + 1 if small else 0]
                t = dict(param=w, grad=grad, copy=copies[len(tensors) % n])
                for name in ("m", "v"):
                    t[name] = torch.zeros(count, dtype=torch.uint8 if small else torch.float32, device=DEV)
                    if small:
                        t[name + "_scale"] = torch.zeros(blocks, device=DEV)
                self.states.append(t)
                tensors.append(dict(count=count, weight_decay=0.01 if small else 0.0, **{name: x.data_ptr() for name, x in t.items()}))
            self.adamw.append(hcclx.AdamWPlan(tensors, T.BFP16, T.FP8E4M3 if small else T.FP32, copy_dtype=T.BFP16))

    @contextlib.contextmanager
    def _launching(self):
        """The layer's stream, behind the caller's work and with the caller's next work behind it."""
        self.stream.wait_stream(torch.cuda.current_stream())
        yield self.stream.cuda_stream
        torch.cuda.current_stream().wait_stream(self.stream)

    def forward(self, dest):
        """result = the experts' outputs for stream_in + added, which total holds.  dest[i]: the expert of every entry of rank i."""
        with self._launching() as stream:
            self.routes.find(dest, stream)
            if self.way_back is not self.routes:
                self.way_back.find(dest, stream)
            self.norm.launch(stream)
            self.routes.there(self.normed, self.topk, self.row_dtype, self.expert_in, stream)
            self.block.launch(stream)
            self.way_back.back(self.expert_out, self.tokens, self.topk, self.result, stream)

    def backward(self):
        """From d_result, which reaches the result and, past the layer, total: d_stream and the weights' gradients."""
        with self._launching() as stream:
            self.routes.there(self.d_result, self.topk, T.BFP16, self.d_expert_out, stream)
            self.block_grad.launch(stream)
            self.way_back.back(self.d_expert_in, self.tokens, self.topk, self.d_normed, stream)
            self.norm_grad.launch(stream)

    def update(self, lr):
        self.steps += 1
        with self._launching() as stream:
            for rank in range(self.n):
                check(self.world.all_reduce(rank, self.grads[0][rank].data_ptr(), self.norm_grad_sum[rank].data_ptr(), self.dim, T.BFP16,
                                            T.SUM, stream))
            for plan in self.adamw:
                plan.step(self.steps, lr, seed=self.steps, stream=stream)


def main(n=8, tokens=512, dim=1024, hidden=512, steps=8):
    world = api.World(n)
    g = torch.Generator(device=DEV).manual_seed(1)
    layer = ExpertLayer(world, tokens, 2, dim, hidden)
    for t in layer.stream_in + layer.added:
        t.copy_(torch.randn(t.shape, device=DEV, generator=g))
    target = [torch.randn(t.shape, device=DEV, generator=g) + t for t in layer.stream_in]
    dest = [torch.randint(0, n, (tokens * 2,), device=DEV, generator=g, dtype=torch.int32) for _ in range(n)]
    losses = []
    for _ in range(steps):
        layer.forward(dest)
        off = [total.float() + result.float() - want for total, result, want in zip(layer.total, layer.result, target)]
        losses.append(float(sum((o * o).sum() for o in off)) / (2 * n * tokens * dim))
        for d, o in zip(layer.d_result, off):
            d.copy_(o / (n * tokens))
        layer.backward()
        layer.update(lr=1e-3)
    torch.cuda.synchronize()
    world.close()
    print("loss " + " ".join(f"{x:.4f}" for x in losses))
    return losses


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:]))
