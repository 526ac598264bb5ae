"""The operators where a launch's buffers are one another's, where values leave the range of ordinary ones, and where one plan meets
different contents from launch to launch: against ops_oracle.py's 64 bits, or bit for bit against what has been compared with those."""
import pytest
import torch

import ops_oracle as O
from hccl_amd import hcclx
from hccl_amd import types as T
from test_gpu_operators import DEV, TD, Ffn, Guarded, gen, normal, ptrs

pytestmark = pytest.mark.gpu


# ---- the norm's gradient on top of its inputs -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [T.FP32, T.BFP16])
@pytest.mark.parametrize("n,rows,elems", [(2, 1, 24), (3, 37, 300), (1, 2100, 136), (2, 9, 8200), (1, 6, 16384)])
@pytest.mark.parametrize("on", ["dy", "total", "dtotal"])
def test_norm_gradient_in_place(n, rows, elems, dtype, on):
    g, td = gen(rows), TD[dtype]
    src = {k: [normal((rows, elems), td, g) for _ in range(n)] for k in ("dy", "total", "dtotal")}
    w = [normal((elems,), td, g) for _ in range(n)]
    dx, dw = [torch.empty_like(t) for t in src["dy"]], [torch.empty_like(t) for t in w]

    def launch(to, to_w):
        hcclx.RmsNormGradPlan(ptrs(src["dy"]), ptrs(src["total"]), ptrs(w), ptrs(to), ptrs(to_w), rows, elems, dtype,
                              dtotal=ptrs(src["dtotal"])).launch()
        torch.cuda.synchronize()
    launch(dx, dw)
    for i in range(n):
        wdx, bdx, wdw, bdw = O.norm_grad(src["dy"][i], src["total"][i], w[i], src["dtotal"][i], 1e-6)
        O.assert_close(dx[i], wdx, bdx)
        O.assert_close(dw[i], wdw, bdw)
    launch(src[on], w)
    assert all(torch.equal(a, b) for a, b in zip(src[on] + w, dx + dw))
