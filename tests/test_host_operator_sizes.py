"""Sizes that no launch of an operator holds are refused when the plan is made (no GPU: the check comes first)."""
import pytest

from hccl_amd import hcclx
from hccl_amd import types as T
from hccl_amd._lib import HcclError


def norm(rows, elems, dtype):
    """The code that a plan of so many rows ends with; 0: it is made."""
    try:
        hcclx.RmsNormPlan([1 << 40], [1 << 55], [1 << 50], rows, elems, dtype)   # addresses that nothing dereferences
    except HcclError as e:
        return e.code
    return 0


# A workgroup takes four rows of up to 512 16-bit elements, and one of 16384 32-bit elements with 1024 threads.
@pytest.mark.parametrize("elems,dtype,most", [(8, T.BFP16, (1 << 28) - 4), (512, T.FP16, (1 << 28) - 4), (256, T.FP32, (1 << 28) - 4),
                                              (7168, T.BFP16, (1 << 24) - 1), (16384, T.FP32, (1 << 22) - 1)])
def test_norm_refuses_more_rows_than_a_launch_holds(elems, dtype, most):
    assert norm(most, elems, dtype) in (0, T.Result.E_RUNTIME)     # (without a GPU)
    assert norm(most + 1, elems, dtype) == 1 and norm(0xFFFFFFFF, elems, dtype) == 1
