"""The operators' Python calls without a GPU: what a call hands to the library is that call's own."""
from hccl_amd import hcclx


def test_adamw_steps_of_one_plan_do_not_share_their_arguments():
    """Another thread steps the plan while the library looks at the first one's arguments."""
    plan = hcclx.AdamWPlan.__new__(hcclx.AdamWPlan)
    plan._h, seen = None, []

    def step(handle, args, stream):
        if not seen:
            seen.append(None)
            plan.step(2, lr=0.5, beta1=0.25, beta2=0.125, eps=0.0, seed=9, grad_scale=64, stream=7)
            seen.pop(0)
        a = args._obj
        seen.append((a.step, a.lr, a.beta1, a.beta2, a.eps, a.seed, a.grad_scale, stream))
        return 0
    plan._step = step
    plan.step(1, lr=1.0, seed=-1, stream=3)
    assert seen == [(2, 0.5, 0.25, 0.125, 0.0, 9, 64, 7), (1, 1.0, 0.9, 0.999, 1e-8, 0xFFFFFFFF, None, 3)]
