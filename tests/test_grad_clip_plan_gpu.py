"""GPU suite: a clipping plan beside gradients that stay, and beside ones that move."""

import time

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _leaves():
    g = torch.Generator().manual_seed(1)
    return [torch.randn(3, n, generator=g).to(DEV).requires_grad_(True) for n in (40, 7, 4096)]


def _backward(leaves, scale):
    sum((scale * p * p).sum() for p in leaves).backward()


def test_a_plan_knows_gradients_that_moved():
    """Gradients that stay in place are clipped step after step; ones that autograd made anew are refused by `check`, as are others than the plan's."""
    from prime_rl_amd import ops
    from prime_rl_amd._lib import PrimeMI355XError

    leaves = _leaves()
    now = lambda: [p.grad[g] if p.grad is not None else None for p in leaves for g in range(3)]  # noqa: E731
    _backward(leaves, 1.0)
    plan = ops.GradClipPlan(now(), groups=[g for _ in leaves for g in range(3)])
    for step in range(3):
        plan.check(now())
        whole = [torch.cat([p.grad[g] for p in leaves]).double() for g in range(3)]
        norms = plan.clip(0.5)
        for g in range(3):
            norm = whole[g].norm()
            assert abs(norms[g].double() - norm) <= 2.0**-23 * norm
            want = whole[g] * (0.5 / (norm + 1e-6))
            got = torch.cat([p.grad[g] for p in leaves]).double()
            assert ((got - want).abs() <= 2.0**-21 * want.abs()).all()  # norm, sum, quotient and product: a rounding of 2^-24 each, and what they carry on
        for p in leaves:
            p.grad.zero_()
        _backward(leaves, step + 2.0)
    held = [p.grad for p in leaves]
    for p in leaves:
        p.grad = None
    with pytest.raises(PrimeMI355XError, match="none"):
        plan.check(now())
    _backward(leaves, 1.0)
    with pytest.raises(PrimeMI355XError, match="not where the plan has it"):
        plan.check(now())
    with pytest.raises(PrimeMI355XError, match="9 gradients"):
        plan.check(now()[:-1])
    with pytest.raises(PrimeMI355XError, match=r"grads\[0\]"):
        plan.check(now()[::-1])
    for p, t in zip(leaves, held):
        p.grad = t
    plan.check(now())
    with pytest.raises(PrimeMI355XError, match="not where the plan has it"):
        plan.check([t.view(torch.int32) for t in now()])


def test_building_and_checking_a_plan_of_many_tensors():
    """What the host spends on a plan of the size of a model's adapters, printed beside a bound that only a blunder passes."""
    from prime_rl_amd import ops

    flat = torch.zeros(2016 * 64, device=DEV)
    grads = list(flat.split(64))
    t0 = time.perf_counter()
    plan = ops.GradClipPlan(grads, groups=[i % 4 for i in range(2016)])
    t1 = time.perf_counter()
    plan.check(grads)
    t2 = time.perf_counter()
    print(f"2016 tensors: plan {1e3 * (t1 - t0):.1f} ms, check {1e3 * (t2 - t1):.2f} ms")
    assert t1 - t0 < 2.0 and t2 - t1 < 0.5
