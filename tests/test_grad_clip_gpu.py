"""GPU suite: gradient norms of many tensors by group and clipping (pm_grad_clip) against 64-bit sums.

The norm is a 64-bit sum rounded once to f32 (2^-24 of it); the factor is one f32 division and the product one f32 (2^-24 each) or bf16 (2^-8) rounding."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def ops():
    from prime_rl_amd import ops as _ops

    return _ops


def _grads(sizes, kinds, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * std).to(kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


def _check(grads, groups, n_groups, max_norm, norms, outs):
    for g in range(n_groups):
        limit = max_norm[g] if isinstance(max_norm, (list, tuple)) else max_norm
        want = math.sqrt(sum(t.double().square().sum().item() for t, k in zip(grads, groups) if k == g))
        got = norms[g].item()
        assert abs(got - want) <= 2 * 2.0**-24 * want, (g, got, want)
        coef = min(1.0, limit / (want + 1e-6)) if limit > 0 else 1.0
        for t, o, k in zip(grads, outs, groups):
            if k == g:
                ref = t.double() * coef
                half = 2.0**-8 if o.dtype == BF16 else 2.0**-24
                assert ((o.double().reshape(-1) - ref.reshape(-1)).abs() <= ref.abs().reshape(-1) * (8 * 2.0**-24 + 2 * half)).all()


SIZES = [1, 2, 3, 7, 8, 9, 1023, 2048, 2049, 4097, 32768, 100003]


@pytest.mark.parametrize("kinds", [(F32,), (BF16,), (F32, BF16)])
@pytest.mark.parametrize("max_norm", [0.7, 1e9, 0.0])
def test_norms_and_clipping_in_place(ops, kinds, max_norm):
    grads = _grads(SIZES, kinds)
    groups = [i % 3 for i in range(len(grads))]
    before = [t.clone() for t in grads]
    norms = ops.GradClipPlan(grads, groups).clip(max_norm)
    _check(before, groups, 3, max_norm, norms, grads)
    if max_norm != 0.7:
        assert all(torch.equal(u, v) for u, v in zip(before, grads))


@pytest.mark.parametrize("src,dst", [(F32, F32), (BF16, F32), (F32, BF16), (BF16, BF16)])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_clipping_into_a_flat_buffer_at_any_offset(ops, src, dst, shift):
    """Outputs (and inputs) that start anywhere in a buffer, each group with its own limit; the gaps between them stay."""
    sizes = [5, 1000, 33, 0, 40961, 16]
    flat_in = torch.randn(sum(sizes) + 64, device=DEV).to(src)
    grads, outs, at = [], [], shift
    flat = torch.full((sum(sizes) + 64,), 7.0, device=DEV).to(dst)
    written = torch.zeros(flat.numel(), dtype=torch.bool, device=DEV)
    for n in sizes:
        grads.append(flat_in[at:at + n])
        outs.append(flat[at:at + n])
        written[at:at + n] = True
        at += n + 3
    groups = [0, 1, 1, 0, 2, 2]
    limits = torch.tensor([0.5, 1e6, 3.0], device=DEV)
    before = flat_in.clone()
    norms = ops.GradClipPlan(grads, groups, out=outs).clip(limits)
    _check(grads, groups, 3, limits.tolist(), norms, outs)
    assert torch.equal(flat_in, before) and (flat[~written] == 7.0).all()


def test_groups_without_gradients_and_unsorted_groups(ops):
    grads = _grads([100, 200, 300, 50], (F32,))
    groups = [4, 1, 4, 0]
    before = [t.clone() for t in grads]
    norms = ops.GradClipPlan(grads, groups, n_groups=6).clip(1.0)
    _check(before, groups, 6, 1.0, norms, grads)
    assert norms[2].item() == norms[3].item() == norms[5].item() == 0.0


def test_many_tensors_and_a_long_one(ops):
    grads = _grads([(i * 37) % 3000 + 1 for i in range(3000)] + [20_000_001], (F32, BF16), std=1e-3)
    groups = [i % 7 for i in range(3000)] + [3]
    before = [t.clone() for t in grads]
    norms = ops.GradClipPlan(grads, groups).clip(1e-2)
    _check(before, groups, 7, 1e-2, norms, grads)


@pytest.mark.parametrize("value", [1e30, 1e-30])
def test_squares_beyond_32_bits(ops, value):
    """Gradients whose squares overflow or vanish in 32 bits have a norm all the same."""
    t = torch.full((1000,), value, device=DEV)
    norm = ops.GradClipPlan([t], out=[torch.empty_like(t)]).clip(1.0)
    want = t[0].double().item() * math.sqrt(1000)
    assert abs(norm.item() - want) <= 2 * 2.0**-24 * want


def test_infinite_and_nan_gradients_follow_clip_grad_norm(ops):
    """An infinite norm makes the factor 0 (infinite elements become NaN, the others 0); a NaN norm makes all NaN; other groups do not notice."""
    a, b, c = (torch.ones(100, device=DEV) for _ in range(3))
    a[3], b[5] = float("inf"), float("nan")
    outs = [torch.empty_like(a) for _ in range(3)]
    norms = ops.GradClipPlan([a, b, c], [0, 1, 2], out=outs).clip(2.0)
    assert torch.isinf(norms[0]) and torch.isnan(norms[1]) and abs(norms[2].item() - 10.0) < 1e-5
    assert torch.isnan(outs[0][3]) and outs[0].nan_to_num(0.0).abs().sum().item() == 0.0
    assert torch.isnan(outs[1]).all()
    torch.testing.assert_close(outs[2], torch.full_like(c, 0.2), rtol=1e-6, atol=0)


def test_sums_of_several_ranks(ops):
    """sumsq() of the parts, added as an all-reduce would, gives the whole's norm; coefs() is what adamw_step takes."""
    whole = _grads([5000, 777], (F32,))
    parts = [[t[: t.numel() // 2].clone() for t in whole], [t[t.numel() // 2:].clone() for t in whole]]
    plans = [ops.GradClipPlan(p, [0, 1]) for p in parts]
    total = plans[0].sumsq() + plans[1].sumsq()
    assert total.dtype == F64
    coefs, norms = plans[0].coefs(1.0, sumsq=total)
    before = [t.clone() for t in parts[1]]
    got = plans[1].clip(1.0, sumsq=total)
    assert torch.equal(got, norms)
    for i, t in enumerate(whole):
        want = t.double().norm().item()
        assert abs(norms[i].item() - want) <= 2 * 2.0**-24 * want
        assert abs(coefs[i].item() - min(1.0, 1.0 / (want + 1e-6))) <= 4 * 2.0**-24
        assert torch.equal(parts[1][i], before[i] * coefs[i])


def test_the_same_bits_every_time_and_in_a_graph(ops):
    grads = _grads([(i * 911) % 70000 + 1 for i in range(60)], (F32, BF16))
    out = [torch.empty(t.numel(), device=DEV) for t in grads]
    plan = ops.GradClipPlan(grads, [i % 2 for i in range(60)], out=out)
    plan.clip(0.3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = plan.clip(0.3)
    for turn in range(3):
        for t in grads:
            t.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        norms, outs = held.clone(), [t.clone() for t in out]
        again = plan.clip(0.3)
        assert torch.equal(norms, again) and all(torch.equal(u, v) for u, v in zip(outs, out)), turn


def test_plans_refuse_what_they_cannot_hold(ops):
    from prime_rl_amd._lib import PrimeMI355XError as E

    t = torch.zeros(100, device=DEV)
    for args in (([t, t], None), ([t, t[50:]], None), ([t], [1], 1), ([t], [-1]), ([t], [0, 0]), ([], None), ([t.half()], None), ([t.double()], None), ([t.view(10, 10).t()], None),
                 ([t], None, None, [t[:50]]), ([t], None, None, []), ([t[:50]], None, None, [t[25:75]]), ([torch.zeros(4)], None)):
        with pytest.raises(E):
            ops.GradClipPlan(*args)
    with pytest.raises(E):
        ops.GradClipPlan([t]).clip(torch.ones(2, device=DEV))
    with pytest.raises(E):
        ops.GradClipPlan([t]).clip(torch.ones(1))
    with pytest.raises(E):
        ops.GradClipPlan([t]).clip(1.0, sumsq=torch.ones(1, device=DEV))


def test_a_plan_that_goes_while_another_stream_runs_it(ops):
    """Its tables' memory, of the stream that made it, is not given to other tensors before the stream that runs the plan has read them."""
    t = torch.full((1 << 20,), 2.0, device=DEV)
    busy, side = torch.randn(4096, 4096, device=DEV), torch.cuda.Stream()
    plan = ops.GradClipPlan([t])
    sizes = [u.numel() for u in (plan._table, plan._pieces)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            busy @ busy
        plan.clip(1024.0)
    del plan
    for _ in range(8):  # the same sizes from the same stream's memory
        others = [torch.zeros(n, dtype=torch.int64, device=DEV) for n in sizes]
    torch.cuda.synchronize()
    assert ((t - 1.0).abs() <= 8 * 2.0**-24).all(), others  # a norm of 2048
