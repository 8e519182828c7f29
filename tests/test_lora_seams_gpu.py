"""GPU suite: adapters on the layer seams and models, and a run of the adapter operators together as a multi-run trainer uses them."""

import math

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E8, E24 = 2.0**-8, 2.0**-24


def _linears(widths, d_in, bias, adjacent, seed):
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(sum(widths) * d_in, generator=g) * d_in**-0.5).to(BF16).to(DEV)
    out, at = [], 0
    for w in widths:
        lin = nn.Linear(d_in, w, bias=bias, device=DEV, dtype=BF16)
        piece = flat[at:at + w * d_in].view(w, d_in)
        lin.weight.data = piece if adjacent else piece.clone()
        at += w * d_in
        for p in lin.parameters():
            p.requires_grad_(False)
        out.append(lin)
    return out


@pytest.mark.parametrize("n,d_in,widths,has,bias,adjacent,mixed", [
    (300, 256, (256, 128, 128), (1, 1, 1), False, True, False),
    (257, 256, (256, 128, 128), (1, 0, 1), True, False, True),
    (64, 512, (128,), (1,), False, False, True),
    (5, 136, (72, 24), (0, 1), False, False, False),  # sizes that the core does not take
])
def test_lora_linear_matches_the_formula_and_its_gradients(n, d_in, widths, has, bias, adjacent, mixed):
    """Tolerances: a bf16 rounding (2^-8 of the value) of the shared product and of each update's sum, and f32 sums; the adapters' gradients are f32 of the rounded dy."""
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters, LoRARows, LoRAState, lora_linear

    g = torch.Generator().manual_seed(4)
    state = LoRAState(3, 8, [8, 16, 12], DEV)
    lins = _linears(widths, d_in, bias, adjacent, 1)
    for lin, h in zip(lins, has):
        if h:
            lin.lora = LoRAAdapters(lin, state)
            lin.lora.b.data.normal_(0, 0.3)
    if mixed:
        ids = torch.randint(-1, 3, (n,), generator=g).to(torch.int32).to(DEV)
        state.set_rows(LoRARows.of(ids, 3))
    else:
        counts = [n // 3, 0, n - n // 3 - 2]
        state.set_rows(LoRARows.packed(counts, DEV))
        ids = torch.tensor([0] * counts[0] + [2] * counts[2] + [-1] * 2, device=DEV)
    x = torch.randn(n, d_in, generator=g).to(BF16).to(DEV).requires_grad_(True)
    y = lora_linear(x, lins)
    dy = torch.randn(y.shape, generator=g).to(BF16).to(DEV)
    y.backward(dy)
    xd, at = x.detach().double(), 0
    dx, dx_tol = torch.zeros(n, d_in, dtype=F64, device=DEV), torch.zeros(n, d_in, dtype=F64, device=DEV)
    for lin, h in zip(lins, has):
        w, part, d = lin.weight.double(), y[:, at:at + lin.out_features].double(), dy[:, at:at + lin.out_features].double()
        at += lin.out_features
        base = xd @ w.t() + (lin.bias.double() if bias else 0.0)
        want = base.clone()
        tol = E8 * base.abs() + 2 * d_in * E24 * (xd.abs() @ w.abs().t())
        step = d @ w
        dx += step
        dx_tol += E8 * step.abs() + 2 * lin.out_features * E24 * (d.abs() @ w.abs())
        for k in range(3 if h else 0):
            rows = ids == k
            a, b, s = lin.lora.a[k].to(BF16).double(), lin.lora.b[k].to(BF16).double(), state.scales[k].double()
            z, za = s * xd[rows] @ a.t(), s * xd[rows].abs() @ a.abs().t()
            dz, dza = s * d[rows] @ b.t(), s * d[rows].abs() @ b.abs().t()
            want[rows] += z @ b
            tol[rows] += (2.0**-16 + 2 * (d_in + 12) * E24) * (za @ b.abs())
            dx[rows] += dz @ a
            dx_tol[rows] += E8 * (dz @ a).abs() + (2.0**-16 + 2 * (lin.out_features + 12) * E24) * (dza @ a.abs())
            for got, ref, mag, terms in ((lin.lora.a.grad[k], dz.t() @ xd[rows], dza.t() @ xd[rows].abs(), lin.out_features), (lin.lora.b.grad[k], z.t() @ d[rows], za.t() @ d[rows].abs(), d_in)):
                assert ((got.double() - ref).abs() <= 2 * (terms + n + 40) * E24 * mag).all()
        assert ((part - want).abs() <= tol + E8 * (want.abs() + tol)).all()
    # every product and update of dx is rounded as it is added: the roundings are of partial sums, at most the sum of the parts' magnitudes each
    roundings = len(lins) + sum(has)
    parts = sum((dy[:, sum(widths[:i]):sum(widths[:i + 1])].double() @ lin.weight.double()).abs() for i, lin in enumerate(lins)) + dx.abs()
    assert ((x.grad.double() - dx).abs() <= dx_tol + roundings * E8 * (parts + dx_tol)).all()


def _one_linear():
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters, LoRARows, LoRAState, lora_linear

    state = LoRAState(2, 8, 16.0, DEV)
    (lin,) = _linears((128,), 256, False, False, 3)
    lin.lora = LoRAAdapters(lin, state)
    lin.lora.b.data.normal_(0, 0.3)
    state.set_rows(LoRARows.packed([40, 30], DEV))
    x = torch.randn(72, 256, device=DEV).to(BF16).requires_grad_(True)
    return lin, state, x, lambda: lora_linear(x, [lin])


def test_a_gradient_that_is_one_row_for_all():
    """The gradient of a sum over rows arrives with a row stride of zero: the same results as from rows of their own."""
    lin, _, x, run = _one_linear()
    v = torch.randn(128, device=DEV).to(BF16)
    leaves = (x, lin.lora.a, lin.lora.b)
    got = torch.autograd.grad(run(), leaves, v.expand(72, 128))
    want = torch.autograd.grad(run(), leaves, v.expand(72, 128).contiguous())
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("what", ["offsets", "weight", "scales"])
def test_a_backward_of_tables_or_weights_changed_since_raises(what):
    lin, state, _, run = _one_linear()
    y = run()
    {"offsets": state.rows.offsets, "weight": lin.weight, "scales": state.scales}[what].mul_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_captured_passes_are_without_gradients():
    """Replays follow what the buffers hold; a captured pass with gradients is refused."""
    _, _, x, run = _one_linear()
    with torch.no_grad():
        run()
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="no_grad"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        run()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        held = run()
    for turn in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(72, 256, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held, run()), turn


def test_gradients_against_differences():
    """d(sum y * dy) / d factor against differences of the whole seam in the factor, in the directions of the gradients themselves."""
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters, LoRARows, LoRAState, lora_linear

    g = torch.Generator().manual_seed(9)
    state = LoRAState(2, 16, 16.0, DEV)
    (lin,) = _linears((256,), 256, False, False, 3)
    lin.weight.data.zero_()  # the shared product is not what is tested: its rounding would hide the differences
    lin.lora = LoRAAdapters(lin, state)
    lin.lora.b.data.copy_(torch.randn(2, 16, 256, generator=g).to(BF16))
    lin.lora.a.data.copy_(torch.randn(2, 16, 256, generator=g).to(BF16))
    state.set_rows(LoRARows.packed([200, 100], DEV))
    x = torch.randn(300, 256, generator=g).to(BF16).to(DEV)
    dy = torch.randn(300, 256, generator=g).to(BF16).to(DEV)
    lora_linear(x, [lin]).backward(dy)
    for p in (lin.lora.a, lin.lora.b):
        way = p.grad.sign()
        slope = (p.grad.double() * way.double()).sum().item()
        start = p.data.clone()
        values = []
        for side in (1.0, -1.0):
            p.data = start + side * 2.0**-3 * way  # the update is linear in each factor: the step may be long, so that roundings stay small beside it
            values.append((lora_linear(x, [lin]).detach().double() * dy.double()).sum().item())
            moved = (p.data.to(BF16).double() - start.double()).abs().mean().item()
            assert 0.9 * 2.0**-3 < moved < 1.1 * 2.0**-3
        p.data = start
        assert abs((values[0] - values[1]) / 2.0**-2 - slope) <= 0.03 * slope


def _tiny(seed=7, chunk=None):
    from prime_rl_amd.trainer.models.layers.lm_head import inject_prime_lm_head
    from prime_rl_amd.trainer.models.qwen3 import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(seed)
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    model = Qwen3ForCausalLM(cfg).to(DEV).to(BF16)
    inject_prime_lm_head(model, chunk_size=chunk)  # None: logits
    return model


def _logits(model, ids, lens):
    out = model(input_ids=ids, seq_lens=torch.tensor(lens, device=DEV))
    return out["logits"].float()


def test_model_with_adapters_that_add_nothing_is_the_model():
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, attach_lora

    model = _tiny()
    ids = torch.randint(0, 512, (1, 200), device=DEV)
    with torch.no_grad():
        before = _logits(model, ids, [120, 80])
        state = attach_lora(model, 3, 8, 16.0)
        state.set_rows(LoRARows.packed([120, 0, 80], DEV))
        assert torch.equal(_logits(model, ids, [120, 80]), before)  # b = 0
        for m in model.modules():
            if hasattr(m, "lora"):
                m.lora.b.data.normal_(0, 0.1)
        state.set_rows(LoRARows.packed([0, 0, 0], DEV))
        assert torch.equal(_logits(model, ids, [120, 80]), before)  # no rows
        state.set_rows(LoRARows.packed([120, 0, 0], DEV))
        after = _logits(model, ids, [120, 80])
        assert torch.equal(after[:, 120:], before[:, 120:]) and not torch.equal(after[:, :120], before[:, :120])  # the other document's rows do not notice


def test_merged_state_dict_is_the_model_with_its_adapter():
    """The merged model against adapters beside the weights: both round every activation to bf16 (2^-8 each) along the 2 x 7 projections, so they may differ by
    2 x 14 x 2^-8 of the logits at most."""
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, attach_lora, merged_state_dict

    model, plain = _tiny(), _tiny(seed=8)
    names = set(model.state_dict())
    state = attach_lora(model, 2, 8, [16.0, 4.0])
    for m in model.modules():
        if hasattr(m, "lora"):
            m.lora.b.data.normal_(0, 0.1)
    ids = torch.randint(0, 512, (1, 100), device=DEV)
    with torch.no_grad():
        for adapter in (0, 1):
            counts = [0, 0]
            counts[adapter] = 100
            state.set_rows(LoRARows.packed(counts, DEV))
            with_adapter = _logits(model, ids, [100])
            sd = merged_state_dict(model, adapter)
            assert set(sd) == names
            plain.load_state_dict(sd)
            merged = _logits(plain, ids, [100])
            state.set_rows(LoRARows.packed([0, 0], DEV))
            base = _logits(model, ids, [100])
            assert (merged - with_adapter).norm() <= 28 * E8 * with_adapter.norm()
            assert (with_adapter - base).norm() > 3 * (merged - with_adapter).norm()  # what the adapter does is well above that


def test_a_training_step_of_two_runs():
    """Forward and backward of two runs' adapters in one pass, each run's gradients clipped into its flat buffer, one AdamW launch for each run, the result merged:
    against the same step written out in 64 bits from the gradients that autograd left."""
    from prime_rl_amd import ops
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, adapter_parameters, attach_lora, merged_state_dict

    model = _tiny(chunk=128)
    state = attach_lora(model, 3, 8, [16.0, 8.0, 16.0])
    params = adapter_parameters(model)
    for i, p in enumerate(params):
        p.data.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) * 0.05)
    frozen = {k: v.clone() for k, v in model.state_dict().items() if ".lora." not in k}
    state.set_rows(LoRARows.packed([90, 0, 60], DEV))
    ids = torch.randint(0, 512, (1, 150), device=DEV)
    out = model(input_ids=ids, seq_lens=torch.tensor([90, 60], device=DEV), labels=ids.roll(-1, 1), temperature=torch.ones(1, 150, device=DEV))
    out["logprobs"].sum().backward()
    assert all(p.grad is not None and p.grad.dtype == F32 for p in params)
    assert all(not p.grad[1].any() for p in params) and any(p.grad[0].any() for p in params) and any(p.grad[2].any() for p in params)
    n = 3
    size = sum(p[0].numel() for p in params)
    flat, master = torch.zeros(n, size, device=DEV), torch.cat([p.data.reshape(n, -1) for p in params], dim=1).contiguous()
    start = master.clone()
    m, v = torch.zeros_like(flat), torch.zeros_like(flat)
    grads = [p.grad[g] for g in range(n) for p in params]
    outs = [o for g in range(n) for o in flat[g].split([p[0].numel() for p in params])]
    plan = ops.GradClipPlan(grads, [g for g in range(n) for _ in params], out=outs)
    limits = torch.tensor([0.5, 0.5, 1e9], device=DEV)
    norms = plan.clip(limits)
    for g in range(n):
        whole = torch.cat([p.grad[g].reshape(-1) for p in params]).double()
        norm = whole.norm().item()
        assert abs(norms[g].item() - norm) <= 4 * E24 * norm
        want = whole * min(1.0, limits[g].item() / (norm + 1e-6))
        assert ((flat[g].double() - want).abs() <= 16 * E24 * want.abs()).all()
        ops.adamw_step(master[g], m[g], v[g], flat[g], None, lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
        moved = torch.where(want == 0, 0.0, 1e-2 * want / (want.abs() + 1e-8))  # a first step of AdamW: bias-corrected moments are g and g^2
        assert ((start[g].double() - master[g].double() - moved).abs() <= 1e-5 * 1e-2 + 4 * E24 * start[g].double().abs()).all()
    assert torch.equal(master[1], start[1])  # a run without rows
    for p, new in zip(params, master.split([p[0].numel() for p in params], dim=1)):
        p.data.copy_(new.reshape(p.shape))
    sd = merged_state_dict(model, 2)
    for name, mod in model.named_modules():
        if hasattr(mod, "lora"):
            delta = state.scales[2].double() * (mod.lora.b[2].to(BF16).double().t() @ mod.lora.a[2].to(BF16).double())
            want = frozen[f"{name}.weight"].double() + delta
            assert ((sd[f"{name}.weight"].double() - want).abs() <= E8 * want.abs() + 2.0**-15 * delta.abs().max()).all()
    assert all(torch.equal(v, model.state_dict()[k]) for k, v in frozen.items())


def test_module_engine_trains_adapters_only():
    from prime_rl_amd.trainer.engine import OptimConfig, pack_micro_batches
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, adapter_parameters, attach_lora
    from prime_rl_amd.trainer.module_engine import ModuleEngine
    from prime_rl_amd.trainer.rl.data import FakeDataLoader, FakeDataLoaderConfig

    model = _tiny(chunk=128)
    state = attach_lora(model, 2, 8, 16.0)
    for p in adapter_parameters(model):
        p.data.normal_(0, 0.05)
    engine = ModuleEngine(model, DEV, optim=OptimConfig(lr=1e-3, weight_decay=0.0, max_norm=1.0))
    frozen = {k: v.clone() for k, v in model.state_dict().items() if ".lora." not in k}
    before = [p.detach().clone() for p in adapter_parameters(model)]
    mbs = FakeDataLoader(FakeDataLoaderConfig(batch_size=2, generate_samples=True), seq_len=160).get_batch()
    for mb in mbs:
        mb["input_ids"] = mb["input_ids"] % 512
    state.set_rows(LoRARows.packed([int(mb["lora_num_tokens"]) for mb in mbs], DEV))  # one run for each micro-batch
    out = engine.step(pack_micro_batches(mbs, DEV))
    assert math.isfinite(out["loss"][0].item()) and out["grad_norm"].item() > 0
    for p, b in zip(adapter_parameters(model), before):
        for g in range(2):
            assert not torch.equal(p[g], b[g])
    assert all(torch.equal(v, model.state_dict()[k]) for k, v in frozen.items())
