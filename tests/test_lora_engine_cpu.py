"""CPU suite: models with adapters in the module engine and its weight push — who is sent what, and which run's update moves what.  The kernels are plain stand-ins; the
model, the engine and the transports are the shipped code."""

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


def _merge(weight, a, b, scale, out=None):
    return (weight.float() + scale * (b.float().t() @ a.float())).to(BF16)


@pytest.fixture
def plain_ops(monkeypatch):
    """The stand-ins of tests/cpu_standin_ops.py in the place of their namesakes, and a plain merge."""
    import inspect

    from prime_rl_amd import ops
    from tests import cpu_standin_ops as S

    for name, fn in inspect.getmembers(S, inspect.isfunction):
        if not name.startswith("_") and hasattr(ops, name):
            monkeypatch.setattr(ops, name, fn)
    monkeypatch.setattr(ops, "lora_merge", _merge)


def _model(moe=False, seed=3):
    from prime_rl_amd.trainer.models.qwen3 import Qwen3Config, Qwen3ForCausalLM
    from prime_rl_amd.trainer.models.qwen3_moe import Qwen3MoeConfig, Qwen3MoeForCausalLM

    torch.manual_seed(seed)
    sizes = dict(vocab_size=64, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, head_dim=128)
    if moe:
        model = Qwen3MoeForCausalLM(Qwen3MoeConfig(**sizes, num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32, mlp_only_layers=[0], use_grouped_mm=False))
    else:
        model = Qwen3ForCausalLM(Qwen3Config(**sizes))
    for p in model.parameters():
        torch.nn.init.normal_(p, std=0.1)
    return model.to(BF16)


ATTENTION = ("q_proj", "k_proj", "v_proj", "o_proj")


def _with_adapters(n, moe=False):
    from prime_rl_amd.trainer.models.layers.lora import adapter_parameters, attach_lora

    model = _model(moe)
    plain = {k: v.clone() for k, v in model.state_dict().items()}
    state = attach_lora(model, n, 4, [8.0 + g for g in range(n)], targets=ATTENTION)
    for i, p in enumerate(adapter_parameters(model)):
        p.data.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) * 0.3)
    return model, plain, state


def _expected(model, plain, adapter):
    """The plain model's tensors with one adapter folded in, from the definition."""
    want = dict(plain)
    for name, m in model.named_modules():
        if hasattr(m, "lora"):
            a, b = m.lora.a[adapter].to(BF16).double(), m.lora.b[adapter].to(BF16).double()
            want[f"{name}.weight"] = plain[f"{name}.weight"].double() + (8.0 + adapter) / 4 * b.t() @ a
    return want


def _same(got, want, folded):
    assert set(got) == set(want)
    for k, w in want.items():
        if w.dtype == torch.float64:  # a rounding to bf16 of sums of four f32 products
            assert got[k].dtype == BF16 and ((got[k].double() - w).abs() <= 2.0**-8 * w.abs() + 2.0**-20).all(), k
            assert not torch.equal(got[k].double(), folded[k].double())
        else:
            assert torch.equal(got[k], w), k


@pytest.mark.parametrize("moe", [False, True])
def test_a_push_carries_the_run_it_is_for(plain_ops, moe):
    """state_dict and the named push have exactly the names of a model without adapters, and the named run's update in the projections."""
    from prime_rl_amd.trainer.engine import OptimConfig
    from prime_rl_amd.trainer.module_engine import ModuleEngine

    model, plain, _ = _with_adapters(2, moe)
    ref = ModuleEngine(_model(moe), "cpu", optim=OptimConfig(type="sign_sgd"))
    names, plan_names = set(ref.state_dict()), [[m.get("names") or m["experts"] for m in g["messages"]] for g in ref.push_plan(1)]
    engine = ModuleEngine(model, "cpu", optim=OptimConfig(type="sign_sgd"))
    for adapter in (0, 1):
        sd = engine.state_dict(adapter)
        assert set(sd) == names
        want = {k: v for k, v in _expected(model, plain, adapter).items() if k in names}  # what MoE models rename carries no adapter here
        _same({k: v for k, v in sd.items() if k in want}, want, plain)
        plan = engine.push_plan(1)
        assert [[m.get("names") or m["experts"] for m in g["messages"]] for g in plan] == plan_names
        sent = {m["names"][0]: t for g, row in zip(plan, engine.push_tensors(plan, 0, adapter)) for m, t in zip(g["messages"], row) if "names" in m}
        assert all(torch.equal(sent[k], sd[k]) for k in sent) and all(f"model.layers.0.self_attn.{p}.weight" in sent for p in ATTENTION)
    for call in (engine.state_dict, lambda adapter=None: engine.push_tensors(engine.push_plan(1), 0, adapter)):
        with pytest.raises(ValueError, match="2 adapters"):
            call()
        for bad in (-1, 2):
            with pytest.raises(ValueError, match=f"adapter {bad}"):
                call(bad)
    with pytest.raises(ValueError, match="without adapters"):
        ref.state_dict(0)


def test_the_only_adapter_needs_no_name(plain_ops, tmp_path):
    """One run: the transports push its merged weights as they push any model's."""
    from safetensors.torch import load_file

    from prime_rl_amd.trainer.engine import OptimConfig
    from prime_rl_amd.trainer.module_engine import ModuleEngine
    from prime_rl_amd.transports.weights import FileSystemWeightBroadcast

    model, plain, _ = _with_adapters(1)
    want = _expected(model, plain, 0)
    engine = ModuleEngine(model, "cpu", optim=OptimConfig(type="sign_sgd"))
    _same(engine.state_dict(), want, plain)
    FileSystemWeightBroadcast(tmp_path).broadcast_weights(engine, 1)
    _same(load_file(tmp_path / "broadcasts" / "step_1" / "model.safetensors"), want, plain)
    FileSystemWeightBroadcast(tmp_path).broadcast_weights(model, 2)  # the model itself
    _same(load_file(tmp_path / "broadcasts" / "step_2" / "model.safetensors"), want, plain)


def test_transports_push_one_of_several_runs(plain_ops, tmp_path):
    from safetensors.torch import load_file

    from prime_rl_amd.trainer.engine import OptimConfig
    from prime_rl_amd.trainer.module_engine import ModuleEngine
    from prime_rl_amd.transports.weights import FileSystemWeightBroadcast

    model, plain, _ = _with_adapters(3)
    want = _expected(model, plain, 2)
    for step, sender in enumerate((model, ModuleEngine(model, "cpu", optim=OptimConfig(type="sign_sgd")))):
        with pytest.raises(ValueError, match="3 adapters"):
            FileSystemWeightBroadcast(tmp_path).broadcast_weights(sender, step)
        FileSystemWeightBroadcast(tmp_path).broadcast_weights(sender, step, adapter=2)
        _same(load_file(tmp_path / "broadcasts" / f"step_{step}" / "model.safetensors"), want, plain)


def test_a_table_of_another_pass_is_refused():
    """A table that is longer than the pass, or was made for one of another length, raises before any kernel runs."""
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, attach_lora, lora_linear
    from prime_rl_amd.trainer.models.layers.mlp import MLP, MLPConfig

    mlp = MLP(MLPConfig(32, 64)).to(BF16)
    state = attach_lora(mlp, 2, 4, 8.0, targets=("up_proj",))
    x = torch.zeros(10, 32, dtype=BF16)

    def run(rows):
        state.set_rows(rows)
        lora_linear(x, [mlp.up_proj])

    offsets = torch.tensor([0, 3, 9], dtype=torch.int32)
    for stale in (LoRARows.packed([6, 5], "cpu"), LoRARows.packed([6, 0], "cpu", n_rows=8), LoRARows.packed(torch.tensor([2, 9]), "cpu"), LoRARows(offsets, n_rows=12),
                  LoRARows(offsets, torch.arange(9, dtype=torch.int32), n_rows=9)):
        with pytest.raises(ValueError, match="set_rows"):
            run(stale)
    for fits in (LoRARows.packed([6, 4], "cpu"), LoRARows.packed([6, 0], "cpu"), LoRARows.packed([1, 2], "cpu", n_rows=10), LoRARows(offsets), LoRARows(offsets, n_rows=10)):
        with pytest.raises(Exception, match="GPU"):  # what the kernels' entry says of tensors in host memory
            run(fits)
    with pytest.raises(ValueError, match="11 rows of adapters in a pass of 10"):
        LoRARows.packed([6, 5], "cpu", n_rows=10)


def _fwd(x, a, b, scales, offsets, base=None, row_ids=None, out=None):
    ends, z = offsets.tolist(), torch.zeros(x.shape[0], (a.shape[1] + 15) // 16 * 16)
    y = base.float().clone()
    for g in range(a.shape[0]):
        rows = slice(ends[g], ends[g + 1])
        z[rows, :a.shape[1]] = scales[g] * (x[rows].float() @ a[g].float().t())
        y[rows] += z[rows, :a.shape[1]] @ b[g].float()
    out = torch.empty_like(base) if out is None else out
    out.copy_(y)
    return out, z


def _bwd(grad_out, x, z, a, b, scales, offsets, base=None, row_ids=None, grad_x=None, grad_a=None, grad_b=None, accumulate=False, want_x=True, want_factors=True):
    ends, r = offsets.tolist(), a.shape[1]
    da, db = torch.zeros(a.shape), torch.zeros(b.shape)
    dx = base.float().clone() if want_x else None
    for g in range(a.shape[0]):
        rows = slice(ends[g], ends[g + 1])
        dz = scales[g] * (grad_out[rows].float() @ b[g].float().t())
        da[g], db[g] = dz.t() @ x[rows].float(), z[rows, :r].t() @ grad_out[rows].float()
        if want_x:
            dx[rows] += dz @ a[g].float()
    if want_x:
        grad_x.copy_(dx)
    return grad_x, da, db


class _Plan:
    """GradClipPlan's factors by group, from the definition."""

    def __init__(self, grads, groups):
        self.grads, self.groups = grads, groups

    def coefs(self, max_norm):
        squares = torch.zeros(max(self.groups) + 1, dtype=torch.float64)
        for t, g in zip(self.grads, self.groups):
            squares[g] += t.double().square().sum()
        norms = squares.sqrt().float()
        return (max_norm / (norms + 1e-6)).clamp(max=1.0) if max_norm > 0 else torch.ones_like(norms), norms


SEQ = 48


@pytest.fixture
def plain_adapters(plain_ops, monkeypatch):
    from prime_rl_amd import ops

    monkeypatch.setattr(ops, "lora_fwd", _fwd)
    monkeypatch.setattr(ops, "lora_bwd", _bwd)
    monkeypatch.setattr(ops, "GradClipPlan", _Plan)


def _engine(n=2, extra=False, dtype=None, dp=None, **optim):
    from prime_rl_amd.trainer.engine import OptimConfig
    from prime_rl_amd.trainer.models.layers.lm_head import inject_prime_lm_head
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters
    from prime_rl_amd.trainer.module_engine import ModuleEngine

    model, _, state = _with_adapters(n)
    if extra:
        model.model.norm.weight.requires_grad_(True)  # a parameter that all runs share
    for m in model.modules():
        if dtype is not None and isinstance(m, LoRAAdapters):
            m.to(dtype)
    inject_prime_lm_head(model, chunk_size=32)
    return model, state, ModuleEngine(model, "cpu", optim=OptimConfig(**{**dict(lr=2e-3, weight_decay=0.01, max_norm=0.01), **optim}), **(dp or {}))


def _batches(step, n=2):
    from prime_rl_amd.trainer.rl.data import FakeDataLoader, FakeDataLoaderConfig

    dl = FakeDataLoader(FakeDataLoaderConfig(batch_size=n, generate_samples=True), seq_len=SEQ)
    dl.batch_counter = step
    mbs = dl.get_batch()
    g = torch.Generator().manual_seed(step)
    for mb in mbs:
        mb["input_ids"] = mb["input_ids"] % 64
        mb["inference_logprobs"] = -torch.rand(1, SEQ, generator=g) * 0.1 - 4.1
    return mbs


def _pass(engine, state, step, counts, mbs=None):
    """Forward and backward of one pass, before the update."""
    from prime_rl_amd.trainer.engine import pack_micro_batches
    from prime_rl_amd.trainer.models.layers.lora import LoRARows

    b = pack_micro_batches(mbs or _batches(step), "cpu")
    state.set_rows(LoRARows.packed(counts, "cpu", n_rows=b.n_tokens))
    engine.backward(engine.forward_loss(b, engine.global_scales(b.local_counts)))


def _run_values(model, run):
    from prime_rl_amd.trainer.models.layers.lora import adapter_parameters

    return torch.cat([p[run].detach().float().reshape(-1) for p in adapter_parameters(model)])


def _region(engine, run):
    return slice(engine.shared_total + run * engine.run_size, engine.shared_total + (run + 1) * engine.run_size)


@pytest.mark.parametrize("kind", ["adamw", "sgd", "sign_sgd"])
@pytest.mark.parametrize("extra,dtype", [(False, None), (True, None), (False, BF16)])
def test_a_run_does_not_notice_the_others(plain_adapters, kind, extra, dtype):
    """Run 0 after two steps is the same to the bit whether run 1 has ordinary gradients, huge ones, none that are numbers, or no rows."""
    results = []
    for how in ("ordinary", "huge", "nan", "no rows"):
        model, state, engine = _engine(extra=extra, dtype=dtype, type=kind)
        for step in range(2):
            _pass(engine, state, step, [SEQ, 0 if how == "no rows" else SEQ])
            if extra:  # what the runs share follows all of them: held still here
                engine.main_grad[:engine.shared_total].zero_()
            before = _run_values(model, 1).clone()
            assert engine.main_grad[_region(engine, 0)].any()
            if how in ("huge", "nan"):
                engine.main_grad[_region(engine, 1)].mul_(1e6 if how == "huge" else float("nan"))
            engine.optimizer_step()
            assert torch.equal(_run_values(model, 1), before) == (how in ("nan", "no rows"))  # of no numbers: nothing is done with them
        assert not engine.main_grad.any() and engine.run_steps == [2, 0 if how in ("nan", "no rows") else 2]
        results.append((_run_values(model, 0), engine.run_norms[0], engine.master[_region(engine, 0)].clone()))
    for other in results[1:]:
        assert all(torch.equal(u, v) for u, v in zip(results[0], other))


def test_a_run_is_clipped_by_its_own_norm(plain_adapters):
    """Two runs' updates against the definition: each with its own norm, factor, and first step of SGD without momentum."""
    model, state, engine = _engine(type="sgd", momentum=0.0, weight_decay=0.0, lr=0.5, max_norm=1e-3)
    _pass(engine, state, 0, [SEQ, SEQ])
    engine.main_grad[_region(engine, 1)].mul_(100.0)
    grads = [engine.main_grad[_region(engine, g)].double() for g in range(2)]
    before = [engine.master[_region(engine, g)].double() for g in range(2)]
    norm = engine.optimizer_step()
    for g in range(2):
        own = grads[g].norm()
        assert own > 1e-3 and abs(engine.run_norms[g].double() - own) <= 1e-6 * own  # f32 sums of squares
        want = before[g] - 0.5 * grads[g] * (1e-3 / (own + 1e-6))
        assert ((engine.master[_region(engine, g)].double() - want).abs() <= 2.0**-23 * before[g].abs() + 1e-6 * (want - before[g]).abs()).all()
    whole = torch.cat(grads).norm()
    assert abs(norm.double() - whole) <= 1e-6 * whole


def test_a_run_that_rests_goes_on_where_it_was(plain_adapters):
    """Run 1 without rows in the second of three steps: its weights and moments wait, and its third update is the second of a run that never rested."""
    model, state, engine = _engine()
    _pass(engine, state, 0, [SEQ, SEQ])
    engine.optimizer_step()
    held = [t[_region(engine, 1)].clone() for t in (engine.master, engine.exp_avg, engine.exp_avg_sq)]
    own = _run_values(model, 0).clone()
    _pass(engine, state, 1, [SEQ, 0])
    engine.optimizer_step()
    assert all(torch.equal(t[_region(engine, 1)], h) for t, h in zip((engine.master, engine.exp_avg, engine.exp_avg_sq), held)) and engine.run_norms[1] == 0
    assert not torch.equal(_run_values(model, 0), own) and engine.run_steps == [2, 1]
    other_model, other_state, other = _engine()
    _pass(other, other_state, 0, [SEQ, SEQ])
    other.optimizer_step()
    for e, st in ((engine, state), (other, other_state)):
        _pass(e, st, 2, [0, SEQ])
        e.optimizer_step()
    assert torch.equal(_run_values(model, 1), _run_values(other_model, 1)) and other.run_steps == [1, 2]


def test_rows_the_device_knows_alone(plain_adapters):
    """A table whose counts the host was not told: the engine reads them."""
    from prime_rl_amd.trainer.models.layers.lora import LoRARows

    model, state, engine = _engine()
    rows = LoRARows(torch.tensor([0, SEQ, SEQ], dtype=torch.int32))
    from prime_rl_amd.trainer.engine import pack_micro_batches

    held = _run_values(model, 1).clone()
    engine.step(pack_micro_batches(_batches(0), "cpu"), rows=[rows])
    assert engine.run_steps == [1, 0] and torch.equal(_run_values(model, 1), held)


def test_passes_of_a_step_have_a_table_each(plain_adapters):
    """Two passes of different rows against one pass of both; without tables, or with too few, the step is refused."""
    from prime_rl_amd._lib import PrimeMI355XError
    from prime_rl_amd.trainer.engine import pack_micro_batches
    from prime_rl_amd.trainer.models.layers.lora import LoRARows

    mbs = _batches(0)
    model, state, engine = _engine(max_norm=1e9)
    passes = [pack_micro_batches([mb], "cpu") for mb in mbs]
    tables = [LoRARows.packed([SEQ, 0], "cpu"), LoRARows.packed([0, SEQ], "cpu")]
    for rows in (None, tables[:1]):
        with pytest.raises(PrimeMI355XError, match="table"):
            engine.step(passes, rows=rows)
    engine.step(passes, rows=tables)
    norms = engine.run_norms
    model, state, engine = _engine(max_norm=1e9)
    engine.step([pack_micro_batches(mbs, "cpu")], rows=[LoRARows.packed([SEQ, SEQ], "cpu")])
    assert ((engine.run_norms - norms).abs() <= 0.05 * norms).all() and engine.run_steps == [1, 1]  # bf16 activations of products of other sizes
    from prime_rl_amd.trainer.engine import OptimConfig
    from prime_rl_amd.trainer.module_engine import ModuleEngine

    with pytest.raises(PrimeMI355XError, match="with adapters"):
        ModuleEngine(_model(), "cpu", optim=OptimConfig()).step([passes[0]], rows=[tables[0]])


def test_adapters_come_before_the_engine(plain_ops):
    from prime_rl_amd._lib import PrimeMI355XError
    from prime_rl_amd.trainer.engine import OptimConfig, pack_micro_batches
    from prime_rl_amd.trainer.models.layers.lora import attach_lora
    from prime_rl_amd.trainer.module_engine import ModuleEngine

    model = _model()
    engine = ModuleEngine(model, "cpu", optim=OptimConfig())
    attach_lora(model, 2, 4, 8.0)
    with pytest.raises(PrimeMI355XError, match="before the engine"):
        engine.step(pack_micro_batches(_batches(0), "cpu"))


def _two_ranks(rank, world, port, out):
    """Rank r has run r's rows only: the ranks hold the same runs after each step, those of one process with both passes."""
    import os

    import torch.distributed as dist

    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch.set_num_threads(2)
    try:
        from prime_rl_amd import ops
        from tests.test_moe_ep_gloo_cpu import _patch_all_ops

        _patch_all_ops()
        ops.lora_fwd, ops.lora_bwd, ops.GradClipPlan = _fwd, _bwd, _Plan
        from prime_rl_amd.trainer.engine import pack_micro_batches
        from prime_rl_amd.trainer.models.layers.lora import LoRARows

        model, _, engine = _engine(n=3, dp=dict(dp_group=dist.group.WORLD, dp_size=world))
        ref_model, _, ref = _engine(n=3)
        for step in range(2):
            mbs = _batches(step)
            tables = [LoRARows.packed([SEQ if g == r else 0 for g in range(3)], "cpu") for r in range(world)]
            engine.step([pack_micro_batches([mbs[rank]], "cpu")], rows=[tables[rank]])
            ref.step([pack_micro_batches([mb], "cpu") for mb in mbs], rows=tables)
            assert engine.run_steps == [step + 1, step + 1, 0] and ref.run_steps == engine.run_steps
            assert torch.equal(engine.run_norms, ref.run_norms), (step, engine.run_norms, ref.run_norms)
        for g in range(3):
            assert torch.equal(_run_values(model, g), _run_values(ref_model, g)), g
    finally:
        dist.destroy_process_group()


def test_runs_on_other_ranks(tmp_path):
    import torch.multiprocessing as mp

    from tests._ports import free_port

    mp.spawn(_two_ranks, args=(2, free_port(), str(tmp_path)), nprocs=2, join=True)


def test_experts_without_adapters_are_named():
    """A MoE model's experts get none: a warning says so where their projections were asked for, and only there."""
    import warnings

    from prime_rl_amd.trainer.models.layers.lora import adapter_linears, attach_lora

    model = _model(moe=True)
    with pytest.warns(UserWarning, match="layers.1.mlp.experts"):
        attach_lora(model, 2, 4, 8.0)
    assert {k.split(".")[-2] for k in adapter_linears(model)} == {*ATTENTION, "gate_proj", "up_proj", "down_proj"}  # layer 0 is dense
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        attach_lora(_model(moe=True), 2, 4, 8.0, targets=ATTENTION)
        attach_lora(_model(), 2, 4, 8.0)


def test_adapters_of_two_states_are_no_set(plain_ops):
    """Adapters hung on by hand with a state each: whose rows a pass has would be guessed, so engine and push refuse them."""
    from prime_rl_amd.trainer.engine import OptimConfig
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters, LoRAState, merged_state_dict
    from prime_rl_amd.trainer.module_engine import ModuleEngine

    model, _, _ = _with_adapters(2)
    mlp = model.model.layers[0].mlp
    mlp.down_proj.lora = LoRAAdapters(mlp.down_proj, LoRAState(2, 4, 8.0, "cpu"))
    for call in (lambda: ModuleEngine(model, "cpu", optim=OptimConfig()), lambda: merged_state_dict(model, 0)):
        with pytest.raises(ValueError, match="2 different states"):
            call()
