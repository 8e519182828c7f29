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
