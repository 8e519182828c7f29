"""GPU suite: several runs' adapters in the module engine — updates by run, and the weights that a run's inference engine is sent."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = torch.bfloat16
SEQ = 160


def _model(n):
    from prime_rl_amd.trainer.models.layers.lm_head import inject_prime_lm_head
    from prime_rl_amd.trainer.models.layers.lora import adapter_parameters, attach_lora
    from prime_rl_amd.trainer.models.qwen3 import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(7)
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    model = Qwen3ForCausalLM(cfg).to(DEV).to(BF16)
    inject_prime_lm_head(model, chunk_size=128)
    names = set(model.state_dict())
    state = attach_lora(model, n, 8, 16.0)
    for i, p in enumerate(adapter_parameters(model)):
        p.data.copy_(torch.randn(p.shape, generator=torch.Generator().manual_seed(i)) * 0.05)
    return model, state, names


def _batches(step, n):
    from prime_rl_amd.trainer.rl.data import FakeDataLoader, FakeDataLoaderConfig

    dl = FakeDataLoader(FakeDataLoaderConfig(batch_size=n, generate_samples=True), seq_len=SEQ)
    dl.batch_counter = step
    mbs = dl.get_batch()
    for mb in mbs:
        mb["input_ids"] = mb["input_ids"] % 512
    return mbs


def _region(engine, run):
    return slice(engine.shared_total + run * engine.run_size, engine.shared_total + (run + 1) * engine.run_size)


def _train(how, steps=2):
    from prime_rl_amd.trainer.engine import OptimConfig, pack_micro_batches
    from prime_rl_amd.trainer.models.layers.lora import LoRARows
    from prime_rl_amd.trainer.module_engine import ModuleEngine

    model, state, names = _model(2)
    engine = ModuleEngine(model, DEV, optim=OptimConfig(lr=1e-3, weight_decay=0.01, max_norm=0.1))
    for step in range(steps):
        b = pack_micro_batches(_batches(step, 2), DEV)
        state.set_rows(LoRARows.packed([SEQ, 0 if how == "no rows" else SEQ], DEV, n_rows=b.n_tokens))
        engine.backward(engine.forward_loss(b, engine.global_scales(b.local_counts)))
        assert engine.main_grad[_region(engine, 0)].any()
        if how in ("huge", "nan"):
            engine.main_grad[_region(engine, 1)].mul_(1e6 if how == "huge" else float("nan"))
        grads = [engine.main_grad[_region(engine, g)].double() for g in range(2)]
        norm = engine.optimizer_step()
        for g in range(2):  # f32 of sums in 64 bits
            assert how == "nan" and g == 1 or abs(engine.run_norms[g].double() - grads[g].norm()) <= 2.0**-23 * grads[g].norm()
        if how != "nan":
            whole = torch.cat(grads).norm()
            assert abs(norm.double() - whole) <= 2.0**-22 * whole
    return model, engine, names


def test_a_run_does_not_notice_the_others():
    """Run 0 after two steps is the same to the bit whether run 1 has ordinary gradients, huge ones, none that are numbers, or no rows; in the last two cases run 1 stays."""
    results = []
    for how in ("ordinary", "huge", "nan", "no rows"):
        _, engine, _ = _train(how)
        assert engine.run_steps == [2, 0 if how in ("nan", "no rows") else 2] and not engine.main_grad.any()
        results.append([t[_region(engine, 0)].clone() for t in (engine.master, engine.exp_avg, engine.exp_avg_sq)] + [engine.run_norms[:1]])
        if how in ("nan", "no rows"):
            start = _model(2)[0]
            from prime_rl_amd.trainer.models.layers.lora import adapter_parameters

            assert all(torch.equal(p[1], q[1]) for p, q in zip(adapter_parameters(engine.model), adapter_parameters(start)))
    for other in results[1:]:
        assert all(torch.equal(u, v) for u, v in zip(results[0], other))


def test_a_push_after_a_step_carries_the_run():
    """The names of the model without adapters; each projection's weight with the run's update as it is after the step, in 64 bits from the factors."""
    model, engine, names = _train("ordinary", steps=1)
    plain = model.state_dict()
    for run in range(2):
        sd = engine.state_dict(run)
        assert set(sd) == names
        plan = engine.push_plan(1)
        sent = {m["names"][0]: t for g, row in zip(plan, engine.push_tensors(plan, 0, run)) for m, t in zip(g["messages"], row)}
        assert set(sent) == names and all(torch.equal(sent[k], sd[k]) for k in names)
        folded = 0
        for name, m in model.named_modules():
            if hasattr(m, "lora"):
                a, b = m.lora.a[run].to(BF16).double(), m.lora.b[run].to(BF16).double()
                want = m.weight.double() + 2.0 * (b.t() @ a)
                tol = (2.0**-16 + 24 * 2.0**-24) * 2.0 * (b.abs().t() @ a.abs())
                assert ((sd[f"{name}.weight"].double() - want).abs() <= tol + 2.0**-8 * (want.abs() + tol)).all(), name
                assert not torch.equal(sd[f"{name}.weight"], m.weight)
                folded += 1
        assert folded == 14
        assert all(torch.equal(sd[k], plain[k]) for k in names if "_proj" not in k)
    with pytest.raises(ValueError, match="2 adapters"):
        engine.state_dict()
