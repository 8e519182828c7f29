"""GPU suite: what a projection with adapters takes that one without takes too."""

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16 = torch.bfloat16


def _linear(d_in=256, d_out=128, device=DEV):
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters, LoRAState

    torch.manual_seed(5)
    lin = nn.Linear(d_in, d_out, bias=False).to(device).to(BF16).requires_grad_(False)
    state = LoRAState(2, 8, [16.0, 4.0], device)
    lin.lora = LoRAAdapters(lin, state)
    lin.lora.b.data.copy_(torch.randn(2, 8, d_out, generator=torch.Generator().manual_seed(6)))
    return lin, state


def test_a_model_that_moved_with_its_adapters():
    """Adapters made in host memory and moved with their projection: the results of ones made in place."""
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, lora_linear

    x = torch.randn(50, 256, device=DEV).to(BF16)
    outs = []
    for device in (DEV, "cpu"):
        lin, state = _linear(device=device)
        if device == "cpu":
            lin.lora.a.data.copy_(outs[0][1])
            lin.weight.data.copy_(outs[0][2])
        lin = lin.to(DEV)
        state.set_rows(LoRARows.packed([20, 28], DEV))
        outs.append((lora_linear(x, [lin]).detach(), lin.lora.a.detach().cpu(), lin.weight.cpu()))
        assert state.scales.device == x.device and state.scales.tolist() == [2.0, 0.5]
    assert torch.equal(outs[0][0], outs[1][0])


@pytest.mark.parametrize("rows", [1, 40])
def test_rows_and_gradients_that_begin_anywhere(rows):
    """Views that begin off a 16-byte boundary: the results of aligned copies."""
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, lora_linear

    lin, state = _linear()
    state.set_rows(LoRARows.packed([rows - 1, 1], DEV))
    x = torch.randn(rows, 256, device=DEV).to(BF16)
    dy = torch.randn(rows, 128, device=DEV).to(BF16)

    def odd(t):
        flat = torch.zeros(t.numel() + 3, dtype=BF16, device=DEV)
        flat[3:] = t.reshape(-1)
        return flat[3:].view(t.shape)

    results = []
    for at in (lambda t: t, odd):
        leaf = at(x).detach().requires_grad_(True)
        y = lora_linear(leaf, [lin])
        results.append((y.detach(), *torch.autograd.grad(y, (leaf, lin.lora.a, lin.lora.b), at(dy))))
    assert all(torch.equal(u, v) for u, v in zip(*results))
