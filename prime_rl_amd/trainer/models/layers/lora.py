"""Low-rank adapters of many runs on the dense projections — the LoRA linears of the reference's multi-run trainer (src/prime_rl/trainer/models/layers/lora) on the
adapter kernels (csrc/lora.hip).

One frozen model serves every run: run g's rows of a pass (the micro-batch's `lora_num_tokens`, trainer/rl/data.py) get `scale[g] * (x A_g^T) B_g` added to the
shared projection's output.  `attach_lora(model, ...)` hangs a `LoRAAdapters` on the chosen `nn.Linear`s as their submodule `lora` (the linear keeps its name and
weight) and freezes everything else; the layer seams (layers/attn.py, layers/mlp.py) then run `lora_linear` in the place of `linear` / `fused_linear`: the products of
layers/linear.py with every adapter's update added in place to its columns, and one autograd node for all of it.

Factors are rank-major, `a [n, rank, in]` and `b [n, rank, out]` (a checkpoint's `lora_B [out, rank]` is `b[g].T`).  Parameters are f32 (the products take them as
bf16): adapters are small, and their gradients arrive in f32 without a rounding."""

from __future__ import annotations

import math
import warnings
from collections.abc import Iterable, Sequence

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from .... import ops
from .linear import _adjacent_view


class LoRARows:
    """Which rows of a pass belong to which adapter: `offsets` i32 [n + 1], adapter g owns positions [offsets[g], offsets[g + 1]); `row_ids` i32 [rows] or None
    (position p is row p).  `n_rows`: the rows of the pass that the table is for, and `counts`: each adapter's rows, where the host knows them; a pass of another
    length is refused by what is known (the kernels clamp a table that does not fit, which would leave rows to the wrong run)."""

    def __init__(self, offsets: Tensor, row_ids: Tensor | None = None, n_rows: int | None = None, counts: list[int] | None = None):
        self.offsets, self.row_ids, self.n_rows, self.counts = offsets, row_ids, n_rows, counts
        self._owned = None if counts is None else sum(counts)
        if n_rows is not None and counts is not None and self._owned > n_rows:
            raise ValueError(f"num_tokens: {self._owned} rows of adapters in a pass of {n_rows}")

    @classmethod
    def packed(cls, num_tokens: Sequence[int] | Tensor, device, n_rows: int | None = None) -> LoRARows:
        """Runs packed one behind the other, `num_tokens[g]` rows of run g (`lora_num_tokens`); rows behind the last run belong to none.  `n_rows`: the rows of the
        pass; without it, and with `num_tokens` on the device, nothing tells a table that was left from another pass."""
        counts = torch.as_tensor(num_tokens, dtype=torch.int32).reshape(-1)
        if not counts.is_cuda and counts.numel() and int(counts.min()) < 0:
            raise ValueError(f"num_tokens: expected no negative counts, got {counts.tolist()}")
        offsets = torch.zeros(counts.numel() + 1, dtype=torch.int32, device=counts.device)
        offsets[1:] = counts.cumsum(0)
        return cls(offsets.to(device), n_rows=n_rows, counts=None if counts.is_cuda else counts.tolist())

    @classmethod
    def of(cls, adapter_ids: Tensor, n_adapters: int) -> LoRARows:
        """Rows in any order, `adapter_ids[row]` their adapter (outside [0, n_adapters): none)."""
        return cls(*ops.lora_rows(adapter_ids, n_adapters), n_rows=adapter_ids.numel())

    def rows_of_adapters(self) -> list[int]:
        """Each adapter's rows; waits for the device where only it knows them."""
        if self.counts is None:
            ends = self.offsets.tolist()
            self.counts = [b - a for a, b in zip(ends, ends[1:])]
        return self.counts

    def check(self, n_rows: int) -> None:
        """Raises where the table is known not to be that of a pass of `n_rows` rows."""
        if self.n_rows is not None and self.n_rows != n_rows:
            raise ValueError(f"the rows' table is for a pass of {self.n_rows} rows, this one has {n_rows}: LoRAState.set_rows comes before each pass")
        if self._owned is not None and self._owned > n_rows:
            raise ValueError(f"the rows' table holds {self._owned} rows of adapters, this pass has {n_rows}: LoRAState.set_rows comes before each pass")


class LoRAState:
    """What all adapters of a model share: their number, rank and scales, and the rows of the pass that is to run."""

    def __init__(self, n_adapters: int, rank: int, alpha: float | Sequence[float], device):
        alphas = list(alpha) if isinstance(alpha, Iterable) else [alpha] * n_adapters
        if n_adapters < 1 or rank < 1 or len(alphas) != n_adapters:
            raise ValueError(f"expected one alpha for each of {n_adapters} adapters of rank {rank}, got {len(alphas)}")
        self.n_adapters, self.rank = n_adapters, rank
        self.scales = torch.tensor([x / rank for x in alphas], dtype=torch.float32, device=device)
        self.rows: LoRARows | None = None

    def set_rows(self, rows: LoRARows) -> None:
        """The rows of the passes that follow, until the next call; where layers are recomputed in the backward, the next call comes after it."""
        if rows.offsets.numel() != self.n_adapters + 1:
            raise ValueError(f"rows of {rows.offsets.numel() - 1} adapters for a model of {self.n_adapters}")
        self.rows = rows

    def scales_on(self, device) -> Tensor:
        """The scales beside the rows of a pass: a model may have moved since it got its adapters."""
        if self.scales.device != device:
            self.scales = self.scales.to(device)
        return self.scales


class LoRAAdapters(nn.Module):
    """The adapters of one projection; `a` starts uniform (as nn.Linear's weight does), `b` at zero: the update starts at zero."""

    def __init__(self, linear: nn.Linear, state: LoRAState):
        super().__init__()
        self.state = state
        device = linear.weight.device
        self.a = nn.Parameter(torch.empty(state.n_adapters, state.rank, linear.in_features, dtype=torch.float32, device=device))
        self.b = nn.Parameter(torch.zeros(state.n_adapters, state.rank, linear.out_features, dtype=torch.float32, device=device))
        nn.init.uniform_(self.a, -1.0 / math.sqrt(linear.in_features), 1.0 / math.sqrt(linear.in_features))


def adapters_of(linears: Sequence[nn.Linear]) -> list[LoRAAdapters | None] | None:
    """The adapters of each projection, None where none of them has any."""
    found = [getattr(lin, "lora", None) for lin in linears]
    return found if any(f is not None for f in found) else None


def _product(x: Tensor, w: Tensor, bias: Tensor | None, out: Tensor) -> None:
    """out = x @ w.T (+ bias) on the core where it takes the shapes."""
    if ops.gemm_supported(x, w, out=out):
        ops.gemm(x, w, out=out, bias=bias)
    else:
        out.copy_(F.linear(x, w, bias))


class _LoRALinearFn(torch.autograd.Function):
    """cat([x @ w_i.T + bias_i + update_i]) over several projections of the same rows; the updates go into the output's columns in place."""

    @staticmethod
    def forward(ctx, x, rows, scales, has_adapter, weights, biases, *factors):
        n, widths = x.shape[0], [w.shape[0] for w in weights]
        y = torch.empty((n, sum(widths)), dtype=x.dtype, device=x.device)
        joined = _adjacent_view(weights)
        if joined is not None and all(b is None for b in biases):
            _product(x, joined, None, y)
        else:
            for w, b, part in zip(weights, biases, y.split(widths, dim=1)):
                _product(x, w, b, part)
        halves = [f.detach().to(torch.bfloat16).contiguous() for f in factors]  # (a trainer engine keeps each run's share in a stretch of its own)
        zs, at = [], 0
        for i, part in enumerate(y.split(widths, dim=1)):
            if has_adapter[i]:
                zs.append(ops.lora_fwd(x, halves[at], halves[at + 1], scales, rows.offsets, base=part, row_ids=rows.row_ids, out=part)[1])
                at += 2
        # the rows' tables and the weights too: changed in place before the backward, they raise there
        ctx.save_for_backward(x, scales, rows.offsets, rows.row_ids, *weights, *halves, *zs)
        ctx.has_adapter, ctx.widths = has_adapter, widths
        ctx.dtypes = [f.dtype for f in factors]
        return y

    @staticmethod
    def backward(ctx, dy):
        x, scales, offsets, row_ids, *rest = ctx.saved_tensors
        n_factors, n_weights = len(ctx.dtypes), len(ctx.widths)
        weights, halves, zs = rest[:n_weights], rest[n_weights:n_weights + n_factors], rest[n_weights + n_factors:]
        joined = _adjacent_view(weights)
        # rows that overlap (a gradient that is one row for all, say) or begin at odd places are written out
        dy = dy if dy.stride(1) == 1 and dy.stride(0) >= dy.shape[1] and dy.stride(0) % 8 == 0 and dy.data_ptr() % 16 == 0 else dy.clone(memory_format=torch.contiguous_format)
        want_x, want_factors = ctx.needs_input_grad[0], any(ctx.needs_input_grad[6:])
        dx, parts = None, dy.split(ctx.widths, dim=1)
        if want_x:
            pairs = [(dy, joined)] if joined is not None else list(zip(parts, weights))
            for d, w in pairs:
                step = ops.gemm(d, w.t()) if ops.gemm_supported(d, w.t()) else d @ w
                dx = step if dx is None else dx.add_(step)
        grads: list[Tensor] = []
        for i, d in enumerate(parts):
            if not ctx.has_adapter[i]:
                continue
            k = len(grads)
            _, da, db = ops.lora_bwd(d, x, zs[k // 2], halves[k], halves[k + 1], scales, offsets, base=dx, row_ids=row_ids, grad_x=dx, want_x=want_x,
                                     want_factors=want_factors)
            grads += [da, db]
        if not want_factors:
            return dx, None, None, None, None, None, *([None] * n_factors)
        return dx, None, None, None, None, None, *(g.to(t) for g, t in zip(grads, ctx.dtypes))


def lora_linear(x: Tensor, linears: Sequence[nn.Linear], adapters: Sequence[LoRAAdapters | None] | None = None) -> Tensor:
    """cat([linear_i(x)], dim=-1) with the projections' adapters for x [N, in] bf16 rows of the pass that `LoRAState.set_rows` described.  The shared weights are
    frozen: gradients go to x and the adapters.  In a captured graph only without gradients: accumulating into leaves that an earlier eager pass holds too would wait for that
    pass' stream, which ends the process (a captured training step calls `ops.lora_fwd` and `ops.lora_bwd` on buffers of its own)."""
    adapters = adapters if adapters is not None else adapters_of(linears)
    if adapters is None:
        raise ValueError("none of the projections has adapters")
    if any(p is not None and p.requires_grad for lin in linears for p in (lin.weight, lin.bias)):
        raise ValueError("the projections beside adapters are frozen: requires_grad_(False) their weight and bias (attach_lora does)")
    state = next(a.state for a in adapters if a is not None)
    if any(a is not None and a.state is not state for a in adapters):
        raise ValueError("the projections' adapters belong to different states")
    if state.rows is None:
        raise ValueError("LoRAState.set_rows says which rows of the pass belong to which adapter: call it before the model")
    if torch.is_grad_enabled() and x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise ValueError("a captured pass through adapters runs under torch.no_grad()")
    state.rows.check(x.shape[0])
    x = x if x.is_contiguous() and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)
    factors = [f for a in adapters if a is not None for f in (a.a, a.b)]
    return _LoRALinearFn.apply(x, state.rows, state.scales_on(x.device), [a is not None for a in adapters], [lin.weight.detach() for lin in linears],
                               [None if lin.bias is None else lin.bias.detach() for lin in linears], *factors)


TARGETS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def attach_lora(model: nn.Module, n_adapters: int, rank: int, alpha: float | Sequence[float], targets: Sequence[str] = TARGETS) -> LoRAState:
    """Hangs adapters on every projection of the attention and dense MLP seams that `targets` names, freezes all other parameters, and returns the state whose
    `set_rows` describes each pass.  A model has one set of adapters: it is attached once.  Experts of MoE layers, routed and shared, get none (a warning says so where
    `targets` names their projections)."""
    from .attn import HipVarlenAttention
    from .mlp import MLP
    from .moe import BCFeedForward, GroupedExperts

    unknown = set(targets) - set(TARGETS)
    if unknown:
        raise ValueError(f"targets: expected names among {TARGETS}, got {sorted(unknown)}")
    if any(isinstance(m, LoRAAdapters) for m in model.modules()):
        raise ValueError("the model has adapters already")
    experts = [name for name, m in model.named_modules() if isinstance(m, (GroupedExperts, BCFeedForward))]
    if experts and set(targets) & {"gate_proj", "up_proj", "down_proj"}:
        warnings.warn(f"attach_lora: {len(experts)} expert modules ({experts[0]}, ...) are frozen without adapters: only attention and dense MLP projections have them", stacklevel=2)
    device = next(model.parameters()).device
    state = LoRAState(n_adapters, rank, alpha, device)
    linears = [lin for m in model.modules() if isinstance(m, (HipVarlenAttention, MLP)) for name, lin in m.named_children() if name in targets]
    if not linears:
        raise ValueError(f"the model has none of the projections {tuple(targets)}")
    for p in model.parameters():
        p.requires_grad_(False)
    for lin in linears:
        lin.lora = LoRAAdapters(lin, state)
    return state


def adapter_parameters(model: nn.Module) -> list[nn.Parameter]:
    """All adapters' factors, in the model's order; run g's share of a factor p (and of its gradient) is p[g]."""
    return [p for m in model.modules() if isinstance(m, LoRAAdapters) for p in (m.a, m.b)]


def adapter_state(model: nn.Module) -> LoRAState | None:
    """The state that the model's adapters share; None for a model without."""
    states = {id(m.state): m.state for m in model.modules() if isinstance(m, LoRAAdapters)}
    if len(states) > 1:
        raise ValueError(f"the model's adapters belong to {len(states)} different states")
    return next(iter(states.values()), None)


def pushed_adapter(model: nn.Module, adapter: int | None) -> int | None:
    """Which adapter a push of `model` folds in: None for a model without adapters, the only one of a model with one, else the one that is named — the inference
    engines know neither a frozen weight without its run's update nor the factors' names."""
    state = adapter_state(model)
    if state is None:
        if adapter is not None:
            raise ValueError(f"adapter {adapter} of a model without adapters")
        return None
    if adapter is None and state.n_adapters > 1:
        raise ValueError(f"the model has {state.n_adapters} adapters: name the one whose run the weights are for (adapter=...)")
    adapter = 0 if adapter is None else adapter
    if not 0 <= adapter < state.n_adapters:
        raise ValueError(f"adapter {adapter} of a model with {state.n_adapters}")
    return adapter


def adapter_linears(model: nn.Module) -> dict[str, nn.Linear]:
    """The projections with adapters, by the names of their weights in the model's state dict."""
    return {f"{name}.weight": m for name, m in model.named_modules(remove_duplicate=False) if isinstance(getattr(m, "lora", None), LoRAAdapters)}


@torch.no_grad()
def merged_weight(linear: nn.Linear, adapter: int) -> Tensor:
    """The projection's weight with one run's adapter folded in (`ops.lora_merge`)."""
    lora = linear.lora
    return ops.lora_merge(linear.weight.detach(), lora.a[adapter].to(torch.bfloat16), lora.b[adapter].to(torch.bfloat16), float(lora.state.scales[adapter]))


@torch.no_grad()
def merged_state_dict(model: nn.Module, adapter: int) -> dict[str, Tensor]:
    """The model's state dict as a model without adapters has it, with one run's adapter folded into the projections (`ops.lora_merge`): what the weight push
    sends to that run's inference engine."""
    adapter = pushed_adapter(model, adapter)
    sd = {k: v.detach() for k, v in model.state_dict().items() if ".lora." not in k}
    sd.update({k: merged_weight(m, adapter) for k, m in adapter_linears(model).items()})
    return sd
