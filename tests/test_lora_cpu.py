"""CPU suite: what the adapter entry points refuse before any device work, and the host side of the adapters."""

import ctypes

import pytest
import torch
from torch import nn

from prime_rl_amd import _lib

P = ctypes.c_void_p(4096)  # never followed: every call here returns before a launch


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        _lib.build()
    return _lib.load()


def _fwd(lib, **kw):
    a = dict(x=P, ldx=64, a=P, b=P, scales=P, offsets=P, row_ids=None, n=10, k=2, d_in=64, d_out=128, rank=8, base=P, ldb=128, out=P, ldo=128, z=P, ws=P, wsb=1 << 30)
    a.update(kw)
    return lib.pm_lora_fwd(a["x"], a["ldx"], a["a"], a["b"], a["scales"], a["offsets"], a["row_ids"], a["n"], a["k"], a["d_in"], a["d_out"], a["rank"], a["base"], a["ldb"], a["out"],
                           a["ldo"], a["z"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(rank=0), -2), (dict(rank=129), -2), (dict(d_in=60), -2), (dict(d_in=0), -2), (dict(d_out=12), -2), (dict(d_out=1 << 23), -2), (dict(n=-1), -1), (dict(n=1 << 31), -1),
    (dict(k=0), -1), (dict(k=70000), -1), (dict(x=None), -1), (dict(a=None), -1), (dict(b=None), -1), (dict(scales=None), -1), (dict(offsets=None), -1), (dict(out=None), -1),
    (dict(z=None), -1), (dict(ldx=56), -1), (dict(ldx=68), -1), (dict(ldo=120), -1), (dict(ldb=130), -1), (dict(x=ctypes.c_void_p(4098)), -1), (dict(out=ctypes.c_void_p(4104)), -1),
    (dict(a=ctypes.c_void_p(4100)), -1), (dict(ldb=256), -1), (dict(n=4, d_in=8192, ldx=8192, wsb=16), -4), (dict(n=4, d_in=8192, ldx=8192, ws=None), -4),
])
def test_forward_refuses(lib, kw, code):
    assert _fwd(lib, **kw) == code and lib.pm_last_error()


def test_no_rows_is_no_work(lib):
    assert _fwd(lib, n=0, x=None, a=None) == 0


def _bwd(lib, **kw):
    a = dict(dy=P, ldg=128, x=P, ldx=64, z=P, a=P, b=P, scales=P, offsets=P, row_ids=None, n=10, k=2, d_in=64, d_out=128, rank=8, base=P, ldb=64, dx=P, ldgx=64, da=P, db=P, acc=0, ws=P,
             wsb=1 << 30)
    a.update(kw)
    return lib.pm_lora_bwd(a["dy"], a["ldg"], a["x"], a["ldx"], a["z"], a["a"], a["b"], a["scales"], a["offsets"], a["row_ids"], a["n"], a["k"], a["d_in"], a["d_out"], a["rank"],
                           a["base"], a["ldb"], a["dx"], a["ldgx"], a["da"], a["db"], a["acc"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(rank=0), -2), (dict(rank=200), -2), (dict(d_in=4), -2), (dict(n=-3), -1), (dict(dy=None), -1), (dict(x=None), -1), (dict(z=None), -1), (dict(da=None), -1), (dict(db=None), -1),
    (dict(offsets=None), -1), (dict(scales=None), -1), (dict(ldg=64), -1), (dict(ldgx=32), -1), (dict(da=ctypes.c_void_p(4100)), -1), (dict(ws=None), -4), (dict(wsb=64), -4),
    (dict(ldb=128), -1),
])
def test_backward_refuses(lib, kw, code):
    assert _bwd(lib, **kw) == code and lib.pm_last_error()


@pytest.mark.parametrize("kw,code", [(dict(w=None), -1), (dict(a=None), -1), (dict(rank=0), -2), (dict(rank=129), -2), (dict(d_out=12), -2), (dict(ldw=60), -1), (dict(out=ctypes.c_void_p(4100)), -1)])
def test_merge_refuses(lib, kw, code):
    a = dict(w=P, ldw=64, a=P, b=P, d_in=64, d_out=128, rank=8, out=P, ldo=64)
    a.update(kw)
    assert lib.pm_lora_merge(a["w"], a["ldw"], a["a"], a["b"], 1.0, a["d_in"], a["d_out"], a["rank"], a["out"], a["ldo"], None) == code


def test_clip_refuses(lib):
    def clip(chunks=P, n=3, offsets=P, groups=1, pieces=P, n_pieces=3, partials=P, sums=None, norms=P, coefs=P):
        return lib.pm_grad_clip(chunks, n, offsets, groups, pieces, n_pieces, None, 1.0, None, partials, sums, norms, coefs, None)

    for kw in (dict(chunks=None), dict(n=-1), dict(n=1 << 32), dict(n_pieces=-1), dict(offsets=None), dict(groups=0), dict(pieces=None), dict(partials=None), dict(coefs=None),
               dict(norms=None, coefs=None), dict(norms=None, coefs=None, sums=P)):
        assert clip(**kw) == -1 and lib.pm_last_error(), kw


def test_more_than_a_launch_holds_is_refused(lib):
    """2^32 threads: 64 x 256 elements for each 256 of them."""
    wide = dict(n=1 << 28, d_in=64, d_out=1 << 22, ldo=1 << 22, ldb=1 << 22)
    assert _fwd(lib, **wide) == -2 and b"too many" in lib.pm_last_error()
    assert _fwd(lib, n=(1 << 28) + 1) == -1
    assert _bwd(lib, n=1 << 28, d_in=1 << 22, ldx=1 << 22, ldb=1 << 22, ldgx=1 << 22) == -2 and b"too many" in lib.pm_last_error()
    assert lib.pm_lora_merge(P, 1 << 22, P, P, 1.0, 1 << 22, 1 << 22, 8, P, 1 << 22, None) == -2 and b"too many" in lib.pm_last_error()
    assert lib.pm_grad_clip(P, 1 << 23, P, 1, P, 3, None, 1.0, None, P, None, P, P, None) == -1
    assert lib.pm_grad_clip(P, 3, P, (1 << 20) + 1, P, 3, None, 1.0, None, P, None, P, P, None) == -1


def test_a_backward_of_nothing_is_no_work(lib):
    assert _bwd(lib, dx=None, da=None, db=None, ws=None) == 0


def test_workspaces_follow_the_sizes(lib):
    assert [lib.pm_lora_z_columns(r) for r in (0, 1, 16, 17, 128, 129)] == [0, 16, 16, 32, 128, 0]
    assert lib.pm_lora_fwd_workspace_bytes(0, 4, 4096, 4096, 16) == 0 and lib.pm_lora_fwd_workspace_bytes(16384, 4, 4096, 4096, 16) == 0  # enough rows: the long axis stays whole
    assert lib.pm_lora_fwd_workspace_bytes(1, 1, 4096, 4096, 16) == 0  # one row of not too many columns: one launch
    assert lib.pm_lora_fwd_workspace_bytes(1, 1, 16384, 4096, 16) == 8 * 16 * 4  # of many: eight parts
    assert lib.pm_lora_bwd_workspace_bytes(0, 4, 4096, 4096, 16, 1) == 0 and lib.pm_lora_bwd_workspace_bytes(100, 4, 4096, 4096, 16, 1) > 100 * 16 * 4


def test_cpu_tensors_are_refused():
    from prime_rl_amd import ops

    bf = dict(dtype=torch.bfloat16)
    x, a, b = torch.zeros(4, 64, **bf), torch.zeros(2, 8, 64, **bf), torch.zeros(2, 8, 128, **bf)
    s, off = torch.ones(2), torch.tensor([0, 2, 4], dtype=torch.int32)
    with pytest.raises(_lib.PrimeMI355XError, match="GPU tensor"):
        ops.lora_fwd(x, a, b, s, off)
    with pytest.raises(_lib.PrimeMI355XError, match="GPU tensor"):
        ops.lora_bwd(torch.zeros(4, 128, **bf), x, torch.zeros(4, 16), a, b, s, off)
    with pytest.raises(_lib.PrimeMI355XError, match="GPU tensor"):
        ops.lora_merge(torch.zeros(128, 64, **bf), a[0], b[0], 1.0)
    with pytest.raises(_lib.PrimeMI355XError, match="GPU tensor"):
        ops.GradClipPlan([torch.zeros(4)])


def test_rows_of_a_pass():
    from prime_rl_amd.trainer.models.layers.lora import LoRARows, LoRAState

    rows = LoRARows.packed([3, 0, 5], "cpu")
    assert rows.offsets.tolist() == [0, 3, 3, 8] and rows.offsets.dtype == torch.int32 and rows.row_ids is None
    assert LoRARows.packed(torch.tensor([4], dtype=torch.int32), "cpu").offsets.tolist() == [0, 4]  # lora_num_tokens of a micro-batch
    with pytest.raises(ValueError, match="negative"):
        LoRARows.packed([3, -1], "cpu")
    state = LoRAState(3, 8, [16, 8, 4], "cpu")
    assert state.scales.tolist() == [2.0, 1.0, 0.5]
    state.set_rows(rows)
    with pytest.raises(ValueError, match="2 adapters"):
        state.set_rows(LoRARows.packed([1, 2], "cpu"))
    for bad in (dict(n_adapters=0), dict(rank=0), dict(alpha=[1.0])):
        with pytest.raises(ValueError):
            LoRAState(**{**dict(n_adapters=2, rank=8, alpha=16.0, device="cpu"), **bad})


def test_attaching_adapters():
    from prime_rl_amd.trainer.models.layers.lora import adapter_parameters, attach_lora, lora_linear
    from prime_rl_amd.trainer.models.layers.mlp import MLP, MLPConfig

    mlp = MLP(MLPConfig(32, 64))
    names = set(mlp.state_dict())
    with pytest.raises(ValueError, match="targets"):
        attach_lora(mlp, 2, 4, 8.0, targets=("w1",))
    with pytest.raises(ValueError, match="none of the projections"):
        attach_lora(nn.Linear(4, 4), 2, 4, 8.0)
    state = attach_lora(mlp, 2, 4, 8.0, targets=("gate_proj", "down_proj"))
    assert set(mlp.state_dict()) - names == {f"{p}_proj.lora.{f}" for p in ("gate", "down") for f in "ab"}
    assert [tuple(p.shape) for p in adapter_parameters(mlp)] == [(2, 4, 32), (2, 4, 64), (2, 4, 64), (2, 4, 32)]
    assert {n for n, p in mlp.named_parameters() if p.requires_grad} == set(mlp.state_dict()) - names
    assert not mlp.gate_proj.lora.b.any() and mlp.gate_proj.lora.a.any() and mlp.gate_proj.lora.a.dtype == torch.float32
    with pytest.raises(ValueError, match="set_rows"):
        lora_linear(torch.zeros(3, 32), [mlp.gate_proj])
    with pytest.raises(ValueError, match="none of the projections has adapters"):
        lora_linear(torch.zeros(3, 32), [mlp.up_proj])
    mlp.gate_proj.weight.requires_grad_(True)
    state.rows = object()
    with pytest.raises(ValueError, match="frozen"):
        lora_linear(torch.zeros(3, 32), [mlp.gate_proj])


def test_a_model_has_one_set_of_adapters():
    from prime_rl_amd.trainer.models.layers.lora import LoRAAdapters, LoRAState, attach_lora, lora_linear
    from prime_rl_amd.trainer.models.layers.mlp import MLP, MLPConfig

    mlp = MLP(MLPConfig(32, 64))
    attach_lora(mlp, 2, 4, 8.0, targets=("gate_proj",))
    with pytest.raises(ValueError, match="already"):
        attach_lora(mlp, 2, 4, 8.0, targets=("down_proj",))
    other = LoRAState(2, 4, 16.0, "cpu")
    mlp.up_proj.lora = LoRAAdapters(mlp.up_proj, other)
    with pytest.raises(ValueError, match="different states"):
        lora_linear(torch.zeros(3, 32), [mlp.gate_proj, mlp.up_proj])
