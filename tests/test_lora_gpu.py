"""GPU suite: the adapter operators (pm_lora_fwd / _bwd / _merge) against their formulas in 64 bits.

Tolerances, element by element, from the roundings: a bf16 result is off by at most half a step, 2^-8 of its value; z and dz are f32 sums over d terms (d 2^-24 of
the sum of magnitudes, doubled for the order of the adds); two bf16 terms carry z into the second product with 2^-16 of it left out, three with 2^-24."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E24, E16, E8 = 2.0**-24, 2.0**-16, 2.0**-8


@pytest.fixture(scope="module")
def ops():
    from prime_rl_amd import ops as _ops

    return _ops


def _rand(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(BF16).to(DEV)


def _case(counts, d_in, d_out, rank, without=0, mixed=False, seed=0):
    """Inputs of `counts[g]` rows for each adapter and `without` rows of none, in the order of the adapters or shuffled."""
    g = torch.Generator().manual_seed(seed)
    n, k = sum(counts) + without, len(counts)
    offsets = torch.tensor([0, *counts]).cumsum(0).to(torch.int32).to(DEV)
    row_ids = torch.randperm(n, generator=g).to(torch.int32).to(DEV) if mixed else None
    return dict(x=_rand(g, n, d_in), a=_rand(g, k, rank, d_in, std=d_in**-0.5), b=_rand(g, k, rank, d_out, std=0.3), scales=(torch.rand(k, generator=g) + 0.5).to(DEV),
                offsets=offsets, base=_rand(g, n, d_out), row_ids=row_ids, dy=_rand(g, n, d_out, std=0.1), bx=_rand(g, n, d_in, std=0.1))


def _rows(c, g):
    lo, hi = c["offsets"][g].item(), c["offsets"][g + 1].item()
    pos = torch.arange(lo, hi, device=DEV)
    return pos, pos if c["row_ids"] is None else c["row_ids"][pos].long()


def _within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {err[bad].max().item():.3e} where {tol[bad].max().item():.3e} is allowed"


def _check_fwd(c, out, z):
    d_in, r = c["x"].shape[1], c["a"].shape[1]
    want = c["base"].double().clone() if c["base"] is not None else torch.zeros(out.shape, dtype=F64, device=DEV)
    tol = torch.zeros_like(want)
    for g in range(c["a"].shape[0]):
        pos, rows = _rows(c, g)
        x, a, b, s = c["x"][rows].double(), c["a"][g].double(), c["b"][g].double(), c["scales"][g].double()
        zg, za = s * (x @ a.t()), s * (x.abs() @ a.abs().t())
        _within(z[pos, :r], zg, 2 * (d_in + 2) * E24 * za, f"z of adapter {g}")
        assert not z[pos, r:].any()
        want[rows] += zg @ b
        tol[rows] += (E16 + 2 * (d_in + r + 4) * E24) * (za @ b.abs())
    _within(out, want, tol + E8 * (want.abs() + tol), "out")


def _check_bwd(c, z, dx, da, db, da0=None, db0=None):
    n, d_in = c["x"].shape
    d_out, r = c["dy"].shape[1], c["a"].shape[1]
    want = c["bx"].double().clone() if c["bx"] is not None else torch.zeros(n, d_in, dtype=F64, device=DEV)
    tol = torch.zeros_like(want)
    for g in range(c["a"].shape[0]):
        pos, rows = _rows(c, g)
        x, dy, a, b, s = c["x"][rows].double(), c["dy"][rows].double(), c["a"][g].double(), c["b"][g].double(), c["scales"][g].double()
        dz, dza = s * (dy @ b.t()), s * (dy.abs() @ b.abs().t())
        want[rows] += dz @ a
        tol[rows] += (E16 + 2 * (d_out + r + 4) * E24) * (dza @ a.abs())
        for got, left, wide, start, what, d in ((da, dz, x, da0, "grad_a", d_out), (db, z[pos, :r].double(), dy, db0, "grad_b", 0)):
            mag = (dza if d else left.abs()).t() @ wide.abs()
            ref = left.t() @ wide + (start[g].double() if start is not None else 0.0)
            _within(got[g], ref, 2 * (d + len(rows) + 40) * E24 * (mag + (start[g].double().abs() if start is not None else 0.0)), f"{what} of adapter {g}")
    if dx is not None:
        _within(dx, want, tol + E8 * (want.abs() + tol), "grad_x")


CASES = [  # rows of each adapter, d_in, d_out, rank, rows of none, in any order
    ([1], 64, 64, 16, 0, False),
    ([1], 4096, 4096, 16, 0, False),
    ([0], 64, 64, 16, 3, False),
    ([1, 1, 1, 1], 2048, 1032, 8, 2, True),
    ([64], 256, 256, 16, 0, False),
    ([63, 65, 0, 1, 130], 256, 384, 16, 5, False),
    ([63, 65, 0, 1, 130], 256, 384, 16, 5, True),
    ([40, 200], 8, 8, 1, 0, False),
    ([33, 31], 72, 24, 5, 1, True),
    ([100, 0, 57], 520, 264, 17, 9, True),
    ([100, 57], 328, 776, 32, 0, False),
    ([70, 90], 584, 136, 48, 7, True),
    ([70, 129], 1096, 648, 64, 7, False),
    ([70, 90], 392, 1048, 100, 0, True),
    ([257, 31], 712, 520, 128, 33, False),
    ([3, 0, 1, 2] * 20, 128, 64, 12, 4, True),  # more adapters than lanes of a wave
    ([9000, 7421, 0, 600], 192, 128, 16, 11, False),
    ([4100, 4097], 256, 512, 64, 1, True),
    # enough of grad_out that dz comes with dB in one pass
    ([9000, 0, 7421, 600], 264, 4104, 16, 11, False),
    ([8000, 33, 9000], 128, 4096, 12, 40, True),
    ([17000], 520, 4008, 1, 0, False),
]


@pytest.mark.parametrize("counts,d_in,d_out,rank,without,mixed", CASES)
def test_lora_fwd_and_bwd_match_the_formula(ops, counts, d_in, d_out, rank, without, mixed):
    c = _case(counts, d_in, d_out, rank, without, mixed)
    out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"], row_ids=c["row_ids"])
    _check_fwd(c, out, z)
    _check_bwd(c, z, *ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"], row_ids=c["row_ids"]))


def test_lora_without_base_starts_from_zero(ops):
    c = _case([50, 14], 128, 256, 16, without=6)
    c["base"] = c["bx"] = None
    out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"])
    _check_fwd(c, out, z)
    assert not out[64:].any()
    _check_bwd(c, z, *ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"]))


def test_lora_in_place_on_column_slices_leaves_everything_else(ops):
    """The update of one projection of a fused q | k | v output: base and out are the same column slice; the columns beside it and rows of no adapter stay."""
    c = _case([75, 0, 90], 256, 128, 16, without=12, mixed=True)
    wide = torch.randn(177, 512, device=DEV).to(BF16)
    c["base"] = wide[:, 128:256].clone()
    whole = wide.clone()
    xw = torch.zeros(177, 264, dtype=BF16, device=DEV)
    xw[:, 8:] = c["x"]
    out, z = ops.lora_fwd(xw[:, 8:], c["a"], c["b"], c["scales"], c["offsets"], base=whole[:, 128:256], out=whole[:, 128:256], row_ids=c["row_ids"])
    assert out.data_ptr() == whole[:, 128:256].data_ptr()
    _check_fwd(c, whole[:, 128:256], z)
    assert torch.equal(whole[:, :128], wide[:, :128]) and torch.equal(whole[:, 256:], wide[:, 256:])
    left = c["row_ids"][165:].long()
    assert torch.equal(whole[left], wide[left])
    # the same to another slice of the buffer that holds the base
    ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=wide[:, 128:256], out=wide[:, 256:384], row_ids=c["row_ids"])
    assert torch.equal(wide[:, 256:384], whole[:, 128:256])


def test_lora_bwd_accumulates_or_overwrites(ops):
    c = _case([130, 0, 31], 136, 264, 24)
    out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"])
    da0, db0 = torch.randn(c["a"].shape, device=DEV), torch.randn(c["b"].shape, device=DEV)
    da, db = da0.clone(), db0.clone()
    dx, ga, gb = ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"], grad_a=da, grad_b=db, accumulate=True)
    assert ga is da and gb is db
    _check_bwd(c, z, dx, da, db, da0, db0)
    assert torch.equal(da[1], da0[1]) and torch.equal(db[1], db0[1])  # no rows: nothing is added
    ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], grad_a=da, grad_b=db, want_x=False)
    _check_bwd(c, z, None, da, db)
    assert not da[1].any() and not db[1].any()


def test_lora_bwd_of_what_is_wanted(ops):
    c = _case([40, 30], 64, 128, 16)
    _, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"])
    args = (c["a"], c["b"], c["scales"], c["offsets"])
    dx, da, db = ops.lora_bwd(c["dy"], c["x"], z, *args, base=c["bx"])
    only_x = ops.lora_bwd(c["dy"], None, None, *args, base=c["bx"], want_factors=False)
    only_w = ops.lora_bwd(c["dy"], c["x"], z, *args, want_x=False)
    assert torch.equal(only_x[0], dx) and only_x[1] is None and only_x[2] is None
    assert only_w[0] is None and torch.equal(only_w[1], da) and torch.equal(only_w[2], db)
    inplace = c["bx"].clone()
    assert torch.equal(ops.lora_bwd(c["dy"], c["x"], z, *args, base=inplace, grad_x=inplace)[0], dx)


@pytest.mark.parametrize("n", [0])
def test_lora_without_rows(ops, n):
    c = _case([0, 0], 64, 128, 16)
    out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"])
    assert out.shape == (0, 128) and z.shape == (0, 16)
    dx, da, db = ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"])
    assert dx.shape == (0, 64) and not da.any() and not db.any()


def test_lora_rows_sorts_any_order(ops):
    ids = torch.tensor([2, -1, 0, 2, 7, 0, 1, 2, 99], dtype=torch.int32, device=DEV)
    offsets, row_ids = ops.lora_rows(ids, 4)
    assert offsets.tolist() == [0, 2, 3, 6, 6] and row_ids.tolist() == [2, 5, 6, 0, 3, 7, 1, 4, 8]


def test_lora_other_rows_and_adapters_do_not_leak(ops):
    """Infinities and NaN of one adapter's rows or factors, or of rows of none, stay where they are; an infinite z is an infinite update and not NaN."""
    c = _case([70, 45, 64], 320, 192, 16, without=10)
    clean, zc = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"])
    gc = ops.lora_bwd(c["dy"], c["x"], zc, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"])
    d = {k: v.clone() if v is not None else None for k, v in c.items()}
    d["x"][70:115] = float("nan")
    d["a"][1] = float("inf")
    d["b"][1] = float("nan")
    d["dy"][70:115] = float("inf")
    d["x"][179:] = float("inf")
    d["dy"][179:] = float("nan")
    out, z = ops.lora_fwd(d["x"], d["a"], d["b"], d["scales"], d["offsets"], base=d["base"])
    g = ops.lora_bwd(d["dy"], d["x"], z, d["a"], d["b"], d["scales"], d["offsets"], base=d["bx"])
    keep = torch.tensor([i for i in range(189) if not 70 <= i < 115], device=DEV)
    assert torch.equal(out[keep], clean[keep]) and torch.equal(g[0][keep], gc[0][keep])
    for k in (1, 2):
        assert torch.equal(g[k][0], gc[k][0]) and torch.equal(g[k][2], gc[k][2])
    assert torch.equal(out[179:], c["base"][179:])
    one = _case([4], 64, 64, 1)
    one["x"][2] = 0
    one["x"][2, 5] = float("inf")
    out, z = ops.lora_fwd(one["x"], one["a"], one["b"], one["scales"], one["offsets"])
    assert torch.isinf(z[2, 0]) and torch.isinf(out[2]).all() and torch.isfinite(out[[0, 1, 3]]).all()


def test_lora_bwd_in_one_pass_keeps_infinities_in_their_rows(ops):
    c = _case([9000, 7000, 500], 128, 4104, 11, without=50, mixed=True)
    args = (c["a"], c["b"], c["scales"], c["offsets"])
    _, z = ops.lora_fwd(c["x"], *args, base=c["base"], row_ids=c["row_ids"])
    clean = ops.lora_bwd(c["dy"], c["x"], z, *args, base=c["bx"], row_ids=c["row_ids"])
    rows = c["row_ids"].long()
    dy = c["dy"].clone()
    dy[rows[9000:9040]] = float("inf")
    dy[rows[9050:9060], 0] = float("nan")
    dy[rows[16500:]] = float("nan")
    got = ops.lora_bwd(dy, c["x"], z, *args, base=c["bx"], row_ids=c["row_ids"])
    keep = torch.cat([rows[:9000], rows[9040:9050], rows[9060:]])
    assert torch.equal(got[0][keep], clean[0][keep])
    for k in (1, 2):
        assert torch.equal(got[k][0], clean[k][0]) and torch.equal(got[k][2], clean[k][2]) and not torch.isfinite(got[k][1]).all()
    dy = c["dy"].clone()
    dy[rows[20], 5] = float("inf")  # an infinite gradient of one column: every column of grad_x that the adapter reaches is infinite, not NaN, where the rank is one
    r1 = (c["a"][:, :1].contiguous(), c["b"][:, :1].contiguous(), c["scales"], c["offsets"])
    _, z1 = ops.lora_fwd(c["x"], *r1, base=c["base"], row_ids=c["row_ids"])
    one = ops.lora_bwd(dy, c["x"], z1, *r1, row_ids=c["row_ids"])[0]
    assert torch.isinf(one[rows[20]]).all() and torch.isfinite(one[rows[21]]).all()


def test_lora_padding_ranks_with_zero_rows_changes_nothing(ops):
    c = _case([80, 33], 256, 128, 12, without=2)
    out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"])
    ref = ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"])
    pad = lambda t: torch.cat([t, torch.zeros(t.shape[0], 28, t.shape[2], dtype=BF16, device=DEV)], dim=1)  # noqa: E731
    a, b = pad(c["a"]), pad(c["b"])
    out2, z2 = ops.lora_fwd(c["x"], a, b, c["scales"], c["offsets"], base=c["base"])
    got = ops.lora_bwd(c["dy"], c["x"], z2, a, b, c["scales"], c["offsets"], base=c["bx"])
    assert not z2[:113, 12:].any() and not got[1][:, 12:].any() and not got[2][:, 12:].any()
    _check_fwd(c, out2, torch.cat([z2[:, :12], torch.zeros(115, 4, device=DEV)], dim=1))
    _check_bwd(c, z2[:, :12], got[0], got[1][:, :12], got[2][:, :12])
    assert ref[1].shape == (2, 12, 256)


def test_lora_gives_the_same_bits_every_time(ops):
    c = _case([700, 1300, 0, 45], 1024, 768, 32, without=3, mixed=True)
    args = (c["a"], c["b"], c["scales"], c["offsets"])
    first = None
    for _ in range(3):
        out, z = ops.lora_fwd(c["x"], *args, base=c["base"], row_ids=c["row_ids"])
        got = (out, *ops.lora_bwd(c["dy"], c["x"], z, *args, base=c["bx"], row_ids=c["row_ids"]))
        assert first is None or all(torch.equal(u, v) for u, v in zip(first, got))
        first = got


def test_lora_offsets_and_row_ids_out_of_range_stay_in_range(ops):
    """Tables that are wrong give wrong rows, never an access outside the tensors (clamped in the kernels)."""
    c = _case([20, 30], 64, 64, 16)
    for offsets in ([0, 1 << 30, 1 << 30], [-5, -3, 2], [40, 10, 90], [0, 50, 50]):
        t = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        ids = torch.full((50,), 1 << 29, dtype=torch.int32, device=DEV)
        ids[:25] = -7
        for rid in (None, ids):
            out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], t, base=c["base"], row_ids=rid)
            ops.lora_bwd(c["dy"], c["x"], torch.zeros_like(z), c["a"], c["b"], c["scales"], t, base=c["bx"], row_ids=rid)
    torch.cuda.synchronize()


def test_lora_rows_past_32_bit_element_offsets(ops):
    """Row tensors of more than 2^31 elements: the last rows, one adapter."""
    n, d = 140_000, 16384
    x = torch.zeros(n, d, dtype=BF16, device=DEV)
    g = torch.Generator().manual_seed(3)
    x[-64:] = _rand(g, 64, d)
    a, b = _rand(g, 1, 8, d, std=d**-0.5), _rand(g, 1, 8, 64, std=0.3)
    offsets = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    out, z = ops.lora_fwd(x, a, b, torch.ones(1, device=DEV), offsets)
    small, zs = ops.lora_fwd(x[-64:].clone(), a, b, torch.ones(1, device=DEV), torch.tensor([0, 64], dtype=torch.int32, device=DEV))
    assert not out[:-64].any()
    torch.testing.assert_close(z[-64:], zs, rtol=0, atol=1e-4)
    torch.testing.assert_close(out[-64:].float(), small.float(), rtol=E8 * 2, atol=1e-4)
    _, da, db = ops.lora_bwd(out, x, z, a, b, torch.ones(1, device=DEV), offsets, want_x=False)
    ref = (out[-64:].double() @ b[0].double().t()).t() @ x[-64:].double()
    assert (da[0].double() - ref).norm() <= 1e-5 * ref.norm()


@pytest.mark.parametrize("d_out,d_in,rank", [(1, 64, 4), (64, 64, 16), (200, 136, 8), (1024, 520, 33), (72, 4096, 64), (640, 264, 128)])
def test_lora_merge_matches_the_formula(ops, d_out, d_in, rank):
    if d_out % 8:
        d_out = 8
    g = torch.Generator().manual_seed(1)
    w, a, b = _rand(g, d_out, d_in), _rand(g, rank, d_in, std=0.2), _rand(g, rank, d_out, std=0.2)
    got = ops.lora_merge(w, a, b, 1.7)
    scale = torch.tensor(1.7, dtype=F32).double().item()
    want = w.double() + scale * (b.double().t() @ a.double())
    tol = (E16 + 2 * (rank + 4) * E24) * scale * (b.double().abs().t() @ a.double().abs())
    _within(got, want, tol + E8 * (want.abs() + tol), "merged")
    wide = torch.zeros(d_out, d_in + 16, dtype=BF16, device=DEV)
    wide[:, 8:-8] = w
    ops.lora_merge(wide[:, 8:-8], a, b, 1.7, out=wide[:, 8:-8])
    assert torch.equal(wide[:, 8:-8], got) and not wide[:, :8].any() and not wide[:, -8:].any()
    assert torch.equal(ops.lora_merge(w, a, b, 0.0), w)


def test_lora_on_another_stream_and_in_graphs(ops):
    """Two graphs of different cases, replayed in turn and with other inputs in the same buffers, against the eager results."""
    cases = [_case([33, 100], 512, 256, 16, without=3, seed=5), _case([1] * 6, 1024, 512, 8, seed=6, mixed=True)]

    def step(c):
        out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"], row_ids=c["row_ids"])
        return (out, *ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"], row_ids=c["row_ids"]))

    graphs = []
    side = torch.cuda.Stream()
    for c in cases:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step(c)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(eager, step(c)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(c)
        graphs.append((graph, c, held))
    for turn in range(3):
        for graph, c, held in graphs:
            c["x"].copy_(torch.randn_like(c["x"]) * (turn + 1))
            c["dy"].copy_(torch.randn_like(c["dy"]))
            graph.replay()
        torch.cuda.synchronize()
        for graph, c, held in graphs:
            assert all(torch.equal(u, v) for u, v in zip(held, step(c))), turn


FEW = [
    ([1], 4096, 520, 16, 0, False),
    ([1], 520, 4096, 16, 0, True),
    ([0, 1, 0, 2], 72, 8, 5, 1, False),
    ([16, 17, 31], 1032, 264, 16, 0, True),
    ([64], 6144, 72, 1, 0, False),
    ([0, 0, 5, 0], 328, 6144, 12, 3, True),
    ([1] * 64, 264, 2056, 16, 0, True),
    ([2] * 25, 512, 1024, 8, 14, False),
    ([63], 64, 64, 16, 1, False),
    ([3, 20, 0, 17], 520, 1032, 32, 2, True),
    ([1, 0, 2], 4096, 520, 48, 1, False),
    ([30, 9], 72, 4096, 64, 0, True),
    ([1] * 40, 136, 2056, 20, 0, False),
    ([1] * 70, 136, 128, 16, 2, True),  # more adapters than outer takes without partials
    ([100, 28], 264, 136, 16, 0, True),  # outer alone without partials
    ([50, 0, 70], 136, 264, 48, 8, False),
    ([129], 72, 136, 16, 0, False),
]


@pytest.mark.parametrize("counts,d_in,d_out,rank,without,mixed", FEW)
def test_lora_of_few_rows(ops, counts, d_in, d_out, rank, without, mixed):
    c = _case(counts, d_in, d_out, rank, without, mixed, seed=9)
    out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"], row_ids=c["row_ids"])
    _check_fwd(c, out, z)
    grads = ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"], row_ids=c["row_ids"])
    _check_bwd(c, z, *grads)
    start = [torch.randn_like(g) for g in grads[1:]]
    into = [t.clone() for t in start]
    dx, *_ = ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"], row_ids=c["row_ids"], grad_a=into[0], grad_b=into[1], accumulate=True)
    _check_bwd(c, z, dx, *into, *start)


@pytest.mark.parametrize("n", [3, 40, 300])
def test_lora_results_in_their_own_inputs_memory(ops, n):
    """out over x, grad_x over grad_out or over x (d_in = d_out): read to the end before they are written."""
    c = _case([n // 2, n - n // 2], 256, 256, 16, seed=4)
    args = (c["a"], c["b"], c["scales"], c["offsets"])
    out, z = ops.lora_fwd(c["x"], *args, base=c["base"])
    x = c["x"].clone()
    over, z2 = ops.lora_fwd(x, *args, base=c["base"], out=x)
    assert over is x
    _check_fwd(c, over, z2)
    for name in ("dy", "x"):
        t = {k: c[k].clone() for k in ("dy", "x")}
        got = ops.lora_bwd(t["dy"], t["x"], z, *args, base=c["bx"], grad_x=t[name])
        assert got[0] is t[name]
        _check_bwd(c, z, *got)


@pytest.mark.parametrize("n,ld,rank", [(40, 1 << 27, 16), (40, 1 << 27, 100), (300, 1 << 24, 16), (300, 1 << 24, 64), (300, 1 << 24, 100)])
def test_lora_rows_gigabytes_apart(ops, n, ld, rank):
    """Column slices of one buffer of more than 2^32 elements, in place."""
    d_in, d_out = 264, 520
    c = _case([n // 3, n - n // 3 - 2], d_in, d_out, rank, 2, True, seed=6)
    storage = torch.empty(n * ld, dtype=BF16, device=DEV)
    wide, at = {}, 0
    for name in ("x", "base", "dy", "bx"):
        w = c[name].shape[1]
        wide[name] = storage.as_strided((n, w), (ld, 1), at)
        wide[name].copy_(c[name])
        at += w
    args = (c["a"], c["b"], c["scales"], c["offsets"])
    out, z = ops.lora_fwd(c["x"], *args, base=c["base"], row_ids=c["row_ids"])
    got, zw = ops.lora_fwd(wide["x"], *args, base=wide["base"], out=wide["base"], row_ids=c["row_ids"])
    assert got is wide["base"]
    _check_fwd(c, got, zw)
    _check_fwd(c, out, z)
    want = ops.lora_bwd(c["dy"], c["x"], z, *args, base=c["bx"], row_ids=c["row_ids"])
    back = ops.lora_bwd(wide["dy"], wide["x"], z, *args, base=wide["bx"], grad_x=wide["bx"], row_ids=c["row_ids"])
    _check_bwd(c, z, *want)
    _check_bwd(c, z, *back)
    assert torch.equal(wide["x"], c["x"]) and torch.equal(wide["dy"], c["dy"])


@pytest.mark.parametrize("counts,d_in,d_out,rank,mixed", [([350, 0, 240], 4096, 1032, 64, True), ([900], 4096, 4096, 64, False), ([500, 400], 4096, 4096, 128, False), ([700, 600], 4096, 4096, 9, True)])
def test_lora_of_long_rows_in_parts(ops, counts, d_in, d_out, rank, mixed):
    """The long axis cut into parts that are added up before they are used; in a graph as well."""
    c = _case(counts, d_in, d_out, rank, 10, mixed, seed=8)

    def step():
        out, z = ops.lora_fwd(c["x"], c["a"], c["b"], c["scales"], c["offsets"], base=c["base"], row_ids=c["row_ids"])
        return (out, z, *ops.lora_bwd(c["dy"], c["x"], z, c["a"], c["b"], c["scales"], c["offsets"], base=c["bx"], row_ids=c["row_ids"]))

    out, z, *grads = step()
    _check_fwd(c, out, z)
    _check_bwd(c, z, *grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        c["x"].copy_(torch.randn_like(c["x"]))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for i in (0, 2, 3, 4):  # (z of rows of no adapter is undefined)
            assert torch.equal(held[i], eager[i]), turn
