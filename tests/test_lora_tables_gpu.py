"""GPU suite: the adapter kernels under wrong tables of rows, with guards around everything they write, and the bits that the factors' gradients keep."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
GUARD, MARK = 4096, -12.5  # elements of each side; in bf16 and f32 the same number


class Guarded:
    """A tensor between two stretches that nobody may write."""

    def __init__(self, *shape, dtype):
        n = 1
        for s in shape:
            n *= s
        self.whole = torch.full((n + 2 * GUARD,), MARK, dtype=dtype, device=DEV)
        self.t = self.whole[GUARD:GUARD + n].view(shape)

    def check(self, what):
        assert (self.whole[:GUARD] == MARK).all() and (self.whole[self.whole.numel() - GUARD:] == MARK).all(), what


def _wrong_tables(n, k):
    rng = random.Random(n)
    return [[rng.randint(-n, 2 * n) for _ in range(k + 1)], [n - g for g in range(k + 1)], [-(1 << 31)] * k + [(1 << 31) - 1], [(1 << 31) - 1] + [-(1 << 31)] * k,
            [0, *[n // 2] * (k - 1), n]]


@pytest.mark.parametrize("n,k,d_in,d_out,rank", [
    (50, 2, 64, 64, 16),  # both products in one launch, factors' gradients without partials
    (100, 3, 264, 136, 40),
    (300, 3, 264, 520, 16),
    (300, 70, 264, 520, 16),  # more adapters than are looked at together
    (300, 3, 1032, 264, 64),
    (300, 3, 264, 1032, 100),
    (900, 2, 4096, 4096, 64),  # the long axis in parts
    (8200, 3, 72, 4104, 12),  # dz beside dB in one pass
])
def test_wrong_tables_write_inside_their_buffers(n, k, d_in, d_out, rank):
    """Offsets and row ids that are no table: results may be anything, what lies around them stays."""
    from prime_rl_amd import _lib

    lib = _lib.load()
    g = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=g).to(BF16).to(DEV)  # noqa: E731
    x, a, b, dy, scales = rand(n, d_in), rand(k, rank, d_in), rand(k, rank, d_out), rand(n, d_out), torch.ones(k, device=DEV)
    rp = lib.pm_lora_z_columns(rank)
    fw, bw = lib.pm_lora_fwd_workspace_bytes(n, k, d_in, d_out, rank), lib.pm_lora_bwd_workspace_bytes(n, k, d_in, d_out, rank, 1)
    out, z, dx = Guarded(n, d_out, dtype=BF16), Guarded(n, rp, dtype=F32), Guarded(n, d_in, dtype=BF16)
    da, db, ws, wsb = Guarded(k, rank, d_in, dtype=F32), Guarded(k, rank, d_out, dtype=F32), Guarded(fw // 4, dtype=F32), Guarded(bw // 4, dtype=F32)
    ids = torch.randint(-2 * n, 3 * n, (n,), generator=g).to(torch.int32).to(DEV)
    stream = torch.cuda.current_stream().cuda_stream
    zeros = torch.zeros(n, rp, device=DEV)
    for offsets in _wrong_tables(n, k):
        t = torch.tensor(offsets, dtype=torch.int64).to(torch.int32).to(DEV)
        for rid in (None, ids):
            for accumulate in (0, 1):
                r = 0 if rid is None else rid.data_ptr()
                _lib.check(lib.pm_lora_fwd(x.data_ptr(), d_in, a.data_ptr(), b.data_ptr(), scales.data_ptr(), t.data_ptr(), r, n, k, d_in, d_out, rank, None, 0, out.t.data_ptr(), d_out,
                                           z.t.data_ptr(), ws.t.data_ptr() if fw else None, fw, stream), "pm_lora_fwd")
                _lib.check(lib.pm_lora_bwd(dy.data_ptr(), d_out, x.data_ptr(), d_in, zeros.data_ptr(), a.data_ptr(), b.data_ptr(), scales.data_ptr(), t.data_ptr(), r, n, k, d_in, d_out,
                                           rank, None, 0, dx.t.data_ptr(), d_in, da.t.data_ptr(), db.t.data_ptr(), accumulate, wsb.t.data_ptr(), bw, stream), "pm_lora_bwd")
                torch.cuda.synchronize()
                for what, m in dict(out=out, z=z, dx=dx, da=da, db=db, ws=ws, wsb=wsb).items():
                    m.check((what, offsets[:5], rid is not None))


@pytest.mark.parametrize("n,d_in,d_out,rank", [(100, 264, 136, 16), (200, 136, 264, 16), (200, 136, 264, 24), (200, 520, 264, 64), (200, 136, 264, 100), (8200, 136, 4104, 12)])
def test_factor_gradients_keep_the_24_bits_of_z_and_dz(n, d_in, d_out, rank):
    """Rows that are powers of two, and one row of each adapter with a gradient: every product is exact in 32 bits and every sum has one term, so the gradients are z's and
    dz's own bits.  Two bf16 terms in the place of three would lose the last eight of them."""
    from prime_rl_amd import ops

    g = torch.Generator().manual_seed(4)
    powers = lambda *s: (2.0 ** torch.randint(-3, 4, s, generator=g)) * (torch.randint(0, 2, s, generator=g) * 2 - 1)  # noqa: E731
    cut = 3 * n // 5
    offsets, live = torch.tensor([0, cut, n], dtype=torch.int32), [cut - 2, cut + 3]
    scales = torch.tensor([1.0 + 2.0**-23 + 2.0**-11, 1.5 - 2.0**-23 - 2.0**-12])
    z = torch.zeros(n, (rank + 15) // 16 * 16)
    z[:, :rank] = torch.randn(n, rank, generator=g)
    x, b, a = powers(n, d_in), powers(2, rank, d_out), powers(2, rank, d_in)
    dy = torch.zeros(n, d_out)
    for row in live:
        dy[row, row % d_out] = 4.0  # one column: dz is the scale's bits times a power of two
    for t in (z[live, :rank], scales):  # what two terms would leave out: one value that needs the third tells, since all are compared for equality
        hi = t.to(BF16).float()
        assert (t != hi + (t - hi).to(BF16).float()).any()
    dev = lambda t: t.to(BF16).to(DEV)  # noqa: E731
    _, da, db = ops.lora_bwd(dev(dy), dev(x), z.to(DEV), dev(a), dev(b), scales.to(DEV), offsets.to(DEV))
    for k, row in enumerate(live):
        dz = scales[k].double() * (b[k].double() @ dy[row].double())
        assert torch.equal(da[k].cpu().double(), dz[:, None] * x[row].double()[None])
        assert torch.equal(db[k].cpu().double(), z[row, :rank].double()[:, None] * dy[row].double()[None])
