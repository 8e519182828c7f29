"""CPU suite: how the adapter kernels cut their work — tiles, ranges and partials — written down a second time and held against the library's workspaces, then walked over
ragged, empty, straddling and wrong tables of rows: every position once, every partial written once and read only where it was written, nothing outside its buffer."""

import random

import pytest

from prime_rl_amd import _lib

KI, MI = 1 << 10, 1 << 20


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        _lib.build()
    return _lib.load()


def cdiv(a, b):
    return -(-a // b)


def padded(rank):
    return cdiv(rank, 16) * 16


def factor_rows(rank):
    return 16 if rank <= 16 else 32 if rank <= 32 else 64 if rank <= 64 else 128


def max_tiles(n, k, rows):
    return min(n // rows + k + 2, n)


def few_rows(n, k, d_in, d_out, rank):
    if n > 64 or rank > 64 or factor_rows(rank) * d_in > 96 * KI:
        return 0
    tiles = max_tiles(n, k, 16)
    return 1 if tiles * cdiv(d_out, 256) <= 256 else 4 if rank <= 32 and tiles * cdiv(d_out, 1024) <= 256 else 0


def shrink_parts(n, k, d, rank):
    narrow, factor = rank <= 16, factor_rows(rank)
    chunks = cdiv(d, 256 if narrow else 128)
    most = min(max(chunks // 2, 1), 8)

    def parts_of(tiles, at_once):
        return most if tiles * most <= at_once else at_once // tiles if tiles < at_once else 1

    if narrow:
        tiles = max_tiles(n, k, 32)
        parts = parts_of(max(tiles, 1), 512)
        if 0 < tiles <= 1024:
            even = min(chunks // 12, 2200 // tiles)
            parts = 8 if even > 8 else max(even, parts)
        return 32, parts
    best = None
    for rows in [16, 32, 48, *range(64, 193, 4)]:
        tiles = min((n + k * (rows - 1)) // rows, n)
        parts = parts_of(max(tiles, 1), 256)
        cost = float((tiles * parts + 255) // 256) * ((rows + factor) * ((chunks + parts - 1) // parts) + 160.0) + (tiles * parts * rows * factor / (256.0 * 32.0) if parts > 1 else 0.0)
        if best is None or cost <= best[0]:
            best = cost, rows, parts
    return best[1:]


def outer_range(n, k, col_tiles, rank):
    best = None
    for rounds in range(1, 9):
        splits = 256 * rounds // col_tiles
        if splits < 1 and rounds > 1:
            continue
        splits = max(1, min(splits, n))
        reach = cdiv(n, splits)
        used = cdiv(n, reach)
        cost = float((used * col_tiles + 255) // 256) * (max(reach, 32) + (4.0 * rank + 96.0) * (1.0 + k / used))
        if best is None or cost < best[0]:
            best = cost, reach
    return best[1]


def bwd_plan(n, k, d_in, d_out, rank, factors):
    """(fused, few, column tiles, ranges and workspace bytes of both sides)."""
    rp, tiles = padded(rank), (cdiv(d_out, 512), cdiv(d_in, 512))
    fused = factors and rank <= 16 and n * d_out >= 32 * MI
    parts = 1 if fused else shrink_parts(n, k, d_out, rank)[1]
    few_tiles = (cdiv(d_out, 128) + cdiv(d_in, 128)) * (rp // 16)
    few = not fused and n <= (128 if k > 1 else 64) and few_tiles * k <= MI
    range0 = outer_range(n, k, tiles[0] if fused else sum(tiles), rank)
    range1 = outer_range(n, k, tiles[1], rank) if fused else range0
    partials = [(cdiv(n, r) + k) * rank * d * 4 if factors and not few else 0 for r, d in ((range0, d_out), (range1, d_in))]
    return dict(fused=fused, few=few, tiles=tiles, ranges=(range0, range1), bytes=parts * n * rp * 4 + (tiles[0] * n * rp * 4 if fused else 0) + sum(partials))


def _sizes(rng):
    spread = lambda lo, hi: max(lo, min(hi, int(lo * (hi / lo) ** rng.random())))  # noqa: E731
    return spread(1, 40000), rng.choice([1, 2, 3, 5, 16, 70, 300]), 8 * spread(1, 1600), 8 * spread(1, 1600), rng.choice([1, 4, 8, 12, 16, 17, 32, 33, 48, 64, 65, 100, 128])


def test_workspaces_are_what_the_plan_says(lib):
    """The second writing of the plan is that of the library: the workspaces follow from parts, ranges and partials."""
    rng = random.Random(5)
    seen = set()
    for n, k, d_in, d_out, rank in [(264, 5, 256, 384, 16), (16384, 4, 4096, 6144, 16), (32768, 8, 4096, 12288, 64)] + [_sizes(rng) for _ in range(3000)]:
        for factors in (0, 1):
            plan = bwd_plan(n, k, d_in, d_out, rank, bool(factors))
            assert lib.pm_lora_bwd_workspace_bytes(n, k, d_in, d_out, rank, factors) == plan["bytes"], (n, k, d_in, d_out, rank, factors)
            seen.add((plan["fused"], plan["few"], rank > 64))
        parts = 1 if few_rows(n, k, d_in, d_out, rank) else shrink_parts(n, k, d_in, rank)[1]
        assert lib.pm_lora_fwd_workspace_bytes(n, k, d_in, d_out, rank) == (parts * n * padded(rank) * 4 if parts > 1 else 0), (n, k, d_in, d_out, rank)
    assert len(seen) == 5  # one pass, few rows and neither, of small and large ranks (one pass: small ones only)


def tables(n, k, rng):
    """Tables of rows that callers hand in, and wrong ones."""
    cuts = sorted(rng.randint(0, n) for _ in range(k - 1))
    yield [0, *cuts, n - rng.choice([0, 0, min(n, 7)])] if not cuts or cuts[-1] <= n - 7 else [0, *cuts, n]
    yield [0] * k + [n]  # all rows at the last adapter
    yield [0] + [n] * k  # at the first
    yield [min(g, n) for g in range(k + 1)]  # a row each
    yield [min(3 * g, n) for g in range(k + 1)]
    yield [0] * (k + 1)  # none


def wrong_tables(n, k, rng):
    yield [rng.randint(-n, 2 * n) for _ in range(k + 1)]
    yield [n - g for g in range(k + 1)]
    yield [-(1 << 31)] * k + [(1 << 31) - 1]
    yield [(1 << 31) - 1] + [-(1 << 31)] * k


def walk_outer(offsets, n, k, reach):
    """What each range of positions sums up: (range, adapter, lo, hi), as a workgroup walks the table (64 adapters are looked at together)."""
    out = []
    for split in range(cdiv(n, reach)):
        begin, end = split * reach, min((split + 1) * reach, n)
        g = next((g for g in range(k) if offsets[g + 1] > begin), k)
        lo = min(max(offsets[g], begin), end) if g < k else end
        while g < k and lo < end:
            hi = min(max(offsets[g + 1], lo), end)
            if hi > lo:
                out.append((split, g, lo, hi))
            lo, g = hi, g + 1
    return out


def joined(offsets, n, g, reach):
    """The partials that the join adds up for adapter g."""
    lo = min(max(offsets[g], 0), n)
    hi = min(max(offsets[g + 1], lo), n)
    return [s + g for s in range(lo // reach, (hi - 1) // reach + 1)] if lo < hi else []


def walk_tiles(offsets, n, k, rows):
    """(adapter, p0, p1) of every tile: the adapters' in turn, then the positions behind the last offset and before the first."""
    out = []
    for e in range(k + 2):
        if e < k:
            lo = min(max(offsets[e], 0), n)
            hi = min(max(offsets[e + 1], lo), n)
        else:
            lo, hi = (min(max(offsets[k], 0), n), n) if e == k else (0, min(max(offsets[0], 0), n))
        out += [(e if e < k else -1, p, min(p + rows, hi)) for p in range(lo, hi, rows)]
    return out


PLANS = [(264, 5, 256, 384, 16), (259, 5, 256, 384, 16), (257, 1, 8, 8, 1), (129, 1, 72, 136, 16), (129, 70, 136, 128, 16), (777, 3, 1024, 2048, 8), (300, 16, 4096, 12288, 64),
         (1000, 300, 64, 64, 128), (17032, 4, 264, 4104, 16), (17000, 1, 520, 4008, 1), (2500, 40, 12800, 8, 100)]


def _plans():
    rng = random.Random(8)
    more = [_sizes(rng) for _ in range(60)]
    return PLANS + [(min(n, 6000), k, d_in, d_out, rank) for n, k, d_in, d_out, rank in more if n > 128]


def test_partials_are_written_once_and_read_where_they_were_written():
    rng = random.Random(6)
    for n, k, d_in, d_out, rank in _plans():
        plan = bwd_plan(n, k, d_in, d_out, rank, True)
        for reach in set(plan["ranges"]):
            held = cdiv(n, reach) + k  # partials of [rank][d] in the workspace
            for offsets in tables(n, k, rng):
                sums = walk_outer(offsets, n, k, reach)
                written = [split + g for split, g, _, _ in sums]
                assert len(set(written)) == len(written) and all(0 <= w < held for w in written), (n, k, reach, offsets)
                covered = sorted((lo, hi, g) for _, g, lo, hi in sums)
                assert [p for lo, hi, _ in covered for p in range(lo, hi)] == list(range(offsets[0], offsets[k])), (n, k, reach, offsets)
                assert all(offsets[g] <= lo and hi <= offsets[g + 1] for lo, hi, g in covered)
                for g in range(k):  # the ranges that meet adapter g, in their order
                    assert joined(offsets, n, g, reach) == [s + h for s, h, _, _ in sums if h == g], (n, k, reach, offsets, g)


def test_wrong_tables_stay_in_their_buffers():
    rng = random.Random(7)
    for n, k, d_in, d_out, rank in _plans():
        plan = bwd_plan(n, k, d_in, d_out, rank, True)
        for offsets in wrong_tables(n, k, rng):
            for reach in set(plan["ranges"]):
                held = cdiv(n, reach) + k
                for split, g, lo, hi in walk_outer(offsets, n, k, reach):
                    assert 0 <= split * reach <= lo < hi <= min((split + 1) * reach, n) and 0 <= split + g < held
                assert all(0 <= w < held for g in range(k) for w in joined(offsets, n, g, reach))
            for rows in (16, 32, 64, 128, shrink_parts(n, k, d_in, rank)[0]):
                assert all(0 <= p0 < p1 <= min(p0 + rows, n) and -1 <= g < k for g, p0, p1 in walk_tiles(offsets, n, k, rows))


def test_tiles_cover_every_position_once():
    rng = random.Random(9)
    for n, k, d_in, d_out, rank in _plans() + [(1, 1, 64, 64, 16), (5, 300, 64, 64, 16), (64, 64, 64, 64, 4)]:
        for offsets in tables(n, k, rng):
            for rows in (16, 32, 64, 128, shrink_parts(n, k, d_in, rank)[0]):
                tiles = walk_tiles(offsets, n, k, rows)
                assert len(tiles) <= max_tiles(n, k, rows), (n, k, rows, offsets)
                assert sorted(p for _, p0, p1 in tiles for p in range(p0, p1)) == list(range(n))
                owner = [next((g for g in range(k) if offsets[g] <= p < offsets[g + 1]), -1) for p in (0, n // 2, n - 1)]
                assert [next(g for g, p0, p1 in tiles if p0 <= p < p1) for p in (0, n // 2, n - 1)] == owner


def test_workgroups_take_every_block_once():
    """The order in which an XCD's workgroups (every eighth) take neighbouring blocks."""
    for grid in [1, 2, 7, 8, 9, 15, 16, 17, 255, 256, 257, 2048, 2051]:
        blocks = [(b & 7) * (grid >> 3) + min(b & 7, grid & 7) + (b >> 3) for b in range(grid)]
        assert sorted(blocks) == list(range(grid))
