"""CPU checks of the library's own division of the paged attention's work (host test hooks): units and tiles
against their definition in whole numbers, up to the largest lengths that the entry takes."""
import ctypes
import random

import pytest

from kernelverse_b200 import _lib

LIMIT = 1 << 30                 # tokens x heads of a group stay below


def units(ql, kl, group, rows, keys, tile):
    out = (ctypes.c_int64 * 3)()
    assert _lib.lib().kvb_selftest_paged_units(ql, kl, group, rows, keys, tile, out) == 0
    return tuple(out)


def units_by_definition(ql, kl, group, rows, keys, tile):
    """The keys 0 .. position of the tile's last row, in units; one at least."""
    last_token = (min((tile + 1) * rows, ql * group) - 1) // group
    return max(1, -(-max(0, kl - ql + last_token + 1) // keys))


@pytest.mark.parametrize("seed", range(60))
def test_units_before_every_tile(seed):
    rng = random.Random(seed)
    rows, keys = rng.choice(((256, 128), (64, 64), (64, 32)))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16, 71))
    ql = rng.choice((1, 2, 5, 64, 100, rng.randrange(1, 1500)))
    kl = rng.choice((0, 1, ql, max(0, ql - rng.randrange(1, 300)), ql + rng.randrange(0, 5000)))
    count, total = -(-ql * group // rows), 0
    for tile in range(count):
        n = units_by_definition(ql, kl, group, rows, keys, tile)
        assert units(ql, kl, group, rows, keys, tile) == (count, n, total)
        total += n
    assert units(ql, kl, group, rows, keys, count) == (count, 0, total)


def floor_sum(n, m, s, b):
    """sum over t < n of (b + s t) // m in whole numbers of any size, by the periods of s t modulo m."""
    total = 0
    while n > 0:
        total += n * (n - 1) // 2 * (s // m) + n * (b // m)
        s, b = s % m, b % m
        n, b, m, s = (s * n + b) // m, (s * n + b) % m, s, m
        if m == 0:
            break
    return total


def test_floor_sum_of_this_file():
    rng = random.Random(1)
    for _ in range(2000):
        n, m, s, b = rng.randrange(0, 50), rng.randrange(1, 40), rng.randrange(0, 90), rng.randrange(0, 90)
        assert floor_sum(n, m, s, b) == sum((b + s * t) // m for t in range(n))


@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 71, 128, 1000, 4099])
@pytest.mark.parametrize("rows,keys", [(256, 128), (64, 64), (64, 32)])
def test_units_of_the_longest_requests(group, rows, keys):
    """Lengths up to the refusal: products and sums that 32 bits barely hold."""
    rng = random.Random(group)
    most = (LIMIT - 1) // group
    for ql, kl in ((most, most), (most, 0), (most, most // 2), (1, most), (most // 3, most), (most - 1, most), (most, 1),
                   (rng.randrange(1, most), rng.randrange(0, most)), (rng.randrange(1, most), rng.randrange(0, most))):
        count = -(-ql * group // rows)
        for tile in {0, 1, count // 2, count - 1, count, rng.randrange(count)}:
            if tile > count:
                continue
            # tiles but the request's last end on whole rows; those whose last row lies before position 0 have one unit
            full = min(tile, count - 1)
            x0 = (kl - ql) * group + rows - 1
            skip = 0 if x0 >= 0 else min(full, (-x0 + rows - 1) // rows)
            before = full + floor_sum(full - skip, group * keys, rows, x0 + skip * rows)
            if tile == count:
                before += units_by_definition(ql, kl, group, rows, keys, count - 1)
            n = units_by_definition(ql, kl, group, rows, keys, tile) if tile < count else 0
            assert units(ql, kl, group, rows, keys, tile) == (count, n, before), (ql, kl, tile)


@pytest.mark.parametrize("seed", range(20))
def test_cta_of_a_unit(seed):
    """CTA c of n holds units [c W / n, (c + 1) W / n)."""
    rng = random.Random(seed)
    f = _lib.lib().kvb_selftest_paged_cta_of
    ctas = rng.choice((1, 7, 148, 296))
    total = rng.choice((ctas, ctas + 1, rng.randrange(ctas, 5000), (1 << 45) + rng.randrange(1 << 20)))
    for unit in [0, total - 1] + [rng.randrange(total) for _ in range(500)] + [
            x for c in range(ctas) for x in (total * c // ctas, total * (c + 1) // ctas - 1)]:
        c = f(unit, total, ctas)
        assert total * c // ctas <= unit < total * (c + 1) // ctas
    assert f(-1, total, ctas) == f(total, total, ctas) == f(0, 0, 1) == -1
