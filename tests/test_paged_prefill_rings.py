"""CPU checks of who has seen what in the tcgen05 paged-attention kernel's rings of K and V tiles, for items
described by the library itself.

A wait on an mbarrier names the parity of a phase, so it cannot tell phase k from phase k - 2: it is sound only
where phase k - 1 of that slot, the copy before it, is over for certain.  Below a warp's knowledge is followed
item by item, copies landing as late as they can: what it has waited for itself, what a product that it saw
finished must have read (codes are converted in order, so all copies before that one too), and what the others
knew when it met them at a barrier.
"""
import ctypes
import random

import pytest

from kernelverse_b200 import _lib

FEW, DEEP, WIDE = 0, 1, 2
ROWS, KEYS = 256, 128          # of a tile of the tcgen05 kernel


def item(ql, kl, group, few_rows, tile, j0, j1):
    out = (ctypes.c_int * 7)()
    assert _lib.lib().kvb_selftest_paged_item(ql, kl, group, few_rows, tile, j0, j1, out) == 0
    return dict(zip(("kind", "rows", "T", "A", "B", "halves_a", "halves_b"), out))


def units(ql, kl, group, rows, keys, tile):
    out = (ctypes.c_int64 * 3)()
    assert _lib.lib().kvb_selftest_paged_units(ql, kl, group, rows, keys, tile, out) == 0
    return tuple(out)


def some_items(seed, few_rows):
    """The items of one CTA: those of consecutive requests, the first and the last one cut."""
    rng = random.Random(seed)
    items = []
    for _ in range(rng.randrange(2, 12)):
        group, ql = rng.choice((1, 2, 4, 5, 8)), rng.choice((1, 1, 2, 4, 20, 33, 64, 130, 300))
        kl = max(0, ql + rng.randrange(-20, 700))
        for tile in range(units(ql, kl, group, ROWS, KEYS, 0)[0]):
            n = units(ql, kl, group, ROWS, KEYS, tile)[1]
            j0 = rng.randrange(n) if not items else 0
            items.append(item(ql, kl, group, few_rows, tile, j0, n if rng.random() < 0.9 else rng.randrange(j0, n) + 1))
    return items


@pytest.mark.parametrize("seed", range(30))
def test_a_chain_leaves_out_one_tile_at_most_and_never_both(seed):
    for few in (0, 1):
        for it in some_items(seed, few):
            if it["kind"] != FEW:
                assert max(it["A"], it["B"]) == it["T"] and min(it["A"], it["B"]) >= it["T"] - 1
                per = 2 if it["kind"] == WIDE else 1
                assert all(0 <= per * it[c] - it[h] <= per - 1 for c, h in (("A", "halves_a"), ("B", "halves_b")))


def unsound_waits_on_codes(items, meet_after_wide, slots=4):
    """Waits of the softmax warps (group A, group B) for a few-row item's tiles in the ring of codes."""
    known, found, u, after_wide = [set(), set()], 0, 0, False
    for it in items:
        n = 2 * it["T"]
        if it["kind"] == FEW:
            if after_wide and meet_after_wide:
                known[0] = known[1] = known[0] | known[1]
            after_wide = False
            for c in range(2):
                for p in range(u, u + n):
                    found += p >= slots and p - slots not in known[c]
                    known[c] = known[c] | {p}
        else:
            for c, tiles in enumerate((it["A"], it["B"])):
                if tiles:
                    known[c] = known[c] | set(range(u + 2 * tiles))
            if it["kind"] == DEEP:
                known[0] = known[1] = known[0] | known[1]
            after_wide = it["kind"] == WIDE
        u += n
    return found


def test_few_row_items_wait_for_no_phase_that_may_lie_two_ahead():
    every = [some_items(seed, 1) for seed in range(400)]
    assert sum(unsound_waits_on_codes(items, False) for items in every) > 0       # what the meeting is for
    assert all(unsound_waits_on_codes(items, True) == 0 for items in every)


def unsound_waits_of_issuers(items, see_all, slots):
    """Waits of the MMA issuers (chain A, chain B) in the ring of 16-bit K and V tiles (K at even positions)."""
    known, found, u = [set(), set()], 0, 0
    for it in items:
        for c, tiles in enumerate((it["A"], it["B"])):
            for p in range(u, u + 2 * (it["T"] if see_all else tiles)):
                found += p >= slots and p - slots not in known[c]
                known[c].add(p)
        # the next item's query rows come once both chains' products of this one's have read them, and every K
        for c in range(2):
            known[c] |= {u + 2 * i for i in range(it["T"])}
        u += 2 * it["T"]
    return found


@pytest.mark.parametrize("slots", [3, 5, 8])
def test_issuers_wait_for_no_phase_that_may_lie_two_ahead(slots):
    every = [some_items(seed, 0) for seed in range(400)]
    assert sum(unsound_waits_of_issuers(items, False, slots) for items in every) > 0
    assert all(unsound_waits_of_issuers(items, True, slots) == 0 for items in every)
