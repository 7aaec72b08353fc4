"""CPU emulation of how the cache's decode kernel cuts its work: every unit is done by exactly one CTA,
and every part of a segment lands in the workspace slot from which the combine kernel reads it.

The arithmetic is the kernel's (csrc/cache_decode.cuh): a segment costs its units and a start of two; the
cost of all segments is cut into equal ranges, one a CTA; a CTA passes over starts."""
import random

import pytest

START = 2       # kCdSegmentCost


def segments_of(lens, rows, heads):
    """(sequence, segment, units) of every segment with units, in the kernel's order."""
    out = []
    for b, (n, r) in enumerate(zip(lens, rows)):
        units = -(-n // 128) if r else 0
        if units:
            out += [(b, s, units) for s in range(heads * -(-r // 8))]
    return out


def walk(segs, grid):
    """What each CTA does: (cta, segment index, units, slot or None), and each segment's (first, last) CTA as noted."""
    base, at = [], 0
    for _, _, units in segs:
        base.append(at)
        at += units + START
    total = at
    ctas = min(grid, total)
    done, info = [], {}
    for c in range(ctas):
        u0, u1 = total * c // ctas, total * (c + 1) // ctas
        for i, (_, _, units) in enumerate(segs):
            first = base[i] + START                     # cost position of the segment's first unit
            a, e = max(first, u0), min(first + units, u1)
            if a >= e:
                continue
            partial = first < u0 or first + units > u1
            slot = 2 * c + (1 if first >= u0 else 0)
            done.append((c, i, range(a - first, e - first), slot if partial else None))
            if a == first:
                info[i] = (c, ((first + units) * ctas - 1) // total)
    return done, info


@pytest.mark.parametrize("seed", range(60))
def test_ranges_cover_every_unit_and_slots_agree(seed):
    rng = random.Random(seed)
    batch, heads = rng.choice([1, 1, 2, 7, 40]), rng.choice([1, 2, 8])
    top = rng.choice([1, 130, 2000, 20000])
    lens = [rng.choice([0, rng.randint(1, top), top]) for _ in range(batch)]
    rows = [rng.choice([0, 1, 4, 8, 9, 20, 32]) for _ in range(batch)]
    segs = segments_of(lens, rows, heads)
    if not segs:
        return
    for grid in (1, 5, 148, 444):
        done, info = walk(segs, grid)
        seen, used = {}, {}
        for c, i, units, slot in done:
            for u in units:
                assert (i, u) not in seen
                seen[i, u] = c
            if slot is not None:
                assert slot not in used, "a slot written twice"
                used[slot] = i
        assert len(seen) == sum(n for _, _, n in segs)
        for i, (_, _, n) in enumerate(segs):
            first, last = info[i]
            assert seen[i, 0] == first and seen[i, n - 1] == last
            if first == last:
                assert i not in used.values()           # written at once
                continue
            # what the combine kernel reads: slot 1 of the first CTA, slot 0 of the others, none of them idle
            read = [2 * (first + c) + (1 if c == 0 else 0) for c in range(last - first + 1)]
            assert sorted(s for s, j in used.items() if j == i) == sorted(read)


def test_a_cta_with_a_start_only_does_nothing():
    done, info = walk([(0, 0, 1)], 444)
    assert len(done) == 1 and info[0] == (2, 2)         # three positions of cost, the unit is the last
