"""How attention's form for steps divides its work, restated: the line of work of a batch, the CTAs' ranges
of it, and the counts by which CTAs that share a sequence and head find the last of them.  A CTA in which
a wait gave up arrives for what it shares all the same, so that every count is zero after every call."""

import random

import pytest

STAGE, ITEM_COST, MIN_STAGES = 128, 3, 2  # keys per stage; what an item costs beside its stages; stages per CTA at least


def plan(stages, kv_heads, grid):
    """(items, ranges): items (first place of its stages, behind its last) in order; ranges [begin, end) of the CTAs."""
    items, at = [], 0
    for st in stages:
        for _ in range(kv_heads if st else 0):
            items.append((at + ITEM_COST, at + ITEM_COST + st))
            at += ITEM_COST + st
    G = min(grid, max(1, at // MIN_STAGES))
    per, rest = divmod(at, G)
    starts = [c * per + min(c, rest) for c in range(G + 1)]

    def cta_of(x):
        return x // (per + 1) if x < rest * (per + 1) else rest + (x - rest * (per + 1)) // per

    return items, list(zip(starts, starts[1:])), cta_of


def shared_of(items, cta_of, begin, end):
    """Parts of a CTA's range and what it shares: [(item, stages, first CTA, contributors)]."""
    out = []
    for i, (a, b) in enumerate(items):
        lo, hi = max(begin, a), min(end, b)
        if lo < hi:
            first = cta_of(a)
            out.append((i, hi - lo, first, cta_of(b - 1) - first + 1))
    return out


def batches():
    rng = random.Random(5)
    yield [32], 8, 444
    yield [1024], 1, 444
    yield [1], 1, 296
    yield [1] * 1000, 8, 444
    yield [0, 0, 1, 0], 3, 7
    for _ in range(60):
        n = rng.randint(1, 200)
        yield [rng.choice([0, 1, 1, 2, rng.randint(1, 70)]) for _ in range(n)], rng.choice([1, 2, 5, 8]), rng.choice([1, 7, 148, 296, 444])


@pytest.mark.parametrize("stages,kv_heads,grid", list(batches()))
def test_ranges_cover_the_work_and_counts_return_to_zero(stages, kv_heads, grid):
    items, ranges, cta_of = plan(stages, kv_heads, grid)
    rng = random.Random(len(items))
    done = [0] * len(items)
    holders = [[] for _ in items]
    parts = []
    for c, (begin, end) in enumerate(ranges):
        mine = shared_of(items, cta_of, begin, end)
        parts.append([p for p in mine if p[3] > 1])
        assert len(parts[-1]) <= 2  # what the kernel has places for
        for i, st, first, n in mine:
            done[i] += st
            holders[i].append(c)
            # record 1 of the first CTA, record 0 of the others: no two items of a CTA in one record
        assert len({c == p[2] for p in parts[-1]}) == len(parts[-1])
    assert done == [b - a for a, b in items]
    firsts = []
    for i, (a, b) in enumerate(items):
        first = cta_of(a)
        assert holders[i] == list(range(first, cta_of(b - 1) + 1))
        if len(holders[i]) > 1:
            firsts.append(first)
    assert len(set(firsts)) == len(firsts)  # a count of its own for every shared item

    def call(count, failing, walk_on):
        """One call; `failing`: CTA -> shared items it has arrived for when a wait gives up."""
        merges = 0
        order = list(range(len(ranges)))
        rng.shuffle(order)
        for c in order:
            owed = parts[c]
            if c in failing and not walk_on:
                owed = owed[:failing[c]]
            for k, (i, _, first, n) in enumerate(owed):
                last = count[first] == n - 1
                count[first] = 0 if last else count[first] + 1
                merges += last and not (c in failing and k >= failing[c])
        return merges

    count = [0] * len(ranges)
    assert call(count, {}, True) == len(firsts) and not any(count)
    failing = {c: rng.randint(0, len(p)) for c, p in enumerate(parts) if rng.random() < 0.3}
    call(count, failing, True)
    assert not any(count)
    assert call(count, {}, True) == len(firsts) and not any(count)  # the call after it merges every item once
    short = {c: k for c, k in failing.items() if k < len(parts[c])}
    if short:  # arriving only for what was finished leaves a remainder to the next call
        call(count, short, False)
        assert any(count)
