"""Where the prefix kernel on tcgen05 leaves its partial results, in whole
numbers: the division of the work into steps on a line, chunks and segments, and
the size of the workspace, as the kernel and the host compute them.  No two
partials share a slot, and none lies behind the workspace, whatever the groups."""

import random

import pytest


def plan(sms, spare, kv, R, sizes, lens, batch, table_pages):
    """(slots of all partials, size of the workspace in slots)."""
    # the host, from what it knows: table width, groups, rows of the batch
    units = kv * (len(sizes) + (batch * R + 255) // 256)
    grid = max(1, min(sms - spare, units * ((table_pages + 1) // 2)))
    room = 3 * grid + units
    # the device, from the lengths
    dims = []
    for s, n in zip(sizes, lens):
        rows = s * R
        mu = (rows + 255) // 256
        dims.append((mu, int(rows - (mu - 1) * 256 <= 128), (n + 127) // 128 if rows else 0))

    def steps(d, blocks):
        return (d[0] - d[1]) * blocks + d[1] * ((blocks + 1) // 2)

    def line(d, share, even):
        n = steps(d, d[2])
        return -(-n // share) * share if even else n
    total = kv * sum(steps(d, d[2]) for d in dims)
    if total == 0:
        return [], room
    share, even = -(-total // grid), False
    for longer in (0, 1):  # heads begin on a CTA of their own where that costs a step at most
        if not even and kv * sum(line(d, share + longer, True) // (share + longer) for d in dims) <= grid:
            share, even = share + longer, True
    slots, lin, seg0 = [], 0, 0
    for mu, single, nb in dims:
        if nb == 0:
            continue
        d, whole = (mu, single, nb), (nb + 1) & ~1
        cl = whole if mu == 1 else min((share + 1) & ~1, whole)
        chunks = -(-nb // cl)
        for h in range(kv):
            for q in range(chunks):
                n = min(cl, nb - q * cl)
                for m in range(mu):
                    first = lin + h * line(d, share, even) + steps(d, q * cl) + m * n
                    last = first + ((n + 1) // 2 if single and m == mu - 1 else n) - 1
                    assert last // share < grid
                    seg = seg0 + (h * chunks + q) * mu + m
                    slots += [c + seg for c in range(first // share, last // share + 1)]
        lin += kv * line(d, share, even)
        seg0 += kv * mu * chunks
    return slots, room


@pytest.mark.parametrize("seed", range(8))
def test_slots_are_distinct_and_within_the_workspace(seed):
    rng = random.Random(seed)
    for _ in range(250):
        groups, kv, pages = rng.choice([1, 1, 2, 3, 5, 12, 40]), rng.choice([1, 2, 3, 8, 20]), \
            rng.choice([5, 6, 7, 33, 130, 513, 1000])
        sizes = [rng.choice([0, 1, 2, 7, 40, 130, 600]) for _ in range(groups)]
        lens = [rng.choice([0, 1, rng.randint(1, pages * 64), pages * 64]) for _ in range(groups)]
        sms = rng.choice([148, 148, 1, 2, 7, 60])
        batch = max(1, sum(sizes) + rng.choice([0, 0, 3]))
        slots, room = plan(sms, rng.choice([0, sms // 3, sms // 2]), kv, rng.choice([1, 2, 4, 16, 17]),
                           sizes, lens, batch, pages)
        assert len(slots) == len(set(slots))
        assert max(slots, default=0) < room
