"""Page plans, releases and slot writes on the device against the same rules
written out one request at a time."""

import pytest
import torch

DEV = "cuda:0"


def plan_by_hand(lens, new, free, count, table, cap, base):
    """The plan of ffai_page_plan, request by request."""
    table = [list(r) for r in table]
    mp = len(table[0])
    out, cu, used = [], [0], 0
    slots, pos = [-1] * cap, [0] * cap
    want_pages = 0
    for b, (n, w) in enumerate(zip(lens, new)):
        ok = n >= 0 and w >= 0 and n + w <= mp * 64
        need = (n + w + 63) // 64 - (n + 63) // 64 if ok else 0
        first = want_pages
        want_pages += need
        start = cu[-1]
        cu.append(start + max(w, 0))
        if not (ok and (need == 0 or want_pages <= count) and cu[-1] <= cap):
            out.append(n)
            continue
        for j in range(need):
            table[b][(n + 63) // 64 + j] = free[count - 1 - first - j]
        if need:
            used = want_pages
        for t in range(w):
            at = n + t
            slots[start + t] = table[b][at // 64] * 64 + at % 64
            pos[start + t] = at + (base[b] if base else 0)
        out.append(n + w)
    return table, out, cu, slots, pos, count - used


def make(B, mp, length, new, seed, spare=None):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, length + 1, (B,), generator=g)
    want = torch.randint(0, new + 1, (B,), generator=g)
    ids = torch.randperm(B * mp, generator=g)
    table = torch.full((B, mp), -1)
    at = 0
    for b in range(B):
        n = (int(lens[b]) + 63) // 64
        table[b, :n] = ids[at:at + n]
        at += n
    free = torch.full((B * mp,), -5)
    rest = ids[at:]
    count = rest.numel() if spare is None else min(spare, rest.numel())
    free[:count] = rest[:count]
    return lens, want, free, count, table


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV).contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("B,mp,length,new,spare,cap_off", [
    (1, 1, 0, 1, None, 0), (1, 4, 63, 2, None, 3), (5, 8, 448, 1, None, 0),
    (32, 16, 900, 70, None, 11), (33, 16, 900, 70, 9, 0), (200, 8, 500, 40, 60, -700),
    (511, 6, 300, 90, None, 1), (513, 6, 300, 90, 300, 0), (3000, 4, 250, 20, None, 100),
    (40, 5, 320, 100, None, 0), (16384, 2, 100, 3, None, 0), (4, 70, 0, 4400, None, 0)])
def test_plan(B, mp, length, new, spare, cap_off):
    from ffai_b200 import kvcache
    lens, want, free, count, table = make(B, mp, length, new, B * 7 + mp, spare)
    base = torch.arange(B) * 3
    cap = max(0, int(want.sum()) + cap_off)
    args = (i32(lens), i32(want), i32(free), i32([count]))
    dev_table = i32(table)
    for _ in range(2):  # a plan can be repeated
        p = kvcache.plan_pages(*args, dev_table, slot_cap=cap, pos_base=i32(base))
        t, out, cu, slots, pos, left = plan_by_hand(lens.tolist(), want.tolist(), free.tolist(),
                                                    count, table.tolist(), cap, base.tolist())
        assert dev_table.tolist() == t
        assert p.lens.tolist() == out
        assert p.cu_new.tolist() == cu
        assert p.slots.tolist() == slots
        assert p.positions.tolist() == pos
        assert p.free_count.tolist() == [left]


@pytest.mark.gpu
def test_plan_without_positions_base():
    from ffai_b200 import kvcache
    table = i32([[3, -1]])
    p = kvcache.plan_pages(i32([63]), i32([2]), i32([9, 8]), i32([2]), table, slot_cap=4, num_pages=10)
    assert p.slots.tolist() == [3 * 64 + 63, 8 * 64, -1, -1]
    assert p.positions.tolist() == [63, 64, 0, 0]
    assert table.tolist() == [[3, 8]] and p.free_count.tolist() == [1]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,count", [([-1], [1], 1), ([1], [-1], 1), ([1], [1], -1),
                                            ([1], [1], 99)])
def test_plan_reports_bad_lengths(lens, new, count):
    from ffai_b200 import attention, kvcache
    kvcache.plan_pages(i32(lens), i32(new), i32([1, 0]), i32([count]), i32([[0, -1]]), slot_cap=2)
    with pytest.raises(attention.AttnError) as e:
        attention.sync(0)
    assert e.value.status == -1


@pytest.mark.gpu
def test_plan_refusals():
    from ffai_b200 import attention, kvcache
    ok = dict(lens=i32([1]), new_tokens=i32([1]), free_pages=i32([1]), free_count=i32([1]),
              block_table=i32([[0, -1]]), slot_cap=1)
    with pytest.raises(ValueError):
        kvcache.plan_pages(**dict(ok, lens=i32([1]).long()))
    with pytest.raises(ValueError):
        kvcache.plan_pages(**dict(ok, new_tokens=i32([1, 2])))
    with pytest.raises(ValueError):
        kvcache.plan_pages(**dict(ok, block_table=i32([[0, -1], [1, 2]]).t()))
    with pytest.raises(attention.AttnError):
        kvcache.plan_pages(**ok, num_pages=0)
    B = 16385
    with pytest.raises(attention.Declined):
        kvcache.plan_pages(i32([0] * B), i32([0] * B), i32([1]), i32([1]),
                           torch.zeros(B, 1, dtype=torch.int32, device=DEV), slot_cap=1)


@pytest.mark.gpu
@pytest.mark.parametrize("B,mp,length,seed", [(1, 1, 64, 0), (5, 8, 448, 1), (513, 6, 300, 2),
                                              (3000, 4, 250, 3), (3, 300, 19200, 4)])
def test_release(B, mp, length, seed):
    from ffai_b200 import kvcache
    lens, _, free, count, table = make(B, mp, length, 1, seed)
    held = sum((n + 63) // 64 for n in lens.tolist())
    count = min(count, B * mp - held)
    g = torch.Generator().manual_seed(seed)
    done = torch.randint(0, 2, (B,), generator=g)
    stack, left = free.tolist(), count
    for b in range(B):
        if done[b]:
            for i in range((int(lens[b]) + 63) // 64):
                stack[left] = int(table[b, i])
                left += 1
    dev_free = i32(free)
    out, n = kvcache.release_pages(i32(lens), i32(done), i32(table), dev_free, i32([count]))
    assert dev_free.tolist() == stack and n.tolist() == [left]
    assert out.tolist() == [0 if d else n for d, n in zip(done.tolist(), lens.tolist())]


@pytest.mark.gpu
def test_release_past_the_stack_is_reported():
    from ffai_b200 import attention, kvcache
    free = i32([7, 7])
    kvcache.release_pages(i32([64, 128]), i32([1, 1]), i32([[0, -1], [1, 2]]), free, i32([0]))
    with pytest.raises(attention.AttnError):
        attention.sync(0)
    assert free.tolist()[0] == 0


@pytest.mark.gpu
def test_release_then_plan_reuses_pages():
    from ffai_b200 import kvcache
    table = i32([[4, 2], [1, -1]])
    free = i32([0, 3, -1, -1, -1])
    lens, count = kvcache.release_pages(i32([100, 5]), i32([1, 0]), table, free, i32([2]))
    p = kvcache.plan_pages(lens, i32([65, 1]), free, count, table, slot_cap=66)
    assert table.tolist() == [[2, 4], [1, -1]]
    assert p.free_count.tolist() == [2] and p.lens.tolist() == [65, 6]


@pytest.mark.gpu
@pytest.mark.parametrize("src,dst", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"),
                                     ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("T,H,form", [(1, 1, "dense"), (7, 3, "fused"), (65, 6, "fused"),
                                      (300, 20, "odd"), (1000, 8, "dense")])
def test_write_slots(src, dst, T, H, form):
    from ffai_b200 import kvcache
    DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
    g = torch.Generator().manual_seed(T + H)
    n_pages = T // 64 + 3
    # fused: two thirds of one row; odd: rows that start between 16-byte lines
    pad = {"dense": 0, "fused": H * 64, "odd": 3}[form]
    rows = torch.randn(T, pad + 2 * H * 64 + (5 if form == "odd" else 0), generator=g).to(DT[src])
    dev = rows.to(DEV)
    if form == "dense":
        k, v = (dev[:, i * H * 64:(i + 1) * H * 64].unflatten(1, (H, 64)).contiguous() for i in (0, 1))
    else:
        k, v = (dev[:, pad + i * H * 64:pad + (i + 1) * H * 64].unflatten(1, (H, 64)) for i in (0, 1))
    slots = torch.randperm(n_pages * 64, generator=g)[:T]
    slots[::5] = -1
    pool = torch.randn(2, n_pages, H, 64, 64, generator=g).to(DT[dst])
    want = pool.clone()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want[0, s // 64, :, s % 64] = k[t].cpu().float().to(DT[dst])
            want[1, s // 64, :, s % 64] = v[t].cpu().float().to(DT[dst])
    kp, vp = pool[0].to(DEV), pool[1].to(DEV)
    kvcache.write_slots(kp, vp, k, v, i32(slots))
    assert torch.equal(kp.cpu(), want[0]) and torch.equal(vp.cpu(), want[1])


@pytest.mark.gpu
def test_write_slots_keeps_bits_and_refuses():
    from ffai_b200 import attention, kvcache
    kp = torch.zeros(2, 1, 64, 64, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    odd = torch.tensor([float("nan"), float("inf"), -0.0, 1e-40], dtype=torch.bfloat16, device=DEV)
    new = odd.repeat(16).view(1, 1, 64)
    kvcache.write_slots(kp, vp, new, new, i32([70]))
    assert torch.equal(kp[1, 0, 6].view(torch.int16), new.view(64).view(torch.int16))
    kvcache.write_slots(kp, vp, new[:0], new[:0], i32([]))
    kvcache.write_slots(kp, vp, new, new, i32([128]))  # past the pool
    with pytest.raises(attention.AttnError):
        attention.sync(0)
    with pytest.raises(attention.Declined):
        kvcache.write_slots(kp, vp, new.half(), new.half(), i32([1]))
    with pytest.raises(ValueError):
        kvcache.write_slots(kp, vp, new.expand(1, 2, 64), new, i32([1]))
    with pytest.raises(ValueError):
        kvcache.write_slots(kp, vp[:1], new, new, i32([1]))


@pytest.mark.gpu
@pytest.mark.parametrize("new,cap", [([5, 1], 2), ([1000], 0), ([3, 700, 2], 9), ([2, 0, 9, 1], 5),
                                     ([-4, 6, 1], 3), ([2 ** 31 - 1, 2 ** 31 - 1, 5], 4)])
def test_plan_sums_requests_that_ask_for_more_than_the_rows(new, cap):
    """cu_new is the running sum whatever fits (of nothing for a negative
    request, and at most the largest int32)."""
    from ffai_b200 import attention, kvcache
    B = len(new)
    p = kvcache.plan_pages(i32([7] * B), i32(new), i32(list(range(8))), i32([8]),
                           i32([[8 + b, -1, -1] for b in range(B)]), slot_cap=cap, num_pages=20)
    want = [0]
    for n in new:
        want.append(want[-1] + max(n, 0))
    assert p.cu_new.tolist() == [min(c, 2 ** 31 - 1) for c in want]
    fits = [n >= 0 and 7 + n <= 192 and want[b + 1] <= cap for b, n in enumerate(new)]
    assert p.lens.tolist() == [7 + n if f else 7 for n, f in zip(new, fits)]
    rows = [(8 + b) * 64 + 7 + i if f else -1 for b, (n, f) in enumerate(zip(new, fits))
            for i in range(min(max(n, 0), cap))]
    assert p.slots.tolist() == (rows + [-1] * cap)[:cap]
    assert p.free_count.tolist() == [8]
    if min(new) < 0:
        with pytest.raises(attention.AttnError):
            attention.sync(0)
    attention.sync(0)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,done,count,cap", [
    ([64, 128], [1, 1], 0, 2), ([64, 128, 5], [1, 1, 1], 0, 2), ([10, 300, 64, 1], [1, 0, 1, 1], 5, 6),
    ([300, 64], [1, 1], 3, 3), ([192, 64], [0, 1], 4, 5), ([640] * 700, [1] * 700, 11, 1003)])
def test_release_counts_the_pages_it_pushed(lens, done, count, cap):
    """Pages past the stack's end are not pushed; the count is of those that
    were, and a plan hands out nothing else."""
    from ffai_b200 import attention, kvcache
    mp = max(1, max((n + 63) // 64 for n in lens))
    table = (torch.arange(len(lens) * mp) + cap).view(len(lens), mp)
    stack = [i if i < count else -9 for i in range(cap)]
    free = i32(stack)
    given = [int(table[b, j]) for b, n in enumerate(lens) if done[b] for j in range((n + 63) // 64)]
    want = (stack[:count] + given)[:cap]
    out, left = kvcache.release_pages(i32(lens), i32(done), i32(table), free, i32([count]))
    assert left.tolist() == [len(want)]
    assert free.tolist() == (want + stack[len(want):])[:cap]
    assert out.tolist() == [0 if d else n for n, d in zip(lens, done)]
    if count + len(given) > cap:
        with pytest.raises(attention.AttnError):
            attention.sync(0)
    attention.sync(0)
    tables = i32(torch.full((cap + 1, 1), -1))
    p = kvcache.plan_pages(i32([0] * (cap + 1)), i32([1] * (cap + 1)), free, left, tables,
                           slot_cap=cap + 1, num_pages=cap + len(lens) * mp)
    got = [t for (t,) in tables.tolist() if t >= 0]
    assert got == want[::-1] and p.lens.tolist() == [1] * len(want) + [0] * (cap + 1 - len(want))
    attention.sync(0)


def refused_plan(lens, new, free, count, table, num_pages, cap):
    """The rule for inputs that hold a bad count or page id: the stack has no
    pages under a bad count and ends at a bad id, and a request whose last page
    is bad and not full takes part as if it outgrew the table."""
    bad = lambda i: not 0 <= i < num_pages  # noqa: E731
    held_bad = [n % 64 != 0 and w > 0 and bad(table[b][n // 64])
                for b, (n, w) in enumerate(zip(lens, new))]
    usable = 0 if not 0 <= count <= len(free) else next(
        (i for i in range(count) if bad(free[count - 1 - i])), count)
    out, want, used = [], 0, 0
    t = [list(r) for r in table]
    slots, cu = [], 0
    for b, (n, w) in enumerate(zip(lens, new)):
        need = 0 if held_bad[b] else (n + w + 63) // 64 - (n + 63) // 64
        first, want, cu = want, want + need, cu + w
        if held_bad[b] or (need and want > usable) or cu > cap:
            out.append(n)
            slots += [-1] * w
            continue
        for j in range(need):
            t[b][(n + 63) // 64 + j] = free[count - 1 - first - j]
        used = max(used, want if need else 0)
        slots += [t[b][(n + i) // 64] * 64 + (n + i) % 64 for i in range(w)]
        out.append(n + w)
    return t, out, (slots + [-1] * cap)[:cap], count - used


@pytest.mark.gpu
@pytest.mark.parametrize("lens,new,free,count,table,cap", [
    # a count that is not one: what needs a page is refused, and the count stays
    ([63, 64], [1, 1], [5, 4], 99, [[0, -1], [1, -1]], 4),
    ([63, 64], [1, 1], [5, 4], -1, [[0, -1], [1, -1]], 4),
    ([0], [200], [5, 4, 3], 4, [[-1] * 4], 200),
    # a bad id on the stack, within, at the end of and behind what is asked for
    ([0, 0, 0], [1, 1, 1], [6, 7, 99, 5], 4, [[-1], [-1], [-1]], 3),
    ([0, 64, 10], [130, 1, 4], [8, 9, -2, 4, 5], 5, [[-1] * 3, [1, -1, -1], [2, -1, -1]], 140),
    ([0, 0], [1, 1], [99, 6, 5], 3, [[-1], [-1]], 2),
    ([0, 0], [64, 64], [5, 20], 2, [[-1], [-1]], 128),
    # a bad id in the table, where new keys go and where none do
    ([10, 10, 64], [1, 1, 1], [5, 4], 2, [[0, -1], [77, -1], [1, -1]], 3),
    ([100, 10], [60, 1], [5, 4], 2, [[0, -1, -1], [2, -1, -1]], 61),
    ([128, 10, 70], [1, 0, 1], [5, 4], 2, [[0, 50, -1], [-3, -1, -1], [60, 3, -1]], 3),
    # and many requests
    ([0] * 1200, [65] * 1200, list(range(700)) + [-1] + list(range(701, 3000)), 3000,
     [[-1, -1]] * 1200, 1200 * 65),
    ([1 + b % 64 for b in range(1200)], [1] * 1200, list(range(1200, 1240)), 40,
     [[b if b % 7 else -1, -1] for b in range(1200)], 1200),
])
def test_plan_refuses_bad_counts_and_pages(lens, new, free, count, table, cap):
    from ffai_b200 import attention, kvcache
    num_pages = 10 if len(lens) < 100 else 3000
    t, out, slots, left = refused_plan(lens, new, free, count, table, num_pages, cap)
    dev = i32(table)
    p = kvcache.plan_pages(i32(lens), i32(new), i32(free), i32([count]), dev, slot_cap=cap,
                           num_pages=num_pages)
    assert p.lens.tolist() == out
    assert p.slots.tolist() == slots
    assert dev.tolist() == t
    assert p.free_count.tolist() == [left]
    met = (out != [n + w for n, w in zip(lens, new)])  # nothing else refuses these
    if met:
        with pytest.raises(attention.AttnError) as e:
            attention.sync(0)
        assert e.value.status == -1
    attention.sync(0)
