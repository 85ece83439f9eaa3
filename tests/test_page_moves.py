"""Forks, compaction and copies of pages (ffai_page_fork, ffai_page_compact,
ffai_kv_copy_keys) against a restatement row by row on the host, number by
number."""

import random

import pytest
import torch

DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def pages(n):
    return (n + 63) // 64


def build(B, mp, length, spare, seed, shared=0.0):
    """(lens, table, stack, count, pool's size): rows of up to `length` keys whose
    pages are shuffled; a share of the rows names whole pages of the row before."""
    rng = random.Random(seed)
    lens = [rng.choice([0, 1, 63, 64, 65, length, rng.randint(0, length)]) for _ in range(B)]
    lens = [min(n, length, mp * 64) for n in lens]
    size = sum(pages(n) for n in lens) + spare + 1
    ids = list(range(size))
    rng.shuffle(ids)
    table = [[rng.choice([-1, 10 ** 9, -7]) for _ in range(mp)] for _ in range(B)]  # stale entries
    named = set()
    for b, n in enumerate(lens):
        for i in range(pages(n)):
            table[b][i] = ids.pop()
        if b and rng.random() < shared:
            for i in range(min(pages(n), pages(lens[b - 1])) - 1):
                ids.append(table[b][i])
                table[b][i] = table[b - 1][i]
        named |= {table[b][i] for i in range(pages(n))}
    free = [p for p in ids if p not in named][:-1]  # one page is someone else's
    return lens, table, free + [-1] * (size - len(free)), len(free), size


def fork(src, lens, table, stack, count, keep=None):
    """The fork row by row."""
    mp, stack = len(table[0]), list(stack)
    rows, ns = [], []
    for b, s in enumerate(src):
        n = lens[s] if s >= 0 else 0
        if keep is not None:
            n = min(n, max(0, keep[b]))
        ns.append(n)
        rows.append((table[s][:pages(n)] if s >= 0 else []))
    refs = {}
    for b, r in enumerate(rows):
        for p in r:
            refs.setdefault(p, []).append(b)
    old = {p for t, n in zip(table, lens) for p in t[:pages(n)]}
    gone = sorted(p for p in old if p not in refs)
    stack[count:count + len(gone)] = gone
    count += len(gone)
    writes = lambda b, p: ns[b] % 64 and rows[b][-1] == p  # noqa: E731
    copies = []
    for b, r in enumerate(rows):
        if not ns[b] % 64:
            continue
        who = refs[r[-1]]
        writers = [x for x in who if writes(x, r[-1])]
        if len(who) > 1 and not (len(writers) == len(who) and writers[0] == b):
            copies.append(b)
    c_src, c_dst, c_keys = [-1] * len(src), [-1] * len(src), [0] * len(src)
    out = [r + [-1] * (mp - len(r)) for r in rows]
    for k, b in enumerate(copies):
        last = len(rows[b]) - 1
        if k < count:
            fresh = stack[count - 1 - k]
            c_src[b], c_dst[b], c_keys[b] = rows[b][-1], fresh, ns[b] % 64
            out[b][last] = fresh
        else:
            out[b][last] = -1
            ns[b] -= ns[b] % 64
    return out, ns, c_src, c_dst, c_keys, max(0, count - len(copies)), stack


def run_fork(src, lens, table, stack, count, keep=None, size=None):
    from ffai_b200 import kvcache
    d = lambda x: i32(x).to(DEV)  # noqa: E731
    free = d(stack)
    f = kvcache.fork_pages(d(src), d(lens), d(table), free, d([count]),
                           keep=None if keep is None else d(keep), num_pages=size)
    return (f.block_table.tolist(), f.lens.tolist(), f.copy_src.tolist(), f.copy_dst.tolist(),
            f.copy_keys.tolist(), f.free_count.item(), free.tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [0.0, 0.7])
@pytest.mark.parametrize("B,mp,length,spare", [(1, 1, 64, 3), (1, 3, 130, 0), (5, 7, 448, 5),
                                               (60, 24, 1500, 40), (33, 2, 100, 1), (513, 6, 300, 600),
                                               (1000, 64, 4096, 10)])
def test_fork(B, mp, length, spare, shared):
    from ffai_b200 import attention
    for seed in range(4):
        rng = random.Random(seed * 100 + B)
        lens, table, stack, count, size = build(B, mp, length, spare, seed, shared)
        kinds = {
            "beams": ([rng.randrange(B) for _ in range(B)], None),
            "cut": (list(range(B)), [max(0, n - rng.randint(0, 9)) for n in lens]),
            "ends": ([-1 if rng.random() < 0.4 else b for b in range(B)], None),
            "more": ([rng.randint(-2, B - 1) for _ in range(2 * B + 1)],
                     [rng.randint(-5, length) for _ in range(2 * B + 1)]),
            "one": ([rng.randrange(B)] * 7, None),
            "none": ([-1], None),
        }
        for name, (src, keep) in kinds.items():
            want = fork(src, lens, table, stack, count, keep)
            got = run_fork(src, lens, table, stack, count, keep)
            for g, w, what in zip(got, want, ("table", "lens", "src", "dst", "keys", "count")):
                assert g == w, (name, seed, what)
            assert got[6][:got[5]] == want[6][:got[5]]
            # the same again: nothing of a call is left for the next
            assert run_fork(src, lens, table, stack, count, keep) == got
    attention.sync(0)


@pytest.mark.gpu
def test_fork_keeps_pages_apart_and_loses_none():
    """Steps of a beam search in a row: every page is named, free or lost to nobody,
    and no two rows write to one page."""
    from ffai_b200 import attention, kvcache
    rng = random.Random(3)
    B, mp = 12, 9
    size = B * mp
    d = lambda x: i32(x).to(DEV)  # noqa: E731
    lens, table = d([0] * B), d([[-1] * mp] * B)
    free, count = d(list(range(size))), d([size])
    for step in range(60):
        plan = kvcache.plan_pages(lens, d([rng.choice([0, 1, 1, 5, 30]) for _ in range(B)]), free, count,
                                  table, slot_cap=400)
        lens, count = plan.lens, plan.free_count
        src = [rng.randrange(B) if rng.random() < 0.5 else b for b in range(B)]
        if step % 7 == 6:
            src[rng.randrange(B)] = -1
        keep = [max(0, int(lens[max(s, 0)]) - rng.choice([0, 0, 0, 3, 90])) for s in src]
        f = kvcache.fork_pages(d(src), lens, table, free, count, keep=d(keep))
        table, lens, count = f.block_table, f.lens, f.free_count
        names = {}
        for b, (row, n) in enumerate(zip(table.tolist(), lens.tolist())):
            for i, p in enumerate(row):
                assert (p >= 0) == (i < pages(n))
                if p >= 0:
                    names.setdefault(p, []).append((b, n % 64 != 0 and i == n // 64))
        for p, who in names.items():
            assert len(who) == 1 or not any(w for _, w in who), p
        left = free.tolist()[:count.item()]
        assert len(set(left)) == len(left) and not set(left) & set(names)
        assert len(left) + len(names) == size
        if step % 5 == 4:
            c = kvcache.compact_pages(lens, table, free, count)
            moves = [(a, b) for a, b in zip(c.copy_src.tolist(), c.copy_dst.tolist()) if a >= 0]
            assert {a for a, _ in moves} <= set(names) and {b for _, b in moves} <= set(left)
            table, free = c.block_table, c.free_pages
            live = {p for row in table.tolist() for p in row if p >= 0}
            assert live == set(range(len(names)))
            assert free.tolist()[:count.item()] == list(range(size - 1, len(names) - 1, -1))
    attention.sync(0)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["src", "length", "page", "stack", "count", "full"])
def test_fork_reports_bad_input(what):
    from ffai_b200 import attention
    lens, table, stack, count = [70, 10], [[0, 1], [2, -1]], [3, 4, -1, -1, -1], 2
    src, want = [0, 0, 1], None
    if what == "src":
        src = [0, 0, 2]
        want = ([[0, 1], [0, 2], [-1, -1]], [70, 70, 0])  # (page 2 went back before)
    elif what == "length":
        lens = [70, 129]
        want = ([[0, 1], [0, 4], [-1, -1]], [70, 70, 0])
    elif what == "page":
        table = [[5, 1], [2, -1]]
        want = ([[-1, 1], [-1, 4], [2, -1]], [70, 70, 10])
    elif what == "stack":
        stack = [3, 5, -1, -1, -1]
        want = ([[0, 1], [0, -1], [2, -1]], [70, 64, 10])
    elif what == "count":
        count = -3
        want = ([[0, 1], [0, -1], [2, -1]], [70, 64, 10])
    else:  # a page that goes back finds the stack full
        src, stack, count = [0], [3, 4], 2
        want = ([[0, 1]], [70])
    try:
        got = run_fork(src, lens, table, stack, count, size=5)
        assert (got[0], got[1]) == want
    finally:
        with pytest.raises(attention.AttnError):
            attention.sync(0)
    # and the next call finds its words clear
    got = run_fork([0, 0, 1], [70, 10], [[0, 1], [2, -1]], [3, 4, -1, -1, -1], 2, size=5)
    assert got[:6] == ([[0, 1], [0, 4], [2, -1]], [70, 70, 10], [-1, 1, -1], [-1, 4, -1], [0, 6, 0], 1)
    attention.sync(0)


def compact(lens, table, stack, count):
    used = [(b, i) for b, n in enumerate(lens) for i in range(pages(n))]
    live = sorted({table[b][i] for b, i in used})
    idle = set(stack[:count])
    every = sorted(set(live) | idle)
    low = set(every[:len(live)])
    movers, holes = [p for p in live if p not in low], [p for p in every if p in low and p in idle]
    to = dict(zip(movers, holes))
    out = [list(r) for r in table]
    for b, i in used:
        out[b][i] = to.get(out[b][i], out[b][i])
    return out, every[len(live):][::-1] + stack[count:], movers, holes


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [0.0, 0.7])
@pytest.mark.parametrize("B,mp,length,spare", [(1, 1, 64, 0), (1, 3, 130, 5), (5, 7, 448, 50),
                                               (60, 24, 1500, 400), (33, 2, 100, 1), (513, 6, 300, 3000),
                                               (1000, 64, 4096, 20000)])
def test_compact(B, mp, length, spare, shared):
    from ffai_b200 import attention, kvcache
    d = lambda x: i32(x).to(DEV)  # noqa: E731
    for seed in range(4):
        lens, table, stack, count, _ = build(B, mp, length, spare, seed, shared)
        want = compact(lens, table, stack, count)
        for _ in range(2):
            c = kvcache.compact_pages(d(lens), d(table), d(stack), d([count]))
            assert c.block_table.tolist() == want[0]
            assert c.free_pages.tolist() == want[1]
            n = len(want[2])
            src, dst = c.copy_src.tolist(), c.copy_dst.tolist()
            assert src[:n] == want[2] and dst[:n] == want[3]
            assert set(src[n:]) | set(dst[n:]) <= {-1}
    attention.sync(0)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["length", "page", "stack", "count", "twice", "both"])
def test_compact_moves_nothing_on_bad_input(what):
    from ffai_b200 import attention, kvcache
    lens, table, stack, count = [70, 10], [[7, 1], [9, -1]], [3, 4, 0, -1, -1, -1, -1, -1, -1, -1], 3
    if what == "length":
        lens[1] = -1
    elif what == "page":
        table[0][0] = 10
    elif what == "stack":
        stack[1] = -2
    elif what == "count":
        count = 11
    elif what == "twice":
        stack[1] = 3
    else:
        stack[1] = 9
    d = lambda x: i32(x).to(DEV)  # noqa: E731
    try:
        c = kvcache.compact_pages(d(lens), d(table), d(stack), d([count]))
        assert c.block_table.tolist() == table and c.free_pages.tolist() == stack
        assert set(c.copy_src.tolist()) | set(c.copy_dst.tolist()) == {-1}
    finally:
        with pytest.raises(attention.AttnError):
            attention.sync(0)
    c = kvcache.compact_pages(d([70, 10]), d([[7, 1], [9, -1]]), d([3, 4, 0, -1, -1, -1, -1, -1, -1, -1]), d([3]))
    assert c.block_table.tolist() == [[0, 1], [3, -1]]
    assert c.copy_src.tolist()[:3] == [7, 9, -1] and c.copy_dst.tolist()[:3] == [0, 3, -1]
    attention.sync(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H,counted", [(1, 1, True), (7, 3, True), (40, 20, False), (700, 2, True),
                                         (3000, 8, False)])
def test_copies(n, H, counted, dtype):
    from ffai_b200 import attention, kvcache
    g = torch.Generator().manual_seed(n)
    N = 2 * n + 3
    perm = torch.randperm(N, generator=g)
    src, dst = perm[:n].to(torch.int32), perm[n:2 * n].to(torch.int32)
    src[torch.rand(n, generator=g) < 0.2] = -1
    dst[torch.rand(n, generator=g) < 0.1] = -5
    keys = torch.randint(0, 65, (n,), generator=g, dtype=torch.int32)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    info = torch.iinfo(bits)  # any bits: NaN and infinities are copied as they are
    k, v = (torch.randint(info.min, info.max, (N, H, 64, 64), generator=g, dtype=bits).view(dtype)
            for _ in range(2))
    kd, vd = k.to(DEV), v.to(DEV)
    kvcache.copy_pages(kd, vd, src.to(DEV), dst.to(DEV), keys=keys.to(DEV) if counted else None)
    for want, got in ((k, kd), (v, vd)):
        want = want.clone()
        for a, b, m in zip(src.tolist(), dst.tolist(), keys.tolist()):
            if a >= 0 and b >= 0:
                m = m if counted else 64
                want[b, :, :m] = want[a, :, :m]
        assert torch.equal(got.cpu().view(bits), want.view(bits))
    attention.sync(0)


@pytest.mark.gpu
def test_copies_past_32_bits():
    """A pool of more than 2^32 bytes."""
    from ffai_b200 import kvcache
    N = (1 << 32) // (64 * 64 * 2 * 4) + 40
    k = torch.zeros((N, 4, 64, 64), dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    k[N - 2], v[N - 2] = 3.0, 4.0
    kvcache.copy_pages(k, v, i32([N - 2, 1]).to(DEV), i32([N - 1, 2]).to(DEV))
    assert (k[N - 1] == 3).all() and (v[N - 1] == 4).all() and (k[0] == 0).all() and (k[N - 3] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("src,dst,keys", [([4], [0], [64]), ([0], [4], [64]), ([0], [1], [65]),
                                          ([0], [1], [-1])])
def test_copies_report_bad_input(src, dst, keys):
    from ffai_b200 import attention, kvcache
    k = torch.arange(4, device=DEV, dtype=torch.float32).view(4, 1, 1, 1).expand(4, 1, 64, 64).contiguous()
    v, d = k.clone(), lambda x: i32(x).to(DEV)
    try:
        kvcache.copy_pages(k, v, d(src), d(dst), keys=d(keys))
        assert [x.unique().item() for x in k] == [0, 1, 2, 3]
    finally:
        with pytest.raises(attention.AttnError):
            attention.sync(0)


@pytest.mark.gpu
def test_streams_and_captures_do_not_share_words():
    """Forks on two streams and in two graphs captured on one stream, replayed
    together, as alone."""
    from ffai_b200 import attention
    from ffai_b200 import kvcache
    d = lambda x: i32(x).to(DEV)  # noqa: E731
    jobs = []
    for seed in (1, 2, 3, 4):
        lens, table, stack, count, _ = build(700, 24, 1500, 800, seed, 0.5)
        rng = random.Random(seed)
        src = [rng.randrange(700) for _ in range(700)]
        want = fork(src, lens, table, stack, count)
        jobs.append((want, (d(src), d(lens), d(table), d(stack), d([count]))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for want, args in jobs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kvcache.fork_pages(*args))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        eager = []
        for s, g, (want, args) in zip(streams, graphs, jobs[2:]):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(kvcache.fork_pages(*args))
        torch.cuda.synchronize()
        for f, (want, _) in zip(outs + eager, jobs):
            assert f.block_table.tolist() == want[0] and f.lens.tolist() == want[1]
            assert f.copy_dst.tolist() == want[3] and f.free_count.item() == want[5]
    attention.sync(0)


def test_refusals_without_a_device():
    from ffai_b200 import kvcache
    t = i32([[0, 1]])
    with pytest.raises(ValueError):
        kvcache.fork_pages(i32([0]), i32([5]), t, i32([2, 3]), i32([2]))
    with pytest.raises(ValueError):
        kvcache.compact_pages(i32([5]), t, i32([2, 3]), i32([2]))
    with pytest.raises(ValueError):
        kvcache.copy_pages(torch.zeros(2, 1, 64, 64), torch.zeros(2, 1, 64, 64), i32([0]), i32([1]))


@pytest.mark.gpu
def test_refusals():
    from ffai_b200 import _abi, attention, kvcache
    d = lambda x: i32(x).to(DEV)  # noqa: E731
    t, lens, free, count = d([[0, 1], [2, 3]]), d([5, 6]), d([4, 5]), d([2])
    with pytest.raises(ValueError):  # lens of another length
        kvcache.fork_pages(d([0]), d([5]), t, free, count)
    with pytest.raises(ValueError):  # 64-bit rows
        kvcache.fork_pages(d([0]).long(), lens, t, free, count)
    with pytest.raises(ValueError):  # one keep for two rows
        kvcache.fork_pages(d([0, 1]), lens, t, free, count, keep=d([1]))
    with pytest.raises(ValueError):  # a strided table
        kvcache.fork_pages(d([0]), lens, t[:, ::2], free, count)
    with pytest.raises(attention.AttnError):  # no new rows
        kvcache.fork_pages(d([]), lens, t, free, count)
    k = torch.zeros(4, 1, 64, 64, device=DEV)
    with pytest.raises(ValueError):
        kvcache.copy_pages(k, k.half(), d([0]), d([1]))
    with pytest.raises(ValueError):
        kvcache.copy_pages(k, k.clone(), d([0]), d([1, 2]))
    kvcache.copy_pages(k, k.clone(), d([]), d([]))
    lib, ctx, p = _abi.load(), attention.context(0), t.data_ptr()
    # outputs over inputs
    assert lib.ffai_page_fork(ctx, 2, 1, 2, 6, lens.data_ptr(), None, lens.data_ptr(), p, free.data_ptr(), 2,
                              count.data_ptr(), p, free.data_ptr(), p, p, p, p, None) == _abi.ERR_INVALID
    assert lib.ffai_page_compact(ctx, 2, 2, 6, lens.data_ptr(), p, free.data_ptr(), 2, count.data_ptr(),
                                 count.data_ptr(), count.data_ptr(), p, p, 1, None) == _abi.ERR_INVALID
