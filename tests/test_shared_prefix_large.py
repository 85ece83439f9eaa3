"""Attention over a shared prefix at the sizes where the prefix has a kernel of
its own, against the formula in 64 bits (computed on the device) on the same
16-bit operands; streams and captured calls.

Tolerances are those of the small sizes: with A = sum_j w_j |v_j| an output
errs by at most (u + 1e-4) A + u |o|, u = 2^-8 (bf16) or 2^-11 (f16, where a
weight below 2^-14 adds 2^-25 |v| a key, |v| < 5.5); the log-sum-exp by 2e-5,
plus 2^-23 of each of up to 18000 weights' sum, which is random: 2e-5 in all.
"""

import pytest
import torch

DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def build(prefix, sizes, own, heads, kv, q_len, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B = sum(sizes)
    pp, sp = max((n + 63) // 64 for n in prefix), max(1, (own + 63) // 64)
    n_pages = len(prefix) * pp + B * sp + 1
    shape = (n_pages, kv, 64, 64)
    kp = (torch.randn(shape, generator=g, device=DEV) * 1.5).to(dtype)
    vp = torch.randn(shape, generator=g, device=DEV).clamp(-5.5, 5.5).to(dtype)
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    ptab = ids[:len(prefix) * pp].view(len(prefix), pp).contiguous()
    stab = ids[len(prefix) * pp:len(prefix) * pp + B * sp].view(B, sp).contiguous()
    lens = [(i * 37) % (own + 1) for i in range(B)]
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    # behind the live keys of a last page: not numbers
    for table, ns in ((ptab, prefix), (stab, lens)):
        for i, n in enumerate(ns):
            if n % 64:
                kp[table[i, n // 64].long(), :, n % 64:] = float("nan")
                vp[table[i, n // 64].long(), :, n % 64:] = float("inf")
    q = torch.randn((B, q_len, heads, 64), generator=g, device=DEV).to(dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(q=q, k_pool=kp, v_pool=vp, prefix_table=ptab, prefix_lens=i32(prefix),
                group_starts=i32(starts), block_table=stab, seq_lens=i32(lens),
                lists=(prefix, lens, starts))


def gather(pool, pages, n):
    """(kv, n, 64) f64: the first n keys of a list of pages."""
    return pool[pages[:(n + 63) // 64].long()].transpose(0, 1).flatten(1, 2)[:, :n].double()


def reference(c, scale):
    prefix, lens, starts = c["lists"]
    B, n, H, _ = c["q"].shape
    kv = c["k_pool"].shape[1]
    o = torch.zeros((B, n, H, 64), dtype=torch.float64, device=DEV)
    a = torch.zeros_like(o)
    lse = torch.full((B, n, H), float("-inf"), dtype=torch.float64, device=DEV)
    for g in range(len(prefix)):
        pk, pv = (gather(c[x], c["prefix_table"][g], prefix[g]) for x in ("k_pool", "v_pool"))
        for b in range(starts[g], starts[g + 1]):
            k = torch.cat([pk, gather(c["k_pool"], c["block_table"][b], lens[b])], 1)
            v = torch.cat([pv, gather(c["v_pool"], c["block_table"][b], lens[b])], 1)
            qb = c["q"][b].double().transpose(0, 1).reshape(kv, H // kv, n, 64)
            s = torch.einsum("hgnd,hkd->hgnk", qb, k) * scale
            for i in range(n):
                s[:, :, i, prefix[g] + max(0, lens[b] - (n - 1 - i)):] = float("-inf")
            l = torch.logsumexp(s, 3)
            w = torch.exp(s - l.unsqueeze(3)).nan_to_num(0.0)
            o[b] = torch.einsum("hgnk,hkd->hgnd", w, v).flatten(0, 1).transpose(0, 1)
            a[b] = torch.einsum("hgnk,hkd->hgnd", w, v.abs()).flatten(0, 1).transpose(0, 1)
            lse[b] = l.flatten(0, 1).transpose(0, 1)
    return o, a, lse


def attend(c, **kw):
    from ffai_b200 import shared_prefix
    return shared_prefix.attend(c["q"], c["k_pool"], c["v_pool"], c["prefix_table"],
                                c["prefix_lens"], c["group_starts"], c["block_table"],
                                c["seq_lens"], scale=0.125, **kw)


CASES = {
    # prefix keys, sequences per group, own keys, heads, kv heads, q_len
    # few rows a KV head: tiles of 16
    "tiles": ([4097, 1, 0, 650], [3, 2, 2, 1], 130, 12, 4, 1),
    "tiles_one_sequence": ([8300], [1], 0, 7, 1, 3),
    "tiles_odd_rows": ([2000, 321], [5, 40], 65, 9, 3, 1),
    # many rows and long prefixes: tcgen05, own keys after it
    "units": ([8300], [50], 70, 12, 4, 2),
    "units_groups": ([8300, 1, 0, 129, 6000], [20, 0, 5, 25, 60], 200, 10, 2, 3),
    "units_one_tile": ([18000, 17999, 127], [33, 30, 1], 33, 15, 5, 1),
    # segments of one key block, that one of the kernel's two chains has no part in
    "units_of_one_block": ([1, 100, 129, 8300], [1, 2, 1, 60], 20, 24, 8, 2),
    "units_many": ([900, 2500], [100, 31], 40, 32, 4, 2),
    # and with long own keys: beside it
    "beside_odd_rows": ([12000], [91], 1600, 9, 3, 1),
    "beside_short": ([7000], [260], 300, 16, 8, 2),
    "beside_groups": ([5000, 0, 6400, 70], [60, 9, 70, 2], 1300, 8, 4, 4),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CASES)
def test_matches_the_formula(name, dtype):
    from ffai_b200 import attention
    attention.sync(0)
    c = build(*CASES[name], dtype, seed=len(name))
    out, lse = attend(c, with_lse=True)
    o, a, want = reference(c, 0.125)
    B, n, H, _ = c["q"].shape
    tol = (U[dtype] + 1e-4) * a + U[dtype] * o.abs() + 1e-7
    if dtype == torch.float16:
        keys = c["lists"][0][0] + max(c["lists"][1])
        tol = tol + keys * 2.0 ** -25 * 5.5 + 2.0 ** -24
    assert torch.isfinite(out).all()
    over = (out.double() - o).abs() - tol
    assert over.max().item() <= 0, f"{over.max():.3e} over"
    got = lse.double().view(H, B, n).permute(1, 2, 0)
    empty = want == float("-inf")
    assert torch.equal(got == float("-inf"), empty)
    assert (got[~empty] - want[~empty]).abs().max().item() <= 2e-5
    assert (out[empty] == 0).all()
    for _ in range(2):
        assert torch.equal(attend(c), out)
    attention.sync(0)  # no wait ran out, no table was out of range


@pytest.mark.gpu
def test_streams_do_not_share_partial_results():
    """Calls queued on two streams without any order between them."""
    cs = [build(*CASES[n], torch.bfloat16, seed=i)
          for i, n in enumerate(("beside_odd_rows", "units_groups"))]
    want = [attend(c) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attend(cs[i]))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for x in outs:
            assert torch.equal(x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiles", "units", "beside_odd_rows"])
def test_captured_and_replayed(name):
    """A capture makes its stream's workspace; replays follow the lengths and
    outlive a larger call on the same stream."""
    c = build(*CASES[name], torch.bfloat16, seed=3)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        g.capture_begin()
        out = attend(c)
        g.capture_end()
    s.synchronize()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attend(c))
    big = build(*CASES["beside_groups"], torch.bfloat16, seed=4)
    with torch.cuda.stream(s):
        attend(big)
    s.synchronize()
    c["seq_lens"] //= 2
    c["prefix_lens"] -= c["prefix_lens"] // 3
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, attend(c))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiles_odd_rows", "units_one_tile", "beside_odd_rows"])
def test_starts_that_do_not_rise_are_reported(name):
    """No group's prefix is attended then: the result is that of no prefixes."""
    from ffai_b200 import attention
    prefix, sizes, own, heads, kv, n = CASES[name]
    c = build([max(16000, prefix[0])] * 4, [1, 2, 3, sum(sizes) - 6], own, heads, kv, n, torch.bfloat16, seed=5)
    B = c["q"].shape[0]
    c["group_starts"].copy_(torch.tensor([3, 2, B, 1, B], dtype=torch.int32))
    out = attend(c)
    with pytest.raises(attention.AttnError) as e:
        attention.sync(0)
    assert e.value.status == -1
    none = dict(c, prefix_lens=torch.zeros_like(c["prefix_lens"]),
                group_starts=torch.tensor([0, 1, 3, 6, B], dtype=torch.int32, device=DEV))
    want = attend(none)
    attention.sync(0)
    U8 = 2.0 ** -7  # two ways to the same sums: each rounds weights and result once
    assert ((out.float() - want.float()).abs() <= U8 * 5.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [
    ([100], [3], 90, 6, 2, 5), ([200, 0], [2, 4], 130, 4, 4, 17), ([300], [9], 40, 10, 1, 3),
    CASES["tiles_one_sequence"], CASES["units"], CASES["beside_groups"],
], ids=["own_prefix", "two_tiles", "ten_heads", "tiles", "units", "beside"])
def test_a_bad_newest_key_reaches_its_own_query_alone(case, dtype):
    """An infinite or NaN key or value of a sequence's newest token: earlier
    queries of the same sequence do not see it, and come out to the bit as
    with a finite one; the newest query's row shows it."""
    prefix, sizes, own, heads, kv, n = case
    c = build(prefix, sizes, max(own, n + 3), heads, kv, n, dtype, seed=11)
    lens = [max(x, n) for x in c["lists"][1]]
    c["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
    # (build leaves NaN behind the lengths it chose: new finite rows for those)
    g = torch.Generator(device=DEV).manual_seed(1)
    for b, ln in enumerate(lens):
        for j in range(c["lists"][1][b], ln):
            page = c["block_table"][b, j // 64].long()
            for pool in ("k_pool", "v_pool"):
                c[pool][page, :, j % 64] = torch.randn((kv, 64), generator=g, device=DEV).to(dtype)
    clean = attend(c)
    assert torch.isfinite(clean).all()
    for pool, value, dims in (("v_pool", float("nan"), slice(5, 6)),
                              ("v_pool", float("inf"), slice(0, 64)),
                              ("k_pool", float("nan"), slice(9, 30))):
        d = dict(c, **{pool: c[pool].clone()})
        for b, ln in enumerate(lens):
            d[pool][c["block_table"][b, (ln - 1) // 64].long(), :, (ln - 1) % 64, dims] = value
        out = attend(d)
        assert torch.equal(out[:, :-1], clean[:, :-1])
        last = out[:, -1, :, dims if pool == "v_pool" else slice(0, 64)]
        assert not torch.isfinite(last).any()
        if pool == "v_pool" and dims == slice(5, 6):
            rest = [x for x in range(64) if x != 5]
            assert torch.equal(out[:, -1][..., rest], clean[:, -1][..., rest])


PREFIXES = {"each": ([250, 140], [3, 4], 40, 6, 2, 2), "tiles": ([4097, 650], [3, 2], 130, 12, 4, 1),
            "units": ([8300, 6000], [30, 40], 70, 12, 4, 2),
            "beside": ([12000, 9000], [50, 41], 1600, 9, 3, 1)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", PREFIXES)
def test_bad_prefix_keys_stay_in_their_group(name, dtype):
    """128 NaN keys in one group's prefix: its rows are NaN, the other group's
    the same to the bit."""
    c = build(*PREFIXES[name], dtype, seed=2)
    clean, lse = attend(c, with_lse=True)
    pages = c["prefix_table"][0, :2].long()
    bad = dict(c, k_pool=c["k_pool"].clone())
    bad["k_pool"][pages] = float("nan")
    out, bad_lse = attend(bad, with_lse=True)
    n, first = c["q"].shape[1], c["lists"][2][1]
    assert torch.isnan(out[:first]).all() and torch.isnan(bad_lse[:, :first * n]).all()
    assert torch.equal(out[first:], clean[first:])
    assert torch.equal(bad_lse[:, first * n:], lse[:, first * n:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", PREFIXES)
def test_scores_of_minus_infinity_weigh_nothing(name, dtype):
    """The first 128 keys' scores are all -inf: the formula's result, without
    them."""
    c = build(*PREFIXES[name], dtype, seed=4)
    c["q"][..., 0] = 1.0
    for g in range(2):
        c["k_pool"][c["prefix_table"][g, :2].long(), :, :, 0] = float("-inf")
    out, lse = attend(c, with_lse=True)
    o, a, want = reference(c, 0.125)
    keys = max(c["lists"][0]) + max(c["lists"][1])
    tol = (U[dtype] + 1e-4) * a + U[dtype] * o.abs() + 1e-7
    if dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * 5.5 + 2.0 ** -24
    assert ((out.double() - o).abs() <= tol).all()
    B, n, H, _ = c["q"].shape
    assert (lse.double().view(H, B, n).permute(1, 2, 0) - want).abs().max().item() <= 2e-5


def captured(call):
    """A graph of `call` (captured on the stream that torch.cuda.graph shares) and its output."""
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


@pytest.mark.gpu
def test_graphs_captured_on_one_stream_do_not_share_state():
    """Attention and sampling captured in the ordinary way, replayed on streams
    without order between them, beside calls on the stream of the captures."""
    from ffai_b200 import attention, sampling
    cs = [build(*CASES[n], torch.bfloat16, seed=i)
          for i, n in enumerate(("beside_odd_rows", "units_groups", "tiles_odd_rows"))]
    g = torch.Generator(device=DEV).manual_seed(1)
    logits = [torch.randn((n, 60001), generator=g, device=DEV) * 3 for n in (90, 33)]
    u = torch.rand(90, generator=g, device=DEV)
    calls = [lambda c=c: attend(c) for c in cs]
    calls += [lambda x=x: sampling.sample(x, u[:x.shape[0]].clone(), top_p=0.9) for x in logits]
    want = [call() for call in calls]
    graphs = [captured(call) for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    shared = torch.cuda.graph.default_capture_stream
    torch.cuda.synchronize()
    for _ in range(20):
        for _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(shared):
            again = [call() for call in calls]
        torch.cuda.synchronize()
        for w, (_, out), a in zip(want, graphs, again):
            assert torch.equal(out, w) and torch.equal(a, w)
    attention.sync(0)


@pytest.mark.gpu
def test_branches_of_one_capture_do_not_share_state():
    cs = [build(*CASES[n], torch.bfloat16, seed=i) for i, n in enumerate(("units", "beside_short"))]
    want = [attend(c) for c in cs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        out = [attend(cs[0])]
        with torch.cuda.stream(side):
            out.append(attend(cs[1]))
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(10):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want))


@pytest.mark.gpu
def test_workspaces_of_graphs_that_are_gone_serve_others():
    import gc
    import time
    c = build(*CASES["units"], torch.bfloat16, seed=3)
    want = attend(c)

    def once():
        graph, out = captured(lambda: attend(c))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del graph, out
        gc.collect()
        torch.cuda.synchronize()
        time.sleep(0.05)
        torch.cuda.empty_cache()
        return torch.cuda.mem_get_info()[0]
    once()
    first = once()
    for _ in range(12):
        last = once()
    # a workspace of this case holds over 30 MB; twelve more would take 360
    assert first - last < 100 * 2 ** 20


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiles", "tiles_odd_rows", "units_groups", "beside_odd_rows"])
@pytest.mark.parametrize("prefix_by,own_by", [(1, 40), (3, 1), (2, 17)])
def test_tables_with_spare_columns(name, prefix_by, own_by):
    """Tables as wide as the longest request may become, what lies behind the
    live pages being anything: the formula's result whichever way is taken."""
    from ffai_b200 import attention
    c = build(*CASES[name], torch.bfloat16, seed=7)
    o, a, want = reference(c, 0.125)

    def wide(table, by):
        t = torch.full((table.shape[0], table.shape[1] * by + 1), 10 ** 9, dtype=torch.int32, device=DEV)
        t[:, :table.shape[1]] = table
        return t
    prefix, lens, _ = c["lists"]
    for table, ns in ((c["prefix_table"], prefix), (c["block_table"], lens)):
        for i, n in enumerate(ns):  # nothing valid behind a row's own pages either
            table[i, (n + 63) // 64:] = -5
    c["prefix_table"], c["block_table"] = wide(c["prefix_table"], prefix_by), wide(c["block_table"], own_by)
    out, lse = attend(c, with_lse=True)
    attention.sync(0)
    B, n, H, _ = c["q"].shape
    u = U[torch.bfloat16]
    assert ((out.double() - o).abs() <= (u + 1e-4) * a + u * o.abs() + 1e-7).all()
    got = lse.double().view(H, B, n).permute(1, 2, 0)
    empty = want == float("-inf")
    assert torch.equal(got == float("-inf"), empty)
    assert (got[~empty] - want[~empty]).abs().max().item() <= 2e-5
