"""Attention of a chunk of new tokens over a paged cache (ffai_attn_chunk_paged)
against the formula in 64 bits on the same 16-bit operands.

Tolerance per element, from the arithmetic: the softmax weights enter the
second product in the cache's type (relative error u = 2^-8 for bf16, 2^-11
for f16, and below 2^-14 an absolute 2^-25 in f16, of up to 2^8 where the
weights are scaled), the output is rounded once to its own type, scores and sums
are f32 (scores of up to 64 products of size about 2: 1e-5 absolute, so 1e-5 of
the weight).  With A = sum_j w_j |v_j|:
    |err| <= (u + 1e-4) A + u_out |o| + n 2^-25 max|v|     (last term f16 only)
The log-sum-exp has no 16-bit step: 2e-5 absolute.

f32 queries with f32 output take no 16-bit step: a query keeps 22 bits at least, a
weight 16 (bf16 twice), and the errors of different keys are independent, so that
they average out: 2^-17 of a weight and 1e-5 of it for its score are within
1e-4 A per element, and within 1e-5 of the result in the 2-norm.
"""

import pytest
import torch

DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SCALE = 0.125


def pages(n):
    return (n + 63) // 64


def build(new, cached, heads, kv_heads, dtype, seed, dead=float("nan"), extra=0, wide=0):
    """Operands on the device: sequence b has cached[b] keys and new[b] tokens with
    theirs; pages are shuffled, what lies behind the live keys is `dead`, table
    entries behind the last page are no pages; `extra` rows of q behind the last
    sequence's, `wide` spare columns in the table."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    B = len(new)
    lens = [a + n for a, n in zip(cached, new)]
    mp = max(1, max(map(pages, lens))) + wide
    size = sum(map(pages, lens)) + 2
    kp = torch.full((size, kv_heads, 64, 64), dead, device=DEV)
    vp = torch.full((size, kv_heads, 64, 64), dead, device=DEV)
    perm = torch.randperm(size, generator=g, device=DEV).tolist()
    table = torch.full((B, mp), -1, dtype=torch.int32)
    kv = []
    for b, n in enumerate(lens):
        ids = [perm.pop() for _ in range(pages(n))]
        table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        k = (torch.randn(kv_heads, n, 64, generator=g, device=DEV) * 1.5).to(dtype)
        v = torch.randn(kv_heads, n, 64, generator=g, device=DEV).to(dtype)
        kv.append((k, v))
        for pool, x in ((kp, k), (vp, v)):
            full = torch.full((kv_heads, len(ids) * 64, 64), dead, device=DEV)
            full[:, :n] = x.float()
            pool[ids] = full.view(kv_heads, len(ids), 64, 64).transpose(0, 1)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + extra, heads, 64, generator=g, device=DEV).to(dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(q=q, k_pool=kp.to(dtype), v_pool=vp.to(dtype), cu_q=i32(cu), block_table=table.to(DEV),
                seq_lens=i32(lens), kv=kv, new=new, lens=lens, cu=cu)


def reference(c, q=None, causal=True):
    """(o, A, lse) in f64: (T, H, 64), (T, H, 64), (T, H)."""
    q = (c["q"] if q is None else q).double()
    T, H, _ = q.shape
    hk = c["k_pool"].shape[1]
    o, a = torch.zeros(T, H, 64, device=DEV).double(), torch.zeros(T, H, 64, device=DEV).double()
    lse = torch.full((T, H), float("-inf"), device=DEV).double()
    for b, (n, total) in enumerate(zip(c["new"], c["lens"])):
        if n == 0 or total == 0:
            continue
        k, v = (x.double().repeat_interleave(H // hk, 0) for x in c["kv"][b])
        rows = slice(c["cu"][b], c["cu"][b + 1])
        s = torch.einsum("thd,hkd->htk", q[rows], k) * SCALE
        limit = total - (n - 1 - torch.arange(n, device=DEV)) if causal else torch.full((n,), total, device=DEV)
        hide = torch.arange(total, device=DEV) >= limit.view(-1, 1)
        s = s.masked_fill(hide, float("-inf"))
        z = torch.logsumexp(s, -1)
        w = torch.exp(s - torch.where(torch.isinf(z), torch.zeros_like(z), z).unsqueeze(-1))
        # 0 times what is not a number is 0 where a key is hidden
        vz = torch.nan_to_num(v, 0, 0, 0)
        o[rows] = torch.einsum("htk,hkd->thd", w, vz)
        a[rows] = torch.einsum("htk,hkd->thd", w, vz.abs())
        odd = ~torch.isfinite(v)
        if odd.any():
            seen = (~hide).double()
            for key in odd.any(-1).any(0).nonzero()[:, 0].tolist():
                o[rows] = torch.where((seen[:, key] > 0).view(-1, 1, 1) & odd[:, key].unsqueeze(0),
                                      torch.full_like(o[rows], float("nan")), o[rows])
        lse[rows] = z.t()
    return o, a, lse


def run(c, **kw):
    from ffai_b200 import chunk_attention
    q = kw.pop("q", c["q"])
    return chunk_attention.attend(q, c["k_pool"], c["v_pool"], c["cu_q"], c["block_table"], c["seq_lens"],
                                  scale=SCALE, **kw)


def check(got, ref, c, dtype, out_dtype):
    o, a, _ = ref
    rows = c["cu"][-1]
    got, o, a = got[:rows].double(), o[:rows], a[:rows]
    tol = (U[dtype] + 1e-4) * a + U[out_dtype] * o.abs() + 1e-7
    if dtype == torch.float16 or out_dtype == torch.float16:
        tol = tol + max(c["lens"]) * 2.0 ** -25 * 5 + 2.0 ** -24
    real = torch.isfinite(o)
    assert torch.equal(torch.isfinite(got), real)
    err = (got - o).abs()[real]
    assert (err <= tol[real]).all(), f"worst {(err - tol[real]).max():.3e} over, err {err.max():.3e}"


def check_lse(lse, ref, c):
    rows = c["cu"][-1]
    got, want = lse[:, :rows].t().double(), ref[2][:rows]
    empty = want == float("-inf")
    assert torch.equal(got == float("-inf"), empty)
    if (~empty).any():
        assert (got[~empty] - want[~empty]).abs().max().item() <= 2e-5


CASES = [
    # new tokens, cached keys, heads, kv heads
    ([1], [0], 1, 1),
    ([1, 1, 1], [0, 63, 64], 6, 6),
    ([5], [127], 12, 12),
    ([1, 2, 3, 4, 5], [448, 0, 129, 64, 300], 12, 12),
    ([17], [0], 1, 1),
    ([16, 0, 33, 1], [100, 50, 0, 1000], 4, 2),
    ([1] * 40, [(37 * i) % 700 for i in range(40)], 8, 2),
    ([8, 1, 3, 8, 6], [2000, 5, 127, 128, 129], 32, 8),
    ([3], [20000], 8, 1),
    ([1], [50000], 28, 4),
    ([64], [64], 2, 1),
    ([128, 129, 127], [0, 0, 0], 2, 2),
    ([300], [0], 6, 6),
    ([257, 1, 500], [1000, 777, 13], 7, 1),
    ([700, 1, 1, 1, 90], [300, 6000, 1, 0, 2500], 28, 4),
    ([1000], [3000], 10, 1),
    ([2049], [100], 16, 2),
    ([0, 0, 5, 0], [10, 0, 7, 64], 4, 4),
    ([7] * 130, [(11 * i) % 90 for i in range(130)], 5, 5),
    ([33], [40000], 16, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_matches_the_formula(case, dtype):
    from ffai_b200 import attention
    new, cached, heads, kv = case
    c = build(new, cached, heads, kv, dtype, seed=len(new) * 31 + heads)
    for causal in (True, False):
        ref = reference(c, causal=causal)
        out, lse = run(c, causal=causal, with_lse=True)
        check(out, ref, c, dtype, dtype)
        check_lse(lse, ref, c)
        # the bound on a sequence's tokens chooses a kernel, not the result's size
        for max_q in (1, max(new)):
            other, olse = run(c, causal=causal, with_lse=True, max_q=max_q)
            check(other, ref, c, dtype, dtype)
            check_lse(olse, ref, c)
            assert torch.equal(other, run(c, causal=causal, max_q=max_q))  # the same bits again
    attention.sync(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_f32_queries_keep_their_bits(case, dtype):
    new, cached, heads, kv = case
    c = build(new, cached, heads, kv, dtype, seed=len(new) * 17 + heads, extra=2)
    q = torch.randn(c["q"].shape, generator=torch.Generator(device=DEV).manual_seed(9), device=DEV)
    for causal in (True, False):
        o, a, lse = reference(c, q=q, causal=causal)
        rows = c["cu"][-1]
        for max_q in (None, 1, max(new)):
            out, got = run(c, q=q, causal=causal, with_lse=True, max_q=max_q)
            assert out.dtype is torch.float32
            err = (out[:rows].double() - o[:rows]).abs()
            assert (err <= 1e-4 * a[:rows] + 1e-7).all()
            assert err.norm() <= 1e-5 * o[:rows].norm() + 1e-7
            check_lse(got, (o, a, lse), c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,cached,heads,kv", [([5, 0, 1, 20], [70, 3, 200, 0], 6, 3),
                                                 ([300, 1], [200, 900], 8, 2)])
def test_layouts_and_output_types(new, cached, heads, kv, dtype):
    c = build(new, cached, heads, kv, dtype, seed=5, extra=3, wide=4)
    ref = reference(c)
    for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
        for q_dtype in (dtype, torch.float32):
            for view in (False, True):
                q = c["q"].to(q_dtype)
                if view:  # a part of a projection's rows
                    wide = torch.full((q.shape[0], heads + 2 * kv, 64), float("nan"), device=DEV, dtype=q_dtype)
                    wide[:, kv:kv + heads] = q
                    q = wide[:, kv:kv + heads]
                out = torch.full(q.shape, 7.0, device=DEV, dtype=out_dtype)
                got = run(c, q=q, out=out)
                assert got is out
                check(out, ref, c, dtype, out_dtype)
                assert (out[c["cu"][-1]:] == 7).all()  # rows behind the last sequence
    # f32 queries are rounded to the cache's type where the output is
    q = torch.randn_like(c["q"].float())
    check(run(c, q=q, out_dtype=dtype), reference(c, q=q.to(dtype)), c, dtype, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,cached,heads,kv,at", [
    ([9], [50], 2, 2, [55]), ([9], [120], 8, 1, [128, 126]), ([300], [100], 4, 4, [399, 250, 130]),
    ([300], [0], 4, 1, [290, 128, 127, 5]), ([140], [500], 2, 2, [510, 600]), ([600], [70], 8, 2, [300, 301, 640]),
    ([256], [0], 1, 1, [255, 128, 129]), ([70, 400], [10, 33], 4, 4, [15, 60])])
def test_what_a_row_does_not_see_does_not_reach_it(new, cached, heads, kv, at, dtype):
    """Keys and values that are not finite at some positions: rows that see them are
    none themselves, rows before them are as if they were not there."""
    for bad in (float("nan"), float("inf"), float("-inf")):
        for which in (0, 1):
            c = build(new, cached, heads, kv, dtype, seed=3)
            b = len(new) - 1
            for pos in at:
                page = int(c["block_table"][b, pos // 64])
                dims = [0, 13, 63] if pos % 2 else [5]
                if which == 0:  # keys: scores that are none
                    c["k_pool"][page, :, pos % 64, dims] = float("nan")
                    c["kv"][b][0][:, pos, dims] = float("nan")
                else:
                    c["v_pool"][page, :, pos % 64, dims] = bad
                    c["kv"][b][1][:, pos, dims] = bad
            o, a, lse = reference(c)
            out = run(c, out_dtype=torch.float32)
            if which == 0:  # a score that is none makes its whole row none
                o = torch.where(torch.isnan(lse).unsqueeze(-1), torch.full_like(o, float("nan")), o)
            check(out, (o, a, lse), c, dtype, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("new,cached", [([5], [-3]), ([200], [-150]), ([400, 3], [-300, -3]), ([1, 2], [-1, -2])])
def test_rows_that_see_no_key(new, cached):
    """Sequences with fewer keys than new tokens: the first tokens see none."""
    for heads, kv in ((4, 2), (1, 1), (16, 1)):
        c = build(new, cached, heads, kv, torch.bfloat16, seed=1)
        ref = reference(c)
        out, lse = run(c, with_lse=True)
        check(out, ref, c, torch.bfloat16, torch.bfloat16)
        check_lse(lse, ref, c)
        assert (out[ref[2] == float("-inf")] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("new,cached", [([1], [3000]), ([4, 1], [900, 4000]), ([300], [1500])])
def test_peaks_after_low_scores(new, cached):
    """Scores that rise by hundreds along the keys: every rescale is taken."""
    c = build(new, cached, 8, 2, torch.bfloat16, seed=8)
    for b, (k, _) in enumerate(c["kv"]):
        ramp = torch.linspace(-1, 6, k.shape[1], device=DEV).view(1, -1, 1)
        k.copy_((k.float() * 0.2 + ramp).to(k.dtype))
        n = k.shape[1]
        ids = c["block_table"][b, :pages(n)].long()
        full = torch.zeros(2, len(ids) * 64, 64, device=DEV, dtype=k.dtype)
        full[:, :n] = k
        c["k_pool"][ids] = full.view(2, len(ids), 64, 64).transpose(0, 1)
    c["q"] = (c["q"].float() + 4).to(torch.bfloat16)
    for max_q in (1, max(new)):
        out, lse = run(c, with_lse=True, max_q=max_q)
        ref = reference(c)
        check(out, ref, c, torch.bfloat16, torch.bfloat16)
        # scores of up to 64 * 4 * 6 / 8 = 192: f32 sums of them to 2^-24 * 64 * 192 at most
        assert (lse.t().double() - ref[2]).abs().max() <= 64 * 192 * 2.0 ** -24


@pytest.mark.gpu
def test_agrees_with_its_neighbours():
    """Single tokens as decode_paged has them, and drafts as shared_prefix's own keys."""
    from ffai_b200 import kvcache, shared_prefix
    c = build([1] * 9, [17 * i for i in range(9)], 6, 6, torch.bfloat16, seed=2)
    out = run(c, out_dtype=torch.float32)
    dec = kvcache.decode_paged(c["q"].view(9, 6, 1, 64), c["k_pool"], c["v_pool"], c["block_table"],
                               c["seq_lens"], scale=SCALE)
    assert (out - dec[:, :, 0]).abs().max() < 2e-2
    c = build([4] * 9, [17 * i for i in range(9)], 6, 2, torch.bfloat16, seed=2)
    none = torch.zeros(0, 1, dtype=torch.int32, device=DEV)
    sp = shared_prefix.attend(c["q"].view(9, 4, 6, 64), c["k_pool"], c["v_pool"], none, none[:, 0],
                              torch.zeros(1, dtype=torch.int32, device=DEV), c["block_table"], c["seq_lens"],
                              scale=SCALE, out_dtype=torch.float32)
    assert (run(c, out_dtype=torch.float32) - sp.view(36, 6, 64)).abs().max() < 2e-2


@pytest.mark.gpu
@pytest.mark.parametrize("new,cached", [([1, 5], [100, 3]), ([300], [200])])
def test_offsets_beyond_32_bits(new, cached):
    """Pages past 2^32 elements of a pool."""
    c = build(new, cached, 4, 2, torch.bfloat16, seed=4)
    shift = (1 << 32) // (2 * 64 * 64) + 5
    n = c["k_pool"].shape[0]
    for name in ("k_pool", "v_pool"):
        big = torch.empty((shift + n, 2, 64, 64), dtype=torch.bfloat16, device=DEV)
        big[shift:] = c[name]
        c[name] = big
    c["block_table"] = torch.where(c["block_table"] >= 0, c["block_table"] + shift, -1).to(torch.int32)
    check(run(c), reference(c), c, torch.bfloat16, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[3, 1, 2], [400, 1, 30]])
@pytest.mark.parametrize("what", ["page", "length", "negative", "falls", "past", "before"])
def test_bad_tables_are_reported_not_read(what, new):
    from ffai_b200 import attention
    c = build(new, [100, 200, 64], 4, 2, torch.bfloat16, seed=6)
    good = run(c)
    attention.sync(0)
    if what == "page":
        c["block_table"][1, 1] = c["k_pool"].shape[0]
    elif what == "length":
        c["seq_lens"][1] = c["block_table"].shape[1] * 64 + 1
    elif what == "negative":
        c["seq_lens"][1] = -5
    elif what == "falls":
        c["cu_q"][2] = c["cu_q"][1] - 1
    elif what == "past":
        c["cu_q"][3] = c["cu"][3] + 1
    else:
        c["cu_q"][0] = -1
    out = torch.full_like(good, 7.0)
    try:
        run(c, out=out)
        if what in ("page", "length", "negative", "past"):  # the first is as it was
            assert torch.equal(out[:c["cu"][1]], good[:c["cu"][1]])
        if what == "past":
            assert (out[c["cu"][2]:] == 7).all()
        if what == "negative":
            assert (out[c["cu"][1]:c["cu"][2]] == 0).all()
    finally:
        with pytest.raises(attention.AttnError) as e:
            attention.sync(0)
        assert "page id outside" in str(e.value)
    c["cu_q"].copy_(torch.tensor(c["cu"], dtype=torch.int32))
    c["seq_lens"].copy_(torch.tensor(c["lens"], dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 300])
def test_tokens_named_many_times_are_refused(new):
    """cu_q that rises and falls over the same tokens: nothing is written."""
    from ffai_b200 import attention
    c = build([new] * 9, [100] * 9, 4, 2, torch.bfloat16, seed=6)
    good = run(c)
    attention.sync(0)
    c["cu_q"].copy_(torch.tensor([0, 9 * new] * 5, dtype=torch.int32))
    out = torch.full_like(good, 7.0)
    run(c, out=out)
    with pytest.raises(attention.AttnError):
        attention.sync(0)
    assert (out == 7).all()
    c["cu_q"].copy_(torch.tensor(c["cu"], dtype=torch.int32))
    assert torch.equal(run(c), good)
    attention.sync(0)


@pytest.mark.gpu
def test_streams_and_captures_do_not_share_partials():
    """Calls on two streams and two graphs captured on one stream, replayed together."""
    jobs = []
    for seed, new, cached in ((1, [1, 1], [30000, 9000]), (2, [2, 300], [20000, 3000]),
                              (3, [1], [40000]), (4, [500, 3], [5000, 12000])):
        c = build(new, cached, 8, 2, torch.bfloat16, seed)
        m = max(new)
        jobs.append((c, m, run(c, max_q=m).clone()))
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for c, m, _ in jobs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(c, max_q=m))
        graphs.append(g)
    for _ in range(10):
        eager = []
        for s, g, (c, m, _) in zip(streams, graphs, jobs[2:]):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(run(c, max_q=m))
        torch.cuda.synchronize()
        for o, (_, _, want) in zip(outs + eager, jobs):
            assert torch.equal(o, want)


@pytest.mark.gpu
def test_no_tokens():
    c = build([0, 0], [5, 70], 4, 2, torch.bfloat16, seed=1)
    assert run(c).shape == (0, 4, 64)


def test_refusals_without_a_device():
    from ffai_b200 import chunk_attention
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        chunk_attention.attend(torch.zeros(1, 2, 64), torch.zeros(1, 2, 64, 64), torch.zeros(1, 2, 64, 64),
                               z, z.view(1, 1), z)


@pytest.mark.gpu
def test_refusals():
    from ffai_b200 import attention
    c = build([3], [70], 4, 2, torch.bfloat16, seed=1)
    with pytest.raises(attention.Declined):  # f32 pools
        run({**c, "k_pool": c["k_pool"].float(), "v_pool": c["v_pool"].float()})
    with pytest.raises(attention.Declined):  # another 16-bit type
        run(c, q=c["q"].half())
    for bad in (dict(k_pool=c["k_pool"].half()), dict(v_pool=c["v_pool"][:, :1]), dict(cu_q=c["cu_q"].long()),
                dict(cu_q=c["cu_q"][:1]), dict(block_table=c["block_table"][0]),
                dict(block_table=c["block_table"].cpu()), dict(seq_lens=c["seq_lens"].repeat(2)),
                dict(q=c["q"].transpose(0, 1)), dict(q=c["q"][..., :32]), dict(q=c["q"][:, :, ::2])):
        with pytest.raises(ValueError):
            run({**c, **bad})
    with pytest.raises(attention.AttnError):  # 3 heads over 2 KV heads
        run(c, q=c["q"][:, :3].contiguous())
    with pytest.raises(ValueError):
        run(c, out=torch.empty(3, 4, 64, device=DEV)[:2])
    with pytest.raises(TypeError):
        run(c, out_dtype=torch.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 1e5, 1e20])
@pytest.mark.parametrize("tokens,heads", [(1, 8), (9, 7), (40, 4), (300, 5)])
def test_f32_queries_of_every_size_and_their_weights(tokens, heads, size, dtype):
    """Two keys, 0 and e_0, with the values 0 and 1, and queries a e_0 (of another size
    beside it, which no key meets): o = w / (1 + w), w = e^(scale a), |scale a| <= 2.
    What a weight loses: its score is off by 2^-22 of it for the query's terms (two in
    f16), 2 * 2^-23 for the matrix instruction's cut sums, 2^-23 for the scale, 2^-24 for
    the last sum: 3 * 2^-22 * 2 at most; e^x by 2^-22, the weight's terms by 2^-22 (f16), the
    sum, the quotient and its rounding by 2^-22 together; its exponent, which is 15 more
    than the score in f16, by 2^-21 ln 2; half a step for what is of second order:
    11 * 2^-22.  (A weight in two bf16 terms is off by 2^-17 = 32 * 2^-22.)"""
    from ffai_b200 import chunk_attention
    g = torch.Generator(device=DEV).manual_seed(tokens)
    pool = torch.full((2, 1, 64, 64), float("nan"), device=DEV, dtype=dtype)
    kp, vp = pool.clone(), pool.clone()
    kp[1, 0, :2], vp[1, 0, :2] = 0, 0
    kp[1, 0, 1, 0] = 1
    vp[1, 0, 1] = 1
    q = torch.zeros(tokens, heads, 64, device=DEV)
    scale = torch.tensor(0.25 / size).item()
    q[:, :, 0] = -(torch.rand(tokens, heads, generator=g, device=DEV) * 8 * size)
    q[:, ::2, 5] = torch.randn(tokens, (heads + 1) // 2, generator=g, device=DEV) * 1000 * size
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    a = q[:, :, 0].double() * torch.tensor(scale, dtype=torch.float32).double().item()
    want = (torch.exp(a) / (1 + torch.exp(a))).unsqueeze(-1).expand(-1, -1, 64)
    for max_q in (None, 1, tokens):
        out = chunk_attention.attend(q, kp, vp, i32(0, tokens), i32(1).view(1, 1), i32(2), scale=scale,
                                     causal=False, max_q=max_q)
        assert ((out.double() - want).abs() <= 11 * 2.0 ** -22 * want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("below", [12.0, 25.6])
def test_many_small_weights_beside_a_large_one(below, dtype):
    """One key of weight 1 and value 0 before 7999 of weight 2^-below and value 1, which
    are rounded alike: o = n w / (1 + n w).  A weight is off by u of it (u = 2^-8, 2^-11; three
    and two terms of f32 queries: 2^-22), in f16 by what half a subnormal step is of the
    largest, 2^-25 / 2^15, or 2^-25 / 2^6 in the kernel for many rows; scores, sums and the
    rest are f32, of 1e-5 together.  Many sequences, so that few are split."""
    from ffai_b200 import chunk_attention
    B, kv, n = 120, 8, 8000
    kp = torch.zeros(125, kv, 64, 64, device=DEV, dtype=dtype)
    vp = torch.ones_like(kp)
    kp[:, :, :, 0], kp[0, :, 0], vp[0, :, 0] = 1, 0, 0
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table, lens, cu = i32(torch.arange(125)).repeat(B, 1), i32([n] * B), i32(torch.arange(B + 1))
    scale = torch.tensor(below * 0.6931471805599453 / 16).item()
    w = torch.exp(torch.tensor(-16 * scale).double()).item()
    want = (n - 1) * w / (1 + (n - 1) * w)
    for q_dtype in (dtype, torch.float32):
        q = torch.zeros(B, 2 * kv, 64, device=DEV, dtype=q_dtype)
        q[:, :, 0] = -16
        for max_q in (1, B):
            out = chunk_attention.attend(q, kp, vp, cu, table, lens, scale=scale, max_q=max_q, out_dtype=torch.float32)
            exact = q_dtype is torch.float32
            u = 2.0 ** -22 if exact else U[dtype]
            floor = 0 if dtype is torch.bfloat16 else 2.0 ** -31 if max_q > 1 and not exact else 2.0 ** -40
            err = (out.double() - want).abs().max().item()
            assert err <= (u + 1e-5) * want + n * floor, (q_dtype, max_q, err / want)
