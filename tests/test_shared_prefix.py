"""Attention over a shared prefix (ffai_attn_shared_prefix) against the
formula in 64 bits on the same 16-bit operands.

Tolerance per element, from the arithmetic: the softmax weights enter the
second product in the cache's type (relative error u = 2^-8 for bf16, 2^-11
for f16, and below 2^-14 an absolute 2^-25 in f16), the output is rounded once
to its own type, scores and sums are f32 (scores of up to 64 products of size
about 2: 1e-5 absolute, so 1e-5 of the weight).  With A = sum_j w_j |v_j|:
    |err| <= (u + 1e-4) A + u_out |o| + n 2^-25 max|v|     (last term f16 only)
The log-sum-exp has no 16-bit step: 2e-5 absolute.
"""

import pytest
import torch

DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def pages(n):
    return (n + 63) // 64


def build(prefix, suffix, sizes, heads, kv_heads, q_len, dtype, seed, extra=0, dead=float("nan")):
    """Operands on the CPU: prefix[g] and suffix[b] keys, sizes[g] sequences a
    group (the last `extra` sequences in no group); pages are shuffled, and
    what lies behind the live keys is `dead`."""
    g = torch.Generator().manual_seed(seed)
    B = len(suffix)
    assert sum(sizes) + extra == B
    pp, sp = max(1, max(map(pages, prefix), default=1)), max(1, max(map(pages, suffix)))
    n_pages = len(prefix) * pp + B * sp + 2
    kp = torch.full((n_pages, kv_heads, 64, 64), dead)
    vp = torch.full((n_pages, kv_heads, 64, 64), dead)
    perm = torch.randperm(n_pages, generator=g).to(torch.int32)
    ptab = perm[:len(prefix) * pp].view(len(prefix), pp)
    stab = perm[len(prefix) * pp:len(prefix) * pp + B * sp].view(B, sp)
    lists = []
    for table, lens in ((ptab, prefix), (stab, suffix)):
        rows = []
        for i, n in enumerate(lens):
            k = (torch.randn(kv_heads, n, 64, generator=g) * 1.5).to(dtype)
            v = torch.randn(kv_heads, n, 64, generator=g).to(dtype)
            for j in range(n):
                kp[table[i, j // 64], :, j % 64] = k[:, j].float()
                vp[table[i, j // 64], :, j % 64] = v[:, j].float()
            rows.append((k, v))
        lists.append(rows)
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    q = torch.randn(B, q_len, heads, 64, generator=g).to(dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=q, k_pool=kp.to(dtype), v_pool=vp.to(dtype), prefix_table=ptab.contiguous(),
                prefix_lens=i32(prefix), group_starts=i32(starts), block_table=stab.contiguous(),
                seq_lens=i32(suffix), pre=lists[0], own=lists[1], starts=starts)


def reference(c, scale, q=None):
    """(o, A, lse) in f64: (B, n, H, 64), (B, n, H, 64), (B, n, H)."""
    q = (c["q"] if q is None else q).double()
    B, n, H, _ = q.shape
    hk = c["k_pool"].shape[1]
    o, a = torch.zeros(B, n, H, 64).double(), torch.zeros(B, n, H, 64).double()
    lse = torch.full((B, n, H), float("-inf")).double()
    for b in range(B):
        g = next((g for g in range(len(c["pre"])) if c["starts"][g] <= b < c["starts"][g + 1]), None)
        pk, pv = c["pre"][g] if g is not None else (c["own"][b][0][:, :0],) * 2
        k = torch.cat([pk, c["own"][b][0]], 1).double()
        v = torch.cat([pv, c["own"][b][1]], 1).double()
        for i in range(n):
            see = pk.shape[1] + max(0, c["own"][b][0].shape[1] - (n - 1 - i))
            if see == 0:
                continue
            for h in range(H):
                kh = h // (H // hk)
                s = (k[kh, :see] @ q[b, i, h]) * scale
                lse[b, i, h] = torch.logsumexp(s, 0)
                w = torch.softmax(s, 0)
                o[b, i, h] = w @ v[kh, :see]
                a[b, i, h] = w @ v[kh, :see].abs()
    return o, a, lse


def run(c, scale, **kw):
    from ffai_b200 import shared_prefix
    t = {k: v.to(DEV) for k, v in c.items() if isinstance(v, torch.Tensor)}
    t["q"] = kw.pop("q", t["q"])
    return shared_prefix.attend(t["q"], t["k_pool"], t["v_pool"], t["prefix_table"],
                                t["prefix_lens"], t["group_starts"], t["block_table"],
                                t["seq_lens"], scale=scale, **kw)


def check(got, ref, c, dtype, out_dtype):
    o, a, _ = ref
    n_keys = max([0] + [p[0].shape[1] for p in c["pre"]]) + max(s[0].shape[1] for s in c["own"])
    tol = (U[dtype] + 1e-4) * a + U[out_dtype] * o.abs() + 1e-7
    if dtype == torch.float16 or out_dtype == torch.float16:
        tol = tol + n_keys * 2.0 ** -25 * 5 + 2.0 ** -24
    err = (got.cpu().double() - o).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {(err - tol).max():.3e} over, err {err.max():.3e}"


CASES = [
    # prefix per group, sequences per group, own keys, heads, kv heads, q_len, in no group
    ([1], [1], [0], 1, 1, 1, 0),
    ([1], [2], [0, 1], 6, 6, 1, 0),
    ([63], [3], [1, 64, 65], 2, 2, 1, 0),
    ([64, 65], [1, 4], [0, 3, 63, 64, 130], 8, 2, 1, 0),
    ([127, 128, 129], [2, 1, 3], [5, 0, 127, 128, 129, 257], 10, 1, 1, 0),
    ([0, 300], [2, 2], [0, 31, 33, 200], 6, 3, 1, 0),
    ([200], [2], [70, 9, 0, 128], 4, 2, 1, 2),
    ([130], [5], [1, 2, 3, 4, 5], 8, 2, 4, 0),
    ([65, 0], [2, 2], [0, 2, 3, 70], 6, 6, 3, 0),
    ([100], [2], [17, 90], 4, 4, 17, 0),
    ([256], [3], [40, 41, 0], 12, 2, 9, 0),
    ([1500], [5], [0, 1, 2, 3, 4], 2, 2, 1, 0),
    ([700], [40], list(range(40)), 8, 2, 1, 0),
    ([257, 900], [33, 2], [(7 * i) % 97 for i in range(35)], 8, 1, 2, 0),
    ([384], [37], [(5 * i) % 61 for i in range(37)], 14, 2, 1, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_matches_the_formula(case, dtype):
    prefix, sizes, suffix, heads, kv, n, extra = case
    c = build(prefix, suffix, sizes, heads, kv, n, dtype, seed=len(suffix) * 31 + heads, extra=extra)
    out, lse = run(c, 0.125, with_lse=True)
    ref = reference(c, 0.125)
    check(out, ref, c, dtype, dtype)
    B = len(suffix)
    got = lse.cpu().double().view(heads, B, n).permute(1, 2, 0)
    empty = ref[2] == float("-inf")
    assert torch.equal(got == float("-inf"), empty)
    assert (got[~empty] - ref[2][~empty]).abs().max().item() <= 2e-5 if (~empty).any() else True
    assert (out.cpu()[empty] == 0).all()
    again = run(c, 0.125)
    assert torch.equal(again, out)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layouts_and_output_types(dtype):
    c = build([190], [0, 5, 77], [3], 8, 4, 2, dtype, seed=5)
    ref = reference(c, 0.2)
    token = run(c, 0.2)
    qh = c["q"].transpose(1, 2).contiguous().to(DEV)
    heads, lse = run(c, 0.2, q=qh, q_layout="heads", out_layout="heads", with_lse=True)
    assert torch.equal(heads.transpose(1, 2), token)
    assert (lse.cpu().double().transpose(1, 2) - ref[2]).abs().max() <= 2e-5
    # q as a view of a fused projection's rows
    B, n, H, _ = c["q"].shape
    fused = torch.randn(B, n, (H + 8) * 64).to(dtype)
    fused[:, :, :H * 64] = c["q"].flatten(2)
    view = fused.to(DEV)[:, :, :H * 64].unflatten(2, (H, 64))
    assert torch.equal(run(c, 0.2, q=view), token)
    for od in (torch.float32, torch.bfloat16, torch.float16):
        check(run(c, 0.2, out_dtype=od), ref, c, dtype, od)
    # f32 queries are rounded to the cache's type
    qf = (c["q"].float() * 1.001)
    check(run(c, 0.2, q=qf.to(DEV), out_dtype=torch.float32), reference(c, 0.2, qf.to(dtype)), c,
          dtype, torch.float32)


@pytest.mark.gpu
def test_no_groups_is_plain_paged_decode():
    from ffai_b200 import kvcache, shared_prefix
    c = build([], [1, 64, 200], [], 6, 6, 1, torch.bfloat16, seed=9, extra=3, dead=0.0)
    t = {k: v.to(DEV) for k, v in c.items() if isinstance(v, torch.Tensor)}
    none = torch.empty(0, 1, dtype=torch.int32, device=DEV)
    out = shared_prefix.attend(t["q"], t["k_pool"], t["v_pool"], none, none[:, 0],
                               torch.zeros(1, dtype=torch.int32, device=DEV), t["block_table"],
                               t["seq_lens"], scale=0.125)
    check(out, reference(c, 0.125), c, torch.bfloat16, torch.bfloat16)
    old = kvcache.decode_paged(t["q"].transpose(1, 2).contiguous(), t["k_pool"], t["v_pool"],
                               t["block_table"], t["seq_lens"], scale=0.125)
    assert (old[:, :, 0] - out[:, 0].float()).abs().max() < 3e-2


@pytest.mark.gpu
def test_peaks_after_low_scores():
    """Keys whose scores rise by hundreds from block to block: the running
    maximum moves every time and old weights vanish."""
    c = build([512], [64, 3], [2], 2, 2, 1, torch.bfloat16, seed=3)
    ramp = torch.linspace(-40, 40, 512)
    q = c["q"].float()
    for kvh in range(2):
        for j in range(512):
            k = (q[0, 0, kvh] * ramp[j] / 8).to(torch.bfloat16)
            c["k_pool"][c["prefix_table"][0, j // 64], kvh, j % 64] = k
            c["pre"][0][0][kvh, j] = k
    check(run(c, 1.0), reference(c, 1.0), c, torch.bfloat16, torch.bfloat16)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Pools of more than 2^32 elements: pages near their end."""
    kv, n_pages = 8, 140000  # 4.6e9 elements, 9.2 GB a pool
    c = build([100], [70, 3], [2], 8, kv, 1, torch.bfloat16, seed=21)
    big_k = torch.empty((n_pages, kv, 64, 64), dtype=torch.bfloat16, device=DEV)
    big_v = torch.empty_like(big_k)
    used = c["k_pool"].shape[0]
    big_k[n_pages - used:] = c["k_pool"].to(DEV)
    big_v[n_pages - used:] = c["v_pool"].to(DEV)
    small = run(c, 0.125)
    moved = dict(c, k_pool=big_k, v_pool=big_v, prefix_table=c["prefix_table"] + (n_pages - used),
                 block_table=c["block_table"] + (n_pages - used))
    assert torch.equal(run(moved, 0.125), small)


@pytest.mark.gpu
def test_runs_on_the_current_stream():
    c = build([130], [5, 70], [2], 4, 2, 1, torch.bfloat16, seed=2)
    want = run(c, 0.125)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(c, 0.125)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_refusals():
    from ffai_b200 import attention
    c = build([64], [3], [1], 4, 2, 1, torch.bfloat16, seed=1)
    with pytest.raises(attention.Declined):
        run(dict(c, k_pool=c["k_pool"].float(), v_pool=c["v_pool"].float()), 0.125)
    with pytest.raises(attention.Declined):
        run(c, 0.125, q=c["q"].half().to(DEV))
    with pytest.raises(attention.AttnError):
        run(c, 0.0)
    with pytest.raises(attention.AttnError):  # 3 heads over 2 KV heads
        run(dict(c, q=c["q"][:, :, :3].contiguous()), 0.125)
    with pytest.raises(ValueError):
        run(dict(c, seq_lens=c["seq_lens"].long()), 0.125)
    with pytest.raises(ValueError):
        run(dict(c, prefix_lens=c["prefix_lens"].repeat(2)), 0.125)
    with pytest.raises(ValueError):
        run(c, 0.125, q=c["q"].to(DEV).expand(1, 2, 4, 64))
    with pytest.raises(ValueError):
        run(c, 0.125, out=torch.empty(1, 1, 4, 32, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["page", "prefix_page", "length", "prefix_length"])
def test_bad_tables_are_reported_not_read(what):
    from ffai_b200 import attention
    c = build([100], [70], [1], 4, 2, 1, torch.bfloat16, seed=4, dead=0.0)
    if what == "page":
        c["block_table"][0, 1] = 10 ** 6
    elif what == "prefix_page":
        c["prefix_table"][0, 0] = -7
    elif what == "length":
        c["seq_lens"][0] = 1000
    else:
        c["prefix_lens"][0] = -1
    run(c, 0.125)
    with pytest.raises(attention.AttnError) as e:
        attention.sync(0)
    assert e.value.status == -1
    attention.sync(0)  # the word is cleared


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 3, 2, 4], [0, 1, 2, 7], [-1, 1, 2, 4], [2, 1, 3, 4], [0, 4, 4, 2]])
@pytest.mark.parametrize("n", [1, 3])
def test_starts_that_do_not_rise_leave_short_prefixes_out_too(starts, n):
    """To the bit the result without prefixes, and an error at the next sync;
    with 40 groups as well, more than a warp has lanes."""
    from ffai_b200 import attention
    for more in (0, 37):
        c = build([70, 0, 9] + [5] * more, [3, 40, 0, 66], [2, 1, 1] + [0] * more, 4, 2, n,
                  torch.bfloat16, seed=len(starts) + n)
        plain = dict(c, prefix_lens=torch.zeros_like(c["prefix_lens"]))
        want = run(plain, 0.125)
        attention.sync(0)
        assert not torch.equal(run(c, 0.125), want)
        bad = dict(c, group_starts=torch.tensor([0] * more + starts, dtype=torch.int32))
        got = run(bad, 0.125)
        with pytest.raises(attention.AttnError) as e:
            attention.sync(0)
        assert e.value.status == -1
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [([130], [2], [64, 70], 2, 1, 64, 0), ([0], [1], [129], 3, 1, 129, 0),
                                  ([65, 300], [1, 2], [100, 5, 33], 4, 2, 33, 0),
                                  ([700], [1], [200], 2, 2, 200, 0)],
                         ids=["whole", "no_prefix", "ragged", "tiles"])
def test_prompts_behind_a_prefix(case, dtype):
    """More new tokens a sequence than a tile has rows, more than it holds keys among them."""
    prefix, sizes, suffix, heads, kv, n, extra = case
    c = build(prefix, suffix, sizes, heads, kv, n, dtype, seed=n, extra=extra)
    out, lse = run(c, 0.125, with_lse=True)
    ref = reference(c, 0.125)
    check(out, ref, c, dtype, dtype)
    got = lse.cpu().double().view(heads, len(suffix), n).permute(1, 2, 0)
    empty = ref[2] == float("-inf")
    assert torch.equal(got == float("-inf"), empty)
    assert (got[~empty] - ref[2][~empty]).abs().max().item() <= 2e-5
    assert (out.cpu()[empty] == 0).all()
