"""Verification of drafted tokens (ffai_verify) against its definition in whole
numbers on the host.

The weights are the one thing computed in floating point: e^d in f32, on the
device by its expf, which the tests take from the device (torch.exp), so tokens
are equal to the last one.  Log-probabilities: x - max is rounded once (2^-24
relative of up to 40), the sum of up to 2^18 terms of 2^-22 each in f32 parts and
its logarithm rounded once: 40 * 2^-24 + 2^-21 + 13 * 2^-24 < 6e-6.
"""

import math

import pytest
import torch

DEV = "cuda:0"
SCALE = 2 ** 36


def weights(x, t):
    """Whole weights (Python integers) of a row of logits on the device."""
    x = x.float()
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x) + 0.0
    top = x.max()
    if top == float("-inf"):
        return [0] * x.numel()
    inv = torch.ones(1, device=x.device) / t if t > 0 else None
    if inv is None or torch.isinf(inv).item():
        w = [0] * x.numel()
        w[int((x == top).nonzero()[0])] = SCALE
        return w
    d = torch.where(x == top, torch.zeros_like(x), x - top) * inv
    w = torch.floor(torch.exp(d).double() * SCALE)
    return [int(v) for v in torch.where(d >= -25, w, torch.zeros_like(w)).tolist()]


def reference(logits, tokens, cu, u, u_last, draft=None, t=None, dt=None):
    """(accepted, next, tokens) by the definition."""
    acc, nxt, out = [], [], [-1] * logits.shape[0]
    V = logits.shape[1]
    for b in range(len(u_last)):
        r0, r1 = cu[b], cu[b + 1]
        if r1 == r0:
            acc.append(0)
            nxt.append(-1)
            continue
        tb = 1.0 if t is None else t[b]
        db = tb if dt is None else dt[b]
        rest, row = None, r0
        while row + 1 < r1:
            x = tokens[row + 1]
            w = weights(logits[row], tb)
            if draft is None:
                v = [0] * V
                if 0 <= x < V:
                    v[x] = 1
                vx, total = 1, 1
            else:
                v = weights(draft[row], db)
                vx, total = (v[x] if 0 <= x < V else 0), sum(v)
            wx = w[x] if 0 <= x < V else 0
            if not (float(u[row]) * float(vx)) * float(sum(w)) < float(wx) * float(total):
                rho = float(sum(w)) / float(total) if total else 0.0
                rest = [max(0, a - math.floor(float(c) * rho)) for a, c in zip(w, v)]
                break
            out[row] = x
            row += 1
        acc.append(row - r0)
        if rest is None or sum(rest) == 0:
            rest = weights(logits[row], tb)
        total, pick = sum(rest), -1
        if total:
            goal = min(math.floor(float(u_last[b]) * float(total)), total - 1)
            run = 0
            for i, w in enumerate(rest):
                run += w
                if run > goal:
                    pick = i
                    break
        nxt.append(pick)
        out[row] = pick
    return acc, nxt, out


def build(B, drafts, V, pad, dtype, seed, kind="normal", with_draft=True, agree=1.0):
    g = torch.Generator().manual_seed(seed)
    rows = [int(torch.randint(0, drafts + 2, (1,), generator=g)) for _ in range(B)]
    rows[0] = drafts + 1
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    T = cu[-1] + 2  # rows behind the last request
    x = torch.randn(T, V + pad, generator=g) * 3
    if kind == "flat":
        x = x * 0
    elif kind == "ties":
        x = x.round()
    elif kind == "low":
        x = x - 60000 if dtype != torch.float16 else x - 6000
    elif kind == "masked":
        x[torch.rand(T, V + pad, generator=g) < 0.7] = float("-inf")
        x[:, 0] = float("nan")
    elif kind == "peak":
        x[:, V // 2] += 30
    y = x + torch.randn(T, V + pad, generator=g) * agree
    x[:, V:] = float("nan")
    y[:, V:] = float("inf")
    x, y = x.to(dtype).to(DEV)[:, :V], y.to(dtype).to(DEV)[:, :V]
    best = torch.nan_to_num(y.float(), nan=-1e30).argmax(1).cpu()
    other = torch.randint(0, V, (T,), generator=g)
    drawn = torch.where(torch.rand(T, generator=g) < 0.7, best, other)
    tokens = torch.cat([drawn[:1], drawn[:-1]]).to(torch.int32)
    u, u_last = torch.rand(T, generator=g), torch.rand(B, generator=g)
    t = torch.tensor([0.0, 0.7, 1.0, 1.6, 1e-39, -1.0])[torch.randint(0, 6, (B,), generator=g)]
    return x, (y if with_draft else None), tokens, cu, u, u_last, t


def run(x, y, tokens, cu, u, u_last, t, dt=None, **kw):
    from ffai_b200 import sampling
    d = lambda v: None if v is None else v.to(DEV)  # noqa: E731
    return sampling.verify(x, d(tokens), d(torch.tensor(cu, dtype=torch.int32)), d(u), d(u_last),
                           draft_logits=y, temperature=d(t), draft_temperature=d(dt), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["normal", "flat", "ties", "low", "masked", "peak"])
@pytest.mark.parametrize("B,drafts,V,pad", [(1, 0, 1, 0), (1, 1, 2, 1), (3, 4, 31, 0), (5, 3, 1000, 3),
                                            (2, 2, 5003, 0)])
def test_matches_the_definition(B, drafts, V, pad, kind, dtype):
    from ffai_b200 import attention
    for with_draft in (True, False):
        x, y, tokens, cu, u, u_last, t = build(B, drafts, V, pad, dtype, B * 7 + V, kind, with_draft)
        for temps, dtemps in ((t, None), (None, None), (t, t.flip(0).contiguous())):
            r = run(x, y, tokens, cu, u, u_last, temps, dtemps, with_logprob=True)
            want = reference(x, tokens.tolist(), cu, u, u_last, y,
                             None if temps is None else temps.tolist(),
                             None if dtemps is None else dtemps.tolist())
            assert r.accepted.tolist() == want[0]
            assert r.next.tolist() == want[1]
            assert r.tokens.tolist() == want[2]
            lp = torch.where(torch.isnan(x), float("-inf"), x.double())
            lp = lp - torch.logsumexp(lp, 1, keepdim=True)
            for i, tok in enumerate(want[2]):
                got = r.logprobs[i].item()
                assert got == 0 if tok < 0 else abs(got - lp[i, tok].item()) <= 6e-6
    attention.sync(0)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [51865, 131072, 200001, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_vocabularies(V, dtype):
    for with_draft, B, drafts in ((True, 3, 2), (False, 2, 1)):
        x, y, tokens, cu, u, u_last, t = build(B, drafts, V, 1, dtype, V, "normal", with_draft, agree=0.3)
        r = run(x, y, tokens, cu, u, u_last, t)
        want = reference(x, tokens.tolist(), cu, u, u_last, y, t.tolist())
        assert (r.accepted.tolist(), r.next.tolist(), r.tokens.tolist()) == want
        assert r.logprobs is None


@pytest.mark.gpu
def test_many_requests():
    x, y, tokens, cu, u, u_last, t = build(700, 3, 97, 0, torch.float32, 5)
    r = run(x, y, tokens, cu, u, u_last, t)
    want = reference(x, tokens.tolist(), cu, u, u_last, y, t.tolist())
    assert (r.accepted.tolist(), r.next.tolist(), r.tokens.tolist()) == want


@pytest.mark.gpu
def test_tokens_are_distributed_as_the_target():
    """The first emitted token over many uniform numbers: its frequencies are the
    target's, whatever the draft; within five standard deviations."""
    from ffai_b200 import sampling
    g = torch.Generator().manual_seed(2)
    V, n = 12, 20000
    x = (torch.randn(V, generator=g) * 1.5).to(DEV)
    y = (torch.randn(V, generator=g) * 1.5).to(DEV)
    p, q = torch.softmax(x.double(), 0).cpu(), torch.softmax(y.double(), 0).cpu()
    drafted = torch.multinomial(q, n, replacement=True, generator=g).to(torch.int32)
    tokens = torch.zeros(2 * n, dtype=torch.int32)
    tokens[1::2] = drafted
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32)
    for draft in (y.expand(2 * n, V).contiguous(), None):
        r = sampling.verify(x.expand(2 * n, V).contiguous(), tokens.to(DEV), cu.to(DEV),
                            torch.rand(2 * n, generator=g).to(DEV), torch.rand(n, generator=g).to(DEV),
                            draft_logits=draft)
        first = torch.bincount(r.tokens[0::2].cpu().long(), minlength=V) / n
        # drafts that were given come from q all the same here: the target's distribution again
        assert ((first - p).abs() <= 5 * (p * (1 - p) / n).sqrt() + 1e-6).all()


@pytest.mark.gpu
def test_rows_that_are_empty_infinite_or_equal():
    inf = float("inf")
    V = 9
    rows = torch.zeros(8, V)
    rows[0] = -inf                       # nothing to choose from: next -1
    rows[1] = float("nan")
    rows[2, 4], rows[2, 7] = inf, inf    # the infinite ones alone
    y = rows.clone()
    y[4] = -inf                          # a draft from nothing does not stand
    tokens = torch.tensor([0, 3, 0, 3, 0, 5, 0, 5], dtype=torch.int32)
    cu = [0, 2, 4, 6, 8]
    x = rows[[0, 5, 2, 2, 4, 5, 6, 7]].to(DEV)
    yd = y[[0, 5, 2, 2, 4, 5, 6, 7]].to(DEV)
    u, u_last = torch.full((8,), 0.99), torch.full((4,), 0.5)
    for draft in (yd, None):
        r = run(x, draft, tokens, cu, u, u_last, None, with_logprob=True)
        want = reference(x, tokens.tolist(), cu, u, u_last, draft)
        assert (r.accepted.tolist(), r.next.tolist(), r.tokens.tolist()) == want
    # equal distributions: everything stands, for any uniform number below 1
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 5000, generator=g).to(DEV)
    u = torch.full((4,), 1 - 2.0 ** -24)
    r = run(x, x.clone(), torch.tensor([7, 8, 9, 10], dtype=torch.int32), [0, 4], u, torch.tensor([0.3]), None)
    assert r.accepted.tolist() == [3] and r.tokens.tolist()[:3] == [8, 9, 10]


@pytest.mark.gpu
def test_drafts_outside_the_vocabulary_and_bad_rows():
    from ffai_b200 import attention
    x, y, _, _, u, u_last, _ = build(3, 3, 50, 0, torch.float32, 9)
    T = x.shape[0]
    tokens = torch.tensor(([0, -1, 50, 2 ** 31 - 1] * T)[:T], dtype=torch.int32)
    for draft in (y, None):
        cu = [0, 2, 3, 4]
        r = run(x, draft, tokens, cu, u, u_last, None)
        want = reference(x, tokens.tolist(), cu, u, u_last, draft)
        assert (r.accepted.tolist(), r.next.tolist()) == want[:2]
        assert r.tokens.tolist() == want[2]
        assert r.accepted.tolist() == [0, 0, 0]
    attention.sync(0)
    for cu in ([0, 3, 2, 4], [-1, 2, 3, 4], [0, 2, 3, T + 1]):
        try:
            r = run(x, y, tokens, cu, u, u_last, None)
            bad = [not (0 <= a <= b <= T) for a, b in zip(cu, cu[1:])]
            assert [n for n, z in zip(r.next.tolist(), bad) if z] == [-1] * sum(bad)
        finally:
            with pytest.raises(attention.AttnError):
                attention.sync(0)


@pytest.mark.gpu
def test_no_rows_at_all():
    x = torch.zeros(0, 10, device=DEV)
    z = torch.zeros(0, device=DEV)
    r = run(x, None, z.int().cpu(), [0, 0, 0], z.cpu(), torch.rand(2), None)
    assert r.accepted.tolist() == [0, 0] and r.next.tolist() == [-1, -1] and r.tokens.numel() == 0


@pytest.mark.gpu
def test_streams_and_captures_do_not_share_state():
    from ffai_b200 import sampling
    jobs = []
    for seed in range(4):
        x, y, tokens, cu, u, u_last, t = build(40, 4, 3001, 0, torch.float32, 60 + seed)
        args = [x, tokens.to(DEV), torch.tensor(cu, dtype=torch.int32, device=DEV), u.to(DEV), u_last.to(DEV)]
        kw = dict(draft_logits=y, temperature=t.to(DEV))
        jobs.append((args, kw, sampling.verify(*args, **kw).tokens.tolist()))
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for args, kw, _ in jobs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sampling.verify(*args, **kw))
        graphs.append(g)
    for _ in range(5):
        eager = []
        for s, g, (args, kw, _) in zip(streams, graphs, jobs[2:]):
            with torch.cuda.stream(s):
                g.replay()
                eager.append(sampling.verify(*args, **kw))
        torch.cuda.synchronize()
        for r, (_, _, want) in zip(outs + eager, jobs):
            assert r.tokens.tolist() == want


def test_refusals_without_a_device():
    from ffai_b200 import sampling
    with pytest.raises(ValueError):
        sampling.verify(torch.zeros(2, 5), torch.zeros(2).int(), torch.zeros(2).int(), torch.zeros(2),
                        torch.zeros(1))


@pytest.mark.gpu
def test_refusals():
    from ffai_b200 import attention, sampling
    x = torch.zeros(4, 20, device=DEV)
    tok, cu = torch.zeros(4, device=DEV).int(), torch.tensor([0, 4], device=DEV).int()
    u, last = torch.zeros(4, device=DEV), torch.zeros(1, device=DEV)
    ok = lambda **k: sampling.verify(**{**dict(logits=x, tokens=tok, cu_rows=cu, u=u, u_last=last), **k})  # noqa: E731
    ok()
    for bad in (dict(tokens=tok.long()), dict(tokens=tok[:3]), dict(cu_rows=cu[:1]), dict(u=u.double()),
                dict(u=u[:2]), dict(logits=x.double()), dict(logits=x.t()), dict(draft_logits=x.half()),
                dict(draft_logits=x[:, :19]), dict(draft_logits=x.cpu()), dict(temperature=u)):
        with pytest.raises(ValueError):
            ok(**bad)
    big = torch.zeros(1, 262145, device=DEV)
    with pytest.raises(attention.Declined):
        sampling.verify(big, tok[:1], torch.tensor([0, 1], device=DEV).int(), u[:1], last)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,B", [(31, 5), (1000, 40), (20011, 3)])
def test_infinite_temperatures_weigh_finite_logits_alike(V, B, dtype):
    """1 / T is 0 there: as for `sample`, every finite logit has the weight of the largest."""
    from ffai_b200 import sampling
    inf = float("inf")
    for kind in ("normal", "masked"):
        for with_draft in (True, False):
            x, y, tokens, cu, u, u_last, _ = build(B, 3, V, 1, dtype, V + B, kind, with_draft)
            hot = torch.full((B,), inf)
            mixed = torch.tensor([inf, 1.0, 0.0])[torch.arange(B) % 3]
            for t, dt in ((hot, hot), (hot, None), (mixed, mixed.flip(0).contiguous()), (torch.ones(B), hot)):
                r = run(x, y, tokens, cu, u, u_last, t, dt, with_logprob=True)
                want = reference(x, tokens.tolist(), cu, u, u_last, y, t.tolist(), None if dt is None else dt.tolist())
                assert (r.accepted.tolist(), r.next.tolist(), r.tokens.tolist()) == want
    # one row of each kind of logit, many uniform numbers: as often as `sample` takes them
    row = torch.tensor([0.5, -inf, 9.0, float("nan"), -70.0, 9.0], device=DEV, dtype=dtype)
    n = 600
    x, u = row.expand(n, 6).contiguous(), (torch.arange(n) / n + 1e-4).to(DEV)
    cu = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    r = sampling.verify(x, torch.zeros(n, dtype=torch.int32, device=DEV), cu, u, u, temperature=inf)
    got, want = (torch.bincount(v.long(), minlength=6).tolist() for v in (r.next, sampling.sample(x, u, temperature=inf)))
    assert got == want == [150, 0, 150, 0, 150, 150]


@pytest.mark.gpu
@pytest.mark.parametrize("with_draft", [True, False])
def test_one_long_request_among_many_without_drafts(with_draft):
    """Far more places than rows: 3000 requests, most without a row, one with 60."""
    g = torch.Generator().manual_seed(4)
    rows = (torch.rand(3000, generator=g) < 0.1).int().tolist()
    rows[1234], rows[7], rows[2999] = 60, 9, 5
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    T, V = cu[-1], 40
    x = torch.randn(T, V, generator=g).to(DEV)
    y = x + 0.05 * torch.randn(T, V, generator=g).to(DEV) if with_draft else None
    best = x.argmax(1).cpu()
    tokens = torch.cat([best[:1], best[:-1]]).to(torch.int32)
    u, u_last = torch.rand(T, generator=g) * (1 if with_draft else 0.1), torch.rand(3000, generator=g)
    r = run(x, y, tokens, cu, u, u_last, None)
    want = reference(x, tokens.tolist(), cu, u, u_last, y)
    assert (r.accepted.tolist(), r.next.tolist(), r.tokens.tolist()) == want
    assert max(want[0]) >= 5
