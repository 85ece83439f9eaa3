"""Sampling (ffai_sample) against its rule written out in whole numbers and 64
bits.  Weights are floor(2^36 e^d) of the f32 exponential of d, taken here
from the same f32 function on the GPU, so tokens must be equal; the
log-probability is f32: a sum of up to 2^18 positive f32 terms per row, in a
tree of at most ~300 sequential additions a thread, and a logarithm: 1e-4.
"""

import math

import pytest
import torch

DEV = "cuda:0"


def rule(x, u, t, k, p, m):
    """(token, logprob) of one row, the rule as written in the header."""
    x = [(-math.inf if v != v else v) for v in x.float().tolist()]
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    top = x[order[0]]
    if top == -math.inf:
        return -1, -math.inf
    f = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
    delta = torch.tensor([0.0 if v == top else v - top for v in x], dtype=torch.float64)
    # (x - max) is rounded once to f32
    delta = torch.where(torch.tensor([v == top for v in x]), torch.zeros(len(x)),
                        f(x) - f(top))
    lp = lambda i: float(delta[i].double() - torch.logsumexp(delta.double(), 0))  # noqa: E731
    inv = f(1.0) / f(t)
    if not t > 0 or math.isinf(float(inv)):
        return order[0], lp(order[0])
    d = torch.where(f(x) == -math.inf, torch.full((len(x),), -math.inf), delta * inv)
    w = (torch.exp(d.to(DEV)) * 2.0 ** 36).long().tolist()
    d = d.tolist()
    cum, run = [], 0
    for i in order:
        run += w[i]
        cum.append(run)
    n = k if 0 < k < len(x) else len(x)
    mass = cum[n - 1]
    if p < 1:
        goal = min(mass, max(1, math.ceil(max(p, 0.0) * float(mass))))
        mass = next(c for c in cum if c >= goal)
    if m > 0:
        floor = min(float(f(math.log(m))), 0.0)
        mass = min(mass, sum(wi for wi, di in zip(w, d) if di >= floor))
    target = max(0, min(mass - 1, math.floor(u * float(mass))))
    at = next(i for i, c in enumerate(cum) if c > target)
    return order[at], lp(order[at])


def f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (0.7, 1, 1.0, 0.0), (0.7, 40, 1.0, 0.0),
            (1.3, 0, 0.9, 0.0), (1.0, 50, 0.95, 0.0), (0.9, 0, 1.0, 0.05), (0.9, 30, 0.8, 0.02),
            (1.0, 0, 0.0, 0.0), (1.0, 0, 1e-6, 0.0), (1.0, 10 ** 6, 2.0, -1.0), (-1.0, 0, 1.0, 0.0),
            (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 7.0), (5.0, 3, 0.999, 0.0), (1e-30, 0, 0.9, 0.0),
            (1e-42, 0, 0.9, 0.0), (1e30, 0, 1.0, 0.0), (0.05, 0, 0.99, 0.0), (1.0, -3, 0.5, 0.5)]


def rows(kind, B, V, g):
    x = torch.randn(B, V, generator=g) * 3
    if kind == "ties":      # many equal logits
        x = (x * 2).round() / 2
    elif kind == "flat":
        x = torch.zeros(B, V)
    elif kind == "peak":
        x[torch.arange(B), torch.randint(0, V, (B,), generator=g)] = 60.0
    elif kind == "masked":  # suppressed tokens, not-numbers, signed zeros
        x[torch.rand(B, V, generator=g) < 0.5] = -math.inf
        x[torch.rand(B, V, generator=g) < 0.05] = math.nan
        x[torch.rand(B, V, generator=g) < 0.1] = -0.0
        x[torch.rand(B, V, generator=g) < 0.1] = 0.0
    elif kind == "tiny":    # neighbours a few units in the last place apart, about zero
        x = (torch.rand(B, V, generator=g) - 0.5) * 1e-6
    elif kind == "low":     # the type's lowest values beside ordinary ones
        x[:, ::2] = torch.finfo(torch.float16).min
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["normal", "ties", "flat", "peak", "masked", "tiny", "low"])
@pytest.mark.parametrize("V,pad", [(1, 0), (2, 1), (31, 0), (1000, 3), (1025, 7), (5003, 0)])
def test_every_setting(kind, V, pad, dtype):
    from ffai_b200 import sampling
    g = torch.Generator().manual_seed(V * 7 + len(kind))
    B = len(SETTINGS)
    full = torch.full((B, V + pad), math.inf)
    full[:, :V] = rows(kind, B, V, g)
    x = full.to(dtype).to(DEV)[:, :V]
    u = torch.rand(B, generator=g)
    u[0], u[4], u[5] = 0.0, 0.99999994, 0.5
    cols = [torch.tensor(c, device=DEV) for c in zip(*SETTINGS)]
    got, lp = sampling.sample(x, u.to(DEV), temperature=cols[0].float(), top_k=cols[1].to(torch.int32),
                              top_p=cols[2].float(), min_p=cols[3].float(), with_logprob=True)
    got, lp = got.tolist(), lp.tolist()
    for b, (t, k, p, m) in enumerate(SETTINGS):
        want, want_lp = rule(x[b].cpu(), float(u[b]), f32(t), k, f32(p), f32(m))
        assert got[b] == want, f"row {b} {SETTINGS[b]}: {got[b]}, rule {want}"
        assert lp[b] == want_lp or abs(lp[b] - want_lp) <= 1e-4 * max(1.0, abs(want_lp))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [51865, 131072, 262144])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_vocabularies(V, dtype):
    from ffai_b200 import sampling
    g = torch.Generator().manual_seed(V)
    use = [0, 3, 4, 5, 7, 10]
    x = (torch.randn(len(use), V, generator=g) * 2.5).to(dtype).to(DEV)
    x[3] = x[3].clamp(max=4.0)  # a crowd of equal maxima
    u = torch.rand(len(use), generator=g)
    cols = [torch.tensor(c, device=DEV) for c in zip(*[SETTINGS[i] for i in use])]
    got = sampling.sample(x, u.to(DEV), temperature=cols[0].float(), top_k=cols[1].to(torch.int32),
                          top_p=cols[2].float(), min_p=cols[3].float()).tolist()
    for b, i in enumerate(use):
        t, k, p, m = SETTINGS[i]
        want, _ = rule(x[b].cpu(), float(u[b]), f32(t), k, f32(p), f32(m))
        assert got[b] == want, f"row {b}"


@pytest.mark.gpu
def test_empty_and_infinite_rows():
    from ffai_b200 import sampling
    x = torch.zeros(5, 40, device=DEV)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 7] = x[2, 30] = math.inf
    x[3, 5] = math.inf
    x[4, :39] = -math.inf
    u = torch.full((5,), 0.6, device=DEV)
    tok, lp = sampling.sample(x, u, with_logprob=True)
    assert tok.tolist() == [-1, -1, 30, 5, 39]
    assert lp[0] == lp[1] == -math.inf and lp[3] == lp[4] == 0
    assert abs(lp[2].item() + math.log(2)) < 1e-6
    assert sampling.sample(x, u, temperature=0.0).tolist() == [-1, -1, 7, 5, 39]


@pytest.mark.gpu
def test_frequencies():
    """Uniform numbers spread evenly over [0, 1) give each kept token its share."""
    from ffai_b200 import sampling
    N = 20000
    x = torch.tensor([1.0, 3.0, 2.0, -1.0, 0.5], device=DEV)
    u = (torch.arange(N, device=DEV) + 0.5) / N
    tok = sampling.sample(x.expand(N, 5).contiguous(), u.float(), temperature=0.8, top_p=0.95)
    share = torch.bincount(tok.long(), minlength=5).double() / N
    w = torch.softmax(x.double() / 0.8, 0)
    keep = torch.zeros(5, device=DEV).double()
    order = w.argsort(descending=True)
    n = int((w[order].cumsum(0) < 0.95).sum()) + 1
    keep[order[:n]] = w[order[:n]]
    assert (share - keep / keep.sum()).abs().max() <= 2 / N + 1e-6


@pytest.mark.gpu
def test_settings_as_numbers_and_streams():
    from ffai_b200 import sampling
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 3001, generator=g).to(DEV)
    u = torch.rand(6, generator=g).to(DEV)
    a = sampling.sample(x, u, temperature=0.7, top_k=20, top_p=0.9, min_p=0.01)
    full = lambda v, dt: torch.full((6,), v, dtype=dt, device=DEV)  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = sampling.sample(x, u, temperature=full(0.7, torch.float32), top_k=full(20, torch.int32),
                            top_p=full(0.9, torch.float32), min_p=full(0.01, torch.float32))
    s.synchronize()
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals():
    from ffai_b200 import attention, sampling
    x = torch.zeros(2, 10, device=DEV)
    u = torch.zeros(2, device=DEV)
    with pytest.raises(attention.Declined):
        sampling.sample(torch.zeros(1, 262145, device=DEV), u[:1])
    with pytest.raises(ValueError):
        sampling.sample(x.double(), u)
    with pytest.raises(ValueError):
        sampling.sample(x.t(), torch.zeros(10, device=DEV))
    with pytest.raises(ValueError):
        sampling.sample(x, u.double())
    with pytest.raises(ValueError):
        sampling.sample(x, u, top_k=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError):
        sampling.sample(x, u[:1])
    with pytest.raises(attention.AttnError):
        sampling.sample(torch.zeros(0, 10, device=DEV), u[:0])


@pytest.mark.gpu
def test_streams_and_captures_do_not_share_state():
    """Calls queued on two streams without order between them, and a capture on
    a stream of its own."""
    from ffai_b200 import sampling
    g = torch.Generator(device="cuda").manual_seed(8)
    sets = [(torch.randn(n, 60001, generator=g, device="cuda") * 3,
             torch.rand(n, generator=g, device="cuda")) for n in (7, 90)]
    want = [sampling.sample(x, u, top_p=0.9) for x, u in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(sampling.sample(*sets[i], top_p=0.9))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sampling.sample(*sets[1], top_p=0.9)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[1])


def logprob_bounds(x, tokens):
    """(log-probabilities of tokens in 64 bits, bounds of the f32 ones).

    A term e^(x - max) is off by the rounding of x - max, 2^-24 |x - max|, an
    f32 exponential, 2^-23, and three additions within a group of four, 3 2^-24;
    what follows is 64 bits, up to the result's own rounding, 2^-24 of it:
    2^-24 (mean of |x - max| under the softmax + 6 + |result|)."""
    x = x.double().cpu()
    d = x - x.amax(1, keepdim=True)
    z = torch.logsumexp(d, 1)
    lp = d.gather(1, tokens.long().cpu().view(-1, 1))[:, 0] - z
    w = torch.softmax(d, 1)
    mean = torch.where(w > 0, w * d.abs(), torch.zeros_like(w)).sum(1)
    return lp, 2.0 ** -24 * (mean + 6 + lp.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [37, 5003, 51865, 131072, 262144])
def test_logprobs_hold_to_f32_rounding(V, dtype):
    from ffai_b200 import sampling
    g = torch.Generator().manual_seed(V + 1)
    kinds = ["normal", "peak", "flat", "ties", "tiny", "low"]
    x = torch.cat([rows(k, 2, V, g) for k in kinds]).to(dtype)
    x[0, ::3] = -math.inf
    x[2] -= 30.0  # a peak that outweighs the rest by far, away from zero
    B = x.shape[0]
    u = torch.rand(B, generator=g).to(DEV)
    temperature = torch.tensor([0.0, 1.0] * (B // 2), device=DEV)
    for settings in (dict(), dict(temperature=0.0), dict(temperature=temperature, top_p=0.9),
                     dict(temperature=2.0, top_k=40, min_p=0.01)):
        tok, lp = sampling.sample(x.to(DEV), u, with_logprob=True, **settings)
        assert (tok >= 0).all()
        want, tol = logprob_bounds(x.float(), tok)
        err = (lp.cpu().double() - want).abs()
        assert (err <= tol).all(), f"{(err / tol).max():.2f} of the bound"
