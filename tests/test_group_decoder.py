"""The batched decode operators chained (ffai_b200.group_decoder) against a
dense computation in 64 bits from the same projected queries, keys and values.

Tolerance of a layer's output y = x + o W^T, per element: attention's own
(2^-8 + 1e-4) A_j + 2^-8 |o_j| (its bf16 output) goes through |W|, the GEMM sums
512 products in f32 (1e-4 of sum |o_j w_j| covers it), and y is rounded to bf16
once, 2^-8 |y|.
"""

import pytest
import torch

DEV = "cuda:0"
H, HK, D, V = 8, 2, 512, 1001


def make(num_pages=40, max_len=200, batch=6, seed=0):
    from ffai_b200.group_decoder import GroupDecoder
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = lambda *s: (torch.randn(s, generator=g, device=DEV) * s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
    dec = GroupDecoder(w((H + 2 * HK) * 64, D), w(D, H * 64), w(V, D), heads=H, kv_heads=HK,
                       batch=batch, max_len=max_len, num_pages=num_pages)
    x = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    return dec, x, g


def expected(dec, x, own, prefix, starts):
    """(y, tolerance) f64 of the layer on x (B, n, D), own[b] = (k, v) of the
    request's keys with the new ones, prefix[g] likewise."""
    B, n, _ = x.shape
    q = dec._project(x.reshape(B * n, D))[0].double().view(B, n, HK, H // HK, 64)
    o = torch.zeros((B, n, H * 64), dtype=torch.float64, device=DEV)
    e = torch.zeros_like(o)
    for b in range(B):
        gi = next((i for i in range(len(prefix)) if starts[i] <= b < starts[i + 1]), None)
        parts = ([prefix[gi]] if gi is not None else []) + [own[b]]
        k, v = (torch.cat([p[i] for p in parts]).double() for i in (0, 1))
        for i in range(n):
            see = k.shape[0] - (n - 1 - i)
            w = torch.softmax(torch.einsum("hgd,khd->hgk", q[b, i], k[:see]) * dec.scale, 2)
            o[b, i] = torch.einsum("hgk,khd->hgd", w, v[:see]).flatten()
            a = torch.einsum("hgk,khd->hgd", w, v[:see].abs()).flatten()
            e[b, i] = (2 ** -8 + 1e-4) * a + 2 ** -8 * o[b, i].abs()
    wo = dec.w_out.double()
    y = x.double() + o @ wo.T
    tol = e @ wo.abs().T + 1e-4 * (o.abs() @ wo.abs().T) + 2 ** -8 * y.abs() + 1e-6
    return y, tol


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3])
def test_steps_match_a_dense_computation(n):
    from ffai_b200 import attention, gemm, sampling
    dec, rand, g = make()
    sizes, starts = [3, 2], [0, 3, 5]  # the sixth request has no prompt
    prompts = [rand(130, D), rand(70, D)]
    dec.open(prompts, sizes)
    prefix = [tuple(t.clone() for t in dec._project(p)[1:]) for p in prompts]
    empty = torch.zeros((0, HK, 64), dtype=torch.bfloat16, device=DEV)
    own = [(empty, empty) for _ in range(6)]
    for step in range(40):
        x = rand(6, n, D)
        on = [1, 1, step % 3 > 0, 1, 1, step > 2]
        active = torch.tensor(on, dtype=torch.int32, device=DEV)
        y, served = dec.hidden(x, active)
        assert served.tolist() == [bool(a) for a in on]
        k, v = (t.view(6, n, HK, 64) for t in dec._project(x.view(6 * n, D))[1:])
        for b in range(6):
            if on[b]:
                own[b] = torch.cat([own[b][0], k[b]]), torch.cat([own[b][1], v[b]])
        assert dec.lens.tolist() == [o[0].shape[0] for o in own]
        if step % 13 == 12 or step < 2:
            rows = [b for b in range(6) if on[b]]
            want, tol = expected(dec, x, own, prefix, starts)
            assert ((y.double() - want).abs() <= tol)[rows].all()
        if step == 20:  # two requests end and start again
            dec.close(torch.tensor([0, 1, 0, 0, 1, 0], dtype=torch.int32, device=DEV))
            own[1] = own[4] = (empty, empty)
    # the step is the layer, the vocabulary projection and the sampler
    x, u = rand(6, n, D), torch.rand(6 * n, generator=g, device=DEV)
    active = torch.tensor([1, 1, 0, 1, 1, 1], dtype=torch.int32, device=DEV)
    lens, free = dec.lens.clone(), dec.free_count.clone()
    y, _ = dec.hidden(x, active)
    dec.lens.copy_(lens)
    dec.free_count.copy_(free)
    tokens = dec.step(x, active, u, temperature=0.7, top_k=50, top_p=0.9)
    logits = gemm.linear(y.view(6 * n, D), dec.w_vocab, out_dtype=torch.float32)[:, :V]
    want = sampling.sample(logits, u, temperature=0.7, top_k=50, top_p=0.9).view(6, n)
    want[2] = -1
    assert torch.equal(tokens, want) and (tokens[[0, 1, 3, 4, 5]] >= 0).all()
    dec.close(torch.ones(6, dtype=torch.int32, device=DEV))
    dec.close_groups()
    assert dec.free_count.item() == 40
    assert sorted(dec.free_pages.tolist()) == list(range(40))
    attention.sync(0)


@pytest.mark.gpu
def test_a_short_pool_refuses_requests_not_others():
    dec, rand, _ = make(num_pages=6, max_len=100)
    dec.open([rand(64, D)], [6])  # five pages left for six requests
    u = torch.full((6,), 0.5, device=DEV)
    active = torch.ones(6, dtype=torch.int32, device=DEV)
    tokens = dec.step(rand(6, 1, D), active, u)
    assert (tokens[:5] >= 0).all() and tokens[5].item() == -1
    assert dec.lens.tolist() == [1, 1, 1, 1, 1, 0] and dec.free_count.item() == 0
    dec.close(torch.tensor([1, 0, 0, 0, 0, 0], dtype=torch.int32, device=DEV))
    tokens = dec.step(rand(6, 1, D), torch.tensor([0, 1, 1, 1, 1, 1], dtype=torch.int32, device=DEV), u)
    assert (tokens[1:] >= 0).all() and tokens[0].item() == -1
    with pytest.raises(MemoryError):
        dec.open([rand(64, D)], [1])
    with pytest.raises(ValueError):
        dec.open([rand(64, D)], [7])


@pytest.mark.gpu
def test_a_captured_step_continues():
    """Replays of one captured step against the same steps one by one."""
    runs = []
    for captured in (False, True):
        dec, rand, g = make(seed=3)
        dec.open([rand(300, D), rand(1, D)], [4, 2])
        active = torch.ones(6, dtype=torch.int32, device=DEV)
        xs = [rand(6, 1, D) for _ in range(8)]
        us = [torch.rand(6, generator=g, device=DEV) for _ in range(8)]
        x, u = xs[0].clone(), us[0].clone()
        out = [dec.step(x, active, u, temperature=0.9, min_p=0.01)]
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = dec.step(x, active, u, temperature=0.9, min_p=0.01)
        for i in range(1, 8):
            x.copy_(xs[i])
            u.copy_(us[i])
            if captured:
                graph.replay()
                out.append(got.clone())
            else:
                out.append(dec.step(x, active, u, temperature=0.9, min_p=0.01))
        runs.append((torch.stack(out), dec.lens.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and runs[0][1].tolist() == runs[1][1].tolist() == [8] * 6


@pytest.mark.gpu
def test_a_captured_step_outlives_its_groups():
    """A step captured over one set of prompts, replayed over others, more and
    fewer, shorter and longer: the tokens of steps that were never captured, to
    the bit, with other work taking the memory that a call sets free."""
    from ffai_b200 import attention
    rounds = [([300, 1], [4, 2]), ([700, 30, 65, 129], [1, 2, 2, 1]), ([64], [5]), ([10, 900], [0, 6])]
    runs = []
    for captured in (False, True):
        dec, rand, g = make(num_pages=60, seed=5)
        held = [(t, t.data_ptr()) for t in (dec.prefix_table, dec.prefix_lens, dec.group_starts,
                                            dec.block_table, dec.lens, dec.free_pages, dec.free_count)]
        active = torch.ones(6, dtype=torch.int32, device=DEV)
        x, u = rand(6, 1, D), torch.rand(6, generator=g, device=DEV)
        tokens, graph = [], None
        for ns, sizes in rounds:
            dec.open([rand(n, D) for n in ns], sizes)
            for _ in range(3):
                x.copy_(rand(6, 1, D))
                u.copy_(torch.rand(6, generator=g, device=DEV))
                noise = [torch.full((2 ** k,), -1, dtype=torch.int32, device=DEV) for k in range(12)]
                if not captured:
                    got = dec.step(x, active, u, temperature=0.9, min_p=0.01)
                else:
                    if graph is None:
                        lens, count = dec.lens.clone(), dec.free_count.clone()
                        table = dec.block_table.clone()
                        dec.step(x, active, u, temperature=0.9, min_p=0.01)
                        for t, v in ((dec.lens, lens), (dec.free_count, count), (dec.block_table, table)):
                            t.copy_(v)
                        graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(graph):
                            out = dec.step(x, active, u, temperature=0.9, min_p=0.01)
                    graph.replay()
                    got = out
                tokens.append(got.clone())
                del noise
            dec.close(active)
            dec.close_groups()
            assert dec.free_count.item() == 60
        assert all(t.data_ptr() == at for t, at in held)
        assert all(a is b for a, (b, _) in zip((dec.prefix_table, dec.prefix_lens, dec.group_starts),
                                               held))
        runs.append(torch.stack(tokens))
    assert (runs[0] >= 0).all() and torch.equal(runs[0], runs[1])
    attention.sync(0)


@pytest.mark.gpu
def test_bounds_on_prompts():
    """Prompts past the bounds are refused before anything changes."""
    from ffai_b200.group_decoder import GroupDecoder
    dec, rand, g = make(num_pages=20)
    w = lambda *s: rand(*s)  # noqa: E731
    tight = GroupDecoder(dec.w_qkv, dec.w_out, w(V, D), heads=H, kv_heads=HK, batch=6, max_len=200,
                         num_pages=20, max_groups=2, max_prompt=100)
    for prompts, sizes in (([rand(101, D)], [1]), ([rand(1, D)] * 3, [1, 1, 1])):
        with pytest.raises(ValueError):
            tight.open(prompts, sizes)
        assert tight.free_count.item() == 20 and tight.group_starts.tolist() == [0, 0, 0]
    prompts = [rand(100, D), rand(65, D)]
    x, active = rand(6, 1, D), torch.ones(6, dtype=torch.int32, device=DEV)
    out = []
    for d in (tight, dec):  # bounds change the layout, not the result
        d.open(prompts, [2, 3])
        out.append(d.hidden(x, active)[0].double())
    prefix = [tuple(t.clone() for t in dec._project(p)[1:]) for p in prompts]
    k, v = dec._project(x.view(6, D))[1:]
    want, tol = expected(dec, x, [(k[b:b + 1], v[b:b + 1]) for b in range(6)], prefix, [0, 2, 5])
    assert all(((y - want).abs() <= tol).all() for y in out)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,sizes", [([], []), ([0], [3]), ([0, 0], [1, 5]), ([0, 70], [2, 2])])
def test_empty_prompts(lens, sizes):
    from ffai_b200 import attention
    dec, rand, _ = make(seed=8)
    prompts = [rand(n, D) for n in lens]
    dec.open(prompts, sizes)
    x, active = rand(6, 1, D), torch.ones(6, dtype=torch.int32, device=DEV)
    y, served = dec.hidden(x, active)
    assert served.all()
    prefix = [tuple(t.clone() for t in dec._project(p)[1:]) if len(p) else
              (torch.zeros((0, HK, 64), dtype=torch.bfloat16, device=DEV),) * 2 for p in prompts]
    starts = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    k, v = dec._project(x.view(6, D))[1:]
    want, tol = expected(dec, x, [(k[b:b + 1], v[b:b + 1]) for b in range(6)], prefix, starts)
    assert ((y.double() - want).abs() <= tol).all()
    dec.close(active)
    dec.close_groups()
    assert dec.free_count.item() == 40
    attention.sync(0)
