"""Steps of drafted tokens chained (ffai_b200.draft_decoder) against a dense
computation in 64 bits from the same projected queries, keys and values.

Tolerance of a layer's output y = x + o W^T, per element: attention's weights are
rounded to bf16 once and so is its output, (2^-8 + 1e-4) A_j + 2^-8 |o_j| with A
the weighted sum of |v|; that goes through |W|, the GEMM sums 512 products in f32
(1e-4 of sum |o_j w_j| covers it), and y is rounded to bf16 once, 2^-8 |y|.
"""

import pytest
import torch

DEV = "cuda:0"
H, HK, D, V, B = 8, 2, 512, 1001, 6


def make(num_pages=40, max_len=400, seed=0):
    from ffai_b200.draft_decoder import DraftDecoder
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    w = lambda *s: x(*s) * s[-1] ** -0.5  # noqa: E731
    dec = DraftDecoder(w((H + 2 * HK) * 64, D), w(D, H * 64), w(V, D), heads=H, kv_heads=HK,
                       batch=B, max_len=max_len, num_pages=num_pages)
    return dec, x, g


def starts(ns):
    cu = [0]
    for n in ns:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def check_layer(dec, x, y, cu, own):
    """y of `hidden` on x; own[b] = (k, v) with the new keys, None: not served."""
    q = dec._project(x)[0].double()
    wo = dec.w_out.double()
    cu = cu.tolist()
    for b in range(B):
        n = cu[b + 1] - cu[b]
        if n == 0 or own[b] is None:
            continue
        k, v = (t.double() for t in own[b])
        qb = q[cu[b]:cu[b + 1]].view(n, HK, H // HK, 64)
        s = torch.einsum("nhgd,khd->nhgk", qb, k) * dec.scale
        see = torch.arange(k.shape[0], device=DEV) < k.shape[0] - n + 1 + torch.arange(n, device=DEV)[:, None]
        w = torch.softmax(s.masked_fill(~see[:, None, None], -torch.inf), 3)
        o = torch.einsum("nhgk,khd->nhgd", w, v).reshape(n, -1)
        a = torch.einsum("nhgk,khd->nhgd", w, v.abs()).reshape(n, -1)
        xb = x[cu[b]:cu[b + 1]].double()
        want = xb + o @ wo.T
        e = (2 ** -8 + 1e-4) * a + 2 ** -8 * o.abs()
        tol = e @ wo.abs().T + 1e-4 * (o.abs() @ wo.abs().T) + 2 ** -8 * want.abs() + 1e-6
        assert ((y[cu[b]:cu[b + 1]].double() - want).abs() <= tol).all(), b


def cached(dec, b):
    """(k, v) of request b as the pools hold them."""
    n = dec.lens[b].item()
    pages = dec.block_table[b, :(n + 63) // 64].long()
    return tuple(p[pages].transpose(1, 2).reshape(-1, HK, 64)[:n] for p in (dec.k_pool, dec.v_pool))


def check_pages(dec, own):
    """Every request holds its keys, and no page is lost or held twice."""
    used = set()
    for b in range(B):
        assert dec.lens[b].item() == own[b][0].shape[0]
        assert all(torch.equal(a, c) for a, c in zip(cached(dec, b), own[b]))
        used.update(dec.block_table[b, :(dec.lens[b].item() + 63) // 64].tolist())
    free = dec.free_pages[:dec.free_count.item()].tolist()
    assert sorted(free + list(used)) == list(range(dec.free_pages.numel()))
    return used


@pytest.mark.gpu
@pytest.mark.parametrize("drafted", [True, False])
def test_steps_match_a_dense_computation(drafted):
    from ffai_b200 import attention, gemm, sampling
    dec, rand, g = make()
    empty = torch.zeros((0, HK, 64), dtype=torch.bfloat16, device=DEV)
    own = [(empty, empty)] * B
    prompts, took = [130, 64, 1, 63, 0, 200], 0
    for step in range(24):
        drafts = [[4, 0, 7, 1, 2, 3], [0, 0, 1, 12, 0, 2], [1] * 6][step % 3]
        if step == 0:  # the prompts, whole
            ns, settled = prompts, [0] * 6
        elif step in (5, 11):  # a chunk beside the others' drafts, one sits out
            ns = [d + 1 for d in drafts]
            ns[1], ns[4] = 70, 0
            settled = [0 if b in (1, 4) else n for b, n in enumerate(ns)]
        else:
            ns = settled = [d + 1 for d in drafts]
        cu, T = starts(ns), sum(ns)
        x = rand(T, D)
        y, served = dec.hidden(x, cu, max_rows=max(ns))
        assert served.tolist() == [n > 0 for n in ns]
        k, v = dec._project(x)[1:]
        new = [(k[a:a + n], v[a:a + n]) for a, n in zip(cu.tolist(), ns)]
        grown = [tuple(torch.cat(p) for p in zip(own[b], new[b])) for b in range(B)]
        check_layer(dec, x, y, cu, grown)
        rows = torch.cat([torch.arange(a, a + j) for a, j in zip(cu.tolist(), settled)]).to(DEV)
        R, cj = rows.numel(), starts(settled)
        tokens = torch.randint(0, V, (R,), generator=g, device=DEV, dtype=torch.int32)
        u, u_last = (torch.rand(n, generator=g, device=DEV) for n in (R, B))
        settings = dict(temperature=0.8, draft_temperature=1.1)
        if drafted:
            settings["draft_logits"] = torch.randn(R, V, generator=g, device=DEV)
        else:
            u *= 2e-3  # (a given draft stands where u < p)
        got = dec.settle(y[rows], tokens, cj, u, u_last, served, **settings)
        if R:
            logits = gemm.linear(y[rows], dec.w_vocab, out_dtype=torch.float32)[:, :V]
            want = sampling.verify(logits, tokens, cj, u, u_last, **settings)
            for a, c in zip(got[:3], want[:3]):
                assert torch.equal(a, torch.where(served, c, -1) if c is want.next else c)
        took += got.accepted.sum().item()
        for b, (j, a) in enumerate(zip(settled, got.accepted.tolist())):
            n = grown[b][0].shape[0] - (j - 1 - a if j else 0)
            own[b] = tuple(t[:n] for t in grown[b])
        check_pages(dec, own)
        if step in (3, 8, 14):  # requests split and end; every second time the pool is made dense
            src = [[0, 0, 2, 2, -1, 5], [1, 1, 1, 1, 4, 5], [5, 4, 3, 2, 1, 0]][step % 3]
            whole = dec.select(torch.tensor(src, dtype=torch.int32, device=DEV))
            assert whole.all()
            own = [own[s] if s >= 0 else (empty, empty) for s in src]
            used = check_pages(dec, own)
            if step != 8:
                dec.compact()
                assert check_pages(dec, own) == set(range(len(used)))
    assert took > 20  # drafts stood, and drafts fell
    assert dec.select(torch.full((B,), -1, dtype=torch.int32, device=DEV)).all()
    assert dec.free_count.item() == 40
    attention.sync(0)


@pytest.mark.gpu
def test_a_short_pool_refuses_requests_not_others():
    from ffai_b200 import attention
    dec, rand, g = make(num_pages=4)
    cu = starts([60, 64, 1, 0, 0, 0])
    _, served = dec.hidden(rand(125, D), cu)
    assert served.tolist() == [True] * 3 + [False] * 3 and dec.free_count.item() == 1
    ns = [6, 3, 2, 0, 0, 2]  # the first takes the last page; two find none
    cu, T = starts(ns), sum(ns)
    tokens = torch.zeros(T, dtype=torch.int32, device=DEV)
    v = dec.step(rand(T, D), tokens, cu, torch.ones(T, device=DEV) * 0.999, torch.zeros(B, device=DEV),
                 with_logprob=True)
    kept = [61, 64, 2, 0, 0, 0]
    assert dec.lens.tolist() == [k + a for k, a in zip(kept, v.accepted.tolist())]
    assert [t >= 0 for t in v.next.tolist()] == [True, False, True, False, False, False]
    rows = [(v.tokens[a:a + n] >= 0).any().item() for a, n in zip(cu.tolist(), ns)]
    assert rows == [True, False, True, False, False, False]
    assert torch.equal(v.logprobs != 0, v.tokens >= 0)
    # a split needs a copy and finds no page: the whole pages stay
    dec.hidden(rand(66, D), starts([0, 0, 60, 0, 0, 6]))
    whole = dec.select(torch.tensor([2, 1, 2, -1, 1, 1], dtype=torch.int32, device=DEV))
    lens = dec.lens.tolist()
    assert lens[1] == lens[4] == lens[5] == 64 and whole[[1, 3, 4, 5]].all()
    assert whole.tolist()[:3:2] == [n > 60 for n in lens[:3:2]]
    attention.sync(0)


@pytest.mark.gpu
def test_a_captured_step_continues():
    """Replays of one captured step, of other lengths each, against the same steps one
    by one: the same tokens."""
    from ffai_b200 import attention
    runs = []
    for captured in (False, True):
        dec, rand, g = make(seed=3)
        dec.hidden(rand(400, D), starts([300, 1, 0, 64, 35, 0]))
        counts = [[5, 1, 3, 2, 4, 1], [1] * 6, [0, 5, 5, 2, 1, 3], [2, 2, 2, 2, 2, 2], [4, 0, 0, 0, 0, 12]]
        x, tokens = torch.zeros((16, D), dtype=torch.bfloat16, device=DEV), torch.zeros(16, dtype=torch.int32, device=DEV)
        u, u_last, cu = torch.zeros(16, device=DEV), torch.zeros(B, device=DEV), starts([0] * B)
        q = torch.zeros((16, V), device=DEV)

        def run():
            return dec.step(x, tokens, cu, u, u_last, draft_logits=q, max_rows=12)

        run()  # nothing: no request has a row
        assert dec.lens.tolist() == [300, 1, 0, 64, 35, 0]
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = run()
        for ns in counts + counts:
            x.copy_(rand(16, D))
            q.copy_(torch.randn(16, V, generator=g, device=DEV))
            tokens.copy_(torch.randint(0, V, (16,), generator=g, device=DEV))
            u.copy_(torch.rand(16, generator=g, device=DEV))
            u_last.copy_(torch.rand(B, generator=g, device=DEV))
            cu.copy_(starts(ns))
            if captured:
                graph.replay()
            else:
                out = run()
            runs.append(torch.cat([out.accepted, out.next, out.tokens, dec.lens]))
    half = len(runs) // 2
    assert all(torch.equal(a, b) for a, b in zip(runs[:half], runs[half:]))
    attention.sync(0)


@pytest.mark.gpu
def test_refusals():
    from ffai_b200.draft_decoder import DraftDecoder
    dec, rand, _ = make()
    for w in ((dec.w_qkv[:64], dec.w_out, dec.w_vocab), (dec.w_qkv, dec.w_out[:, :64], dec.w_vocab),
              (dec.w_qkv, dec.w_out, dec.w_vocab[:, :64])):
        with pytest.raises(ValueError):
            DraftDecoder(*w, heads=H, kv_heads=HK, batch=B, max_len=64, num_pages=6)


def on_the_host():
    """A decoder whose tensors lie on the host; its operators are the caller's to replace."""
    from ffai_b200.draft_decoder import DraftDecoder
    w = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    return DraftDecoder(w((H + 2 * HK) * 64, D), w(D, H * 64), w(V, D), heads=H, kv_heads=HK, batch=B,
                        max_len=128, num_pages=12)


def test_a_selection_of_no_request_is_not_looked_up(monkeypatch):
    """An index past the batch would end the process on a device."""
    from ffai_b200 import kvcache
    dec = on_the_host()
    dec.lens.copy_(torch.arange(B, dtype=torch.int32) + 10)

    def fork(src, lens, table, free_pages, free_count, keep=None):
        real = (src >= 0) & (src < B)
        return kvcache.Fork(table, torch.where(real, lens[src.clamp(0, B - 1)], 0), None, None, None, free_count)

    monkeypatch.setattr(kvcache, "fork_pages", fork)
    monkeypatch.setattr(kvcache, "copy_pages", lambda *a, **k: None)
    for src in ([0, B, 2 ** 31 - 1, -5, 1, 1], [B] * B):
        whole = dec.select(torch.tensor(src, dtype=torch.int32))
        assert whole.tolist() == [s < B for s in src]
    lens = dec.lens.clone()
    for n in (B - 1, B + 1):
        with pytest.raises(ValueError):
            dec.select(torch.zeros(n, dtype=torch.int32))
    assert torch.equal(dec.lens, lens)


@pytest.mark.gpu
def test_a_selection_of_no_request_is_reported():
    from ffai_b200 import attention
    dec, rand, _ = make()
    dec.hidden(rand(110, D), starts([10, 70, 0, 30, 0, 0]))
    whole = dec.select(torch.tensor([1, B, 2 ** 31 - 1, 3, -1, 0], dtype=torch.int32, device=DEV))
    assert whole.tolist() == [True, False, False, True, True, True]
    assert dec.lens.tolist() == [70, 0, 0, 30, 0, 10]
    with pytest.raises(attention.AttnError):
        attention.sync(0)
    attention.sync(0)


def test_rows_outside_every_request_get_no_slot(monkeypatch):
    """Rows before the first request and behind the last are nobody's: their keys go nowhere."""
    from ffai_b200 import chunk_attention, draft_decoder, kvcache
    dec, written = on_the_host(), []
    monkeypatch.setattr(draft_decoder, "linear", lambda x, w, **k: torch.zeros(x.shape[0], w.shape[0], dtype=x.dtype))
    monkeypatch.setattr(kvcache, "plan_pages", lambda lens, n, pages, count, table, slot_cap: kvcache.PagePlan(
        lens=lens + n, cu_new=torch.cat([n.new_zeros(1), n.cumsum(0, dtype=torch.int32)]),
        slots=torch.arange(100, 100 + slot_cap, dtype=torch.int32), positions=None, free_count=count))
    monkeypatch.setattr(kvcache, "write_slots", lambda kp, vp, k, v, slots: written.append(slots.tolist()))
    monkeypatch.setattr(chunk_attention, "attend", lambda q, *a, **k: torch.zeros(q.shape, dtype=q.dtype))
    for first, last in ((0, 0), (3, 0), (0, 2), (5, 4)):
        cu = torch.tensor([0, 2, 2, 3, 7, 8, 9], dtype=torch.int32) + first
        T = first + 9 + last
        _, served = dec.hidden(torch.zeros(T, D, dtype=torch.bfloat16), cu)
        assert served.tolist() == [True, False, True, True, True, True]
        assert written.pop() == [-1] * first + list(range(100, 109)) + [-1] * last


@pytest.mark.gpu
def test_rows_before_the_first_request_change_nothing():
    from ffai_b200 import attention
    dec, rand, _ = make(seed=1)
    ns, first = [30, 70, 1, 0, 64, 5], 3
    x, cu = rand(first + sum(ns) + 4, D), starts(ns) + first
    y, served = dec.hidden(x, cu)
    assert served.tolist() == [n > 0 for n in ns]
    k, v = dec._project(x)[1:]
    own = [(k[a:a + n], v[a:a + n]) for a, n in zip(cu.tolist(), ns)]
    check_pages(dec, own)
    check_layer(dec, x, y, cu, own)
    attention.sync(0)
