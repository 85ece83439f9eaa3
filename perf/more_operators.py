"""Operators of a server that checks drafted tokens and reuses pages, measured:
attention of a chunk of new tokens over a paged cache, verification of drafted
tokens, forks of requests that share pages, and compaction of a pool.

A case is a dict of plain values.  `op` names the operator:

  chunk    ffai_b200.chunk_attention.attend
  verify   ffai_b200.sampling.verify
  fork     ffai_b200.kvcache.fork_pages, then copy_pages
  compact  ffai_b200.kvcache.compact_pages, then copy_pages

With `own` true, `run` makes the framework's calls; with `own` false it
computes the same in elementary torch operations.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 64
HD = 64
DEV = "cuda:0"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ES = {"f32": 4, "bf16": 2, "f16": 2}
W_SCALE = 2.0 ** 36  # probabilities are whole multiples of 2^-36 of the row's largest


# ---------------------------------------------------------------- cases

def listed():
    return [
        # Five beams of one utterance, each with its last token and up to four drafted ones: the
        # smallest step, where latency counts.
        dict(name="chunk_drafts", op="chunk", batch=5, ones=0, new=5, cached=448, heads=12,
             kv_heads=12, dtype="bf16", q="bf16", causal=True, lse=False),
        # 24 requests with long histories, one token each.
        dict(name="chunk_single", op="chunk", batch=24, ones=24, new=1, cached=30000, heads=32,
             kv_heads=8, dtype="f16", q="f16", causal=True, lse=False),
        # A serving batch whose drafts are checked: up to eight tokens a request.
        dict(name="chunk_verify", op="chunk", batch=64, ones=0, new=8, cached=2000, heads=32,
             kv_heads=8, dtype="bf16", q="bf16", causal=True, lse=True),
        # A step of continuous batching: chunks of four prompts beside 32 single tokens.
        dict(name="chunk_mixed", op="chunk", batch=36, ones=32, new=700, cached=6000, heads=28,
             kv_heads=4, dtype="bf16", q="f32", causal=True, lse=False),
        # Two long prompts, a chunk of each: the largest.
        dict(name="chunk_prompt", op="chunk", batch=2, ones=0, new=8192, cached=24000, heads=32,
             kv_heads=8, dtype="bf16", q="bf16", causal=True, lse=False),
        # Five beams over Whisper's vocabulary, drafted by a smaller model.
        dict(name="verify_beams", op="verify", batch=5, drafts=4, vocab=51865, ld=51872,
             dtype="f32", draft=True, greedy=False, logprob=True),
        # A serving batch whose drafts were looked up in the text before: no draft model.
        dict(name="verify_lookup", op="verify", batch=64, drafts=7, vocab=51865, ld=51865,
             dtype="bf16", draft=False, greedy=False, logprob=False),
        # A large batch over a large vocabulary, with the draft model's logits.
        dict(name="verify_large", op="verify", batch=96, drafts=4, vocab=128000, ld=128000,
             dtype="f32", draft=True, greedy=False, logprob=False),
        # Beam search: twelve utterances of five beams continue each other's histories.
        dict(name="fork_beams", op="fork", batch=60, group=5, length=448, max_pages=7, kv_heads=20,
             dtype="f16", keep=False),
        # A server's step: requests cut back to what was accepted, some ended, some forked.
        dict(name="fork_requests", op="fork", batch=1000, group=8, length=1500, max_pages=32,
             kv_heads=4, dtype="bf16", keep=True),
        # A small pool, a few requests left in it.
        dict(name="compact_few", op="compact", batch=16, length=448, max_pages=7, kv_heads=12,
             dtype="bf16", load=0.5),
        # A large pool, a third of it in use, made dense.
        dict(name="compact_pool", op="compact", batch=300, length=1900, max_pages=32, kv_heads=8,
             dtype="bf16", load=0.35),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["chunk"] * 6 + ["verify"] * 4 + ["fork"] * 2 + ["compact"] * 2)
    if op == "chunk":
        heads, kv = rng.choice([(6, 6), (8, 8), (12, 12), (20, 20), (32, 8), (16, 2), (28, 4),
                                (10, 1), (24, 8), (40, 8)])
        batch = _log_int(rng, 1, 128)
        ones = rng.choice([0, batch, batch // 2, batch - 1])
        # no more multiply-adds than the largest listed case, and no more keys than any
        cached = _log_int(rng, 1, max(2, min(60000, 6_000_000 // (batch * kv))))
        room = 100_000_000 // (heads * max(cached, 2000)) // max(1, batch - ones) * 25
        new = 1 if ones == batch else _log_int(rng, 1, max(2, min(8192, room)))
        dtype = rng.choice(["bf16", "f16"])
        return dict(op=op, batch=batch, ones=ones, new=new, cached=cached, heads=heads,
                    kv_heads=kv, dtype=dtype, q=rng.choice([dtype, dtype, "f32"]),
                    causal=rng.random() < 0.8, lse=rng.random() < 0.5)
    if op == "verify":
        vocab = _log_int(rng, 1000, 200000)
        drafts = rng.choice([1, 2, 3, 4, 5, 7, 12])
        batch = _log_int(rng, 1, max(2, min(300, 96 * 3 * 128000 // vocab // (drafts + 1))))
        return dict(op=op, batch=batch, drafts=drafts, vocab=vocab,
                    ld=vocab + rng.choice([0, 0, 1, 7, 32]), dtype=rng.choice(["f32", "bf16", "f16"]),
                    draft=rng.random() < 0.6, greedy=rng.random() < 0.2,
                    logprob=rng.random() < 0.5)
    kv = rng.choice([1, 4, 6, 8, 12, 20])
    dtype = rng.choice(["bf16", "f16", "f32"])
    max_pages = _log_int(rng, 2, 40)
    batch = _log_int(rng, 1, min(1000, 300 * 32 * 8 * 2 // (kv * max_pages * ES[dtype])))
    length = rng.randint(1, max_pages * PAGE)
    case = dict(op=op, batch=batch, length=length, max_pages=max_pages, kv_heads=kv, dtype=dtype)
    if op == "fork":
        case.update(group=rng.choice([1, 2, 5, 8, 30]), keep=rng.random() < 0.5)
    else:
        case["load"] = rng.choice([0.05, 0.3, 0.5, 0.8, 0.95])
    return case


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 29)
    return g


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced: a ragged batch whose sum is known."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _shuffled(vals, g):
    t = torch.tensor(vals, dtype=torch.int32, device=DEV)
    return t[torch.randperm(len(vals), generator=g, device=DEV)].contiguous()


def _new_counts(case):
    many = case["batch"] - case["ones"]
    return [1] * case["ones"] + (_spread((case["new"] + 2) // 3, case["new"], many) if many else [])


def _cached_lens(case):
    return _spread(case["cached"] // 8, case["cached"], case["batch"])


def _prepare_chunk(case, seed):
    g = _gen(seed)
    dt, hk, h, b = DT[case["dtype"]], case["kv_heads"], case["heads"], case["batch"]
    new, cached = _shuffled(_new_counts(case), g), _shuffled(_cached_lens(case), g)
    lens = new + cached
    mp = _pages(case["cached"] + case["new"])
    held = _pages(lens)
    n_pages = int(held.sum()) + 3
    shape = (n_pages, hk, PAGE, HD)
    k_pool = (torch.randn(shape, generator=g, device=DEV) * 1.5).to(dt)
    v_pool = torch.randn(shape, generator=g, device=DEV).to(dt)
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, mp), -1, dtype=torch.int32, device=DEV)
    live = torch.arange(mp, device=DEV) < held.view(-1, 1)
    table[live] = ids[:n_pages - 3]
    # what lies behind a last page's live keys is whatever was there: not numbers, in places
    last = table.gather(1, (held - 1).view(-1, 1).long())[:, 0].long()
    used = lens - (held - 1) * PAGE
    dead = torch.arange(PAGE, device=DEV).view(1, 1, PAGE, 1) >= used.view(-1, 1, 1, 1)
    for pool in (k_pool, v_pool):
        pool[last] = torch.where(dead, torch.full_like(pool[last], float("nan")), pool[last])
    counts = new.tolist()
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    # queries are a part of one projection's output rows
    qkv = torch.randn((cu[-1], h + 2 * hk, HD), generator=g, device=DEV).to(DT[case["q"]])
    return dict(q=qkv[:, :h], k_pool=k_pool, v_pool=v_pool, block_table=table, seq_lens=lens,
                cu_q=torch.tensor(cu, dtype=torch.int32, device=DEV), scale=0.125, starts=cu,
                host_lens=lens.tolist(), max_q=max(counts))


def _row_counts(case):
    """Rows of each request: its last token and its drafts."""
    return [1 + n for n in _spread(0 if case["batch"] > 3 else 1, case["drafts"], case["batch"])]


def _prepare_verify(case, seed):
    g = _gen(seed)
    b, v = case["batch"], case["vocab"]
    rows = _shuffled(_row_counts(case), g)
    cu = [0]
    for n in rows.tolist():
        cu.append(cu[-1] + n)
    t = cu[-1]
    x = torch.randn((t, case["ld"]), generator=g, device=DEV) * 2.5
    # a few tokens stand out, as a model's do, by more in some rows than in others
    hot = torch.randint(0, v, (t, 12), generator=g, device=DEV)
    lift = torch.rand((t, 12), generator=g, device=DEV) * 10 + 4 * torch.rand((t, 1), generator=g, device=DEV)
    x.scatter_add_(1, hot, lift)
    # the smaller model agrees more or less
    y = None
    if case["draft"]:
        noise = torch.randn((t, case["ld"]), generator=g, device=DEV)
        y = x + noise * (0.2 + 1.5 * torch.rand((t, 1), generator=g, device=DEV))
    # suppressed tokens, and what lies in the padding
    gone = torch.randint(0, v, (max(1, v // 60),), generator=g, device=DEV)
    for z in (x, y):
        if z is not None:
            z[:, gone] = float("-inf")
            z[:, v:] = float("nan")
    temp = torch.tensor([0.0] if case["greedy"] else [0.0, 0.6, 0.8, 1.0, 1.0, 1.3], device=DEV)
    temp = temp[torch.randint(0, temp.numel(), (b,), generator=g, device=DEV)].contiguous()
    # each row's draft is drawn from the smaller model, or is one of the tokens that stand out
    if y is not None:
        scale = 1 / temp.clamp(min=0.05).repeat_interleave(rows.long()).view(-1, 1)
        noise = -torch.log(-torch.log(torch.rand((t, v), generator=g, device=DEV).clamp(1e-20, 1 - 1e-7)))
        drawn = (y[:, :v] * scale + noise).argmax(1)
    else:
        best = x[:, :v].argmax(1)
        drawn = torch.where(torch.rand(t, generator=g, device=DEV) < 0.6, best, hot[:, 0])
    tokens = torch.zeros(t, dtype=torch.int32, device=DEV)
    tokens[1:] = drawn[:-1].to(torch.int32)
    st = dict(logits=x.to(DT[case["dtype"]])[:, :v], tokens=tokens,
              cu_rows=torch.tensor(cu, dtype=torch.int32, device=DEV),
              u=torch.rand(t, generator=g, device=DEV), u_last=torch.rand(b, generator=g, device=DEV),
              draft_logits=None, temperature=temp)
    if y is not None:
        st["draft_logits"] = y.to(DT[case["dtype"]])[:, :v]
    return st


def _pools(case, n_pages, g):
    shape = (n_pages, case["kv_heads"], PAGE, HD)
    return [torch.randn(shape, generator=g, device=DEV).to(DT[case["dtype"]]) for _ in range(2)]


def _prepare_fork(case, seed):
    g = _gen(seed)
    b, mp = case["batch"], case["max_pages"]
    lens = _shuffled(_spread(0, case["length"], b), g)
    held = _pages(lens)
    n_pages = int(held.sum()) + b + 2
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, mp), -1, dtype=torch.int32, device=DEV)
    live = torch.arange(mp, device=DEV) < held.view(-1, 1)
    n = int(held.sum())
    table[live] = ids[:n]
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:n_pages - n] = ids[n:]
    k, v = _pools(case, n_pages, g)
    # a row continues one of its group: itself, in a server's step, three times in four
    at = torch.arange(b, device=DEV)
    base = at // case["group"] * case["group"]
    size = torch.minimum(torch.tensor(case["group"], device=DEV), b - base)
    src = base + (torch.rand(b, generator=g, device=DEV) * size).long().clamp(max=size - 1)
    keep = None
    if case["keep"]:
        luck = torch.rand(b, generator=g, device=DEV)
        src = torch.where(luck < 0.75, at, src)
        src = torch.where(luck > 0.95, -1, src)
        cut = torch.randint(0, 9, (b,), generator=g, device=DEV)
        keep = (lens[src.clamp(min=0)].long() - cut).clamp(min=0).to(torch.int32)
    return dict(src=src.to(torch.int32), lens=lens, block_table=table, free_pages=free,
                free_count=torch.tensor([n_pages - n], dtype=torch.int32, device=DEV), keep=keep,
                k_pool=k, v_pool=v)


def _prepare_compact(case, seed):
    g = _gen(seed)
    b, mp = case["batch"], case["max_pages"]
    lens = _shuffled(_spread(0, case["length"], b), g)
    held = _pages(lens)
    n = int(held.sum())
    n_pages = max(n, 1) + int(n / case["load"] * (1 - case["load"])) + 2
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((b, mp), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(mp, device=DEV) < held.view(-1, 1)] = ids[:n]
    # every fifth request shares the pages of the one before it, as far as both have any
    both = torch.minimum(held[4::5], held[3::5][:held[4::5].numel()])
    share = torch.arange(mp, device=DEV) < (both - 1).view(-1, 1)
    table[4::5] = torch.where(share, table[3::5][:both.numel()], table[4::5])
    used = torch.zeros(n_pages, dtype=torch.bool, device=DEV)
    used[table[table >= 0].long()] = True
    spare = ids[~used[ids.long()]]
    spare = spare[:max(1, spare.numel() - 1)]  # a page belongs to someone else
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free[:spare.numel()] = spare
    k, v = _pools(case, n_pages, g)
    return dict(lens=lens, block_table=table, free_pages=free,
                free_count=torch.tensor([spare.numel()], dtype=torch.int32, device=DEV),
                k_pool=k, v_pool=v)


def prepare(case, seed):
    make = {"chunk": _prepare_chunk, "verify": _prepare_verify, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["op"]]
    st = make(case, seed)
    st["case"] = case
    return st


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_chunk(s):
    from ffai_b200 import chunk_attention
    return chunk_attention.attend(s["q"], s["k_pool"], s["v_pool"], s["cu_q"], s["block_table"],
                                  s["seq_lens"], scale=s["scale"], causal=s["case"]["causal"],
                                  max_q=s["max_q"], with_lse=s["case"]["lse"])


def _own_verify(s):
    from ffai_b200 import sampling
    r = sampling.verify(s["logits"], s["tokens"], s["cu_rows"], s["u"], s["u_last"],
                        draft_logits=s["draft_logits"], temperature=s["temperature"],
                        with_logprob=s["case"]["logprob"])
    return (r.accepted, r.next, r.tokens) + ((r.logprobs,) if s["case"]["logprob"] else ())


def _own_fork(s):
    from ffai_b200 import kvcache
    f = kvcache.fork_pages(s["src"], s["lens"], s["block_table"], s["free_pages"], s["free_count"],
                           keep=s["keep"])
    kvcache.copy_pages(s["k_pool"], s["v_pool"], f.copy_src, f.copy_dst, keys=f.copy_keys)
    return (f.block_table, f.lens, f.copy_src, f.copy_dst, f.copy_keys, f.free_count,
            s["free_pages"], s["k_pool"], s["v_pool"])


def _own_compact(s):
    from ffai_b200 import kvcache
    c = kvcache.compact_pages(s["lens"], s["block_table"], s["free_pages"], s["free_count"])
    kvcache.copy_pages(s["k_pool"], s["v_pool"], c.copy_src, c.copy_dst)
    return c.block_table, c.free_pages, c.copy_src, c.copy_dst, s["k_pool"], s["v_pool"]


# ---- the plain forms

def _plain_chunk(s):
    q, hk = s["q"], s["k_pool"].shape[1]
    t, h, _ = q.shape
    grp = h // hk
    out = torch.empty((t, h, HD), dtype=q.dtype, device=q.device)
    lse = torch.empty((h, t), dtype=torch.float32, device=q.device) if s["case"]["lse"] else None
    for b, n_keys in enumerate(s["host_lens"]):
        t0, t1 = s["starts"][b], s["starts"][b + 1]
        n = t1 - t0
        pages = s["block_table"][b, :_pages(n_keys)].long()
        hide = None
        if s["case"]["causal"]:
            limit = n_keys - n + 1 + torch.arange(n, device=q.device)
            hide = torch.arange(n_keys, device=q.device) >= limit.view(-1, 1)
            hide = hide.repeat_interleave(grp, dim=0)
        step = max(1, (1 << 30) // (n * grp * n_keys))
        for h0 in range(0, hk, step):
            h1 = min(hk, h0 + step)
            k, v = (p[pages, h0:h1].transpose(0, 1).reshape(h1 - h0, -1, HD)[:, :n_keys].float()
                    for p in (s["k_pool"], s["v_pool"]))
            qg = q[t0:t1, h0 * grp:h1 * grp].float().unflatten(1, (h1 - h0, grp))
            qg = qg.transpose(0, 1).flatten(1, 2) * s["scale"]         # (heads, n G, 64)
            sc = qg @ k.transpose(1, 2)
            if hide is not None:
                sc.masked_fill_(hide, float("-inf"))
            m = sc.amax(-1, keepdim=True)
            p = sc.sub_(m).exp_()
            l = p.sum(-1, keepdim=True)
            o = (p @ v / l).unflatten(1, (n, grp)).transpose(0, 1).flatten(1, 2)
            out[t0:t1, h0 * grp:h1 * grp] = o.to(q.dtype)
            if lse is not None:
                z = (m + torch.log(l))[..., 0].unflatten(1, (n, grp))
                lse[h0 * grp:h1 * grp, t0:t1] = z.transpose(1, 2).reshape(-1, n)
    return out if lse is None else (out, lse)


def _weights(x, temp):
    """Whole weights (R, V) of rows of logits at temperatures (R,), f32 exponents; and the maxima."""
    x = x.float()
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    top, first = x.max(1, keepdim=True)
    first = (x == top).to(torch.int8).argmax(1, keepdim=True)
    greedy = ~(temp > 0)
    inv = 1.0 / torch.where(greedy, torch.ones_like(temp), temp)
    d = torch.where(x == top, torch.zeros_like(x), x - top) * inv.view(-1, 1)
    w = (torch.exp(d) * W_SCALE).long()
    one = torch.zeros_like(w).scatter_(1, first, int(W_SCALE))
    w = torch.where(greedy.view(-1, 1), one, w)
    return torch.where(top == float("-inf"), torch.zeros_like(w), w), x, top


def _plain_verify(s):
    dev = s["logits"].device
    cu = s["cu_rows"].long()
    b, (t, v) = cu.numel() - 1, s["logits"].shape
    row = torch.arange(t, device=dev)
    who = torch.searchsorted(cu[1:], row, right=True)
    w, x, top = _weights(s["logits"], s["temperature"][who])
    mass = w.sum(1)
    # the draft that row i's distribution is asked about, if it has one
    is_draft = row + 1 < cu[who + 1]
    tok = torch.where(is_draft, s["tokens"].roll(-1).long(), 0)
    if s["draft_logits"] is not None:
        q, _, _ = _weights(s["draft_logits"], s["temperature"][who])
    else:
        q = torch.zeros_like(w).scatter_(1, tok.view(-1, 1), 1)
    q_mass = q.sum(1)
    wx, qx = (z.gather(1, tok.view(-1, 1))[:, 0].double() for z in (w, q))
    ok = is_draft & (s["u"].double() * qx * mass.double() < wx * q_mass.double())
    # rows before the first that fails
    fails = torch.where(ok, t, row)
    first = torch.full((b,), t, device=dev).scatter_reduce(0, who, fails, "amin")
    accepted = first - cu[:-1]
    wf, qf = w[first], q[first]
    rho = mass[first].double() / q_mass[first].double()
    less = torch.floor(qf.double() * rho.view(-1, 1))
    less = torch.where(q_mass[first].view(-1, 1) > 0, less, torch.zeros_like(less)).long()
    rest = (wf - less).clamp(min=0)
    use = (is_draft[first] & (rest.sum(1) > 0)).view(-1, 1)
    rest = torch.where(use, rest, wf)
    cum = rest.cumsum(1)
    total = cum[:, -1:]
    goal = torch.floor(s["u_last"].double().view(-1, 1) * total.double()).long()
    goal = torch.minimum(goal, total - 1).clamp(min=0)
    pick = torch.searchsorted(cum, goal, right=True).clamp(max=v - 1)[:, 0]
    pick = torch.where(total[:, 0] > 0, pick, torch.full_like(pick, -1))
    out = torch.where(row < first[who], tok, torch.full_like(tok, -1))
    out = torch.where(row == first[who], pick[who], out).to(torch.int32)
    res = (accepted.to(torch.int32), pick.to(torch.int32), out)
    if s["case"]["logprob"]:
        z = torch.log(torch.exp(x - top).sum(1))
        lp = x.gather(1, out.long().clamp(min=0).view(-1, 1))[:, 0] - top[:, 0] - z
        res += (torch.where(out >= 0, lp, torch.zeros_like(lp)),)
    return res


def _copy(s, src, dst, keys):
    """Page contents copied, in place: copies that are none rewrite a row with itself."""
    have = src >= 0
    key = torch.arange(PAGE, device=src.device)
    a = src.long().clamp(min=0)
    for pool in (s["k_pool"], s["v_pool"]):
        for i in range(0, a.numel(), 4096):
            live = have[i:i + 4096].nonzero()[:, 0] + i
            d = dst[live].long()
            take = (key < keys[live].view(-1, 1)).view(-1, 1, PAGE, 1)
            pool[d] = torch.where(take, pool[a[live]], pool[d])


def _plain_fork(s):
    table, lens, free = s["block_table"], s["lens"].long(), s["free_pages"]
    dev, mp, n_pages = table.device, table.shape[1], s["k_pool"].shape[0]
    src = s["src"].long()
    n = torch.where(src >= 0, lens[src.clamp(min=0)], torch.zeros_like(src))
    if s["keep"] is not None:
        n = torch.minimum(n, s["keep"].long().clamp(min=0))
    slot = torch.arange(mp, device=dev).view(1, -1)
    rows = table[src.clamp(min=0)].long()
    rows = torch.where(slot < _pages(n).view(-1, 1), rows, torch.full_like(rows, -1))
    # references after the fork; the pages that end in the middle are written by who holds them
    place = torch.where(rows >= 0, rows, n_pages)
    refs = torch.zeros(n_pages + 1, dtype=torch.long, device=dev)
    refs.scatter_add_(0, place.flatten(), torch.ones_like(place).flatten())
    part = n % PAGE > 0
    last = rows.gather(1, (n // PAGE).clamp(max=mp - 1).view(-1, 1))[:, 0]
    last = torch.where(part, last, n_pages)
    writers = torch.zeros_like(refs).scatter_add_(0, last, torch.ones_like(last))
    who = torch.arange(src.numel(), device=dev)
    first = torch.full_like(refs, src.numel()).scatter_reduce(0, last, who, "amin")
    alone = (refs[last] == 1) | ((refs[last] == writers[last]) & (first[last] == who))
    copies = part & ~alone
    # pages that no row names any more are pushed in the order of their numbers
    old = torch.zeros(n_pages + 1, dtype=torch.bool, device=dev)
    old[torch.where(slot < _pages(lens).view(-1, 1), table.long(), n_pages).flatten()] = True
    gone = old[:-1] & (refs[:-1] == 0)
    count = s["free_count"].long()
    at = torch.where(gone, count + gone.long().cumsum(0) - 1, free.numel())
    pad = torch.cat([free, free[:1]])
    pad.scatter_(0, at, torch.arange(n_pages, dtype=torch.int32, device=dev))
    free.copy_(pad[:-1])
    count = count + gone.sum()
    # then each copy takes one, in row order; who finds none keeps its whole pages
    order = copies.long().cumsum(0)
    found = copies & (order <= count)
    fresh = free[(count - order).clamp(0, free.numel() - 1)].long()
    none = torch.full_like(last, -1)
    new_last = torch.where(found, fresh, torch.where(copies, none, last))
    j = (n // PAGE).clamp(max=mp - 1).view(-1, 1)
    rows.scatter_(1, j, torch.where(part, new_last, rows.gather(1, j)[:, 0]).view(-1, 1))
    out_lens = torch.where(copies & ~found, n // PAGE * PAGE, n)
    c_src = torch.where(found, last, none).to(torch.int32)
    c_dst = torch.where(found, fresh, none).to(torch.int32)
    c_keys = torch.where(found, n % PAGE, torch.zeros_like(n)).to(torch.int32)
    _copy(s, c_src, c_dst, c_keys)
    return (rows.to(torch.int32), out_lens.to(torch.int32), c_src, c_dst, c_keys,
            (count - found.sum()).to(torch.int32), free, s["k_pool"], s["v_pool"])


def _plain_compact(s):
    table, lens, free = s["block_table"], s["lens"].long(), s["free_pages"]
    dev, mp, n_pages = table.device, table.shape[1], s["k_pool"].shape[0]
    used = torch.arange(mp, device=dev).view(1, -1) < _pages(lens).view(-1, 1)
    live = torch.zeros(n_pages + 1, dtype=torch.bool, device=dev)
    live[torch.where(used, table.long(), n_pages).flatten()] = True
    live = live[:-1]
    spot = torch.arange(free.numel(), device=dev)
    idle = torch.zeros(n_pages + 1, dtype=torch.bool, device=dev)
    idle[torch.where(spot < s["free_count"], free.long(), n_pages)] = True
    idle = idle[:-1]
    # the live pages belong on the lowest numbers of both
    target = (live | idle) & ((live | idle).long().cumsum(0) <= live.sum())
    page = torch.arange(n_pages, device=dev)
    movers, holes = live & ~target, idle & target
    cap = min(table.numel(), free.numel())
    pairs = []
    for which in (movers, holes):
        at = torch.where(which, which.long().cumsum(0) - 1, cap)
        pairs.append(torch.full((cap + 1,), -1, dtype=torch.int32, device=dev)
                     .scatter_(0, at, page.to(torch.int32))[:-1])
    src, dst = pairs
    moved = page.clone()
    keep = torch.cat([moved, moved[:1]])
    keep.scatter_(0, torch.where(src >= 0, src.long(), n_pages), dst.long())
    out = torch.where(used, keep[table.long().clamp(min=0)].to(torch.int32), table)
    # the stack, lowest number on top
    left = (live | idle) & ~target
    rank = left.long().flip(0).cumsum(0).flip(0) - 1
    stack = torch.cat([free, free[:1]])
    stack.scatter_(0, torch.where(left, rank, free.numel()), page.to(torch.int32))
    _copy(s, src, dst, torch.full_like(src, PAGE))
    return out, stack[:-1], src, dst, s["k_pool"], s["v_pool"]


_OWN = dict(chunk=_own_chunk, verify=_own_verify, fork=_own_fork, compact=_own_compact)
_PLAIN = dict(chunk=_plain_chunk, verify=_plain_verify, fork=_plain_fork, compact=_plain_compact)


# ---------------------------------------------------------------- work and exact values

def work(case):
    op = case["op"]
    if op == "chunk":
        n, cached = _new_counts(case), _cached_lens(case)
        es, eq = ES[case["dtype"]], ES[case["q"]]
        keys = (sum(cached) + sum(n)) * case["kv_heads"]
        rows = sum(n) * case["heads"]
        # chunks meet the caches in any order: the mean
        pairs = sum(x * (sum(cached) / len(cached) + (x / 2 if case["causal"] else x)) for x in n)
        return dict(bytes=2 * HD * (es * keys + eq * rows) + (4 * rows if case["lse"] else 0),
                    flops=int(4 * HD * case["heads"] * pairs))
    if op == "verify":
        rows, b = sum(_row_counts(case)), case["batch"]
        # the draft's distribution is asked for at every row but a request's last
        n = (rows + (rows - b if case["draft"] else 0)) * case["vocab"]
        return dict(bytes=n * ES[case["dtype"]] + 20 * rows + 24 * b, flops=4 * n)
    lens = _spread(0, case["length"], case["batch"])
    held = sum(_pages(n) for n in lens)
    page = PAGE * HD * case["kv_heads"] * ES[case["dtype"]]
    if op == "fork":
        # of the rows that share a last page that is not full all but one copy its keys; half of
        # what random beams share, an eighth of a server's requests
        part = sum(n % PAGE for n in lens) / PAGE
        share = (0.1 if case["keep"] else 0.37) if case["group"] > 1 else 0.0
        return dict(bytes=4 * (3 * held + 6 * case["batch"]) + int(4 * page * part * share), flops=0)
    # about 1 - load of the pages lie too high
    return dict(bytes=4 * (4 * held) + int(4 * page * held * (1 - case["load"])), flops=0)


def exact(case, seed):
    if case["op"] == "chunk":
        return _exact_chunk(prepare(case, seed))
    if case["op"] == "verify":
        return _exact_verify(prepare(case, seed))
    return None  # whole numbers and copies throughout


def _exact_chunk(s):
    t, h, _ = s["q"].shape
    hk = s["k_pool"].shape[1]
    dev = s["q"].device
    out = torch.zeros((t, h, HD), dtype=torch.float64, device=dev)
    lse = torch.full((h, t), float("-inf"), dtype=torch.float64, device=dev)
    for b, n_keys in enumerate(s["host_lens"]):
        t0, n = s["starts"][b], s["starts"][b + 1] - s["starts"][b]
        table = s["block_table"][b, :_pages(n_keys)].long()
        pos = torch.arange(n_keys, device=dev)
        for g in range(hk):
            k = s["k_pool"][table, g].reshape(-1, HD)[:n_keys].double().t()
            v = s["v_pool"][table, g].reshape(-1, HD)[:n_keys].double()
            step = max(1, (1 << 28) // n_keys)
            for head in range(g * (h // hk), (g + 1) * (h // hk)):
                for i in range(0, n, step):
                    j = min(n, i + step)
                    sc = s["scale"] * (s["q"][t0 + i:t0 + j, head].double() @ k)
                    if s["case"]["causal"]:
                        own_pos = n_keys - n + torch.arange(i, j, device=dev)
                        sc[pos > own_pos.view(-1, 1)] = float("-inf")
                    z = torch.logsumexp(sc, 1)
                    out[t0 + i:t0 + j, head] = torch.exp(sc - z.view(-1, 1)) @ v
                    lse[head, t0 + i:t0 + j] = z
    return (out, lse) if s["case"]["lse"] else out


def _exact_row(x, temp):
    """Whole weights (f64) of one row, from exponents in 32 bits and powers rounded to 32."""
    x = torch.nan_to_num(x.float(), nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    if not temp > 0:
        w = torch.zeros(x.numel(), dtype=torch.float64, device=x.device)
        w[(x == x.max()).to(torch.int8).argmax()] = W_SCALE
        return w
    d = (x - x.max()) * (torch.ones(1, device=x.device) / temp)
    return torch.floor(torch.exp(d.double()).float().double() * W_SCALE)


def _exact_verify(s):
    dev = s["logits"].device
    cu, temps = s["cu_rows"].tolist(), s["temperature"].tolist()
    toks, u, last = s["tokens"].tolist(), s["u"].tolist(), s["u_last"].tolist()
    accepted, chosen = [], []
    out = [-1] * s["logits"].shape[0]
    logprob = [0.0] * len(out)
    for b, temp in enumerate(temps):
        at = cu[b]
        rest = None
        while at + 1 < cu[b + 1]:
            x = toks[at + 1]
            w = _exact_row(s["logits"][at], temp)
            if s["draft_logits"] is not None:
                q = _exact_row(s["draft_logits"][at], temp)
            else:
                q = torch.zeros_like(w)
                q[x] = 1
            p, r = w / w.sum(), q / q.sum()
            if not u[at] * float(r[x]) < float(p[x]):
                rest = torch.clamp(p - r, min=0)
                # probabilities below the whole weights' step are none
                rest = torch.where(rest * w.sum() > 1, rest, torch.zeros_like(rest))
                break
            out[at] = x
            at += 1
        if rest is None or not float(rest.sum()) > 0:
            rest = _exact_row(s["logits"][at], temp)
        cum = (rest / rest.sum()).cumsum(0)
        pick = int((cum > last[b]).to(torch.int8).argmax())
        accepted.append(at - cu[b])
        chosen.append(pick)
        out[at] = pick
    if s["case"]["logprob"]:
        for i, x in enumerate(out):
            if x >= 0:
                row = torch.nan_to_num(s["logits"][i].double(), nan=float("-inf"),
                                       neginf=float("-inf"))
                logprob[i] = float(row[x] - torch.logsumexp(row, 0))
    res = tuple(torch.tensor(z, dtype=torch.int32, device=dev) for z in (accepted, chosen, out))
    if s["case"]["logprob"]:
        res += (torch.tensor(logprob, dtype=torch.float64, device=dev),)
    return res
