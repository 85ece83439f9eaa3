"""The operators of a batched decode step, measured: attention over a shared
prefix, page tables and slot maps, the scatter of new keys and values, and
sampling.

A case is a dict of plain values.  `op` names the operator:

  attend   ffai_b200.shared_prefix.attend
  plan     ffai_b200.kvcache.plan_pages
  release  ffai_b200.kvcache.release_pages
  write    ffai_b200.kvcache.write_slots
  sample   ffai_b200.sampling.sample

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
W_SCALE = 2.0 ** 36  # sampling weights are whole multiples of 2^-36 of the largest


# ---------------------------------------------------------------- cases

def listed():
    return [
        # Five beams of one utterance over its prompt of 224 tokens, 12 heads: the smallest
        # decode step, where latency counts.
        dict(name="attend_beams", op="attend", groups=1, batch=5, q_len=1, heads=12, kv_heads=12,
             prefix=224, suffix=224, dtype="bf16", lse=False),
        # Twelve utterances of five beams, each over its own 1500 shared keys (the length of a
        # window's encoder output) and up to 448 keys of its own, 20 heads.
        dict(name="attend_utterances", op="attend", groups=12, batch=60, q_len=1, heads=20,
             kv_heads=20, prefix=1500, suffix=448, dtype="f16", lse=False),
        # 64 requests behind one long common prompt, shared key heads.
        dict(name="attend_prompt", op="attend", groups=1, batch=64, q_len=1, heads=32, kv_heads=8,
             prefix=8200, suffix=1000, dtype="bf16", lse=True),
        # Three long prompts, 96 requests, four tokens a request (drafted tokens being checked):
        # the largest.
        dict(name="attend_drafts", op="attend", groups=3, batch=96, q_len=4, heads=32, kv_heads=8,
             prefix=32768, suffix=700, dtype="bf16", lse=False),
        # One decode step of 32 requests: one new token each.
        dict(name="plan_step", op="plan", batch=32, new=1, length=448, max_pages=16),
        # Admission of many requests, prompts and single tokens mixed.
        dict(name="plan_prompts", op="plan", batch=2000, new=130, length=1500, max_pages=64),
        # Requests that end hand their pages back.
        dict(name="release", op="release", batch=500, length=1500, max_pages=64),
        # The new keys and values of one decode step.
        dict(name="write_step", op="write", tokens=60, kv_heads=20, src="bf16", dtype="bf16",
             pages=600),
        # The keys and values of a chunk of prompts, from a f32 projection.
        dict(name="write_prompts", op="write", tokens=20001, kv_heads=8, src="f32", dtype="bf16",
             pages=1500),
        # Five beams over Whisper's vocabulary.
        dict(name="sample_beams", op="sample", batch=5, vocab=51865, ld=51872, dtype="f32",
             mode="mixed", logprob=True),
        # A serving batch, each request with its own settings.
        dict(name="sample_batch", op="sample", batch=64, vocab=51865, ld=51865, dtype="bf16",
             mode="mixed", logprob=True),
        # A large batch over a large vocabulary, nucleus sampling throughout.
        dict(name="sample_large", op="sample", batch=300, vocab=128000, ld=128000, dtype="f32",
             mode="top_p", logprob=False),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["attend"] * 5 + ["sample"] * 4 + ["plan", "plan", "release", "write", "write"])
    if op == "attend":
        heads, kv = rng.choice([(6, 6), (8, 8), (12, 12), (16, 16), (20, 20), (32, 8), (16, 2),
                                (28, 4), (10, 1), (24, 8)])
        q_len = rng.choice([1, 1, 1, 2, 3, 4, 8, 17])
        batch = _log_int(rng, 1, 128)
        groups = min(batch, rng.choice([1, 1, 2, 3, 5, 12]))
        # no more multiply-adds than the largest listed case, and no more keys
        rows = batch * q_len * heads
        top = min(60000, 400_000_000 // rows, 800_000 // (kv * groups))
        prefix = _log_int(rng, 1, max(2, top))
        suffix = _log_int(rng, 1, max(2, min(2000, 2_000_000 // (batch * kv), 60_000_000 // rows)))
        return dict(op=op, groups=groups, batch=batch, q_len=q_len, heads=heads, kv_heads=kv,
                    prefix=prefix, suffix=suffix, dtype=rng.choice(["bf16", "f16"]),
                    lse=rng.random() < 0.5)
    if op == "sample":
        vocab = _log_int(rng, 1000, 200000)
        batch = _log_int(rng, 1, min(500, 300 * 128000 // vocab))
        return dict(op=op, batch=batch, vocab=vocab, ld=vocab + rng.choice([0, 0, 1, 7, 32]),
                    dtype=rng.choice(["f32", "bf16", "f16"]),
                    mode=rng.choice(["mixed", "mixed", "top_p", "top_k", "plain"]),
                    logprob=rng.random() < 0.5)
    if op in ("plan", "release"):
        max_pages = _log_int(rng, 4, 64)
        case = dict(op=op, batch=_log_int(rng, 1, 2000),
                    length=rng.randint(1, max_pages * PAGE * 3 // 4), max_pages=max_pages)
        if op == "plan":
            case["new"] = _log_int(rng, 1, min(130, max_pages * PAGE - case["length"]))
        return case
    kv = rng.choice([1, 4, 6, 8, 12, 20])
    tokens = _log_int(rng, 1, 20001 * 8 // max(kv, 8))
    dtype = rng.choice(["bf16", "f16", "f32"])
    return dict(op=op, tokens=tokens, kv_heads=kv, src=rng.choice(["f32", dtype]), dtype=dtype,
                pages=tokens // PAGE + rng.randint(2, 200))


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 17)
    return g


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced: a ragged batch whose sum is known."""
    if n == 1:
        return [hi]
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _ragged(case):
    """(sequences, prefix keys) of each group: uneven, fixed by the case."""
    g, b = case["groups"], case["batch"]
    cuts = [b * (i * (i + 3 * g)) // (g * 4 * g) for i in range(g + 1)]
    for i in range(1, g + 1):  # at least one sequence a group
        cuts[i] = max(cuts[i], cuts[i - 1] + 1)
    for i in range(g, -1, -1):
        cuts[i] = min(cuts[i], b - (g - i))
    sizes = [cuts[i + 1] - cuts[i] for i in range(g)]
    return sizes, _spread(max(1, case["prefix"] * 2 // 3), case["prefix"], g)


def _suffix_lens(case):
    return _spread(0 if case["batch"] > 3 else 1, case["suffix"], case["batch"])


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _prepare_attend(case, seed):
    g = _gen(seed)
    dt, hk = DT[case["dtype"]], case["kv_heads"]
    sizes, plens = _ragged(case)
    order = torch.randperm(case["groups"], generator=g, device=DEV).tolist()
    plens = [plens[i] for i in order]
    lens = torch.tensor(_suffix_lens(case), dtype=torch.int32, device=DEV)
    lens = lens[torch.randperm(case["batch"], generator=g, device=DEV)].contiguous()
    pp, sp = max(_pages(n) for n in plens), _pages(case["suffix"])
    n_pages = case["groups"] * pp + case["batch"] * sp + 3
    shape = (n_pages, hk, PAGE, HD)
    k_pool = (torch.randn(shape, generator=g, device=DEV) * 1.5).to(dt)
    v_pool = torch.randn(shape, generator=g, device=DEV).to(dt)
    perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    ptab = perm[:case["groups"] * pp].view(case["groups"], pp).contiguous()
    stab = perm[case["groups"] * pp:case["groups"] * pp + case["batch"] * sp]
    stab = stab.view(case["batch"], sp).contiguous()
    # what lies behind a last page's live keys is whatever was there: not numbers, in places
    key = torch.arange(PAGE, device=DEV)
    for table, n in ((ptab, torch.tensor(plens, device=DEV)), (stab, lens)):
        used = n.long()
        last = table.gather(1, ((used - 1).clamp(min=0) // PAGE).view(-1, 1))[:, 0].long()
        dead = (key.view(1, 1, PAGE, 1) >= (used - (used - 1).clamp(min=0) // PAGE * PAGE).view(-1, 1, 1, 1))
        for pool in (k_pool, v_pool):
            pool[last] = torch.where(dead, torch.full_like(pool[last], float("nan")), pool[last])
    q = torch.randn((case["batch"], case["q_len"], case["heads"], HD), generator=g, device=DEV).to(dt)
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    return dict(q=q, k_pool=k_pool, v_pool=v_pool, prefix_table=ptab,
                prefix_lens=torch.tensor(plens, dtype=torch.int32, device=DEV),
                group_starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
                block_table=stab, seq_lens=lens, scale=0.125, starts=starts, plens=plens)


def _prepare_pages(case, seed):
    g = _gen(seed)
    b, mp = case["batch"], case["max_pages"]
    perm = torch.randperm(b, generator=g, device=DEV)
    lens = torch.tensor(_spread(0, case["length"], b), dtype=torch.int32, device=DEV)[perm].contiguous()
    held = (lens + PAGE - 1) // PAGE
    n_pages = b * mp
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = ids.view(b, mp).clone()
    slot = torch.arange(mp, device=DEV).view(1, mp)
    free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    live = slot < held.view(-1, 1)
    table[~live] = -1
    st = dict(lens=lens, block_table=table, free_pages=free)
    if case["op"] == "plan":
        spare = ids.view(b, mp)[~live]
        # one request in twenty finds the pool short: the last ones in a batch of many
        count = int(spare.numel())
        free[:count] = spare
        want = torch.tensor(_spread(1, case["new"], b), dtype=torch.int32, device=DEV)
        new = want[torch.randperm(b, generator=g, device=DEV)].contiguous()
        need = int(((lens + new + PAGE - 1) // PAGE - held).sum())
        if b >= 20 and need >= 20:
            count = min(count, need - need // 20)
        st.update(new=new, slot_cap=int(sum(_spread(1, case["new"], b))) + 5,
                  pos_base=torch.randint(0, 5000, (b,), generator=g, device=DEV).to(torch.int32))
    else:
        count = n_pages // 7
        count = min(count, n_pages - int(held.sum()))
        free[:count] = ids.view(b, mp)[~live][:count]
        st["done"] = (torch.rand(b, generator=g, device=DEV) < 0.3).to(torch.int32)
    st["free_count"] = torch.tensor([count], dtype=torch.int32, device=DEV)
    return st


def _prepare_write(case, seed):
    g = _gen(seed)
    t, hk, n = case["tokens"], case["kv_heads"], case["pages"]
    # keys and values are two thirds of one projection's output rows
    qkv = torch.randn((t, 3 * hk * HD), generator=g, device=DEV).to(DT[case["src"]])
    slots = torch.randperm(n * PAGE, generator=g, device=DEV)[:t].to(torch.int32)
    if t >= 8:
        slots[torch.randint(0, t, (max(1, t // 50),), generator=g, device=DEV)] = -1
    shape = (n, hk, PAGE, HD)
    return dict(k_pool=torch.zeros(shape, dtype=DT[case["dtype"]], device=DEV),
                v_pool=torch.zeros(shape, dtype=DT[case["dtype"]], device=DEV),
                k_new=qkv[:, hk * HD:2 * hk * HD].unflatten(1, (hk, HD)),
                v_new=qkv[:, 2 * hk * HD:].unflatten(1, (hk, HD)), slots=slots)


def _prepare_sample(case, seed):
    g = _gen(seed)
    b, v = case["batch"], case["vocab"]
    x = torch.randn((b, case["ld"]), generator=g, device=DEV) * 2.5
    # a few tokens stand out, as a model's do, by more in some rows than in others
    hot = torch.randint(0, v, (b, 12), generator=g, device=DEV)
    lift = torch.rand((b, 12), generator=g, device=DEV) * 10 + 4 * torch.rand((b, 1), generator=g, device=DEV)
    x.scatter_add_(1, hot, lift)
    # suppressed tokens, and what lies in the padding
    x[:, torch.randint(0, v, (max(1, v // 60),), generator=g, device=DEV)] = float("-inf")
    x[:, v:] = float("nan")
    x = x.to(DT[case["dtype"]])
    st = dict(logits=x[:, :v], u=torch.rand(b, generator=g, device=DEV), temperature=None,
              top_k=None, top_p=None, min_p=None)
    pick = lambda vals: torch.tensor(vals, device=DEV)[  # noqa: E731
        torch.randint(0, len(vals), (b,), generator=g, device=DEV)].contiguous()
    mode = case["mode"]
    if mode == "mixed":
        st["temperature"] = pick([0.0, 0.2, 0.6, 0.8, 1.0, 1.0, 1.3])
        st["top_k"] = pick([0, 0, 1, 5, 40, 50, 1000]).to(torch.int32)
        st["top_p"] = pick([1.0, 1.0, 0.5, 0.9, 0.95])
        st["min_p"] = pick([0.0, 0.0, 0.02, 0.1])
    elif mode == "top_p":
        st["temperature"] = pick([0.7, 0.9, 1.0])
        st["top_p"] = pick([0.8, 0.9, 0.95, 0.99])
    elif mode == "top_k":
        st["temperature"] = pick([0.7, 1.0])
        st["top_k"] = pick([1, 10, 50, 200, 5000]).to(torch.int32)
    return st


def prepare(case, seed):
    make = {"attend": _prepare_attend, "plan": _prepare_pages, "release": _prepare_pages,
            "write": _prepare_write, "sample": _prepare_sample}[case["op"]]
    st = make(case, seed)
    st["case"] = case
    return st


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_attend(s):
    from ffai_b200 import shared_prefix
    return shared_prefix.attend(s["q"], s["k_pool"], s["v_pool"], s["prefix_table"],
                                s["prefix_lens"], s["group_starts"], s["block_table"],
                                s["seq_lens"], scale=s["scale"], with_lse=s["case"]["lse"])


def _own_plan(s):
    from ffai_b200 import kvcache
    p = kvcache.plan_pages(s["lens"], s["new"], s["free_pages"], s["free_count"], s["block_table"],
                           slot_cap=s["slot_cap"], pos_base=s["pos_base"])
    return s["block_table"], p.lens, p.cu_new, p.slots, p.positions, p.free_count


def _own_release(s):
    from ffai_b200 import kvcache
    lens, count = kvcache.release_pages(s["lens"], s["done"], s["block_table"], s["free_pages"],
                                        s["free_count"])
    return s["free_pages"], lens, count


def _own_write(s):
    from ffai_b200 import kvcache
    kvcache.write_slots(s["k_pool"], s["v_pool"], s["k_new"], s["v_new"], s["slots"])
    return s["k_pool"], s["v_pool"]


def _own_sample(s):
    from ffai_b200 import sampling
    return sampling.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                           top_p=s["top_p"], min_p=s["min_p"], with_logprob=s["case"]["logprob"])


# ---- the plain forms

def _plain_attend(s):
    q, hk = s["q"], s["k_pool"].shape[1]
    b, n, h, _ = q.shape
    grp = h // hk
    out = torch.empty_like(q)
    lse = torch.empty((h, b * n), dtype=torch.float32, device=q.device) if s["case"]["lse"] else None
    sp = s["block_table"].shape[1]
    slot = torch.arange(sp * PAGE, device=q.device)
    tok = torch.arange(n, device=q.device)
    for g, plen in enumerate(s["plens"]):
        b0, b1 = s["starts"][g], s["starts"][g + 1]
        pages = s["prefix_table"][g, :_pages(plen)].long()
        table = s["block_table"][b0:b1].clamp(min=0).long()
        lens = s["seq_lens"][b0:b1]
        # query i of a sequence sees its own keys up to its own position
        limit = lens.view(-1, 1) - (n - 1) + tok                       # (s, n)
        seen = slot < limit.unsqueeze(-1)                              # (s, n, L)
        kp = s["k_pool"][pages].transpose(0, 1).reshape(hk, -1, HD)[:, :plen].float()
        vp = s["v_pool"][pages].transpose(0, 1).reshape(hk, -1, HD)[:, :plen].float()
        ks = s["k_pool"][table].transpose(1, 2).reshape(b1 - b0, hk, -1, HD).float()
        vs = s["v_pool"][table].transpose(1, 2).reshape(b1 - b0, hk, -1, HD).float()
        live = (slot < lens.view(-1, 1)).view(b1 - b0, 1, -1, 1)
        ks = torch.where(live, ks, torch.zeros_like(ks))
        vs = torch.where(live, vs, torch.zeros_like(vs))
        qg = q[b0:b1].float().unflatten(2, (hk, grp)).permute(2, 0, 1, 3, 4) * s["scale"]
        sa = qg.flatten(1, 3) @ kp.transpose(1, 2)                     # (Hkv, s n G, P)
        sb = qg.flatten(2, 3) @ ks.permute(1, 0, 3, 2)                 # (Hkv, s, n G, L)
        hide = ~seen.repeat_interleave(grp, dim=1)
        sb = sb.masked_fill(hide, float("-inf"))
        sa = sa.view(hk, b1 - b0, n * grp, plen)
        m = torch.maximum(sa.amax(-1), sb.amax(-1)).unsqueeze(-1)
        pa, pb = torch.exp(sa - m), torch.exp(sb - m)
        l = pa.sum(-1, keepdim=True) + pb.sum(-1, keepdim=True)
        o = (pa.flatten(1, 2) @ vp).view_as(qg.flatten(2, 3)) + pb @ vs.transpose(0, 1)
        o = (o / l).unflatten(2, (n, grp)).permute(1, 2, 0, 3, 4).flatten(2, 3)
        out[b0:b1] = o.to(q.dtype)
        if lse is not None:
            z = (m + torch.log(l))[..., 0].unflatten(2, (n, grp))
            lse[:, b0 * n:b1 * n] = z.permute(0, 3, 1, 2).reshape(h, -1)
    return out if lse is None else (out, lse)


def _plain_plan(s):
    lens, new = s["lens"].long(), s["new"].long()
    table, cap = s["block_table"], s["slot_cap"]
    b, mp = table.shape
    held, total = _pages(lens), lens + new
    fits = total <= mp * PAGE
    need = torch.where(fits, _pages(total) - held, torch.zeros_like(held))
    incl = need.cumsum(0)
    cu = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    ok = fits & ((need == 0) | (incl <= s["free_count"].long())) & (cu[1:] <= cap)
    need = torch.where(ok, need, torch.zeros_like(need))
    first = incl - torch.where(fits, _pages(total) - held, torch.zeros_like(held))
    page = torch.arange(mp, device=lens.device)
    j = page.view(1, -1) - held.view(-1, 1)
    take = (j >= 0) & (j < need.view(-1, 1))
    src = (s["free_count"].long() - 1 - first.view(-1, 1) - j).clamp(0, s["free_pages"].numel() - 1)
    table.copy_(torch.where(take, s["free_pages"][src], table))
    t = torch.arange(cap, device=lens.device)
    who = torch.searchsorted(cu[1:], t, right=True).clamp(max=b - 1)
    at = lens[who] + t - cu[who]
    good = (t < cu[-1]) & ok[who]
    slots = table[who, (at // PAGE).clamp(0, mp - 1)].long() * PAGE + at % PAGE
    slots = torch.where(good, slots, -1).to(torch.int32)
    positions = torch.where(good, at + s["pos_base"].long()[who], 0).to(torch.int32)
    lens_out = torch.where(ok, total, lens).to(torch.int32)
    count = (s["free_count"].long() - need.sum()).to(torch.int32)
    return table, lens_out, cu.to(torch.int32), slots, positions, count


def _plain_release(s):
    lens, done, table, free = s["lens"].long(), s["done"] != 0, s["block_table"], s["free_pages"]
    give = torch.where(done, _pages(lens), torch.zeros_like(lens))
    incl = give.cumsum(0)
    page = torch.arange(table.shape[1], device=lens.device).view(1, -1)
    live = page < give.view(-1, 1)
    at = s["free_count"].long() + (incl - give).view(-1, 1) + page
    # entries that are not handed back go to a place past the end
    pad = torch.cat([free, free[:1]])
    pad.scatter_(0, torch.where(live, at, free.numel()).flatten(), table.flatten())
    free.copy_(pad[:-1])
    return (free, torch.where(done, torch.zeros_like(lens), lens).to(torch.int32),
            (s["free_count"].long() + incl[-1:]).to(torch.int32))


def _plain_write(s):
    keep = s["slots"] >= 0
    # rows without a slot rewrite, in place, the row of the first token that has one
    first = keep.to(torch.int32).argmax()
    src = torch.where(keep, torch.arange(keep.numel(), device=keep.device), first)
    slot = s["slots"].long()[src]
    for pool, new in ((s["k_pool"], s["k_new"]), (s["v_pool"], s["v_new"])):
        pool[slot // PAGE, :, slot % PAGE] = new[src].float().to(pool.dtype)
    return s["k_pool"], s["v_pool"]


def _settings(s):
    b, dev = s["logits"].shape[0], s["logits"].device
    full = lambda v, dt: torch.full((b,), v, dtype=dt, device=dev)  # noqa: E731
    t = s["temperature"] if s["temperature"] is not None else full(1.0, torch.float32)
    k = s["top_k"] if s["top_k"] is not None else full(0, torch.int32)
    p = s["top_p"] if s["top_p"] is not None else full(1.0, torch.float32)
    m = s["min_p"] if s["min_p"] is not None else full(0.0, torch.float32)
    return t, k, p, m


def _choose(x, u, t, k, p, m, weights):
    """Tokens of logits x (B, V), f32 without NaN; `weights(d)` gives whole weights of d <= 0."""
    v = x.shape[1]
    xs, idx = torch.sort(x, dim=1, descending=True, stable=True)
    top = xs[:, :1]
    greedy = ~(t > 0)
    inv = 1.0 / torch.where(greedy, torch.ones_like(t), t)
    d = (xs - top) * inv.view(-1, 1)
    d = torch.where(xs == float("-inf"), torch.full_like(d, float("-inf")), d)
    w = weights(d)
    cum = w.cumsum(1)
    k = torch.where((k <= 0) | (k > v), torch.full_like(k, v), k).long()
    mass_k = cum.gather(1, (k - 1).view(-1, 1))
    want = torch.ceil(p.double().clamp(0, 1).view(-1, 1) * mass_k.double()).long()
    want = torch.minimum(want, mass_k).clamp(min=1)
    mass_p = cum.gather(1, torch.searchsorted(cum, want).clamp(max=v - 1))
    floor = torch.log(m.double().clamp(min=0)).float().clamp(max=0)
    mass_m = torch.where(d >= floor.view(-1, 1), w, torch.zeros_like(w)).sum(1, keepdim=True)
    mass = torch.minimum(mass_p, mass_m)
    target = torch.floor(u.double().view(-1, 1) * mass.double()).long()
    target = torch.minimum(target, mass - 1).clamp(min=0)
    at = torch.searchsorted(cum, target, right=True).clamp(max=v - 1)
    at = torch.where(greedy.view(-1, 1), torch.zeros_like(at), at)
    token = idx.gather(1, at)[:, 0]
    return torch.where(top[:, 0] == float("-inf"), torch.full_like(token, -1), token).to(torch.int32)


def _plain_sample(s):
    t, k, p, m = _settings(s)
    x = s["logits"].float()
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    token = _choose(x, s["u"], t, k, p, m, lambda d: (torch.exp(d) * W_SCALE).long())
    if not s["case"]["logprob"]:
        return token
    top = x.amax(1, keepdim=True)
    z = torch.log(torch.exp(x - top).sum(1))
    return token, x.gather(1, token.long().clamp(min=0).view(-1, 1))[:, 0] - top[:, 0] - z


_OWN = dict(attend=_own_attend, plan=_own_plan, release=_own_release, write=_own_write,
            sample=_own_sample)
_PLAIN = dict(attend=_plain_attend, plan=_plain_plan, release=_plain_release, write=_plain_write,
              sample=_plain_sample)


# ---------------------------------------------------------------- work and exact values

def work(case):
    op = case["op"]
    if op == "attend":
        sizes, plens = _ragged(case)
        # groups meet the prefix lengths in any order: the mean
        prefix_rows = sum(plens) / len(plens) * case["batch"]
        suffix = sum(_suffix_lens(case))
        es = ES[case["dtype"]]
        rows = case["batch"] * case["q_len"] * case["heads"]
        keys = (sum(plens) + suffix) * case["kv_heads"]
        return dict(bytes=2 * HD * es * (keys + rows) + (4 * rows if case["lse"] else 0),
                    flops=4 * HD * case["heads"] * case["q_len"] * (prefix_rows + suffix))
    if op == "plan":
        tokens, b = sum(_spread(1, case["new"], case["batch"])), case["batch"]
        return dict(bytes=4 * (5 * b + 2 * (tokens + 5) + 2 * (tokens // PAGE)), flops=0)
    if op == "release":
        held = sum(_pages(n) for n in _spread(0, case["length"], case["batch"])) * 0.3
        return dict(bytes=4 * (3 * case["batch"] + 2 * int(held)), flops=0)
    if op == "write":
        n = 2 * case["tokens"] * case["kv_heads"] * HD
        return dict(bytes=n * (ES[case["src"]] + ES[case["dtype"]]) + 4 * case["tokens"], flops=0)
    n = case["batch"] * case["vocab"]
    return dict(bytes=n * ES[case["dtype"]] + case["batch"] * 24, flops=4 * n)


def exact(case, seed):
    if case["op"] == "attend":
        return _exact_attend(prepare(case, seed))
    if case["op"] == "sample":
        return _exact_sample(prepare(case, seed))
    if case["op"] == "write":
        return _exact_write(prepare(case, seed))
    return None  # whole numbers throughout


def _exact_attend(s):
    q = s["q"].double()
    b, n, h, _ = q.shape
    hk = s["k_pool"].shape[1]
    out = torch.zeros((b, n, h, HD), dtype=torch.float64, device=q.device)
    lse = torch.full((b, n, h), float("-inf"), dtype=torch.float64, device=q.device)
    lens = s["seq_lens"].tolist()
    for g, plen in enumerate(s["plens"]):
        pages = s["prefix_table"][g, :_pages(plen)].long()
        pk = s["k_pool"][pages].transpose(0, 1).reshape(hk, -1, HD)[:, :plen].double()
        pv = s["v_pool"][pages].transpose(0, 1).reshape(hk, -1, HD)[:, :plen].double()
        for i in range(s["starts"][g], s["starts"][g + 1]):
            pages = s["block_table"][i, :_pages(lens[i])].long()
            own_k = s["k_pool"][pages].transpose(0, 1).reshape(hk, -1, HD)[:, :lens[i]].double()
            own_v = s["v_pool"][pages].transpose(0, 1).reshape(hk, -1, HD)[:, :lens[i]].double()
            qi = q[i].reshape(n, hk, h // hk, HD).permute(1, 0, 2, 3).reshape(hk, -1, HD)
            sc = torch.cat([qi @ pk.transpose(1, 2), qi @ own_k.transpose(1, 2)], -1) * s["scale"]
            sc = sc.reshape(hk, n, h // hk, -1)
            for j in range(n):
                seen = plen + max(0, lens[i] - (n - 1 - j))
                sc[:, j, :, seen:] = float("-inf")
            z = torch.logsumexp(sc, -1)
            pr = torch.exp(sc - z.unsqueeze(-1)).reshape(hk, -1, sc.shape[-1])
            o = pr[..., :plen] @ pv + pr[..., plen:] @ own_v
            out[i] = o.reshape(hk, n, h // hk, HD).permute(1, 0, 2, 3).reshape(n, h, HD)
            lse[i] = z.permute(1, 0, 2).reshape(n, h)
    lse = lse.permute(2, 0, 1).reshape(h, b * n)
    return (out, lse) if s["case"]["lse"] else out


def _exact_write(s):
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    pools = []
    for pool, new in ((s["k_pool"], s["k_new"]), (s["v_pool"], s["v_new"])):
        flat = pool.double().transpose(1, 2).flatten(0, 1)             # (slots, Hkv, 64)
        flat[at] = new[keep].double()
        pools.append(flat.unflatten(0, (-1, PAGE)).transpose(1, 2))
    return tuple(pools)


def _exact_sample(s):
    t, k, p, m = (v.tolist() for v in _settings(s))
    u = s["u"].double()
    x = s["logits"]
    tokens, logprobs = [], []
    for i in range(x.shape[0]):
        row = torch.nan_to_num(x[i].float(), nan=float("-inf"), posinf=float("inf"),
                               neginf=float("-inf"))
        xs, idx = torch.sort(row, descending=True, stable=True)
        if not t[i] > 0:
            at = 0
        else:
            # the exponent is defined in 32 bits, its power rounded to 32 bits
            d = (xs - xs[0]) * (torch.ones(1, device=x.device) / t[i])
            w = torch.floor(torch.exp(d.double()).float().double() * W_SCALE)
            cum = w.cumsum(0)
            n = k[i] if 0 < k[i] <= xs.numel() else xs.numel()
            mk = cum[n - 1]
            mass = cum[(cum >= mk * min(max(p[i], 0.0), 1.0)).to(torch.int8).argmax()]
            if m[i] > 0:
                mass = torch.minimum(mass, w[d.double() >= min(math.log(m[i]), 0.0)].sum())
            at = int((cum > torch.floor(u[i] * mass)).to(torch.int8).argmax())
        tokens.append(int(idx[at]))
        logprobs.append(float(xs[at].double() - torch.logsumexp(row.double(), 0)))
    tok = torch.tensor(tokens, dtype=torch.int32, device=x.device)
    if not s["case"]["logprob"]:
        return tok
    return tok, torch.tensor(logprobs, dtype=torch.float64, device=x.device)
