"""Decode steps of a batch whose requests share prompts, on the device from
hidden states to sampled tokens: the batched decode operators as a caller
chains them, around one attention layer.

A step is seven calls without a host round trip:

  1. the fused q/k/v projection (`gemm.linear`) of the step's tokens;
  2. `kvcache.plan_pages`: pages and slots for them, from lengths on the device;
  3. `kvcache.write_slots`: their keys and values, read in place from the
     projection's rows, into the page pools;
  4. `shared_prefix.attend`: every request over its group's prompt, read once a
     group, and its own keys, q likewise in place;
  5. the out-projection with the residual in its epilogue;
  6. the vocabulary projection;
  7. `sampling.sample`.

The state lives in tensors that are made once and that every call, `open` and
`close_groups` too, updates in place: a step captured in a CUDA graph can be
replayed for the decoder's whole life.  Requests that end hand their pages
back (`kvcache.release_pages`).  Layer norms, the MLP and embeddings stay with
the caller, as in `encoder_attention`; a model with more layers keeps pools per
layer and shares the plan.  No reference counterpart (its decoder serves one
utterance at a time and clones its caches, text_decoder.rs:1363-1381).

    python -m ffai_b200.group_decoder        # a timed run on synthetic weights
"""

from __future__ import annotations

import torch

from . import kvcache, sampling, shared_prefix
from .gemm import linear

HD = 64


class GroupDecoder:
    """One attention layer and the vocabulary projection for up to `batch`
    requests: w_qkv ((heads + 2 kv_heads) * 64, D), w_out (D, heads * 64),
    w_vocab (V, D), bf16 on the device.  At most max_groups prompts at a time
    (default: `batch`) of max_prompt tokens (default: what num_pages hold);
    attention is laid out for these bounds, so close ones make it faster."""

    def __init__(self, w_qkv, w_out, w_vocab, *, heads: int, kv_heads: int, batch: int,
                 max_len: int, num_pages: int, scale: float = HD ** -0.5,
                 max_groups: int | None = None, max_prompt: int | None = None):
        if w_qkv.shape != ((heads + 2 * kv_heads) * HD, w_out.shape[0]) or \
                w_out.shape[1] != heads * HD or w_vocab.shape[1] != w_out.shape[0]:
            raise ValueError("group decoder: w_qkv ((heads + 2 kv_heads) * 64, D), "
                             "w_out (D, heads * 64), w_vocab (V, D)")
        dev = w_qkv.device
        self.w_qkv, self.w_out, self.vocab = w_qkv, w_out, w_vocab.shape[0]
        # the GEMM writes whole groups of 32 columns: rows of zeros behind the vocabulary
        pad = -self.vocab % 32
        self.w_vocab = torch.cat([w_vocab, w_vocab.new_zeros(pad, w_vocab.shape[1])])
        self.heads, self.kv_heads, self.scale, self.batch = heads, kv_heads, scale, batch
        shape = (num_pages, kv_heads, kvcache.PAGE_KEYS, HD)
        self.k_pool = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
        self.v_pool = torch.zeros_like(self.k_pool)
        i32 = dict(dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(num_pages, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)
        pages = (max_len + kvcache.PAGE_KEYS - 1) // kvcache.PAGE_KEYS
        self.block_table = torch.full((batch, pages), -1, **i32)
        self.lens = torch.zeros(batch, **i32)
        self.max_groups = batch if max_groups is None else max_groups
        self.max_prompt = num_pages * kvcache.PAGE_KEYS if max_prompt is None else max_prompt
        pages = max(1, (self.max_prompt + kvcache.PAGE_KEYS - 1) // kvcache.PAGE_KEYS)
        self.prefix_table = torch.full((self.max_groups, pages), -1, **i32)
        self.prefix_lens = torch.zeros(self.max_groups, **i32)
        self.group_starts = torch.zeros(self.max_groups + 1, **i32)

    def _project(self, x):
        """(T, D) -> q (T, heads, 64), k, v (T, kv_heads, 64): views of one buffer."""
        qkv = linear(x, self.w_qkv).unflatten(1, (-1, HD))
        H, hk = self.heads, self.kv_heads
        return qkv[:, :H], qkv[:, H:H + hk], qkv[:, H + hk:]

    def open(self, prompts, sizes) -> None:
        """Start groups: prompts[g] (n_g, D) bf16 hidden states (after the
        caller's norm) of group g's prompt, shared by sizes[g] consecutive
        requests.  The requests and groups before must have been closed."""
        ns = [p.shape[0] for p in prompts]
        if len(ns) != len(sizes) or sum(sizes) > self.batch:
            raise ValueError("group decoder: a size for each prompt, at most `batch` requests")
        if len(ns) > self.max_groups or max(ns, default=0) > self.max_prompt:
            raise ValueError(f"group decoder: at most {self.max_groups} prompts of "
                             f"{self.max_prompt} tokens")
        i32 = dict(dtype=torch.int32, device=self.lens.device)
        none = self.max_groups - len(ns)  # groups without requests, behind the others
        starts = [0]
        for s in list(sizes) + [0] * none:
            starts.append(starts[-1] + s)
        self.group_starts.copy_(torch.tensor(starts, **i32))
        want = torch.tensor(ns + [0] * none, **i32)
        plan = kvcache.plan_pages(torch.zeros_like(want), want, self.free_pages, self.free_count,
                                  self.prefix_table, slot_cap=sum(ns))
        self.free_count.copy_(plan.free_count)
        self.prefix_lens.copy_(plan.lens)
        if not torch.equal(plan.lens, want):
            self.close_groups()
            raise MemoryError("group decoder: no free pages for the prompts")
        if sum(ns) > 0:
            _, k, v = self._project(torch.cat(list(prompts)))
            kvcache.write_slots(self.k_pool, self.v_pool, k, v, plan.slots)

    def hidden(self, x, active):
        """The layer on x (B, n, D) bf16, n new tokens of every request with
        active[b] = 1 (int32; others 0): (x + attention's output, served), served[b]
        false for requests that were not active or found no page (nothing of
        them is kept)."""
        B, n, D = x.shape
        q, k, v = self._project(x.view(B * n, D))
        plan = kvcache.plan_pages(self.lens, active * n, self.free_pages, self.free_count,
                                  self.block_table, slot_cap=B * n)
        # packed rows of the plan to rows of x: the same unless a request sits out
        at = (plan.cu_new[:-1, None] + torch.arange(n, device=x.device)).clamp_(max=B * n - 1)
        served = (active > 0) & (plan.lens != self.lens)
        slots = torch.where(served[:, None], plan.slots[at], -1).flatten()
        self.lens.copy_(plan.lens)
        self.free_count.copy_(plan.free_count)
        kvcache.write_slots(self.k_pool, self.v_pool, k, v, slots)
        o = shared_prefix.attend(q.unflatten(0, (B, n)), self.k_pool, self.v_pool,
                                 self.prefix_table, self.prefix_lens, self.group_starts,
                                 self.block_table, self.lens, scale=self.scale)
        y = linear(o.view(B * n, -1), self.w_out, residual=x.view(B * n, D))
        return y.view(B, n, D), served

    def step(self, x, active, u, **settings):
        """One step: tokens (B, n) int32 sampled after each new token with
        u (B * n,) in [0, 1) and `sampling.sample`'s settings; -1 where a request
        was not served."""
        B, n, D = x.shape
        y, served = self.hidden(x, active)
        logits = linear(y.view(B * n, D), self.w_vocab, out_dtype=torch.float32)[:, :self.vocab]
        tokens = sampling.sample(logits, u, **settings).view(B, n)
        return torch.where(served[:, None], tokens, -1)

    def close(self, done) -> None:
        """Requests with done[b] != 0 (int32) hand their pages back."""
        lens, count = kvcache.release_pages(self.lens, done, self.block_table, self.free_pages,
                                            self.free_count)
        self.lens.copy_(lens)
        self.free_count.copy_(count)

    def close_groups(self) -> None:
        """All prompts' pages go back."""
        lens, count = kvcache.release_pages(self.prefix_lens, torch.ones_like(self.prefix_lens),
                                            self.prefix_table, self.free_pages, self.free_count)
        self.prefix_lens.copy_(lens)
        self.free_count.copy_(count)


def main(groups: int = 12, beams: int = 5, prompt: int = 1500, steps: int = 64) -> None:
    """Twelve utterances of five beams at Whisper-large's width, each group over
    its own 1500 shared keys; a captured step replayed."""
    D, heads, vocab, B = 1280, 20, 51865, groups * beams
    g = torch.Generator(device="cuda:0").manual_seed(0)
    w = lambda *s: (torch.randn(s, generator=g, device="cuda:0") * s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
    dec = GroupDecoder(w(3 * D, D), w(D, D), w(vocab, D), heads=heads, kv_heads=heads, batch=B,
                       max_len=448, num_pages=groups * 24 + B * 7, max_groups=groups,
                       max_prompt=prompt)
    dec.open([w(prompt, D) * D ** 0.5 for _ in range(groups)], [beams] * groups)
    table = w(vocab, D) * D ** 0.5  # embeddings
    active = torch.ones(B, dtype=torch.int32, device="cuda:0")
    u = torch.zeros(B, device="cuda:0")
    tokens = torch.randint(0, vocab, (B, 1), generator=g, device="cuda:0", dtype=torch.int32)

    def step():
        tokens.copy_(dec.step(table[tokens.clamp(min=0)], active, u, temperature=0.8, top_p=0.95))

    for _ in range(3):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    for _ in range(steps):
        u.uniform_(generator=g)
        graph.replay()
    b.record()
    torch.cuda.synchronize()
    us = a.elapsed_time(b) * 1e3 / steps
    print(f"{B} requests in {groups} groups, {prompt} + up to {steps + 4} keys, vocabulary {vocab}: "
          f"{us:.0f} us a step, {B / us * 1e6:.0f} tokens/s")


if __name__ == "__main__":
    main()
