"""Decode steps of a batch that verifies drafted tokens, on the device from hidden
states to emitted tokens: the operators of ragged steps as a caller chains them,
around one attention layer.

A step's rows are packed, cu_rows[b] .. cu_rows[b + 1] request b's: a chunk of its
prompt, its last token with any number of drafts, or nothing.  It is eight calls
without a host round trip:

  1. the fused q/k/v projection (`gemm.linear`) of all rows;
  2. `kvcache.plan_pages`: pages and slots for them, from lengths on the device;
  3. `kvcache.write_slots`: their keys and values into the page pools;
  4. `chunk_attention.attend`: each row over its request's keys up to its own;
  5. the out-projection with the residual in its epilogue;
  6. the vocabulary projection of the rows that are to be verified;
  7. `sampling.verify`: the drafts that stand, and a token behind them;
  8. `kvcache.fork_pages`: the keys of the others are cut off, and pages that
     became empty go back.

`select` reorders, splits and ends requests (beams, best-of-n) on shared pages,
`compact` moves the pages in use to the front of the pools.  The state lives in
tensors that are made once and that every call updates in place: a step captured
in a CUDA graph can be replayed for the decoder's whole life.  Layer norms, the
MLP, embeddings and the drafts themselves stay with the caller; a model with more
layers keeps pools per layer and shares the plan, the fork and the compaction.  No
reference counterpart (its decoder takes one token a step, text_decoder.rs:926-941).

    python -m ffai_b200.draft_decoder        # a timed run on synthetic weights
"""

from __future__ import annotations

import torch

from . import chunk_attention, kvcache, sampling
from .gemm import linear

HD = 64


class DraftDecoder:
    """One attention layer and the vocabulary projection for up to `batch`
    requests: w_qkv ((heads + 2 kv_heads) * 64, D), w_out (D, heads * 64),
    w_vocab (V, D), bf16 on the device."""

    def __init__(self, w_qkv, w_out, w_vocab, *, heads: int, kv_heads: int, batch: int,
                 max_len: int, num_pages: int, scale: float = HD ** -0.5):
        if w_qkv.shape != ((heads + 2 * kv_heads) * HD, w_out.shape[0]) or \
                w_out.shape[1] != heads * HD or w_vocab.shape[1] != w_out.shape[0]:
            raise ValueError("draft decoder: w_qkv ((heads + 2 kv_heads) * 64, D), "
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
        self.rows = torch.arange(batch, **i32)

    def _project(self, x):
        """(T, D) -> q (T, heads, 64), k, v (T, kv_heads, 64): views of one buffer."""
        qkv = linear(x, self.w_qkv).unflatten(1, (-1, HD))
        H, hk = self.heads, self.kv_heads
        return qkv[:, :H], qkv[:, H:H + hk], qkv[:, H + hk:]

    def hidden(self, x, cu_rows, *, max_rows: int | None = None):
        """The layer on x (T, D) bf16, request b's rows cu_rows[b] .. cu_rows[b + 1]
        (batch + 1, int32), whose keys and values are kept: (x + attention's
        output, served (batch,)), served[b] false for requests that brought
        nothing or found no page (nothing of them is kept).  Rows of those, and
        before the first or behind the last request, hold nothing of use.  max_rows: the most rows of
        a request, if known."""
        T = x.shape[0]
        q, k, v = self._project(x)
        n = cu_rows.diff()
        plan = kvcache.plan_pages(self.lens, n, self.free_pages, self.free_count,
                                  self.block_table, slot_cap=T)
        served = plan.lens != self.lens
        # packed rows of the plan to rows of x: the same unless a request sits out
        i = torch.arange(T, device=x.device, dtype=torch.int32)
        b = torch.searchsorted(cu_rows[1:], i, right=True).clamp_(max=self.batch - 1)
        at = plan.cu_new[b] + i - cu_rows[b]
        here = served[b] & (i >= cu_rows[0]) & (i < cu_rows[-1])
        slots = torch.where(here, plan.slots[at.clamp_(0, max(T - 1, 0))], -1)
        self.lens.copy_(plan.lens)
        self.free_count.copy_(plan.free_count)
        kvcache.write_slots(self.k_pool, self.v_pool, k, v, slots)
        o = chunk_attention.attend(q, self.k_pool, self.v_pool, cu_rows, self.block_table,
                                   self.lens, scale=self.scale, max_q=max_rows)
        return linear(o.view(T, -1), self.w_out, residual=x), served

    def settle(self, y, tokens, cu_rows, u, u_last, served, **settings) -> sampling.Verified:
        """`sampling.verify` (its arguments and settings) on the layer's output
        rows y (R, D) of the last tokens and drafts that the last call of `hidden`
        took in, cu_rows[b] .. cu_rows[b + 1] request b's; the keys of the drafts
        that do not stand are cut off.  Requests that were not served accept
        nothing, and their next token is -1."""
        if y.shape[0]:
            logits = linear(y, self.w_vocab, out_dtype=torch.float32)[:, :self.vocab]
        else:  # a step of prompts only
            logits = y.new_empty((0, self.vocab), dtype=torch.float32)
        v = sampling.verify(logits, tokens, cu_rows, u, u_last, **settings)
        accepted = torch.where(served, v.accepted, 0)
        n = cu_rows.diff()
        keep = torch.where(served & (n > 0), self.lens - n + 1 + accepted, self.lens)
        # (no copies: a key that a request wrote itself lies in a page of its own)
        self._take(kvcache.fork_pages(self.rows, self.lens, self.block_table, self.free_pages,
                                      self.free_count, keep=keep))
        i = torch.arange(tokens.numel(), device=y.device, dtype=torch.int32)
        b = torch.searchsorted(cu_rows[1:], i, right=True).clamp_(max=self.batch - 1)
        logprobs = None if v.logprobs is None else torch.where(served[b], v.logprobs, 0.0)
        return v._replace(accepted=accepted, next=torch.where(served, v.next, -1),
                          tokens=torch.where(served[b], v.tokens, -1), logprobs=logprobs)

    def step(self, x, tokens, cu_rows, u, u_last, *, max_rows: int | None = None,
             **settings) -> sampling.Verified:
        """A step in which every request brings its last token and its drafts
        (tokens (T,) int32, x their hidden states): `hidden` and `settle` of all
        rows."""
        y, served = self.hidden(x, cu_rows, max_rows=max_rows)
        return self.settle(y, tokens, cu_rows, u, u_last, served, **settings)

    def _take(self, f: kvcache.Fork) -> None:
        self.block_table.copy_(f.block_table)
        self.lens.copy_(f.lens)
        self.free_count.copy_(f.free_count)

    def select(self, src):
        """Request b continues request src[b] (batch, int32; -1: it ends), sharing
        its pages.  Returns (batch,) bool: false where no page was left for the
        copy of a last one, and the request was cut back to whole pages, or where
        src[b] is no request (b is empty then; `attention.sync` reports it)."""
        if src.shape != self.rows.shape:
            raise ValueError(f"draft decoder: src must be ({self.batch},)")
        old = self.lens[src.clamp(0, self.batch - 1)]
        f = kvcache.fork_pages(src, self.lens, self.block_table, self.free_pages, self.free_count)
        kvcache.copy_pages(self.k_pool, self.v_pool, f.copy_src, f.copy_dst, keys=f.copy_keys)
        self._take(f)
        return (src < 0) | (src < self.batch) & (f.lens == old)

    def compact(self) -> None:
        """The pages in use move to the front of the pools, in order."""
        c = kvcache.compact_pages(self.lens, self.block_table, self.free_pages, self.free_count)
        kvcache.copy_pages(self.k_pool, self.v_pool, c.copy_src, c.copy_dst)
        self.block_table.copy_(c.block_table)
        self.free_pages.copy_(c.free_pages)


def main(batch: int = 64, prompt: int = 1500, drafts: int = 4, steps: int = 64) -> None:
    """64 requests at Whisper-large's width behind prompts of 1500 tokens, fed in
    chunks, four drafts each a step; a captured step replayed."""
    D, heads, vocab, dev = 1280, 20, 51865, "cuda:0"
    g = torch.Generator(device=dev).manual_seed(0)
    w = lambda *s: (torch.randn(s, generator=g, device=dev) * s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
    rows = drafts + 1
    most = prompt + rows * (steps + 8)
    dec = DraftDecoder(w(3 * D, D), w(D, D), w(vocab, D), heads=heads, kv_heads=heads, batch=batch,
                       max_len=most, num_pages=batch * ((most + 63) // 64))
    left, chunk = prompt, 512
    while left > 0:
        n = min(chunk, left)
        cu = torch.arange(batch + 1, dtype=torch.int32, device=dev) * n
        dec.hidden(w(batch * n, D) * D ** 0.5, cu, max_rows=n)
        left -= n
    table = w(vocab, D) * D ** 0.5  # embeddings
    cu = torch.arange(batch + 1, dtype=torch.int32, device=dev) * rows
    u = torch.zeros(batch * rows, device=dev)
    u_last = torch.zeros(batch, device=dev)
    tokens = torch.randint(0, vocab, (batch, rows), generator=g, device=dev, dtype=torch.int32)
    emitted = torch.zeros((), dtype=torch.int64, device=dev)

    def step():
        v = dec.step(table[tokens.flatten()], tokens.flatten(), cu, u, u_last, max_rows=rows,
                     temperature=1.0)
        tokens[:, 0] = v.next.clamp(min=0)
        emitted.add_(v.accepted.sum() + batch)

    for _ in range(3):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    emitted.zero_()
    torch.cuda.synchronize()
    a.record()
    for _ in range(steps):
        u.uniform_(generator=g)
        u_last.uniform_(generator=g)
        graph.replay()
    b.record()
    torch.cuda.synchronize()
    us = a.elapsed_time(b) * 1e3 / steps
    print(f"{batch} requests of {drafts} drafts behind {prompt} keys, vocabulary {vocab}: {us:.0f} us "
          f"a step, {emitted.item() / steps / us * 1e6:.0f} tokens/s")


if __name__ == "__main__":
    main()
