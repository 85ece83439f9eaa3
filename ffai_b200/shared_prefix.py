"""Attention of a batch whose sequences share long prefixes, over a paged KV
cache: each group's prefix is read once for all its sequences
(ffai_attn_shared_prefix).

Group g is the consecutive sequences [group_starts[g], group_starts[g + 1])
and shares the first prefix_lens[g] keys of the pages in prefix_table[g];
sequence b adds seq_lens[b] keys of its own in the pages of block_table[b].
Query i of a sequence's q_len sees the whole prefix and its own keys up to its
own position (the last query is the newest key).  Pools are those of
kvcache.PagedKVCache, (num_pages, kv_heads, 64, 64); heads may be a multiple
of kv_heads.  No reference counterpart: its beams clone whole caches
(text_decoder.rs:1363-1381).
"""

from __future__ import annotations

import ctypes

import torch

from . import _abi
from .attention import _DT, _LAYOUT, _check, _ptr, _stream, _token_stride, context
from .kvcache import PAGE_KEYS


def _int32(t: torch.Tensor, name: str, shape, dev: torch.device) -> None:
    if t.dtype != torch.int32 or t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"shared prefix: {name} must be contiguous int32 {tuple(shape)} on {dev}")


def attend(q, k_pool, v_pool, prefix_table, prefix_lens, group_starts, block_table, seq_lens, *,
           scale: float = 1.0, q_layout="token", out_layout="token", out_dtype=None,
           with_lse=False, out=None):
    """q (B, q_len, H, 64) ("token", possibly a view of a fused projection) or
    (B, H, q_len, 64) ("heads"); prefix_table (groups, pages), prefix_lens
    (groups,), group_starts (groups + 1,), block_table (B, pages), seq_lens
    (B,): int32 on the device.  Returns out in `out_layout` and `out_dtype`
    (default: q's) [, lse f32 (H, B * q_len) or (B, H, q_len)]."""
    dev = q.device
    if dev.type != "cuda":
        raise ValueError("operands must be CUDA tensors")
    if q.dim() != 4 or q.shape[-1] != 64:
        raise ValueError(f"expected a 4-d (..., 64) q, got {tuple(q.shape)}")
    if q_layout not in ("token", "heads") or out_layout not in ("token", "heads"):
        raise ValueError("shared prefix: layouts are 'token' or 'heads'")
    B, n, H = (q.shape[0], q.shape[1], q.shape[2]) if q_layout == "token" else (
        q.shape[0], q.shape[2], q.shape[1])
    ts = 0
    if not q.is_contiguous():
        if q_layout == "token":  # one token a sequence: the sequences are the tokens
            ts = _token_stride(q[:, 0] if n == 1 else q)
        if q_layout != "token" or ts is None or ts < H * 64:
            raise ValueError("q must be contiguous, or a token-major view with dense heads and "
                             "one token stride")
    pool = k_pool.shape
    if (len(pool) != 4 or pool[2] != PAGE_KEYS or pool[3] != 64 or v_pool.shape != pool
            or v_pool.dtype != k_pool.dtype or k_pool.device != dev or v_pool.device != dev
            or not k_pool.is_contiguous() or not v_pool.is_contiguous()):
        raise ValueError("shared prefix: k and v pools contiguous (num_pages, kv_heads, 64, 64) "
                         "of one type on q's device")
    groups = prefix_table.shape[0]
    if prefix_table.dim() != 2 or block_table.dim() != 2:
        raise ValueError("shared prefix: tables are 2-d (rows, pages)")
    _int32(prefix_table, "prefix_table", prefix_table.shape, dev)
    _int32(prefix_lens, "prefix_lens", (groups,), dev)
    _int32(group_starts, "group_starts", (groups + 1,), dev)
    _int32(block_table, "block_table", (B, block_table.shape[1]), dev)
    _int32(seq_lens, "seq_lens", (B,), dev)
    shape = (B, n, H, 64) if out_layout == "token" else (B, H, n, 64)
    if out is None:
        out = torch.empty(shape, dtype=q.dtype if out_dtype is None else out_dtype, device=dev)
    elif out.shape != shape or out.device != dev or not out.is_contiguous():
        raise ValueError(f"shared prefix: out must be contiguous {shape} on {dev}")
    lse = None
    if with_lse:
        lse = torch.empty((H, B * n) if out_layout == "token" else (B, H, n),
                          dtype=torch.float32, device=dev)
    if any(t.dtype not in _DT for t in (q, k_pool, out)):
        raise TypeError("shared prefix: f32, bf16 or f16 operands")
    d = _abi.new_desc(batch=B, heads=H, q_len=n, q_dtype=_DT[q.dtype], kv_dtype=_DT[k_pool.dtype],
                      out_dtype=_DT[out.dtype], q_layout=_LAYOUT[q_layout],
                      out_layout=_LAYOUT[out_layout], scale=scale, token_stride=ts)
    ctx = context(dev.index)
    st = _abi.load().ffai_attn_shared_prefix(
        ctx, ctypes.byref(d), pool[1], _ptr(q), _ptr(k_pool), _ptr(v_pool), pool[0],
        _ptr(group_starts), groups, _ptr(prefix_table), _ptr(prefix_lens), prefix_table.shape[1],
        _ptr(block_table), _ptr(seq_lens), block_table.shape[1], _ptr(out), _ptr(lse),
        _stream(dev))
    _check(st, ctx)
    return (out, lse) if with_lse else out
