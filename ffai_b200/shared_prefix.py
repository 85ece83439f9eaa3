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
from .attention import _DT, _LAYOUT, _check, _raw_stream, _token_stride, context
from .kvcache import PAGE_KEYS


def _int32(t: torch.Tensor, name: str, shape, index: int) -> int:
    """Address of a contiguous int32 device tensor of this shape."""
    if (t.dtype is not torch.int32 or t.shape != shape or t.get_device() != index
            or not t.is_contiguous()):
        raise ValueError(f"shared prefix: {name} must be contiguous int32 {tuple(shape)} on "
                         f"cuda:{index}")
    return t.data_ptr()


def attend(q, k_pool, v_pool, prefix_table, prefix_lens, group_starts, block_table, seq_lens, *,
           scale: float = 1.0, q_layout="token", out_layout="token", out_dtype=None,
           with_lse=False, out=None):
    """q (B, q_len, H, 64) ("token", possibly a view of a fused projection) or
    (B, H, q_len, 64) ("heads"); prefix_table (groups, pages), prefix_lens
    (groups,), group_starts (groups + 1,), block_table (B, pages), seq_lens
    (B,): int32 on the device.  Returns out in `out_layout` and `out_dtype`
    (default: q's) [, lse f32 (H, B * q_len) or (B, H, q_len)]."""
    if not q.is_cuda:
        raise ValueError("operands must be CUDA tensors")
    if q.dim() != 4 or q.shape[3] != 64:
        raise ValueError(f"expected a 4-d (..., 64) q, got {tuple(q.shape)}")
    if q_layout not in ("token", "heads") or out_layout not in ("token", "heads"):
        raise ValueError("shared prefix: layouts are 'token' or 'heads'")
    index = q.get_device()
    token = q_layout == "token"
    B, n, H, _ = q.shape
    if not token:
        n, H = H, n
    ts = 0
    if not q.is_contiguous():
        if token:  # one token a sequence: the sequences are the tokens
            ts = _token_stride(q[:, 0] if n == 1 else q)
        if not token or ts is None or ts < H * 64:
            raise ValueError("q must be contiguous, or a token-major view with dense heads and "
                             "one token stride")
    pool = k_pool.shape
    if (len(pool) != 4 or pool[2] != PAGE_KEYS or pool[3] != 64 or v_pool.shape != pool
            or v_pool.dtype is not k_pool.dtype or k_pool.get_device() != index
            or v_pool.get_device() != index or not k_pool.is_contiguous()
            or not v_pool.is_contiguous()):
        raise ValueError("shared prefix: k and v pools contiguous (num_pages, kv_heads, 64, 64) "
                         "of one type on q's device")
    if prefix_table.dim() != 2 or block_table.dim() != 2:
        raise ValueError("shared prefix: tables are 2-d (rows, pages)")
    groups, prefix_pages = prefix_table.shape
    max_pages = block_table.shape[1]
    tables = (_int32(group_starts, "group_starts", (groups + 1,), index), groups,
              _int32(prefix_table, "prefix_table", (groups, prefix_pages), index),
              _int32(prefix_lens, "prefix_lens", (groups,), index), prefix_pages,
              _int32(block_table, "block_table", (B, max_pages), index),
              _int32(seq_lens, "seq_lens", (B,), index), max_pages)
    shape = (B, n, H, 64) if out_layout == "token" else (B, H, n, 64)
    if out is None:
        out = q.new_empty(shape) if out_dtype is None else q.new_empty(shape, dtype=out_dtype)
    elif out.shape != shape or out.get_device() != index or not out.is_contiguous():
        raise ValueError(f"shared prefix: out must be contiguous {shape} on cuda:{index}")
    lse = None
    if with_lse:
        lse = q.new_empty((H, B * n) if out_layout == "token" else (B, H, n), dtype=torch.float32)
    dt = _DT.get(q.dtype), _DT.get(k_pool.dtype), _DT.get(out.dtype)
    if None in dt:
        raise TypeError("shared prefix: f32, bf16 or f16 operands")
    d = _abi.Desc(batch=B, heads=H, q_len=n, head_dim=64, q_dtype=dt[0], kv_dtype=dt[1],
                  out_dtype=dt[2], q_layout=_LAYOUT[q_layout], out_layout=_LAYOUT[out_layout],
                  scale=scale, token_stride=ts)
    ctx = context(index)
    st = _abi.load().ffai_attn_shared_prefix(
        ctx, ctypes.byref(d), pool[1], q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), pool[0],
        *tables, out.data_ptr(), None if lse is None else lse.data_ptr(), _raw_stream(index))
    if st:
        _check(st, ctx)
    return (out, lse) if with_lse else out
