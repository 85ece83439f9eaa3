"""Attention of a chunk of new tokens over a paged KV cache
(ffai_attn_chunk_paged): a prompt's next chunk, a last token with its drafts, or
a single token, any mix of them in one call.

Sequence b brings the packed tokens cu_q[b] .. cu_q[b + 1] of q, the newest of
the seq_lens[b] keys in the pages of block_table[b]; each sees the keys up to its
own (all of them without `causal`).  Pools are those of kvcache.PagedKVCache,
(num_pages, kv_heads, 64, 64); heads may be a multiple of kv_heads.  No reference
counterpart: prompts there run whole (text_decoder.rs:904-923).
"""

from __future__ import annotations

import ctypes

import torch

from . import _abi
from .attention import _DT, _check, _raw_stream, _token_stride, context
from .kvcache import PAGE_KEYS


def _int32(t: torch.Tensor, name: str, shape, index: int) -> int:
    """Address of a contiguous int32 device tensor of this shape."""
    if (t.dtype is not torch.int32 or t.shape != shape or t.get_device() != index
            or not t.is_contiguous()):
        raise ValueError(f"chunk: {name} must be contiguous int32 {tuple(shape)} on cuda:{index}")
    return t.data_ptr()


def attend(q, k_pool, v_pool, cu_q, block_table, seq_lens, *, scale: float = 1.0,
           causal: bool = True, max_q: int | None = None, out_dtype=None, with_lse=False, out=None):
    """q (T, H, 64), possibly a view of a fused projection; cu_q (B + 1,),
    block_table (B, pages), seq_lens (B,) int32 on the device, seq_lens with the
    new tokens.  max_q: the most tokens of a sequence, if known (it helps
    to choose the kernel, one for all of them).  Returns out (T, H, 64) of out_dtype (default: q's) [, lse f32
    (H, T)]; rows outside every sequence are left as they are in `out`."""
    if not q.is_cuda:
        raise ValueError("operands must be CUDA tensors")
    if q.dim() != 3 or q.shape[2] != 64:
        raise ValueError(f"expected a 3-d (T, H, 64) q, got {tuple(q.shape)}")
    index = q.get_device()
    T, H, _ = q.shape
    ts = _token_stride(q)
    if ts is None or (ts != 0 and T > 1 and ts < H * 64):
        raise ValueError("q must be contiguous, or a view with dense heads and one token stride")
    pool = k_pool.shape
    if (len(pool) != 4 or pool[2] != PAGE_KEYS or pool[3] != 64 or v_pool.shape != pool
            or v_pool.dtype is not k_pool.dtype or k_pool.get_device() != index
            or v_pool.get_device() != index or not k_pool.is_contiguous()
            or not v_pool.is_contiguous()):
        raise ValueError("chunk: k and v pools contiguous (num_pages, kv_heads, 64, 64) of one "
                         "type on q's device")
    if block_table.dim() != 2:
        raise ValueError("chunk: block_table is 2-d (rows, pages)")
    B, max_pages = block_table.shape
    starts = _int32(cu_q, "cu_q", (B + 1,), index)
    tables = (_int32(block_table, "block_table", (B, max_pages), index),
              _int32(seq_lens, "seq_lens", (B,), index), max_pages)
    if out is None:
        out = q.new_empty((T, H, 64)) if out_dtype is None else q.new_empty((T, H, 64), dtype=out_dtype)
    elif out.shape != (T, H, 64) or out.get_device() != index or not out.is_contiguous():
        raise ValueError(f"chunk: out must be contiguous {(T, H, 64)} on cuda:{index}")
    lse = q.new_empty((H, T), dtype=torch.float32) if with_lse else None
    dt = _DT.get(q.dtype), _DT.get(k_pool.dtype), _DT.get(out.dtype)
    if None in dt:
        raise TypeError("chunk: f32, bf16 or f16 operands")
    token = _abi.LAYOUT_TOKEN_MAJOR
    d = _abi.Desc(batch=B, heads=H, q_len=max_q or 0, head_dim=64, q_dtype=dt[0], kv_dtype=dt[1],
                  out_dtype=dt[2], q_layout=token, out_layout=token, causal=int(causal),
                  scale=scale, token_stride=ts if T > 1 else 0)
    ctx = context(index)
    st = _abi.load().ffai_attn_chunk_paged(
        ctx, ctypes.byref(d), pool[1], q.data_ptr(), T, starts, k_pool.data_ptr(),
        v_pool.data_ptr(), pool[0], *tables, out.data_ptr(),
        None if lse is None else lse.data_ptr(), _raw_stream(index))
    if st:
        _check(st, ctx)
    return (out, lse) if with_lse else out
