"""Sampling of one token per row of logits on the device: temperature, top-k,
top-p and min-p from given uniform numbers (ffai_sample).

    tokens = sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)

The settings are per row (device tensors), one number for all rows, or None
for off.  Equal inputs give equal tokens: weights are whole numbers, so every
sum is exact.  No reference counterpart: the reference's decoder takes the
largest logit on the host.

`verify` checks drafted tokens against the target's distribution in the same
whole weights (ffai_verify).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _abi
from .attention import _DT, _check, _raw_stream, context


def _setting(v, name: str, dtype: torch.dtype, batch: int, dev: torch.device):
    """A row setting as a device vector (a number is spread over the rows)."""
    if not isinstance(v, torch.Tensor):
        return torch.full((batch,), v, dtype=dtype, device=dev)
    if (v.dtype is not dtype or v.dim() != 1 or v.numel() != batch
            or v.get_device() != dev.index or not v.is_contiguous()):
        raise ValueError(f"sample: {name} must be contiguous {dtype} ({batch},) on {dev}")
    return v


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature=None, top_k=None, top_p=None,
           min_p=None, with_logprob: bool = False, out: torch.Tensor | None = None):
    """logits (B, V) f32 / bf16 / f16 with unit column stride, u (B) f32 in
    [0, 1).  Returns tokens (B) int32 [, log-probabilities (B) f32 of the
    tokens under the softmax of the logits as they are]; -1 for a row with
    nothing above -inf."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DT:
        raise ValueError("sample: logits (B, V) f32, bf16 or f16 on a CUDA device")
    B, V = logits.shape
    ld, unit = logits.stride()
    if unit != 1 and V > 1:
        raise ValueError("sample: logits with unit column stride")
    dev = logits.device
    f32 = torch.float32
    u = _setting(u, "u", f32, B, dev)
    # (held by name until the call is made: a number becomes a tensor here)
    t = None if temperature is None else _setting(temperature, "temperature", f32, B, dev)
    k = None if top_k is None else _setting(top_k, "top_k", torch.int32, B, dev)
    p = None if top_p is None else _setting(top_p, "top_p", f32, B, dev)
    m = None if min_p is None else _setting(min_p, "min_p", f32, B, dev)
    if out is None:
        out = u.new_empty(B, dtype=torch.int32)
    elif out.shape != (B,) or out.dtype != torch.int32 or out.device != dev or not out.is_contiguous():
        raise ValueError(f"sample: out must be contiguous int32 ({B},) on {dev}")
    logprob = u.new_empty(B) if with_logprob else None
    index = dev.index
    ctx = context(index)
    st = _abi.load().ffai_sample(
        ctx, logits.data_ptr(), ld if B > 1 else V, _DT[logits.dtype], B, V, u.data_ptr(),
        None if t is None else t.data_ptr(), None if k is None else k.data_ptr(),
        None if p is None else p.data_ptr(), None if m is None else m.data_ptr(), out.data_ptr(),
        None if logprob is None else logprob.data_ptr(), _raw_stream(index))
    if st:
        _check(st, ctx)
    return (out, logprob) if with_logprob else out


class Verified(NamedTuple):
    """What becomes of a step's drafts (verify): device tensors."""
    accepted: torch.Tensor  # (B,) int32 drafts of each request that stand
    next: torch.Tensor      # (B,) int32 the token behind them, -1: none
    tokens: torch.Tensor    # (T,) int32 both, at each request's first rows; -1 elsewhere
    logprobs: torch.Tensor | None  # (T,) f32 of those tokens, 0 elsewhere


def _logits(x: torch.Tensor, name: str):
    """Rows' stride of logits (T, V) with unit column stride."""
    if x.dim() != 2 or not x.is_cuda or x.dtype not in _DT:
        raise ValueError(f"verify: {name} (T, V) f32, bf16 or f16 on a CUDA device")
    ld, unit = x.stride()
    if unit != 1 and x.shape[1] > 1:
        raise ValueError(f"verify: {name} with unit column stride")
    return ld if x.shape[0] > 1 else x.shape[1]


def verify(logits: torch.Tensor, tokens: torch.Tensor, cu_rows: torch.Tensor, u: torch.Tensor,
           u_last: torch.Tensor, *, draft_logits=None, temperature=None, draft_temperature=None,
           with_logprob: bool = False) -> Verified:
    """Request b has the rows cu_rows[b] .. cu_rows[b + 1] (B + 1, int32): its
    last token and its drafts, `tokens` (T,) int32 being what was fed at each.
    The draft of row i + 1 is weighed by row i's logits (T, V) with u[i] (T,) f32
    in [0, 1): it stands if u q(x) < p(x).  q comes from row i of draft_logits
    (logits' shape and type; default: the drafts were given, q = 1).  Behind the
    last that stands, u_last[b] (B,) picks a token from what p leaves of q, or
    from p after the last row.  Temperatures as in `sample`, by request;
    draft_temperature is `temperature` unless given."""
    ld = _logits(logits, "logits")
    T, V = logits.shape
    dev = logits.device
    if draft_logits is not None:
        draft_ld = _logits(draft_logits, "draft_logits")
        if (draft_logits.shape != logits.shape or draft_logits.dtype is not logits.dtype
                or draft_logits.device != dev):
            raise ValueError("verify: draft_logits of logits' shape, type and device")
    B = u_last.numel()
    f32, i32 = torch.float32, torch.int32
    for v, name, dtype, n in ((tokens, "tokens", i32, T), (cu_rows, "cu_rows", i32, B + 1),
                              (u, "u", f32, T), (u_last, "u_last", f32, B)):
        if (v.dtype is not dtype or v.dim() != 1 or v.numel() != n or v.device != dev
                or not v.is_contiguous()):
            raise ValueError(f"verify: {name} must be contiguous {dtype} ({n},) on {dev}")
    t = None if temperature is None else _setting(temperature, "temperature", f32, B, dev)
    d = t if draft_temperature is None else _setting(draft_temperature, "draft_temperature", f32, B, dev)
    buf = tokens.new_empty(2 * B + T)
    at = buf.data_ptr()
    logprobs = u.new_empty(T) if with_logprob else None
    index = dev.index
    ctx = context(index)
    st = _abi.load().ffai_verify(
        ctx, logits.data_ptr(), ld, None if draft_logits is None else draft_logits.data_ptr(),
        0 if draft_logits is None else draft_ld, _DT[logits.dtype], B, T, V, cu_rows.data_ptr(),
        tokens.data_ptr(), u.data_ptr(), u_last.data_ptr(), None if t is None else t.data_ptr(),
        None if d is None else d.data_ptr(), at, at + 4 * B, at + 8 * B,
        None if logprobs is None else logprobs.data_ptr(), _raw_stream(index))
    if st:
        _check(st, ctx)
    return Verified(*buf.unsafe_split_with_sizes((B, B, T)), logprobs)
