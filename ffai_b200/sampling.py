"""Sampling of one token per row of logits on the device: temperature, top-k,
top-p and min-p from given uniform numbers (ffai_sample).

    tokens = sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)

The settings are per row (device tensors), one number for all rows, or None
for off.  Equal inputs give equal tokens: weights are whole numbers, so every
sum is exact.  No reference counterpart: the reference's decoder takes the
largest logit on the host.
"""

from __future__ import annotations

import torch

from . import _abi
from .attention import _DT, _check, _ptr, _stream, context


def _setting(v, name: str, dtype: torch.dtype, batch: int, dev: torch.device):
    if v is None:
        return None
    if not isinstance(v, torch.Tensor):
        return torch.full((batch,), v, dtype=dtype, device=dev)
    if v.dtype != dtype or v.shape != (batch,) or v.device != dev or not v.is_contiguous():
        raise ValueError(f"sample: {name} must be contiguous {dtype} ({batch},) on {dev}")
    return v


def sample(logits: torch.Tensor, u: torch.Tensor, *, temperature=None, top_k=None, top_p=None,
           min_p=None, with_logprob: bool = False, out: torch.Tensor | None = None):
    """logits (B, V) f32 / bf16 / f16 with unit column stride, u (B) f32 in
    [0, 1).  Returns tokens (B) int32 [, log-probabilities (B) f32 of the
    tokens under the softmax of the logits as they are]; -1 for a row with
    nothing above -inf."""
    if logits.dim() != 2 or logits.device.type != "cuda" or logits.dtype not in _DT:
        raise ValueError("sample: logits (B, V) f32, bf16 or f16 on a CUDA device")
    B, V = logits.shape
    if logits.stride(1) != 1 and V > 1:
        raise ValueError("sample: logits with unit column stride")
    dev = logits.device
    u = _setting(u, "u", torch.float32, B, dev)
    temperature = _setting(temperature, "temperature", torch.float32, B, dev)
    top_k = _setting(top_k, "top_k", torch.int32, B, dev)
    top_p = _setting(top_p, "top_p", torch.float32, B, dev)
    min_p = _setting(min_p, "min_p", torch.float32, B, dev)
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=dev)
    elif out.shape != (B,) or out.dtype != torch.int32 or out.device != dev or not out.is_contiguous():
        raise ValueError(f"sample: out must be contiguous int32 ({B},) on {dev}")
    logprob = torch.empty(B, dtype=torch.float32, device=dev) if with_logprob else None
    ctx = context(dev.index)
    st = _abi.load().ffai_sample(ctx, _ptr(logits), logits.stride(0) if B > 1 else V,
                                 _DT[logits.dtype], B, V, _ptr(u), _ptr(temperature), _ptr(top_k),
                                 _ptr(top_p), _ptr(min_p), _ptr(out), _ptr(logprob), _stream(dev))
    _check(st, ctx)
    return (out, logprob) if with_logprob else out
