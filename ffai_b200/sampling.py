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
