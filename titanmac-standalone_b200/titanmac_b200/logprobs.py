"""What rows of logits say of tokens: their log-probabilities, the entropy, the most likely alternatives (``tmw_token_logprobs``).

The model's own loss is the mean of the first with the opposite sign; here every token's value is kept, and all three can be
trained on.
"""

from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

_DESC = struct.Struct("@6iQ2q6Q")  # tmw_logprobs_desc
_STRIDES = struct.Struct("@2q")
MAX_TOP = 32


class TokenLogprobs(NamedTuple):
    """``logprobs`` and ``entropy`` of the shape of the targets, ``top_ids`` (int64) and ``top_logprobs`` with one more axis of the
    alternatives, the most likely first and the lower id first among equals (None without alternatives).  fp32."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def _rows(t: torch.Tensor):
    """``(tensor with the same values, batch, tokens, strides)`` of ``[.., V]``: rows in two steps, one behind the other inside."""
    shape, strides = t.shape, t.stride()
    if (strides[-1] != 1 and shape[-1] != 1) or len(shape) > 3:
        t = t.contiguous()
        strides = t.stride()
    if len(shape) == 3:
        return t, shape[0], shape[1], strides[0], strides[1]
    if len(shape) == 2:
        return t, shape[0], 1, strides[0], 0
    return t, t.numel() // shape[-1], 1, shape[-1], 0


def _forward(logits: torch.Tensor, targets: torch.Tensor, n_top: int, with_lse: bool):
    """``(logprobs, entropy, top_ids, top_logprobs, lse)``; without alternatives the ids and their values are None."""
    device, shape = logits.device, targets.shape
    logprobs = torch.empty_like(targets, dtype=torch.float32)
    entropy = torch.empty_like(logprobs)
    lse = torch.empty(*shape, 2, dtype=torch.float32, device=device) if with_lse else None
    top_ids = top_logprobs = None
    if n_top:
        top_ids = torch.empty(*shape, n_top, dtype=torch.int64, device=device)
        top_logprobs = torch.empty_like(top_ids, dtype=torch.float32)
    if targets.numel():
        t, batch, tokens, s0, s1 = _rows(logits)
        desc = _DESC.pack(_native._DTYPES[t.dtype], batch, tokens, t.shape[-1], n_top, 0, t.data_ptr(), s0, s1, targets.data_ptr(),
                          logprobs.data_ptr(), entropy.data_ptr(), lse.data_ptr() if with_lse else 0,
                          top_logprobs.data_ptr() if n_top else 0, top_ids.data_ptr() if n_top else 0)
        _native.launch(t.get_device(), _native.lib().tmw_token_logprobs, desc)
    return logprobs, entropy, top_ids, top_logprobs, lse


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, targets: torch.Tensor, n_top: int):
        logprobs, entropy, top_ids, top_logprobs, lse = _forward(logits, targets, n_top, True)
        ctx.set_materialize_grads(False)
        if n_top:
            ctx.mark_non_differentiable(top_ids)
        ctx.save_for_backward(logits, targets, lse, entropy, top_ids)
        return logprobs, entropy, top_ids, top_logprobs

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprobs, d_entropy, _, d_top):
        logits, targets, lse, entropy, top_ids = ctx.saved_tensors
        device = logits.device
        d_logits = torch.empty(*logits.shape, dtype=logits.dtype, device=device)
        given = [None if g is None else g.contiguous() for g in (d_logprobs, d_entropy, d_top)]
        if targets.numel():
            t, batch, tokens, s0, s1 = _rows(logits)
            n_top = 0 if top_ids is None else top_ids.shape[-1]
            desc = _DESC.pack(_native._DTYPES[t.dtype], batch, tokens, t.shape[-1], n_top, 0, t.data_ptr(), s0, s1, targets.data_ptr(),
                              0, entropy.data_ptr(), lse.data_ptr(), 0, top_ids.data_ptr() if n_top else 0)
            _native.launch(t.get_device(), _native.lib().tmw_token_logprobs_backward, desc,
                           *[None if g is None else g.data_ptr() for g in given], d_logits.data_ptr(),
                           _STRIDES.pack(*_rows(d_logits)[3:]))
        return d_logits, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, n_top: int = 0) -> TokenLogprobs:
    """Log-probabilities of ``targets [..]`` (int64) under ``logits [.., V]``, the entropy of every row, and its ``n_top`` (at most
    32) most likely ids.  Differentiable in the logits, backwards and once; a forward-mode derivative is refused.

    A target of -100 counts as none: its value is 0 and no gradient comes from it.  A target outside the vocabulary has NaN and
    ``_native.poll_status`` raises.  A row without a distribution (a NaN, +inf or nothing but -inf among its logits) has NaN, and
    ids of -1."""
    if not logits.is_cuda or targets.get_device() != logits.get_device():
        _native._require_cuda(logits, targets)
        raise ValueError("token_logprobs: logits and targets must be on one device")
    if logits.dtype not in _native._DTYPES or targets.dtype is not torch.int64:
        raise TypeError("token_logprobs: logits in fp32, bf16 or fp16 and targets in int64 expected")
    shape = logits.shape
    if not shape or shape[:-1] != targets.shape or shape[-1] == 0:
        raise ValueError("token_logprobs: logits [.., vocabulary] and targets [..] must agree in the axes in front")
    if not 0 <= n_top <= min(MAX_TOP, shape[-1]):
        raise ValueError(f"token_logprobs: n_top must be in 0 .. {min(MAX_TOP, shape[-1])}, got {n_top}")
    _native.refuse_tangents("token_logprobs", logits)
    targets = targets.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, n_top))
    return TokenLogprobs(*_forward(logits, targets, n_top, False)[:4])
