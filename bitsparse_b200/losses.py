"""Log probabilities of given tokens, with entropy and top alternatives.

``token_logprobs`` reads the logits once in their own type -- no fp32 copy, no
materialised softmax -- and its backward writes their gradient in one more
pass.  ``-token_logprobs(...).logprobs.sum()`` is the summed cross entropy.
The kernels are in csrc/logprobs.cu.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from . import _runtime as R

MAX_TOP = 64
_TYPES = {torch.bfloat16: _lib.BS_BF16, torch.float32: _lib.BS_F32}


class TokenLogprobs(NamedTuple):
    logprobs: Tensor                    # [...] fp32: log p(target)
    entropy: Tensor                     # [...] fp32
    top_logprobs: Tensor | None = None  # [..., top] fp32, best first (not differentiable)
    top_indices: Tensor | None = None   # [..., top] int64


def _rows(t: Tensor, V: int) -> tuple[Tensor, int]:
    """(`t` or a copy, row stride): rows of V with unit column stride."""
    if t.is_contiguous():
        return t, V
    t = t.reshape(-1, V)
    if (V > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < V):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else V


def _forward(logits, targets, top, temperature, ignore, save):
    lead, V, dev = targets.shape, logits.shape[-1], logits.device
    n = targets.numel()
    lp = targets.new_empty(lead, dtype=torch.float32)
    ent = torch.empty_like(lp)
    stats = lp.new_empty((n, 2)) if save else None
    top_lp = top_ix = None
    if top:
        top_lp = lp.new_empty((*lead, top))
        top_ix = torch.empty_like(top_lp, dtype=torch.int64)
    x, ld = _rows(logits, V)
    if n:
        R.launch(dev, "bs_token_logprobs", x.data_ptr(), _TYPES[x.dtype], n, V, ld,
                 targets.data_ptr(), ignore, temperature, top, lp.data_ptr(), ent.data_ptr(),
                 R.ptr(top_lp), R.ptr(top_ix), R.ptr(stats), R.status_word(dev).data_ptr(),
                 R.stream_handle(dev))
    return lp, ent, top_lp, top_ix, stats, x


def _grads(ctx, d_lp, d_ent, *_):
    logits, targets, ent, stats = ctx.saved_tensors
    n, V, dt, dev = targets.numel(), ctx.shape[-1], logits.dtype, logits.device
    d = torch.empty_like(logits) if logits.shape == ctx.shape and logits.is_contiguous() else \
        logits.new_empty(ctx.shape)
    if n:
        d_lp = None if d_lp is None else d_lp.contiguous()
        d_ent = None if d_ent is None else d_ent.contiguous()
        x, ld = _rows(logits, V)
        R.launch(dev, "bs_token_logprobs_backward", x.data_ptr(), _TYPES[dt], n, V, ld,
                 targets.data_ptr(), ctx.ignore, ctx.temperature, stats.data_ptr(),
                 ent.data_ptr(), R.ptr(d_lp), R.ptr(d_ent), d.data_ptr(), V,
                 R.stream_handle(dev))
    return d, None, None, None, None


_grads_once = once_differentiable(_grads)


class _TokenLogprobs(Function):
    @staticmethod
    def forward(ctx, logits, targets, top, temperature, ignore):
        lp, ent, top_lp, top_ix, stats, x = _forward(logits, targets, top, temperature, ignore,
                                                     True)
        ctx.set_materialize_grads(False)
        ctx.temperature, ctx.ignore, ctx.shape = temperature, ignore, logits.shape
        ctx.save_for_backward(x, targets, ent, stats)
        if top:
            ctx.mark_non_differentiable(top_lp, top_ix)
            return lp, ent, top_lp, top_ix
        return lp, ent

    @staticmethod
    def backward(ctx, *grads):
        # the wrapper is for a graph of the gradients alone
        return (_grads_once if torch.is_grad_enabled() else _grads)(ctx, *grads)


def token_logprobs(logits: Tensor, targets: Tensor, *, top: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of `targets` [...] under softmax(logits / temperature),
    the distribution's entropy and its `top` most likely tokens.

    logits [..., V] bf16 or fp32; targets int64 or int32.  Equal logits are
    ordered by the lowest index.  Positions whose target is ``ignore_index``
    are not read: 0, indices -1, no gradient.  Where every logit is -inf, log
    probabilities are -inf and the entropy 0; where one is NaN or +inf, all is
    NaN.  A target outside the vocabulary gives NaN and no gradient, and
    ``check_status()`` reports it.  Rows may have any one stride; rows that have
    none, as those of a batch's ``logits[:, :-1]``, are copied first (to ignore
    each sequence's last position instead reads the logits where they are).
    """
    R.require_cuda(logits, "logits")
    if logits.dtype not in _TYPES:
        raise TypeError(f"logits must be bfloat16 or float32, not {logits.dtype}")
    if logits.dim() == 0 or logits.shape[-1] == 0 or logits.shape[:-1] != targets.shape:
        raise ValueError(f"logits [..., V] and targets [...] do not fit: {tuple(logits.shape)} "
                         f"and {tuple(targets.shape)}")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, not {targets.dtype}")
    if targets.device != logits.device:
        raise RuntimeError(f"targets must be on {logits.device}")
    V = logits.shape[-1]
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must lie in 0..{min(MAX_TOP, V)}, not {top}")
    if not 1e-10 <= temperature <= 1e10:
        raise ValueError("temperature must be positive (1e-10 to 1e10)")
    R.refuse_tangents(logits)
    t = targets.to(torch.int64).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, t, top, float(temperature),
                                                   int(ignore_index)))
    return TokenLogprobs(*_forward(logits, t, top, float(temperature), int(ignore_index),
                                   False)[:4])
