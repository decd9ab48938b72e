"""Norms around a block, fused with its gate and the residual join.

``residual_norm`` takes a block's output into the residual stream and
normalises the stream for the next block in one pass:

    u = rms_norm(y) * post_weight     (post_norm) or y
    stream = skip_scale * x + branch_scale * act(gate) * u
    normed = rms_norm(stream) * weight

with ``rms_norm(v) = v / sqrt(mean(v^2) + eps)``.  Both outputs are
differentiable in x, y, both weights and the gate.  ``rms_norm`` is the norm
alone (before a first block).  The kernels are in csrc/norm.cu; arithmetic is
fp32 whatever the types, and every output is rounded once.
"""
from __future__ import annotations

import functools
import math

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from . import _runtime as R

_ACTS = {"none": 0, "sigmoid": 1}
_TYPES = {torch.bfloat16: _lib.BS_BF16, torch.float32: _lib.BS_F32}


def _rows(t: Tensor, D: int) -> tuple[Tensor, int]:
    """(`t` or a copy, row stride): rows of D with unit column stride."""
    if t.is_contiguous():
        return t, D
    t = t.reshape(-1, D)
    if (D > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < D):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else D


def _param(t: Tensor | None, name: str, device, D: int) -> Tensor | None:
    if t is None:
        return None
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be bfloat16 or float32, not {t.dtype}")
    if t.shape != (D,):
        raise ValueError(f"{name} must have shape ({D},), not {tuple(t.shape)}")
    return t.contiguous()


@functools.lru_cache(maxsize=256)
def _gate_rows(gate: torch.Size, lead: torch.Size, D: int) -> tuple[int, bool]:
    """(rows of y that share a row of a gate of this shape, whether it has D columns)."""
    shape = tuple(gate) or (1,)
    wide = shape[-1] == D and D > 1
    if not wide and shape[-1] != 1:
        raise ValueError(f"gate must have {D} columns or one, not {shape[-1]}")
    own = shape[:-1]
    if len(own) > len(lead):
        raise ValueError(f"gate of shape {tuple(gate)} has more dimensions than y")
    own = (1,) * (len(lead) - len(own)) + own
    shared = False  # once a dimension is broadcast, the ones after it have to be
    for g, n in zip(own, lead):
        if g != n and g != 1 or shared and g != 1:
            raise ValueError(f"gate of shape {tuple(gate)} must be given for leading dimensions "
                             f"of {tuple(lead) + (D,)} and broadcast over the rest")
        shared = shared or g != n
    return math.prod(lead) // max(1, math.prod(own)), wide


@functools.lru_cache(maxsize=256)
def _workspace_floats(index: int, *args) -> int:
    with torch.cuda.device(index):
        return _lib.load().bs_residual_norm_workspace_bytes(*args) // 4


def _forward(x, y, w, pw, gate, cfg, save):
    """(stream, normed) of x and y's shape, r_post, r_pre, and x and y as the
    rows that were read."""
    post, gate_rows, wide, act, skip, branch, eps, out_dtype = cfg
    shape, x_t, dev = x.shape, x.dtype, x.device
    D = shape[-1]
    T = x.numel() // D
    x, ldx = _rows(x, D)
    ldy = y_at = s_at = 0
    s = r = None
    r_at = rp_at = 0
    if y is not None:
        y, ldy = _rows(y, D)
        y_at = y.data_ptr()
        s = _new(x, shape, x_t)
        s_at = s.data_ptr()
    h = _new(x, shape, out_dtype)
    if save:
        r = x.new_empty(2 * T if post else T, dtype=torch.float32)
        r_at = r.data_ptr()
        rp_at = r_at + 4 * T if post else 0
    if T:
        R.launch(dev, "bs_residual_norm", x.data_ptr(), _TYPES[x_t], ldx, y_at,
                 _TYPES[out_dtype], ldy, T, D, *_at(w), post, *_at(pw), *_at(gate), gate_rows,
                 wide, act, skip, branch, eps, s_at, h.data_ptr(), rp_at, r_at,
                 R.status_word(dev).data_ptr(), R.stream_handle(dev))
    return s, h, r, x, y


def _new(like: Tensor, shape: torch.Size, dtype: torch.dtype) -> Tensor:
    """A contiguous tensor (by the cheapest call where `like` has its shape and type)."""
    if like.dtype == dtype and like.shape == shape and like.is_contiguous():
        return torch.empty_like(like)
    return like.new_empty(shape, dtype=dtype)


def _at(t: Tensor | None) -> tuple[int, int]:
    """(address, type code) of a parameter."""
    return (0, 0) if t is None else (t.data_ptr(), _TYPES[t.dtype])


def _backward(ds, dh, s, y, w, pw, gate, r, shape, cfg, wants):
    """Gradients (dx, dy, dw, dpw, dgate) of the wanted ones, None for others."""
    post, gate_rows, wide, act, skip, branch, eps, out_dtype = cfg
    D = shape[-1]
    T = r.numel() // 2 if post else r.numel()
    s_t, dev = s.dtype, s.device
    want_x, want_y, want_w, want_pw, want_gate = wants
    # without a norm or gate on the branch its gradient is the stream's, scaled
    shared = (want_x and want_y and not post and gate is None and skip == branch
              and s_t == out_dtype)
    dx = dy = dw = dpw = dgate = None
    dx_at = dy_at = 0
    if want_x:
        dx = _new(s, shape, s_t)
        dx_at = dx.data_ptr()
    if want_y and not shared:
        dy = _new(s, shape, out_dtype)
        dy_at = dy.data_ptr()
    if want_w:
        dw = torch.empty_like(w)
    if want_pw:
        dpw = torch.empty_like(pw)
    if want_gate:
        dgate = torch.empty_like(gate)
    if T == 0:
        for t in (dw, dpw, dgate):
            if t is not None:
                t.zero_()
        return dx, dx if shared else dy, dw, dpw, dgate
    n = _workspace_floats(dev.index, T, D, post, gate is not None, gate_rows, wide)
    ws = r.new_empty(n)
    s, lds = _rows(s, D)
    ldy = y_at = 0
    if y is not None:
        y, ldy = _rows(y, D)
        y_at = y.data_ptr()
    r_at = r.data_ptr()
    R.launch(dev, "bs_residual_norm_backward", 0 if ds is None else ds.data_ptr(),
             0 if dh is None else dh.data_ptr(), s.data_ptr(), _TYPES[s_t], lds, y_at,
             _TYPES[out_dtype], ldy, T, D, *_at(w), post, *_at(pw), *_at(gate), gate_rows, wide,
             act, skip, branch, eps, r_at + 4 * T if post else 0, r_at, dx_at, dy_at,
             R.ptr(dw), R.ptr(dpw), R.ptr(dgate), ws.data_ptr(), n * 4,
             R.status_word(dev).data_ptr(), R.stream_handle(dev))
    return dx, dx if shared else dy, dw, dpw, dgate


def _grads(ctx, *grads):
    s, y, w, pw, gate, r = ctx.saved_tensors
    ds, dh = grads if len(grads) == 2 else (None, grads[0])
    ds = None if ds is None else ds.contiguous()
    dh = None if dh is None else dh.contiguous()
    return (*_backward(ds, dh, s, y, w, pw, gate, r, ctx.shape, ctx.cfg,
                       ctx.needs_input_grad[:5]), None)


_grads_once = once_differentiable(_grads)


class _ResidualNorm(Function):
    @staticmethod
    def forward(ctx, x, y, w, pw, gate, cfg):
        s, h, r, x, y = _forward(x, y, w, pw, gate, cfg, True)
        ctx.cfg, ctx.shape = cfg, h.shape
        ctx.set_materialize_grads(False)
        # a norm or gate on the branch needs y, and the stream is formed again
        # from x and y.  Else the stream alone is kept, as it was stored: half the
        # memory and four arrays to read and write in place of five, for a bf16
        # weight's gradient 2.4e-3 off in 2-norm where its own rounding is 1.7e-3
        branch = cfg[0] or gate is not None
        ctx.save_for_backward(x if branch or y is None else s, y if branch else None, w, pw, gate,
                              r)
        return (s, h) if y is not None else h

    @staticmethod
    def backward(ctx, *grads):
        # the wrapper is for a graph of the gradients alone
        return (_grads_once if torch.is_grad_enabled() else _grads)(ctx, *grads)


def _check_eps(eps: float) -> float:
    if not eps > 0:
        raise ValueError("eps must be positive")
    return float(eps)


def residual_norm(x: Tensor, y: Tensor, weight: Tensor | None = None, *, post_norm: bool = False,
                  post_weight: Tensor | None = None, gate: Tensor | None = None,
                  gate_act: str = "none", skip_scale: float = 1.0, branch_scale: float = 1.0,
                  eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """Join a block's output `y` with the residual stream `x` and normalise.

    x, y [..., D]; x may be fp32 with bf16 y (a 32-bit residual stream), else
    both have one type (bf16 or fp32).  weight, post_weight [D] (bf16 or
    fp32; None: ones).  gate: shape broadcastable to y's with trailing
    dimensions broadcast -- a value for each element [..., D], token [..., 1],
    sequence and channel [B, 1, D], channel [D], or one scalar; ``gate_act``
    "none" or "sigmoid".  Returns (stream, normed): x's and y's type.
    """
    R.require_cuda(x, "x")
    shape, x_t, y_t, dev = x.shape, x.dtype, y.dtype, x.device
    if shape != y.shape or len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"x and y must have one shape [..., D], not {tuple(x.shape)} and "
                         f"{tuple(y.shape)}")
    if x_t not in _TYPES or y_t not in (x_t, torch.bfloat16):
        raise TypeError(f"x and y must be bfloat16 or float32 (or a float32 x with a bfloat16 "
                        f"y), not {x_t} and {y_t}")
    if y.device != dev:
        raise RuntimeError(f"y must be on {dev}")
    if gate_act not in _ACTS:
        raise ValueError(f"gate_act must be one of {sorted(_ACTS)}, not {gate_act!r}")
    if post_weight is not None and not post_norm:
        raise ValueError("post_weight needs post_norm=True")
    D = shape[-1]
    w = _param(weight, "weight", dev, D)
    pw = _param(post_weight, "post_weight", dev, D)
    gate_rows, wide = 1, False
    if gate is not None:
        if gate.device != dev:
            raise RuntimeError(f"gate must be on {dev}")
        if gate.dtype not in _TYPES:
            raise TypeError(f"gate must be bfloat16 or float32, not {gate.dtype}")
        gate_rows, wide = _gate_rows(gate.shape, shape[:-1], D)
        gate = gate.contiguous()
    R.refuse_tangents(x, y, w, pw, gate)
    cfg = (bool(post_norm), gate_rows, wide, _ACTS[gate_act], float(skip_scale),
           float(branch_scale), _check_eps(eps), y_t)
    if torch.is_grad_enabled() and (
            x.requires_grad or y.requires_grad or (w is not None and w.requires_grad)
            or (pw is not None and pw.requires_grad)
            or (gate is not None and gate.requires_grad)):
        return _ResidualNorm.apply(x, y, w, pw, gate, cfg)
    return _forward(x, y, w, pw, gate, cfg, False)[:2]


def rms_norm(x: Tensor, weight: Tensor | None = None, *, eps: float = 1e-6,
             dtype: torch.dtype | None = None) -> Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in
    `dtype` (default x's; bfloat16 from a float32 x is allowed)."""
    R.require_cuda(x, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must have shape [..., D], not {tuple(x.shape)}")
    dtype = x.dtype if dtype is None else dtype
    if x.dtype not in _TYPES or dtype not in (x.dtype, torch.bfloat16):
        raise TypeError(f"no norm of {x.dtype} in {dtype}")
    D = x.shape[-1]
    w = _param(weight, "weight", x.device, D)
    R.refuse_tangents(x, w)
    cfg = (False, 1, False, 0, 1.0, 1.0, _check_eps(eps), dtype)
    if torch.is_grad_enabled() and (x.requires_grad or (w is not None and w.requires_grad)):
        return _ResidualNorm.apply(x, None, w, None, None, cfg)
    return _forward(x, None, w, None, None, cfg, False)[1]
