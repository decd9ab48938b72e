"""Orthogonalised updates: the Newton-Schulz operator and the Muon optimiser.

``orthogonalize`` replaces a matrix (or a batch of equal ones) by one with the
same singular vectors and singular values near 1.  The products run on the
tensor cores with fp16 operands scaled by powers of two and fp32 accumulation
(csrc/orthogonal.cu).  ``Muon`` steps matrix parameters by the orthogonalised
momentum, all parameters of one shape in one batch.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Iterable, Sequence

import torch
from torch import Tensor

from . import _lib
from . import _runtime as R

# The quintic whose steps take singular values of (0, 1] near 1 fastest: its
# slope at 0 is large, at the price of a result in about [0.7, 1.2].
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 32


@functools.lru_cache(maxsize=64)
def _coefficients(coefficients: tuple, steps: int):
    """The C entry point's float[steps][3]."""
    if len(coefficients) == 3 and not any(isinstance(c, tuple) for c in coefficients):
        coefficients = (coefficients,) * steps
    if len(coefficients) != steps or any(len(c) != 3 for c in coefficients):
        raise ValueError("coefficients must be (a, b, c), or one such triple for each step")
    flat = [float(v) for c in coefficients for v in c]
    if not all(math.isfinite(v) for v in flat):
        raise ValueError("coefficients must be finite")
    return (ctypes.c_float * (3 * steps))(*flat)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, rows: int, cols: int) -> int:
    return int(_lib.load().bs_orthogonalize_workspace_bytes(batch, rows, cols))


def orthogonalize(update: Tensor, *, steps: int = 5,
                  coefficients: Sequence = COEFFICIENTS, eps: float = 1e-7) -> Tensor:
    """Newton-Schulz orthogonalisation of `update` [..., rows, cols].

    X = update / (its Frobenius norm + eps), then `steps` times
    X = a X + b (X X^T) X + c (X X^T)^2 X with ``coefficients`` (a, b, c), or
    one triple for each step.  bf16 or fp32 input, any row or batch stride;
    the result is a contiguous bf16 tensor.  Not differentiable.  A zero
    matrix stays zero.
    """
    R.require_cuda(update, "update")
    if update.dim() < 2:
        raise ValueError(f"update must be [..., rows, cols], not {tuple(update.shape)}")
    if update.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"update must be bfloat16 or float32, not {update.dtype}")
    steps = int(steps)
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"steps must lie in 1..{MAX_STEPS}, not {steps}")
    if not eps > 0:
        raise ValueError("eps must be positive")
    key = tuple(tuple(c) if isinstance(c, (list, tuple)) else c for c in coefficients)
    coef = _coefficients(key, steps)
    shape, dev = update.shape, update.device
    rows, cols = shape[-2:]
    out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    if out.numel() == 0:
        return out
    g = update.detach()
    if g.dim() != 3:
        g = g.reshape(-1, rows, cols)
    if (cols > 1 and g.stride(2) != 1) or (rows > 1 and g.stride(1) < cols):
        g = g.contiguous()
    batch = g.shape[0]
    ws = torch.empty(_workspace_bytes(batch, rows, cols), dtype=torch.uint8, device=dev)
    R.launch(dev, "bs_orthogonalize", g.data_ptr(), R.dtype_code(g.dtype), batch, rows, cols,
             g.stride(1) if rows > 1 else cols, g.stride(0) if batch > 1 else rows * cols, steps,
             ctypes.addressof(coef), eps, out.data_ptr(), ws.data_ptr(), ws.numel(),
             R.status_word(dev).data_ptr(), R.stream_handle(dev))
    return out


class Muon(torch.optim.Optimizer):
    """Momentum, orthogonalised: for each matrix parameter

        buf = momentum * buf + grad
        p -= lr * (scale * orthogonalize(grad + momentum * buf) + weight_decay * p)

    (without ``nesterov``: orthogonalize(buf)), scale = sqrt(max(1, rows /
    cols)).  Parameters (bf16 or fp32) of more dimensions are matrices of their
    first one by the rest.  For a model's matrices; embeddings, norms and biases
    belong to another optimiser.

    The state is fp32 whatever the parameters' type.  A bf16 parameter is the
    rounding of a fp32 value, and what that rounding left is kept beside the
    momentum (``remainder``): a decay or update far below a bf16 step adds up
    over the steps.  Where someone else changed a parameter in between, its
    remainder no longer belongs to it and is dropped.
    """

    def __init__(self, params: Iterable, lr: float = 0.02, momentum: float = 0.95,
                 nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 coefficients: Sequence = COEFFICIENTS):
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError("lr and weight_decay must not be negative, momentum in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)  # (makes the parameters a list)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError(f"Muon steps matrices; a parameter has {p.dim()} dimension(s)")

    def load_state_dict(self, state_dict):
        """The state is copied, in fp32: the base class would cast it to the
        parameters' type."""
        seen = []
        hook = self.register_load_state_dict_pre_hook(lambda _, d: seen.append(d))
        try:  # (the last hook of those that may have changed the dictionary)
            super().load_state_dict(state_dict)
        finally:
            hook.remove()
        state_dict = seen[-1]
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                for name in ("momentum_buffer", "remainder"):
                    value = state_dict["state"].get(key, {}).get(name)
                    if value is not None:
                        self.state[p][name] = value.to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []  # (group, matrices of one shape and type)
        for group in self.param_groups:
            same: dict = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    if p.dtype not in (torch.bfloat16, torch.float32):
                        raise TypeError(f"Muon steps bfloat16 or float32 parameters, not {p.dtype}")
                    rows = p.shape[0]
                    same.setdefault((rows, p.numel() // rows, p.dtype, p.device), []).append(p)
            work += [(group, params, key[0], key[1]) for key, params in same.items()]
        for args in work:
            self._step_shape(*args)
        return loss

    def _states(self, params, name):
        for p in params:
            if name not in self.state[p]:
                self.state[p][name] = torch.zeros_like(p, dtype=torch.float32)
        return [self.state[p][name] for p in params]

    def _step_shape(self, group, params, rows, cols):
        momentum, lr = group["momentum"], group["lr"]
        narrow = params[0].dtype != torch.float32

        def batch_of(tensors):
            return torch.stack([t.reshape(rows, cols) for t in tensors])

        def views(batch):
            return [t.view(p.shape) for t, p in zip(batch.unbind(), params)]

        grads = [p.grad for p in params]
        if narrow:
            batch = batch_of(grads).float()
            grads = views(batch)
        bufs = self._states(params, "momentum_buffer")
        torch._foreach_mul_(bufs, momentum)
        torch._foreach_add_(bufs, grads)
        if group["nesterov"] and narrow:
            torch._foreach_add_(grads, bufs, alpha=momentum)  # in the batch
        else:
            batch = batch_of(torch._foreach_add(grads, bufs, alpha=momentum)
                             if group["nesterov"] else bufs)
        o = orthogonalize(batch, steps=group["steps"], coefficients=group["coefficients"])
        decay, rate = 1 - lr * group["weight_decay"], -lr * max(1.0, rows / cols) ** 0.5
        if not narrow:
            if decay != 1:
                torch._foreach_mul_(params, decay)
            torch._foreach_add_(params, views(o.float()), alpha=rate)
            return
        rest = self._states(params, "remainder")
        own, values = batch_of(params), batch_of(rest)
        values.add_(own)  # what the parameters are the roundings of
        torch.where(values.to(own.dtype) == own, values, own, out=values)
        if decay != 1:
            values.mul_(decay)
        values.add_(o, alpha=rate)
        own.copy_(values)  # rounded once; the difference is exact
        torch._foreach_copy_(params, views(own))
        torch._foreach_copy_(rest, views(values.sub_(own)))
