"""Global gradient norm and clipping, between `backward()` (and `distributed.all_reduce_gradients`) and
`optimizer.step()` (the place of /root/reference/3D-Reconstruction-main/models/trainers/base.py:502-516): two launches over
all tensors instead of several per tensor.

    loss.backward()
    norm = clip_grad_norm(params, max_norm=1.0)
    optimizer.step()

The norm is a 64-bit sum in an order that sizes, layouts and alignment fix: ranks that hold equal gradients in equal
layouts get equal bits.
"""
from __future__ import annotations

from typing import Iterable, List, Tuple

import torch
from torch import Tensor

from . import _backend as B

EPS = 1.0e-6  # added to the norm that max_norm is divided by


def _listed(grads) -> List[Tensor]:
    return [grads] if isinstance(grads, Tensor) else list(grads)  # (a tensor is one gradient, not its rows)


def grad_norm(grads: Iterable[Tensor]) -> Tensor:
    """sqrt of the sum of squares over all tensors (fp32, bf16 and fp16, any mix) as a 0-d fp32 tensor on their device."""
    grads = _listed(grads)
    with B.timed("gs_grad_norm", grads[0].device if grads else None):
        return B.ops().grad_norm(grads)


def clip_gradients(grads: Iterable[Tensor], max_norm: float, inplace: bool = False,
                   error_if_nonfinite: bool = False) -> Tuple[List[Tensor], Tensor]:
    """Scales the gradients by `min(1, max_norm / (norm + 1e-6))`, `norm` being the one over all of them.  Returns (the
    scaled gradients, norm as a 0-d fp32 tensor): new tensors, or with `inplace` the same ones, which are neither read a
    second time nor written when the norm is within `max_norm` (views with gaps are, through a copy).  Small new tensors
    are pieces of one allocation, as those of `torch.split` are: `resize_` to more elements would reach into the next.  A
    NaN norm makes every gradient NaN, and so does an infinite one with an infinite `max_norm`; with a finite one it makes
    the finite values 0.  `error_if_nonfinite` raises instead, before anything is changed (one host synchronisation and one
    more read of the gradients).  No two gradients may share memory when they are scaled in place."""
    grads = _listed(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    if error_if_nonfinite and not bool(torch.isfinite(grad_norm(grads))):
        raise RuntimeError("the total norm of the gradients is not finite: they are left as they are")
    with B.timed("gs_grad_clip", grads[0].device if grads else None):
        scaled, norm = B.ops().clip(grads, max_norm, EPS, inplace)
    return (grads if inplace else scaled), norm


def clip_grad_norm(params: Iterable[Tensor], max_norm: float, error_if_nonfinite: bool = False) -> Tensor:
    """Scales `.grad` of every parameter that has one in place, as `clip_gradients(..., inplace=True)` does, and returns
    their norm (a 0-d fp32 tensor; 0 where no parameter has a gradient).  A parameter named twice counts once."""
    if isinstance(params, Tensor):
        params = [params]
    seen, grads, dev = set(), [], None
    for p in params:
        dev = p.device
        if p.grad is not None and id(p) not in seen:
            seen.add(id(p))
            grads.append(p.grad)
    if not grads:
        return torch.zeros((), device=dev)
    return clip_gradients(grads, max_norm, inplace=True, error_if_nonfinite=error_if_nonfinite)[1]
