"""Global gradient norm and clipping, between `backward()` (and `distributed.all_reduce_gradients`) and
`optimizer.step()` (the place of /root/reference/3D-Reconstruction-main/models/trainers/base.py:502-516): two launches over
all tensors instead of several per tensor.

    loss.backward()
    norm = clip_grad_norm(params, max_norm=1.0)
    optimizer.step()

The norm is a 64-bit sum in an order that the sizes alone fix: ranks that hold equal gradients get equal bits.
"""
from __future__ import annotations

from ctypes import c_int32, c_int64, c_void_p
from typing import Iterable, List, Sequence, Tuple

import torch
from torch import Tensor

from . import _backend as B

EPS = 1.0e-6  # added to the norm that max_norm is divided by


def _tables(src: Sequence[Tensor], dst: Sequence[Tensor]):
    n = len(src)
    return ((c_void_p * n)(*[t.data_ptr() for t in src]), (c_void_p * n)(*[t.data_ptr() for t in dst]),
            (c_int64 * n)(*[t.numel() for t in src]), (c_int32 * n)(*[B.dtype_code(t) for t in src]))


def _dense(t: Tensor) -> bool:
    """Whether the tensor's values fill its memory without gaps or overlaps, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    expect = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda d: d[1]):
        if stride != expect:
            return False
        expect *= size
    return True


def _check(grads: Sequence[Tensor]) -> torch.device:
    for t in grads:
        if t.layout != torch.strided:
            raise TypeError("gsplat (MI355X build): dense gradients expected, got a sparse one")
    return B.require_gpu(*grads)


def _workspace(n: int, dev: torch.device) -> Tuple[Tensor, int]:
    nbytes = int(B.lib().gs_grad_norm_workspace_bytes(n))
    return torch.empty(nbytes // 8, device=dev, dtype=torch.float64), nbytes


def grad_norm(grads: Iterable[Tensor]) -> Tensor:
    """sqrt of the sum of squares over all tensors (fp32, bf16 and fp16, any mix) as a 0-d fp32 tensor on their device."""
    grads = [g.detach() for g in grads]
    dev = _check(grads)
    src = [g if _dense(g) else g.contiguous() for g in grads]
    norm = torch.empty((), device=dev, dtype=torch.float32)
    ws, nbytes = _workspace(len(src), dev)
    ps, _, pn, pt = _tables(src, src)
    with B.device_guard(dev), B.timed("gs_grad_norm", dev):
        B.check(B.lib().gs_grad_norm(len(src), ps, pn, pt, B.ptr(ws), nbytes, B.ptr(norm), B.stream_handle(dev)),
                "gs_grad_norm")
    return norm


def clip_gradients(grads: Iterable[Tensor], max_norm: float, inplace: bool = False,
                   error_if_nonfinite: bool = False) -> Tuple[List[Tensor], Tensor]:
    """Scales the gradients by `min(1, max_norm / (norm + 1e-6))`, `norm` being the one over all of them.  Returns (the
    scaled gradients, norm as a 0-d fp32 tensor): new tensors, or with `inplace` the same ones, which are neither read a
    second time nor written when the norm is within `max_norm`.  A NaN norm makes every gradient NaN and an infinite one
    makes the finite ones 0; `error_if_nonfinite` raises instead, before anything is changed (one host synchronisation and
    one more read of the gradients).  No two gradients may share memory when they are scaled in place."""
    grads = list(grads)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    if not grads:
        raise ValueError("no gradients given")
    with torch.no_grad():
        raw = [g.detach() for g in grads]
        dev = _check(raw)
        if error_if_nonfinite and not bool(torch.isfinite(grad_norm(raw))):
            raise RuntimeError("the total norm of the gradients is not finite: they are left as they are")
        if inplace and any(st == 0 and n > 1 for g in raw for n, st in zip(g.shape, g.stride())):
            raise ValueError("a gradient whose values share memory (an expanded one) cannot be scaled in place")
        src = [g if _dense(g) else g.contiguous() for g in raw]
        dst = src if inplace else [torch.empty_like(g) for g in src]
        norm = torch.empty((), device=dev, dtype=torch.float32)
        ws, nbytes = _workspace(len(src), dev)
        ps, pd, pn, pt = _tables(src, dst)
        with B.device_guard(dev), B.timed("gs_grad_clip", dev):
            B.check(B.lib().gs_grad_clip(len(src), ps, pd, pn, pt, max_norm, EPS, B.ptr(ws), nbytes, B.ptr(norm),
                                         B.stream_handle(dev)), "gs_grad_clip")
        if not inplace:
            return dst, norm
        for r, s in zip(raw, src):
            if s is not r:
                r.copy_(s)
    torch.autograd.graph.increment_version(grads)  # written behind autograd's back
    return grads, norm


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
