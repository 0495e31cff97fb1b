"""The norm of a model's gradients taken as one vector, and their clipping to a limit (no counterpart in the reference)."""

from __future__ import annotations

import math
from collections.abc import Iterable

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _dense(t: torch.Tensor) -> bool:
    """The elements fill a range of memory, each its own place."""
    step = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != step:
            return False
        step *= size
    return True


def _check(name: str, grads: list[torch.Tensor], in_place: bool, memory: bool) -> None:
    """`memory`: the tensors have some, whose places are compared."""
    for g in grads:
        assert g.dtype in _TYPES
        assert g.device == grads[0].device
        if in_place and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
            raise ValueError(f"{name}: an expanded tensor cannot be clipped in place")
    _native._require_cuda(*grads)
    if in_place and memory:
        ranges = sorted((g.data_ptr(), g.data_ptr() + g.numel() * g.element_size()) for g in grads if g.numel() and _dense(g))
        if any(first[1] > second[0] for first, second in zip(ranges, ranges[1:])):
            raise ValueError(f"{name}: gradients that share memory cannot be clipped in place")


def _checked(name: str, grads: torch.Tensor | Iterable[torch.Tensor | None], norm_type: float, in_place: bool) -> tuple[list[torch.Tensor], bool]:
    grads = [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]
    if norm_type not in (2, math.inf):
        raise ValueError(f"{name}: norm_type is 2 or infinity, got {norm_type!r}")
    if in_place:
        for g in grads:
            if g.requires_grad:
                raise ValueError(f"{name}: a gradient that requires a gradient itself cannot be clipped in place")
            if not torch.compiler.is_compiling() and unpack_dual(g).tangent is not None:
                raise ValueError(f"{name}: a gradient with a forward-mode tangent cannot be clipped in place")
    _check(name, grads, in_place, not torch.compiler.is_compiling())
    return grads, norm_type != 2


def clip_grad_norm_(grads: torch.Tensor | Iterable[torch.Tensor | None], max_norm: float, *, norm_type: float = 2.0) -> torch.Tensor:
    """Scale the CUDA tensors `grads` in place so that their common norm is at most `max_norm`; returns that norm as it was.

    The norm is that of all elements of all tensors taken as one vector: the root of the sum of squares, or with `norm_type=math.inf`
    the largest magnitude.  Every element is multiplied by min(1, max_norm / (norm + 1e-6)); where that is 1 nothing is written.
    The tensors are float32, bfloat16 or float16, mixed as they come, of any number, shape and alignment (dense ones in
    place, views with gaps through a copy); None and empty ones are skipped.  They may not share memory, require a gradient or
    have a forward-mode tangent.  The sum of squares is held in 64 bits and added in a fixed order.  The result is a float32 tensor of no dimensions on the same device: nothing is waited for.  A NaN or an
    infinity among the gradients makes it NaN or infinite, and the gradients NaN or (but for the infinite ones) zero."""
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm is not negative, got {max_norm!r}")
    max_norm, norm_type = float(max_norm), float(norm_type)
    if not torch.compiler.is_compiling():
        out = _native.HOST.clip_grad_norm(grads, max_norm, norm_type, True)  # None: not an ordinary call
        if out is not None:
            return out
    grads, largest = _checked("clip_grad_norm_", grads, norm_type, True)
    impl = _native.clip_grad_norm_op if torch.compiler.is_compiling() else _native._clip_grad_norm_impl
    return impl(grads, max_norm, largest)


def grad_norm(grads: torch.Tensor | Iterable[torch.Tensor | None], *, norm_type: float = 2.0) -> torch.Tensor:
    """The norm that `clip_grad_norm_` returns, and nothing else.  It carries no graph: it is not differentiable."""
    norm_type = float(norm_type)
    if not torch.compiler.is_compiling():
        out = _native.HOST.clip_grad_norm(grads, 0.0, norm_type, False)
        if out is not None:
            return out
    grads, largest = _checked("grad_norm", grads, norm_type, False)
    impl = _native.grad_norm_op if torch.compiler.is_compiling() else _native._grad_norm_impl
    return impl(grads, largest)
