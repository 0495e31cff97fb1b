"""Cross entropy of a linear layer over many symbols, with its gradients: how a network that predicts symbols is trained (no counterpart
in the reference)."""

from __future__ import annotations

import torch

from . import _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_TARGETS = (torch.int64, torch.int32)
_REDUCTIONS = ("none", "mean", "sum")  # by their codes in the library


def _reduction(name: str, reduction: str) -> int:
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{name}: Unknown reduction {reduction!r} (expected 'none', 'mean' or 'sum')")
    return _REDUCTIONS.index(reduction)


def _check_code(reduction: int) -> None:
    if not 0 <= reduction < len(_REDUCTIONS):
        raise ValueError(f"linear_cross_entropy: Unknown reduction code {reduction!r}")


def _check_operands(name: str, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int) -> None:
    assert len(x.shape) >= 1
    assert len(weight.shape) == 2 and weight.shape[1] == x.shape[-1]
    assert x.dtype in _TYPES and weight.dtype == x.dtype
    assert target.shape == x.shape[:-1]
    assert target.dtype in _TARGETS
    assert x.device == weight.device == target.device
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{name}: a weight of {weight.shape[0]} rows of {weight.shape[1]} elements is not supported")
    if not (_native._whole(ignore_index) and -(2**63) <= ignore_index < 2**63):
        raise ValueError(f"{name}: ignore_index must be a whole number of 64 bits, got {ignore_index!r}")


def _check(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int) -> None:
    _check_operands("linear_cross_entropy", x, weight, target, ignore_index)
    _native._require_cuda(x)


def _check_backward(
    dloss: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, lse: torch.Tensor, reduction: int, ignore_index: int
) -> None:
    _check_operands("linear_cross_entropy_backward", x, weight, target, ignore_index)
    assert dloss.shape == (target.shape if reduction == 0 else ())
    assert lse.shape == target.shape
    assert dloss.dtype == lse.dtype == torch.float32
    assert dloss.device == lse.device == x.device
    _native._require_cuda(x)


def linear_cross_entropy(
    x: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    *,
    reduction: str = "mean",
    ignore_index: int = -100,
    return_lse: bool = False,
):
    """The cross entropy of the logits z = x weight^T against the symbols `target`, without the logits in memory:
    lse = log sum_v exp(z[..., v]), loss = lse - z[..., target].

    x [..., D] and weight [V, D] are CUDA tensors of one type, float32, bfloat16 or float16; target [...] is int64 or int32.  Positions whose target
    is `ignore_index` have no loss and no gradient; one whose target is no symbol otherwise has a loss and gradients of NaN.  The loss is float32:
    `reduction="none"` gives that of each position (0 for ignored ones), "sum" their sum and "mean" the sum over the number of positions that are not
    ignored, 0 where there is none.  `return_lse=True` returns (loss, lse) with the float32 lse of shape target.shape, which
    `linear_cross_entropy_backward` takes; -loss of "none" is the log-probability of the target.

    Products of 16-bit elements are exact and added in 32 bits.  float32 is taken apart into three bfloat16 parts, whose six largest products have about
    the accuracy of 32-bit arithmetic whatever `set_tf32_enabled` says; an infinity in float32 counts as NaN.  Logits may be as large as 32 bits
    hold, one of +infinity gives NaN, and symbols of -infinity have probability 0.

    x and weight may have any strides.  Rows of consecutive elements that do not overlap are read in place where they begin on 16-byte boundaries:
    of 16 bits, from 2048 positions on only on 128-byte ones, and weight of float32 with up to 192 positions.  Everything else is copied first,
    float32 (but for weight with so few positions) as its parts, of 6 bytes for an element.  The loss is differentiable in x and weight, once and backwards; lse is not.  A tensor with a forward-mode
    tangent is refused."""
    code = _reduction("linear_cross_entropy", reduction)
    if not torch.compiler.is_compiling() and not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):
        out = _native.HOST.linear_cross_entropy(x, weight, target, code, ignore_index, _native._status_address(x))  # None: not an ordinary call
        if out is not None:
            return out if return_lse else out[0]
    _check(x, weight, target, ignore_index)
    if torch.compiler.is_compiling():
        loss, lse = _native.linear_cross_entropy_op(x, weight, target, code, ignore_index)
    else:
        loss, lse = _LinearCrossEntropy.apply(x, weight, target, code, ignore_index)
    return (loss, lse) if return_lse else loss


def linear_cross_entropy_backward(
    dloss: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    lse: torch.Tensor,
    *,
    reduction: str = "mean",
    ignore_index: int = -100,
    x_grad: bool = True,
    weight_grad: bool = True,
):
    """(dx, dweight) of `linear_cross_entropy` for the gradient dloss of its result (float32, of its shape) and the lse that it returned.

    With g the share of dloss in each position (0 for ignored ones) and d = g (exp(z - lse) - [target]): dx = d weight, dweight = d^T x, of x's type;
    None where `x_grad` or `weight_grad` is False.  The logits are computed once more, for a piece of the symbols at a time, and d is rounded
    to 16 bits for its two products where x has 16, without what is common to all positions: in float16 relative to the largest finite |dloss|.
    Sums are in 32 bits in a fixed order.  The operands are read in place or copied as in the forward call, but x is copied whenever weight_grad is
    set (and has its room in the workspace in any case).

    What x holds in ignored positions does not count, NaN or not; dx is zero there, whatever weight holds.  An infinite element of weight makes its
    column of dx NaN in the other positions, 0 times infinity, also where it makes a symbol impossible (in float32, which counts it as NaN, all
    columns).  The results carry no graph, and tensors with a forward-mode tangent are refused."""
    code = _reduction("linear_cross_entropy_backward", reduction)
    if not torch.compiler.is_compiling():
        out = _native.HOST.linear_cross_entropy_backward(
            x, weight, target, dloss, lse, code, ignore_index, bool(x_grad), bool(weight_grad), _native._status_address(x)
        )
        if out is not None:
            return out
    _check_backward(dloss, x, weight, target, lse, code, ignore_index)
    impl = _native.linear_cross_entropy_backward_op if torch.compiler.is_compiling() else _native._linear_cross_entropy_backward_impl
    dx, dweight = impl(dloss, x, weight, target, lse, code, ignore_index, bool(x_grad), bool(weight_grad))
    return dx if x_grad else None, dweight if weight_grad else None


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, reduction, ignore_index):
        loss, lse = _native._linear_cross_entropy_impl(x, weight, target, reduction, ignore_index)
        ctx.save_for_backward(x, weight, target, lse)
        ctx.args = reduction, ignore_index
        ctx.mark_non_differentiable(lse)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, _dlse):
        return _gradients(ctx, dloss, _native._linear_cross_entropy_backward_impl)


def _gradients(ctx, dloss, impl):
    need_x, need_weight = ctx.needs_input_grad[:2]
    dx, dweight = impl(dloss, *ctx.saved_tensors, *ctx.args, need_x, need_weight)
    return dx if need_x else None, dweight if need_weight else None, None, None, None


def _setup_context(ctx, inputs, output):
    x, weight, target, reduction, ignore_index = inputs
    _loss, lse = output
    ctx.mark_non_differentiable(lse)
    ctx.save_for_backward(x, weight, target, lse)
    ctx.args = reduction, ignore_index


def _op_backward(ctx, dloss, _dlse):
    return _gradients(ctx, dloss, _native.linear_cross_entropy_backward_op)


_native.linear_cross_entropy_op.register_autograd(_op_backward, setup_context=_setup_context)
