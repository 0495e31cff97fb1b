"""Layer norm with its gradients, for the networks that predict a circuit's weights (no counterpart in the reference)."""

from __future__ import annotations

import torch

from . import _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None) -> None:
    assert len(x.shape) >= 1
    assert x.dtype in _TYPES
    _check_weights("layer_norm", x, weight, bias)
    _native._require_cuda(x)


def _check_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None) -> None:
    assert len(x.shape) >= 1
    assert x.dtype in _TYPES
    assert dy.shape == x.shape and dy.dtype == x.dtype
    assert mean.shape == rstd.shape == x.shape[:-1]
    assert mean.dtype == rstd.dtype == torch.float32
    assert dy.device == x.device == mean.device == rstd.device
    _check_weights("layer_norm_backward", x, weight)
    _native._require_cuda(x)


def _check_weights(name: str, x: torch.Tensor, *weights: torch.Tensor | None) -> None:
    kinds = set()
    for t in weights:
        if t is not None:
            assert t.shape == x.shape[-1:]
            assert t.device == x.device
            kinds.add(t.dtype)
    assert len(kinds) <= 1
    assert kinds <= {x.dtype, torch.float32}
    if x.shape[-1] == 0:
        raise ValueError(f"{name}: rows of no elements are not supported")


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-5,
    return_stats: bool = False,
):
    """y = (x - mean) * rstd * weight + bias over the last dimension of a CUDA tensor x [..., D] in float32, bfloat16 or float16,
    with mean = sum(x) / D and rstd = 1 / sqrt(sum((x - mean)^2) / D + eps).

    weight and bias [D] are optional and float32 or of x's type, both the same.  The sums are in 32 bits whatever x's type; y has x's
    type and shape and is contiguous.  x may have any strides: rows of consecutive elements at one distance are read in
    place, other views are copied first.  `return_stats=True` returns (y, mean, rstd) with float32 statistics of shape x.shape[:-1],
    which `layer_norm_backward` takes.  y is differentiable in x, weight and bias, once and backwards; a tensor with a forward-mode
    tangent is refused."""
    if not torch.compiler.is_compiling() and not (
        torch.is_grad_enabled()
        and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad))
    ):
        out = _native.HOST.layer_norm(x, weight, bias, eps, return_stats)  # None: not an ordinary call
        if out is not None:
            return out
    _check(x, weight, bias)
    if torch.compiler.is_compiling():
        out = _native.layer_norm_op(x, weight, bias, float(eps))
    else:
        out = _LayerNorm.apply(x, weight, bias, float(eps))
    return out if return_stats else out[0]


def layer_norm_backward(
    dy: torch.Tensor,
    x: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor | None = None,
    *,
    weight_grad: bool = True,
    bias_grad: bool = True,
):
    """(dx, dweight, dbias) of `layer_norm` for the gradient dy of its result (x's shape and type) and the mean and rstd that it returned.

    With g = dy * weight and h = (x - mean) * rstd: dx = rstd * (g - sum(g) / D - h * sum(g * h) / D), dweight = sum over rows of dy * h,
    dbias = sum over rows of dy.  dx has x's type, the other two weight's (x's without a weight); they are None where `weight_grad` or
    `bias_grad` is False.  The sums are in 32 bits and added in a fixed order.  The results carry no graph."""
    if not torch.compiler.is_compiling():
        out = _native.HOST.layer_norm_backward(dy, x, mean, rstd, weight, weight_grad, bias_grad)
        if out is not None:
            return out
    _check_backward(dy, x, mean, rstd, weight)
    impl = _native.layer_norm_backward_op if torch.compiler.is_compiling() else _native._layer_norm_backward_impl
    dx, dweight, dbias = impl(dy, x, mean, rstd, weight, bool(weight_grad), bool(bias_grad))
    return dx, dweight if weight_grad else None, dbias if bias_grad else None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _native._layer_norm_impl(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_type = None if bias is None else bias.dtype
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _dmean, _drstd):
        return (*_gradients(ctx, dy, *ctx.saved_tensors, _native._layer_norm_backward_impl), None)


def _gradients(ctx, dy, x, mean, rstd, weight, impl):
    need_x, need_weight, need_bias = ctx.needs_input_grad[:3]
    wide = ctx.bias_type == torch.float32  # (a bias in 32 bits, without a weight to say so)
    dx, dweight, dbias = impl(dy, x, mean, rstd, weight, need_weight, need_bias, wide)
    return dx if need_x else None, dweight if need_weight else None, dbias if need_bias else None


def _setup_context(ctx, inputs, output):
    x, weight, bias, _eps = inputs
    _y, mean, rstd = output
    ctx.mark_non_differentiable(mean, rstd)
    ctx.save_for_backward(x, mean, rstd, weight)
    ctx.bias_type = None if bias is None else bias.dtype


def _op_backward(ctx, dy, _dmean, _drstd):
    return (*_gradients(ctx, dy, *ctx.saved_tensors, _native.layer_norm_backward_op), None)


_native.layer_norm_op.register_autograd(_op_backward, setup_context=_setup_context)
