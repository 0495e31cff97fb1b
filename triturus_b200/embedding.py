"""Rows of a table by symbol, with the table's gradient: how a network reads symbols (no counterpart in the reference)."""

from __future__ import annotations

import math

import torch

from . import _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_TOKENS = (torch.int64, torch.int32)


def _check(tokens: torch.Tensor, weight: torch.Tensor, scale: float, padding_idx: int | None) -> None:
    assert tokens.dtype in _TOKENS
    assert len(weight.shape) == 2
    assert weight.dtype in _TYPES
    assert tokens.device == weight.device
    _check_numbers("embedding", weight.shape[0], weight.shape[1], scale, padding_idx)
    _native._require_cuda(weight)


def _check_backward(dy: torch.Tensor, tokens: torch.Tensor, symbols: int, scale: float, padding_idx: int | None) -> None:
    assert tokens.dtype in _TOKENS
    assert len(dy.shape) >= 1 and dy.shape[:-1] == tokens.shape
    assert dy.dtype in _TYPES
    assert tokens.device == dy.device
    _check_numbers("embedding_backward", symbols, dy.shape[-1], scale, padding_idx)
    _native._require_cuda(dy)


def _check_numbers(name: str, symbols: int, width: int, scale: float, padding_idx: int | None) -> None:
    if not _native._whole(symbols):
        raise ValueError(f"{name}: symbols must be a whole number, got {symbols!r}")
    if symbols < 1 or width < 1:
        raise ValueError(f"{name}: a table of {symbols} rows of {width} elements is not supported")
    if not (math.isfinite(scale) and abs(scale) <= torch.finfo(torch.float32).max):
        raise ValueError(f"{name}: scale must be a finite number of 32 bits, got {scale!r}")
    if padding_idx is not None and not (_native._whole(padding_idx) and 0 <= padding_idx < symbols):
        raise ValueError(f"{name}: padding_idx is no symbol of the table, got {padding_idx!r}")


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[tokens]: the rows of a table `weight` [V, D] (float32, bfloat16 or float16) for the symbols of the CUDA tensor `tokens`
    [...] (int64 or int32), as a contiguous tensor [..., D] of weight's type.

    A symbol that is not in 0 ... V - 1 (a negative one is none that counts from the end) gives a row of NaN and has no gradient; nothing is
    read for it.  The product with a scale other than 1 is taken in 32 bits and rounded to weight's type.  weight may have any strides: rows of
    consecutive elements at one distance are read in place, other views are copied first.

    Differentiable in weight, once and backwards: the gradient is that of `embedding_backward`, where positions of the symbol `padding_idx`
    count as nothing.  A tensor with a forward-mode tangent is refused."""
    if not torch.compiler.is_compiling() and not (torch.is_grad_enabled() and weight.requires_grad):
        out = _native.HOST.embedding(tokens, weight, scale, padding_idx)  # None: not an ordinary call
        if out is not None:
            return out
    _check(tokens, weight, scale, padding_idx)
    if torch.compiler.is_compiling():
        return _native.embedding_op(tokens, weight, float(scale), padding_idx)
    return _Embedding.apply(tokens, weight, float(scale), padding_idx)


def embedding_backward(
    dy: torch.Tensor, tokens: torch.Tensor, symbols: int, *, scale: float = 1.0, padding_idx: int | None = None
) -> torch.Tensor:
    """The gradient [symbols, D] of the table of `embedding` for the gradient dy [..., D] of its result: row v is
    scale * sum of dy over the positions of symbol v, zero where there is none and for v = padding_idx.

    Of dy's type; the sums are in 32 bits, taken in an order that depends on `tokens` alone, so that the same call gives the same result.
    The positions are sorted by symbol on the device, or compared with each other where there are few.  The result carries no graph, and a tensor with a
    forward-mode tangent is refused."""
    if not torch.compiler.is_compiling():
        out = _native.HOST.embedding_backward(dy, tokens, symbols, scale, padding_idx)
        if out is not None:
            return out
    _check_backward(dy, tokens, symbols, scale, padding_idx)
    impl = _native.embedding_backward_op if torch.compiler.is_compiling() else _native._embedding_backward_impl
    return impl(dy, tokens, symbols, float(scale), padding_idx)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.args = weight.shape[0], scale, padding_idx
        return _native._embedding_impl(tokens, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return None, _native._embedding_backward_impl(dy, *ctx.saved_tensors, *ctx.args), None, None


def _setup_context(ctx, inputs, output):
    tokens, weight, scale, padding_idx = inputs
    ctx.save_for_backward(tokens)
    ctx.args = weight.shape[0], scale, padding_idx


def _op_backward(ctx, dy):
    return None, _native.embedding_backward_op(dy, *ctx.saved_tensors, *ctx.args), None, None


_native.embedding_op.register_autograd(_op_backward, setup_context=_setup_context)
