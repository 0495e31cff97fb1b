"""Sampling of symbols from the log-probabilities that a circuit gives them (no counterpart in the reference)."""

from __future__ import annotations

import math

import torch

from . import _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(logits: torch.Tensor, noise: torch.Tensor, temperature, top_k, top_p, min_p) -> None:
    """The parameters as tensors, or anything else for numbers."""
    assert len(logits.shape) >= 1
    assert logits.dtype in _TYPES
    assert noise.shape == logits.shape
    assert noise.dtype == torch.float32
    assert noise.device == logits.device
    for value, kind in ((temperature, torch.float32), (top_k, torch.int32), (top_p, torch.float32), (min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            assert value.dtype == kind
            assert value.shape == logits.shape[:-1]
            assert value.device == logits.device


def _check_device(logits: torch.Tensor) -> None:
    _native._require_cuda(logits)
    if logits.shape[-1] == 0:
        raise ValueError("sample: rows of no symbols are not supported")


def _parameter(name: str, value, off, valid):
    """(tensor or None, number)"""
    if isinstance(value, torch.Tensor):
        return value, off
    if value is None:
        return None, off
    if not valid(value):
        raise ValueError(f"sample: {name} is out of range, got {value!r}")
    return None, type(off)(value)


def sample(
    logits: torch.Tensor,
    noise: torch.Tensor,
    *,
    temperature: float | torch.Tensor = 1.0,
    top_k: int | torch.Tensor | None = None,
    top_p: float | torch.Tensor | None = None,
    min_p: float | torch.Tensor | None = None,
    return_logprob: bool = False,
):
    """One symbol for each row of the CUDA tensor `logits` [..., V] (float32, bfloat16 or float16; log-probabilities or any others) from
    given random numbers: `noise` of the same shape in float32, positive and exponentially distributed
    (`torch.empty(shape, device="cuda").exponential_()`).  Returns int64 tokens of shape logits.shape[:-1].

    With p_i = exp((x_i - max x) / temperature), and the symbols in the order of falling x, equal ones by index, the filters keep in turn
      top_k: the first top_k;
      top_p: of these the fewest whose sum of p reaches top_p times theirs (the first in any case);
      min_p: of these the ones with p_i >= min_p, that is min_p times the probability of the most probable one.
    The token is the kept symbol with the largest p_i / noise_i (the lower index of equal ones): symbol i with probability
    p_i / sum of the p kept.  `return_logprob=True` returns (token, logprob) with the float32 logarithm of that probability.

    A parameter is a number, None (no filter) or a tensor of the rows' shape (float32, top_k int32), where a top_k below 1, a top_p of 1
    and a min_p of 0 are no filter.  A temperature of 0 (in a tensor: any that is not positive) gives the first of the largest
    logits with logprob 0.  Symbols of -inf are impossible and never given; a row of nothing else gives token -1 and logprob
    -inf, a row with a NaN -1 and NaN.  Infinity counts as the largest number.  logits and noise may have any strides: rows of consecutive elements
    at one distance are read in place, other views are copied first.  Only the noise of kept symbols counts, though that of others may be
    read.

    The same call gives the same result each time.  The number of rows decides how many blocks share one, and with that the order in which its p
    are added: in another batch a row's logprob may differ in its last bits, and its token where a sum is that close to top_p.  The results
    carry no graph: logprob is not differentiable."""
    if not torch.compiler.is_compiling():
        out = _native.HOST.sample(logits, noise, temperature, top_k, top_p, min_p, return_logprob)  # None: not an ordinary call
        if out is not None:
            return out
    _check(logits, noise, temperature, top_k, top_p, min_p)
    params = (
        *_parameter("temperature", temperature, 1.0, lambda v: 0.0 <= v < math.inf),
        *_parameter("top_k", top_k, 0, lambda v: 1 <= v == int(v)),
        *_parameter("top_p", top_p, 1.0, lambda v: 0.0 <= v <= 1.0),
        *_parameter("min_p", min_p, 0.0, lambda v: 0.0 <= v <= 1.0),
    )
    _check_device(logits)
    params = (*params[:3], min(params[3], 2**31 - 1), *params[4:])
    token, logprob = (_native.sample_op if torch.compiler.is_compiling() else _native._sample_impl)(logits, noise, *params)
    return (token, logprob) if return_logprob else token
