"""GPU: clip_grad_norm_ at the ends of the range of 32-bit numbers, and on tensors that it cannot clip."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fw

import triturus_b200 as tb
from test_clip_grad_norm_gpu import BF16, F32, LAST, U, norm_of, some

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("numbers", [1000, 40_000, 900_001])
@pytest.mark.parametrize("limit", [1.0, 1e-3, 1e-9, 1e-20])
def test_factors_below_the_least_normal_number(numbers, limit, norm_type):
    """The factor is limit / norm whatever its size: 16 u of each element, as for others, and what a result below the least normal
    number (2^-126 = 1.2e-38) loses."""
    for scale in (1e36, 3e37):
        for kinds in ((F32,), (F32, BF16)):
            grads = [some((numbers,), kind, i, scale) for i, kind in enumerate(kinds)]
            want = norm_of(grads, norm_type)
            before = [g.double().cpu() for g in grads]
            tb.clip_grad_norm_(grads, limit, norm_type=norm_type)
            for g, b in zip(grads, before):
                target = b * (limit / (want + 1e-6))
                assert bool(((g.double().cpu() - target).abs() <= (16 * U + LAST[g.dtype]) * target.abs() + 2.0**-126).all())


def test_tangents_are_refused():
    """A tensor is scaled in place with its tangent only by a derivative that there is not."""
    with fw.dual_level():
        dual = fw.make_dual(some((30,), F32, 1), some((30,), F32, 2))
        kept = dual.clone()
        for form in ([dual], (some((4,), F32, 3), dual), iter([dual.view(5, 6)])):
            with pytest.raises(ValueError, match="tangent"):
                tb.clip_grad_norm_(form, 0.1)
        assert torch.equal(dual, kept)
        tb.clip_grad_norm_([some((30,), F32, 1)], 0.1)
