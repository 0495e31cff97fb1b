"""GPU: the end of what top_k and top_p keep, where it falls among symbols far below the others; against the definition of test_sample_gpu."""

import pytest
import torch

from test_sample_gpu import BF16, F32, check

pytestmark = pytest.mark.gpu

LEAST = -3.4028234663852886e38


def rows_of(first, last, symbols, some, kind, seed):
    """`some` symbols near `first` among ones of `last`."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((2, symbols), last)
    for row in x:
        row[torch.randperm(symbols, generator=g)[:some]] = first * (1 - 1e-3 * torch.rand(some, generator=g))
    return x.to(kind).cuda(), torch.empty(2, symbols).exponential_(generator=g).cuda()


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("last", [LEAST, -2e38, -1e5])
@pytest.mark.parametrize("first", [0.25, 1.0, 5.0, 16.0, 100.0])
def test_masks_of_the_least_number_at_high_temperatures(first, last, kind):
    """A range of keys from a positive value to one near the least number is more than half of all keys."""
    if kind == BF16 and last == LEAST:
        last = float(torch.finfo(BF16).min)
    for temperature in (20.0, 300.0):
        x, q = rows_of(first, last, 300, 10, kind, 1)
        for given in (dict(top_k=200), dict(top_k=9), dict(top_k=299, top_p=0.99)):
            check(x, q, temperature=temperature, **given)
        x, q = rows_of(first, last, 1500, 100, kind, 2)
        for given in (dict(top_k=700), dict(top_k=1499, top_p=0.99), dict(top_p=0.5, min_p=0.2)):
            check(x, q, temperature=temperature, **given)
        x, q = rows_of(first, last, 6000, 100, kind, 3)
        for given in (dict(top_k=3500), dict(top_k=5999), dict(top_k=5000, top_p=0.99)):
            check(x, q, temperature=temperature, **given)
