"""GPU: the end of what top_k and top_p keep, where it falls among symbols far below the others; against the definition of test_sample_gpu."""

import math

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


ALL_BUT = 1 - 2**-24  # the largest top_p that is a filter


def hardly_reached(top, low, symbols, below, seed):
    """A row whose sum of p in 32 bits is above what it is by more than 2^-24 of it, so that what top_p asks for is not reached: the largest
    symbol, and one of p = 0.51 x 2^-23 for each level of a warp's tree of sums (symbols 4 apart are of neighbouring threads), each of
    which is rounded up.  All else is -inf but `below` symbols of the value `low`."""
    g = torch.Generator().manual_seed(seed)
    x = torch.full((2, symbols), -math.inf)
    x[:, 0] = top
    for level in (4, 8, 16, 32, 64):
        x[:, level] = top + math.log(0.51 * 2.0**-23)
    free = 65 + torch.randperm(symbols - 65, generator=g)[:below]
    x[:, free] = low
    return x.cuda(), torch.empty(2, symbols).exponential_(generator=g).cuda()


@pytest.mark.parametrize("top", [16.8, 16.9, 17.0, 18.5, 20.5, 25.0])
@pytest.mark.parametrize("symbols,below", [(400, 200), (3000, 1900), (9000, 6000)])
def test_masses_that_32_bits_do_not_hold(top, symbols, below):
    """Symbols of p = 0 in 32 bits in a bin whose upper end has p > 0: the end among them is one of them, and no empty bin."""
    for gap in (86.5, 87.2, 87.4, 88.0, 88.7, 90.5, 104.0):
        x, q = hardly_reached(top, top - gap, symbols, below, 7)
        for given in (dict(top_p=ALL_BUT), dict(top_p=torch.full((2,), ALL_BUT, device="cuda")), dict(top_k=symbols - 1, top_p=ALL_BUT)):
            check(x, q, **given)
        # where nothing but such symbols has little noise, one of the six above them is the answer: none of p = 0 is ever given
        q[:, 65:] = 1e-30
        token, _ = check(x, q, top_p=ALL_BUT)
        assert int(token.max()) <= 64


def test_rows_of_ever_smaller_symbols():
    """Every p from 1 down to none, in steps of the order of the bins and of half a binade."""
    for step in (0.05, 0.35, 0.7, 30.0):
        x = 60.0 - step * torch.arange(5000, dtype=torch.float32)
        x = torch.stack([x, x.flip(0), torch.where(x > -math.inf, x.clamp(min=-27.4), x)]).cuda()
        q = torch.empty(3, 5000).exponential_(generator=torch.Generator().manual_seed(1)).cuda()
        for temperature in (0.05, 1.0, 40.0):
            for top_p in (ALL_BUT, 0.999, 0.3, 0.0):
                check(x, q, temperature=temperature, top_p=top_p)
                check(x, q, temperature=temperature, top_p=top_p, top_k=3000)
