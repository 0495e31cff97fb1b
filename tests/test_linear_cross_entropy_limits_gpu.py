"""GPU: linear_cross_entropy and its gradients with logits from thousands to the largest numbers of 32 bits, on both sides of where the exchanged forms begin.

Bounds, beside those of test_linear_cross_entropy_gpu.  The logits here are products of one element of x and one of weight, of at most 11 digits each,
and zeros: exact.  lse is rounded (4 u |lse| counts its arguments too); beyond thousands that is more than a unit of an exponent, so the gradients are compared with
their formula at the lse that the forward call returned, as they are defined.  Their exponents (z - lse) log2 e have three roundings (difference, constant,
product), 3 u |z - lse|, and the exponential has 2^-22."""

import math

import pytest
import torch
from test_linear_cross_entropy_gpu import HALF, IDS, IGNORE, KINDS, LARGEST, LEAST, U, expected, inputs, product_error

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

ROWS = [1, 64, 65, 300]


def close(name, got, want, bound, kind=torch.float32):
    got, want = got.double(), want.double()
    off = (got - want).abs()
    beyond = (got == torch.copysign(torch.full_like(want, math.inf), want)) & (want.abs() + bound >= LARGEST[kind])
    assert bool(((off <= bound) | beyond).all()), (name, float((off / bound).nan_to_num(math.inf).max()))


def check_exact_logits(x, w, t, z):
    """z: the logits, exactly, in float64."""
    kind, n = x.dtype, len(x)
    given, at = t != IGNORE, torch.where(t == IGNORE, 0, t)[:, None]
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    want = torch.logsumexp(z, -1)
    elo = 4 * U * want.abs() + 2.0**-15
    close("lse", lse, want, elo)
    want = torch.where(given, want - z.gather(1, at).squeeze(1), 0.0)
    close("loss", loss, want, elo + U * want.abs())
    one = torch.ones((), device="cuda")
    dx, dw = tb.linear_cross_entropy_backward(one, x, w, t, lse)
    tb.check_status()
    share = given.double()[:, None] / max(1, int(given.sum()))
    far = z - lse.double()[:, None]
    p = torch.exp(far)
    d = share * (p - torch.zeros_like(z).scatter_(1, at, 1.0))
    half = 2 * U if kind == torch.float32 else HALF[kind]
    ed = share * torch.where(p > 0, p * torch.expm1((3 * U * far.abs() + 2.0**-21).clamp(max=1.0)), 0.0) + (half + 4 * U) * d.abs()
    ed = ed + share * (2.0**-126 + (2.0**-40 if kind == torch.float16 else 0.0)) + 2.0**-132
    xd, wd = x.double(), w.double()
    want = d @ wd
    close("dx", dx, want, ed @ wd.abs() + (product_error(kind, len(w)) + 8 * U) * (d.abs() @ wd.abs()) + HALF[kind] * want.abs() + LEAST[kind], kind)
    want = d.t() @ xd
    close("dweight", dw, want, ed.t() @ xd.abs() + (product_error(kind, n) + 8 * U) * (d.abs().t() @ xd.abs()) + HALF[kind] * want.abs() + LEAST[kind], kind)


# powers of two of the elements: x is 1, 1.25, 1.5 or 1.75 of the first, weight a whole number up to 255 of the second
POWERS = {torch.float16: [(2, 0), (7, 5), (15, 8)], torch.bfloat16: [(2, 0), (10, 10), (15, 8), (40, 52), (60, 59)]}
POWERS[torch.float32] = POWERS[torch.bfloat16]


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("n", ROWS)
def test_logits_of_any_size(n, kind):
    """Up to 3.7e9 in float16 and 2.97e38 otherwise (log2 e times as much is beyond 32 bits), of both signs, all logits of a row large or some."""
    g = torch.Generator().manual_seed(n)
    a = 1 + torch.randint(4, (n,), generator=g) / 4
    for first, last in ((-44, 255), (200, 255)):
        k = first + torch.randperm(last - first + 1, generator=g)
        t = torch.randint(len(k), (n,), generator=g)
        t[::3] = int(k.argmax())
        t[5::7] = IGNORE
        for px, pw in POWERS[kind]:
            for sign in (1.0, -1.0):
                x, w = torch.zeros(n, 24), 2 * torch.rand(len(k), 24, generator=g) - 1
                x[:, 0], w[:, 0] = sign * a * 2.0**px, k * 2.0**pw
                x, w = x.to(kind).cuda(), w.to(kind).cuda()
                z = x[:, :1].double() * w[:, 0].double()
                assert torch.equal(z, z.float().double())
                check_exact_logits(x, w, t.cuda(), z)


@pytest.mark.parametrize("kind", KINDS[1:], ids=IDS[1:])
@pytest.mark.parametrize("n", ROWS)
def test_symbols_masked_by_the_least_number(n, kind):
    """Symbols whose logits are the type's lowest number, in runs that fill whole tiles: as if they were not there."""
    x, w, t = inputs(n, 1500, 48, kind)
    x[:, 0], w[:, 0] = 1.0, 0.0
    at = torch.arange(1500, device="cuda")
    for masked in (at < 600, at >= 900, at // 300 % 2 == 0, at % 2 == 1, (at != 777) & (at != 778)):
        some = (~masked).nonzero().squeeze(1)
        table = w.clone()
        table[masked, 0] = torch.finfo(kind).min
        among = torch.where(t == IGNORE, IGNORE, t % len(some))
        target = torch.where(t == IGNORE, IGNORE, some[among.clamp(min=0)])
        loss, lse = tb.linear_cross_entropy(x, table, target, return_lse=True)
        dloss = torch.tensor(64.0, device="cuda")
        dx, dw = tb.linear_cross_entropy_backward(dloss, x, table, target, lse)
        tb.check_status()
        want, bound = expected(x, table[some], among, dloss, "mean")
        for name, got, e, b in zip(("loss", "lse", "dx", "dweight"), (loss, lse, dx, dw[some]), want, bound):
            close(name, got, e, b, kind)
        assert not dw[masked].any()
