"""GPU: the gradients of linear_cross_entropy where weight or dloss hold infinities or NaN."""

import pytest
import torch
from test_linear_cross_entropy_gpu import IDS, IGNORE, KINDS, expected, inputs

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("n,v,d", [(30, 700, 96), (64, 5003, 513), (200, 700, 96), (300, 300, 40), (1000, 10_007, 200)])
def test_ignored_positions_beside_infinite_weights(n, v, d, bad, kind):
    """dx is zero where there is no loss, whatever weight holds: 0 times infinity does not reach it, with and without dweight."""
    x, w, t = inputs(n, v, d, kind)
    t[::4] = IGNORE
    w[7, 3], w[v - 1, d - 1] = bad, bad
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    assert not loss[t == IGNORE].any()
    for weight_grad in (True, False):
        dx, _ = tb.linear_cross_entropy_backward(torch.ones(n, device="cuda"), x, w, t, lse, reduction="none", weight_grad=weight_grad)
        assert not dx[t == IGNORE].any() and bool(dx[t != IGNORE].isnan().any())
    tb.check_status()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [64, 700])
def test_ignored_positions_beside_infinite_weights_in_pieces(n, kind):
    """More logits than a piece of the symbols holds, so that dx is added to from piece to piece."""
    v = 140_001 if kind == torch.float32 else 400_003
    v = v if n == 700 else v * 11
    x, w, t = inputs(n, v, 8, kind)
    t[::4] = IGNORE
    for at in (5, v // 2, v - 1):
        w[at, at % 8] = INF
    lse = tb.linear_cross_entropy(x, w, t, return_lse=True)[1]
    dx, _ = tb.linear_cross_entropy_backward(torch.ones((), device="cuda"), x, w, t, lse)
    tb.check_status()
    assert not dx[t == IGNORE].any() and bool(dx[t != IGNORE].isnan().any())


@pytest.mark.parametrize("kind", KINDS[1:], ids=IDS[1:])
@pytest.mark.parametrize("n", [30, 64, 65, 300])
def test_gradients_with_impossible_symbols(n, kind):
    """Symbols of -infinity through one column of weight: that column of dx is 0 times infinity, NaN; the others, and dweight, are as if the symbols were not
    there."""
    x, w, t = inputs(n, 700, 72, kind)
    x[:, 0], w[:, 0] = 1.0, 0.0
    w[::2, 0] = -INF
    among = torch.where(t == IGNORE, IGNORE, t // 2)
    t = torch.where(t == IGNORE, IGNORE, t // 2 * 2 + 1)
    loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
    dloss = torch.tensor(32.0, device="cuda")
    dx, dw = tb.linear_cross_entropy_backward(dloss, x, w, t, lse)
    tb.check_status()
    want, bound = expected(x, w[1::2], among, dloss, "mean")
    assert bool(dx[t != IGNORE, 0].isnan().all()) and not dx[t == IGNORE].any() and not dw[::2].any()
    for name, got, e, b in zip(("loss", "lse", "dx", "dweight"), (loss, lse, dx[:, 1:], dw[1::2]), want, bound):
        e, b = (e[:, 1:], b[:, 1:]) if name == "dx" else (e, b)
        assert bool(((got.double() - e).abs() <= b).all()), name


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [60, 300])
def test_losses_that_are_no_numbers(n, kind):
    """Such a dloss reaches dx of all positions that count and of none that are ignored, and dweight; one of them for a single position reaches that row alone."""
    x, w, t = inputs(n, 1000, 64, kind)
    t[::9] = IGNORE
    lse = tb.linear_cross_entropy(x, w, t, return_lse=True)[1]
    for bad in (INF, -INF, NAN):
        dx, dw = tb.linear_cross_entropy_backward(torch.tensor(bad, device="cuda"), x, w, t, lse)
        assert not dx[t != IGNORE].isfinite().any()
        assert not dx[t == IGNORE].any()
        assert not dw.isfinite().any()
        dloss = torch.ones(n, device="cuda")
        dloss[5] = bad
        dx, dw = tb.linear_cross_entropy_backward(dloss, x, w, t, lse, reduction="none")
        assert int(t[5]) != IGNORE and not dx[5].isfinite().any()
        assert bool(dx[:5].isfinite().all()) and bool(dx[6:].isfinite().all()) and bool(dx[6:].any())
    tb.check_status()
