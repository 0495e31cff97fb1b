"""GPU: linear_cross_entropy and its gradients against their formulas in float64, elementwise.

Bounds.  u = 2^-24.  S = sum_d |x_d w_d|.
Logits, 16-bit operands: products are exact; each MMA adds 16 of them and cuts off below a unit of the last place, 2 u of at most S, for up to 512 terms, which
are then added up with a rounding: E_z = (min(D / 16, 32) + 8) 2 u S + D / 512 u S.  float32: what the six products of parts leave out is below 2^-22.9 = 2.2 u of each product, the MMAs of the first
parts of 32 or 64 terms are cut off (2 u each, up to four), those of the others by 2^-8 of that, and the sums of D / 32 of them rounded: E_z = (16 + D / 32) u S.
lse: max E_z, the exponentials (2^-22 each), their arguments (4 u of the numbers, as far as those count), and some 320 additions in a row: E_lse = max E_z + 2^-15 + 4 u |lse|.
loss: E_lse + E_z of the target, and u of both for the difference.
d = g (p - [target]): p is off by exp(E_z + E_lse + 2^-21) - 1 at most, and d is rounded by half a step h of its type (2^-8, 2^-11; float32: 2 u, cut off), in float16 at
least by 2^-25 2^-15 of the largest g.  A p below 2^-126, the least normal number, is 0, and so are parts of d below 2^-133, the least bfloat16: 2^-126 |g| + 2^-132.  Its products: as for the logits, with K terms and their own S = sum |d| |w|, 16384 of 16 bits in an accumulator, summed again for each piece.
The result is rounded by half a step of its type: to infinity from the largest number and half a step of it on (in float16 65520, of the bfloat16 and
float32 numbers here none comes near)."""

import math

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0**-24
KINDS = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
HALF = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}
LARGEST = {k: torch.finfo(k).max * (1 + torch.finfo(k).eps / 4) for k in KINDS}
IGNORE = -100


def product_error(kind, terms, together=16_384):
    return (16 + terms / 32) * U if kind == torch.float32 else (min(terms, together) / 16 + 8) * 2 * U + terms / together * U


def expected(x, weight, target, dloss, reduction, ignore=IGNORE):
    """loss, lse, dx, dweight, and how far each may be off; on x's device, in float64."""
    kind, symbols = x.dtype, weight.shape[0]
    D = x.shape[-1]
    x, w, t = x.double().reshape(-1, D), weight.double(), target.long().reshape(-1)
    given = t != ignore
    n = len(t)
    z = x @ w.t()
    ez = product_error(kind, D, 512) * (x.abs() @ w.abs().t())
    lse = torch.logsumexp(z, -1)
    elo = ez.amax(-1) + 2.0**-15 + 4 * U * lse.abs()
    at = torch.where(given, t, 0)[:, None]
    loss = torch.where(given, lse - z.gather(1, at).squeeze(1), 0.0)
    eloss = torch.where(given, elo + ez.gather(1, at).squeeze(1) + U * (lse.abs() + z.gather(1, at).squeeze(1).abs()) + U * loss, 0.0)
    share = torch.where(given, 1.0, 0.0)
    count = max(1, int(given.sum()))
    if reduction == "none":
        g = share * dloss.double().reshape(-1)
    else:
        g = share * dloss.double() / (count if reduction == "mean" else 1)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at, given.double()[:, None])
    d = g[:, None] * (p - hot)
    half = 2 * U if kind == torch.float32 else HALF[kind]
    ed = g.abs()[:, None] * p * torch.expm1(ez + elo[:, None] + 2.0**-21) + (half + 4 * U) * d.abs()
    ed = ed + 2.0**-126 * g.abs()[:, None] + 2.0**-132
    if kind == torch.float16:
        ed = ed + 2.0**-40 * g.abs().amax() * given[:, None]
    dx, dw = d @ w, d.t() @ x
    edx = (ed @ w.abs()) + (product_error(kind, symbols) + 8 * U) * (d.abs() @ w.abs()) + HALF[kind] * dx.abs() + LEAST[kind]
    edw = (ed.t() @ x.abs()) + (product_error(kind, n) + 8 * U) * (d.abs().t() @ x.abs()) + HALF[kind] * dw.abs() + LEAST[kind]
    if reduction == "none":
        total, etotal = loss, eloss
    else:
        total, etotal = loss.sum(), eloss.sum()
        if reduction == "mean":
            total, etotal = total / count, etotal / count
        etotal = etotal + 2 * U * total.abs()
    return (total, lse, dx, dw), (etotal, elo, edx, edw)


def check(x, weight, target, dloss=None, reduction="mean", ignore=IGNORE):
    loss, lse = tb.linear_cross_entropy(x, weight, target, reduction=reduction, ignore_index=ignore, return_lse=True)
    assert lse.shape == target.shape and lse.dtype == loss.dtype == torch.float32
    assert loss.shape == (target.shape if reduction == "none" else ())
    if dloss is None:
        dloss = torch.full_like(loss, 2.0**10 if x.dtype == torch.float16 else 1.0)
    dx, dw = tb.linear_cross_entropy_backward(dloss, x, weight, target, lse, reduction=reduction, ignore_index=ignore)
    tb.check_status()
    assert dx.shape == x.shape and dw.shape == weight.shape and dx.dtype == dw.dtype == x.dtype
    assert dx.is_contiguous() and dw.is_contiguous()
    want, bound = expected(x, weight, target, dloss, reduction, ignore)
    for name, got, w, b in zip(("loss", "lse", "dx", "dweight"), (loss, lse, dx, dw), want, bound):
        got = got.double().reshape(w.shape)
        off = (got - w).abs()
        beyond = (got == torch.copysign(torch.full_like(w, math.inf), w)) & (w.abs() + b >= LARGEST[x.dtype])
        assert bool(((off <= b) | beyond).all()), (name, float((off / b).nan_to_num(math.inf).max()))
    again = tb.linear_cross_entropy(x, weight, target, reduction=reduction, ignore_index=ignore, return_lse=True)
    assert torch.equal(again[0], loss) and torch.equal(again[1], lse)
    again = tb.linear_cross_entropy_backward(dloss, x, weight, target, lse, reduction=reduction, ignore_index=ignore)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    return loss, lse, dx, dw


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed * 7919 + shape[0])).cuda()


def inputs(n, v, d, kind, seed=0, scale=3.0):
    """Logits of a few units' spread, rows that point at their targets, a few positions ignored."""
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + v)
    w = torch.randn(v, d, generator=g) / math.sqrt(d)
    t = torch.randint(v, (n,), generator=g)
    x = scale * torch.randn(n, d, generator=g) + 4.0 * torch.rand(n, 1, generator=g) * w[t]
    t[torch.rand(n, generator=g) < 0.1] = IGNORE
    return x.to(kind).cuda(), w.to(kind).cuda(), t.cuda()


SIZES = [(1, 1, 1), (1, 2, 3), (5, 3, 8), (7, 1000, 256), (31, 130, 17), (128, 256, 64), (129, 257, 65), (255, 129, 1024), (256, 512, 72), (300, 1000, 200), (513, 2003, 513), (40, 20_011, 24), (3000, 300, 130), (600, 4096, 640)]


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("n,v,d", SIZES)
def test_matches_definition(n, v, d, kind):
    check(*inputs(n, v, d, kind))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions(reduction, kind):
    x, w, t = inputs(200, 500, 64, kind)
    shape = (200,) if reduction == "none" else ()
    for scale in (1.0, -300.0, 0.0):
        g = torch.full(shape, scale, device="cuda")
        if reduction == "none":
            g = g * torch.exp(2.0 * rand(200, seed=3))
        check(x, w, t, g, reduction)
    check(x.view(4, 50, 64), w, t.view(4, 50), None, reduction)
    check(x, w, t.int(), None, reduction)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_pieces_of_the_symbols(kind):
    """More logits than a piece holds: many row tiles (dx is added to from piece to piece), and few (its contraction is split as well)."""
    few = 2 if kind == torch.float32 else 1
    check(*inputs(20_000 // few, 14_001 // few + 1, 64, kind))
    check(*inputs(700, (400_003 if kind != torch.float32 else 140_001), 72, kind), reduction="sum")


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_many_rows_and_few_symbols(kind):
    """dweight's contraction is split among the CTAs."""
    check(*inputs(30_000, 100, 40, kind))
    check(*inputs(70_001, 3, 8, kind))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [2, 15, 16, 17, 32, 33, 48, 49, 63, 64, 65, 96, 127, 128, 129, 191, 192, 193])
def test_few_rows(n, kind):
    """On both sides of where rows of x become rows and no columns of the MMAs, and where another one begins."""
    for v, d, reduction in ((1003, 200, "mean"), (130, 513, "none"), (20_000, 72, "sum")):
        check(*inputs(n, v, d, kind), reduction=reduction)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("n", [30, 60, 120])
def test_few_rows_with_masks(n, kind):
    x, w, t = inputs(n, 700, 96, kind)
    t[::4] = IGNORE
    g = torch.exp(rand(n, seed=4)) * (256.0 if kind == torch.float16 else 1.0)
    want = check(x, w, t, g, "none")
    check(x, w, torch.full_like(t, IGNORE))
    check(x, w, t.int())
    g[::4], x[::4] = float("nan"), float("nan")
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    dx, _ = tb.linear_cross_entropy_backward(g, x, w, t, lse, reduction="none", weight_grad=False)
    assert torch.equal(loss, want[0]) and torch.equal(dx, want[2]) and bool(lse[::4].isnan().all())
    dx, dw = tb.linear_cross_entropy_backward(g, x, w, t, lse, reduction="none")
    assert torch.equal(dx, want[2]) and torch.equal(dw, want[3])
    x, w, t = inputs(n, 700, 96, kind)
    t[3], t[n - 1] = 700, -1
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    dx, dw = tb.linear_cross_entropy_backward(torch.ones_like(loss), x, w, t, lse, reduction="none")
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[[3, n - 1]] = True
    assert torch.equal(loss.isnan(), bad) and torch.equal(dx.isnan().all(1), bad) and torch.equal(dx.isnan().any(1), bad) and bool(dw.isnan().all())
    if kind != torch.float32:
        w[::2] = float("-inf")
        x, t = x.abs() + 0.1, torch.where(t < 0, t, t // 2 * 2 + 1).clamp(max=699)
        loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
        some = tb.linear_cross_entropy(x, w[1::2].contiguous(), torch.where(t < 0, t, t // 2), reduction="none", return_lse=True)
        assert torch.allclose(lse, some[1], rtol=0, atol=1e-4)
        w[1::2] = float("-inf")  # nothing is possible
        loss, lse = tb.linear_cross_entropy(x, w, t.clamp(min=0), reduction="none", return_lse=True)
        assert bool((lse == float("-inf")).all()) and bool(loss.isnan().all())


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_few_rows_and_pieces_of_the_symbols(kind):
    check(*inputs(64, 1_500_001 if kind == torch.float32 else 4_300_001, 8, kind))


@pytest.mark.parametrize("kind", KINDS[1:], ids=IDS[1:])
@pytest.mark.parametrize("n", [6, 70, 333])
def test_common_factors_are_not_rounded(n, kind):
    """Where the targets have no probability the gradient of a row is -dloss / n of its target's row, however dloss and 1 / n are rounded to 16 bits: d is exact then, four
    roundings in 32 bits and half a step of the result are left, and the n symbols of probability e^-32 < 2^-46."""
    v, d = n + 1, 64
    w = torch.zeros(v, d, device="cuda")
    x = torch.zeros(n, d, device="cuda")
    w[n, 0] = 32.0  # the last symbol has all of the probability
    x[:, 0] = 1.0
    w[:n, 1:] = rand(n, d - 1)
    w, x = w.to(kind), x.to(kind)
    t = torch.arange(n, device="cuda")
    loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
    dloss = torch.tensor(0.3, device="cuda")
    dx, _ = tb.linear_cross_entropy_backward(dloss, x, w, t, lse)
    g = float(dloss) / n
    want = -g * w[:n, 1:].double()
    rest = n * 2.0**-46 * g * float(w[:n, 1:].abs().max())
    assert bool(((dx[:, 1:].double() - want).abs() <= (HALF[kind] + 5 * U) * want.abs() + rest + LEAST[kind]).all())


@pytest.mark.parametrize("n", [16, 80])
def test_large_offsets(n):
    """A table beyond 2^31 elements: its last rows are read and their gradients written at 64-bit offsets."""
    v, d = 270_001, 8192
    w = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 5, 131_072, 262_143, 262_144, v - 2, v - 1], device="cuda")
    w[some] = (rand(len(some), d) / 90.0).bfloat16()
    x = rand(n, d, seed=1).bfloat16()
    t = some[torch.arange(n, device="cuda") % len(some)]
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="sum", return_lse=True)
    dx, dw = tb.linear_cross_entropy_backward(torch.ones((), device="cuda"), x, w, t, lse, reduction="sum")
    tb.check_status()
    z = x.double() @ w[some].double().t()  # (all other logits are 0)
    want = torch.logsumexp(torch.cat([z, torch.full((n, 1), math.log(v - len(some)), device="cuda", dtype=torch.float64)], 1), 1)
    assert bool(((lse.double() - want).abs() <= 1e-4).all())
    p = torch.exp(z - want[:, None]) - (t[:, None] == some).double()
    for got, exact in ((dx, p @ w[some].double()), (dw[some], p.t() @ x.double())):
        assert float((got.double() - exact).norm()) <= 2.0**-7 * float(exact.norm())
    rest = torch.exp(-want) @ x.double()  # every other row's gradient
    for row in (2, 200_000, 262_145, v - 3):
        assert float((dw[row].double() - rest).norm()) <= 2.0**-7 * float(rest.norm())


def test_wide_rows():
    check(*inputs(64, 700, 8192, torch.bfloat16))
    check(*inputs(64, 700, 8192, torch.float32))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_ignored_positions(kind):
    x, w, t = inputs(300, 400, 48, kind)
    t[:] = IGNORE
    for reduction in ("none", "sum", "mean"):
        loss, _, dx, dw = check(x, w, t, None, reduction)
        assert not loss.any() and not dx.any() and not dw.any()
    t[17] = 5
    _, _, dx, _ = check(x, w, t)
    assert not dx[:17].any() and not dx[18:].any()
    # another mark, which is also a symbol; and none that occurs
    t = torch.arange(300, device="cuda") % 400
    check(x, w, t, ignore=7)
    check(x, w, t, ignore=-(2**63))
    # dloss of ignored positions does not count, whatever it is
    t[::3] = IGNORE
    g = torch.ones(300, device="cuda")
    want = check(x, w, t, g, "none")
    g[::6], g[3::6] = float("nan"), float("inf")
    lse = want[1]
    got = tb.linear_cross_entropy_backward(g, x, w, t, lse, reduction="none")
    assert torch.equal(got[0], want[2]) and torch.equal(got[1], want[3])
    # nor does what x holds there
    x[::3] = float("nan")
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    assert torch.equal(loss, want[0]) and bool(lse[::3].isnan().all())
    dx, none = tb.linear_cross_entropy_backward(torch.ones(300, device="cuda"), x, w, t, lse, reduction="none", weight_grad=False)
    assert torch.equal(dx, want[2]) and none is None
    dx, dw = tb.linear_cross_entropy_backward(torch.ones(300, device="cuda"), x, w, t, lse, reduction="none")
    assert torch.equal(dx, want[2]) and torch.equal(dw, want[3])


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_targets_that_are_no_symbols(kind):
    x, w, t = inputs(300, 400, 48, kind)
    good = check(x, w, t, reduction="none")
    t[3], t[200], t[299] = 400, -1, 2**40
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    bad = torch.zeros(300, dtype=torch.bool, device="cuda")
    bad[[3, 200, 299]] = True
    assert bool(loss[bad].isnan().all()) and torch.equal(loss[~bad], good[0][~bad]) and torch.equal(lse, good[1])
    assert bool(tb.linear_cross_entropy(x, w, t).isnan())
    dx, dw = tb.linear_cross_entropy_backward(torch.full_like(loss, 1024.0 if kind == torch.float16 else 1.0), x, w, t, lse, reduction="none")
    assert bool(dx[bad].isnan().all()) and torch.equal(dx[~bad], good[2][~bad]) and bool(dw.isnan().all())


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_strides(kind):
    big = rand(700, 300).to(kind)
    t = torch.randint(200, (60,), generator=torch.Generator().manual_seed(2)).cuda()
    t[::9] = IGNORE
    views = [lambda n, d: big[3 : 3 + n, 8 : 8 + d], lambda n, d: big[: 2 * n : 2, :d], lambda n, d: big[:n, 5 : 5 + d], lambda n, d: big.flip(0)[:n, :d],
             lambda n, d: big.t()[:n, :d], lambda n, d: big[:n, ::2][:, :d], lambda n, d: big[:1, :d].expand(n, d), lambda n, d: big[1 : 1 + n, 1 : 1 + d]]  # fmt: skip
    for d in (64, 50):
        for fx in views:
            check(fx(60, d), big[:200, 100 : 100 + d], t)
        for fw in views:
            check(big[:60, 200 : 200 + d], fw(200, d), t)
    check(big[:60, :64].view(6, 10, 64).transpose(0, 1), big[:200, :64], t.view(6, 10).t())


def test_memory_around_the_results():
    """dx and dweight are written to the last element and no further, at odd sizes."""
    from triturus_b200 import _native

    x, w, t = inputs(130, 259, 67, torch.bfloat16)
    loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
    want = tb.linear_cross_entropy_backward(torch.ones_like(loss), x, w, t, lse)
    flat = torch.full((130 * 67 + 259 * 67 + 96,), 7.0, dtype=torch.bfloat16, device="cuda")
    dx, dw = flat[32 : 32 + 130 * 67], flat[64 + 130 * 67 : 64 + 130 * 67 + 259 * 67]
    sizes = 130, 259, 67, 67, 67, 1
    nbytes = _native.LIB.triturus_b200_linear_cross_entropy_backward_workspace_bytes(x.data_ptr(), w.data_ptr(), *sizes)
    space = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    one = torch.ones((), device="cuda")
    rc = _native.LIB.triturus_b200_linear_cross_entropy_backward(
        one.data_ptr(), x.data_ptr(), w.data_ptr(), t.data_ptr(), 8, lse.data_ptr(), dx.data_ptr(), dw.data_ptr(), *sizes, 1, IGNORE, space.data_ptr(), nbytes,
        None, torch.cuda.current_stream().cuda_stream)  # fmt: skip
    assert rc == 0
    assert torch.equal(dx.view(130, 67), want[0]) and torch.equal(dw.view(259, 67), want[1])
    assert bool((flat[:32] == 7).all()) and bool((flat[32 + 130 * 67 : 64 + 130 * 67] == 7).all()) and bool((flat[-32:] == 7).all())


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_large_and_impossible_logits(kind):
    """Logits of thousands, whose exponentials 32 bits do not hold; symbols of -infinity, which 16-bit operands can give; NaN."""
    x, w, t = inputs(100, 300, 32, kind, scale=1.0)
    check(x * 300, w, t)
    if kind == torch.float32:
        return
    x[:, 0], w[:, 0] = 1.0, 0.0
    w[::2, 0] = float("-inf")  # half of the symbols are impossible
    t = torch.where(t == IGNORE, t, t // 2 * 2 + 1).clamp(max=299)
    loss, lse = tb.linear_cross_entropy(x, w, t, reduction="none", return_lse=True)
    some = check(x, w[1::2].contiguous(), torch.where(t == IGNORE, t, t // 2), reduction="none")
    assert torch.allclose(lse, some[1], rtol=0, atol=1e-4) and torch.allclose(loss, some[0], rtol=0, atol=1e-4)
    w[::2, 0] = 0.0
    w[5, 3] = float("nan")
    assert bool(tb.linear_cross_entropy(x, w, t).isnan())


def test_scaled_losses_of_float16():
    """Gradients of any dloss keep their digits: d is held relative to the largest."""
    x, w, t = inputs(300, 1000, 64, torch.float16)
    lse = tb.linear_cross_entropy(x, w, t, return_lse=True)[1]
    one = tb.linear_cross_entropy_backward(torch.tensor(2.0**14, device="cuda"), x, w, t, lse)
    for power in (8, 16):
        got = tb.linear_cross_entropy_backward(torch.tensor(2.0**power, device="cuda"), x, w, t, lse)
        for a, b in zip(got, one):
            normal = (a.abs() >= 2.0**-14) & (b.abs() >= 2.0**-14)
            assert bool(normal.any()) and torch.equal(a[normal].double(), (b.double() * 2.0 ** (power - 14))[normal])
    for bad in (float("inf"), float("nan")):
        dx, dw = tb.linear_cross_entropy_backward(torch.tensor(bad, device="cuda"), x, w, t, lse)
        assert not dx[t != IGNORE].isfinite().any() and not dx[t == IGNORE].isfinite().logical_not().any() or not dw.isfinite().all()
    g = torch.ones(300, device="cuda")
    g[5] = float("inf")
    t[5] = 3
    dx, _ = tb.linear_cross_entropy_backward(g, x, w, t, lse, reduction="none")
    assert not dx[5].isfinite().any() and bool(dx[6:].isfinite().all()) and bool(dx[6:].any())


def test_no_positions():
    w = rand(50, 16)
    for shape in ((0,), (3, 0)):
        x, t = torch.empty(*shape, 16, device="cuda"), torch.empty(shape, dtype=torch.int64, device="cuda")
        loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
        assert loss.shape == () and float(loss) == 0 and lse.shape == shape
        assert tb.linear_cross_entropy(x, w, t, reduction="none").shape == shape
        dx, dw = tb.linear_cross_entropy_backward(torch.ones((), device="cuda"), x, w, t, lse)
        assert dx.shape == x.shape and dw.shape == w.shape and not dw.any()
    one = tb.linear_cross_entropy(rand(16), w, torch.tensor(3, device="cuda"), reduction="none")  # one position without a dimension
    assert one.shape == ()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_autograd(kind):
    x, w, t = inputs(300, 500, 64, kind)
    for reduction in ("mean", "sum", "none"):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = tb.linear_cross_entropy(a, b, t, reduction=reduction)
        g = torch.full((), 64.0, device="cuda").expand(loss.shape)  # (as sum() gives it: no memory of its own)
        loss.backward(g)
        lse = tb.linear_cross_entropy(x, w, t, return_lse=True)[1]
        dx, dw = tb.linear_cross_entropy_backward(g, x, w, t, lse, reduction=reduction)
        assert torch.equal(a.grad, dx) and torch.equal(b.grad, dw)
    a = x.clone().requires_grad_()
    (only,) = torch.autograd.grad(tb.linear_cross_entropy(a, w, t), a)
    assert torch.equal(only, tb.linear_cross_entropy_backward(torch.ones((), device="cuda"), x, w, t, lse, weight_grad=False)[0])
    loss, lse = tb.linear_cross_entropy(a, w, t, return_lse=True)
    assert loss.requires_grad and not lse.requires_grad


def test_gradients_against_differences():
    """Central differences of the float32 loss: its rounding, 2 E_z / step, and the third derivative, below step^2."""
    x, w, t = inputs(20, 30, 16, torch.float32)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    tb.linear_cross_entropy(a, b, t, reduction="sum").backward()
    f = lambda p, q: float(tb.linear_cross_entropy(p, q, t, reduction="none").double().sum())  # noqa: E731
    step = 2.0**-6
    for grad, base, call in ((a.grad, x, lambda y: f(y, w)), (b.grad, w, lambda y: f(x, y))):
        for i, j in ((0, 0), (7, 15), (19, 3)):
            up, down = base.clone(), base.clone()
            up[i, j] += step
            down[i, j] -= step
            assert abs((call(up) - call(down)) / (2 * step) - float(grad[i, j])) <= 5e-3


def test_streams_and_graphs():
    x, w, t = inputs(600, 3001, 72, torch.bfloat16)

    def both():
        loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
        return loss, lse, *tb.linear_cross_entropy_backward(torch.ones_like(loss), x, w, t, lse)

    want = both()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other.wait_stream(torch.cuda.current_stream())
    got = []
    for stream in (side, other, side, other):  # calls beside each other, each with its own workspace
        with torch.cuda.stream(stream):
            got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        graphs.append((graph, out))
    x.copy_(x.flip(0).clone())
    t.copy_(t.flip(0).clone())
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = both()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    tb.check_status()
