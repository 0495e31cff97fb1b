"""GPU: clip_grad_norm_ and grad_norm against the definition in float64.

Bounds.  u = 2^-24.  The norm: up to 8 squares are added in 32 bits (8 u), all else in 64, the root halves that and rounds once: below 8 u.
The factor adds two roundings and the product one: below 16 u of each element, and for 16-bit elements half a unit of their last place,
2^-9 (bfloat16) or 2^-12 (float16), doubled here, and float16's smallest step."""

import math

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0**-24
LAST = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def norm_of(grads, norm_type):
    flat = [g.detach().double().cpu().reshape(-1) for g in grads if g is not None]
    flat = torch.cat(flat) if flat else torch.zeros(0, dtype=torch.float64)
    if norm_type == 2:
        return float(flat.square().sum().sqrt())
    return float(flat.abs().max()) if flat.numel() else 0.0


def check(grads, share, norm_type=2.0):
    """Clip to `share` of the norm."""
    want = norm_of(grads, norm_type)
    before = [None if g is None else g.detach().double().cpu() for g in grads]
    bits = [None if g is None else g.clone() for g in grads]
    alone = tb.grad_norm(grads, norm_type=norm_type)
    limit = share * want
    norm = tb.clip_grad_norm_(grads, limit, norm_type=norm_type)
    assert norm.shape == () and norm.dtype == F32 and torch.equal(norm, alone)
    rounded = float(torch.tensor(want, dtype=F32))  # (infinite where 32 bits cannot hold it)
    assert float(norm) == rounded or abs(float(norm) - want) <= 8 * U * want
    factor = min(1.0, limit / (want + 1e-6))
    for g, b, kept in zip(grads, before, bits):
        if g is None:
            continue
        if factor == 1.0:
            assert torch.equal(g, kept)
        else:
            target = b * factor
            assert bool(((g.detach().double().cpu() - target).abs() <= (16 * U + LAST[g.dtype]) * target.abs() + LEAST[g.dtype]).all())


def some(shape, kind, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(kind).cuda()


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("share", [0.3, 1.5])
def test_lists(share, norm_type):
    check([some((1,), F32, 0)], share, norm_type)
    check([some((3, 5), kind, 1) for kind in (F32, BF16, F16)], share, norm_type)
    check([some((n,), (F32, BF16, F16)[n % 3], n) for n in (1, 2, 7, 8, 9, 4095, 4096, 8191, 8192, 8193, 16384, 16385, 70001)], share, norm_type)
    check([some((1000, 1003), F32, 2), some((2_000_001,), BF16, 3, 0.01), None, some((0,), F32, 4), some((5,), F16, 5, 100.0)], share, norm_type)


@pytest.mark.parametrize("count", [63, 64, 65, 300, 1024, 1025, 2100])
def test_many_tensors(count):
    check([some((1 + (37 * i) % 101,), (F32, BF16)[i % 2], i) for i in range(count)], 0.5)


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_views_of_one_buffer_and_what_lies_beside_them(kind):
    flat = some((100_000,), kind, 8)
    kept = flat.clone()
    places = [(1, 2), (3, 40), (44, 1000), (1051, 16_400), (17_460, 60_001), (80_000, 3)]
    grads = [flat[a : a + n] for a, n in places]
    check(grads, 0.5)
    inside = torch.zeros(100_000, dtype=torch.bool)
    for a, n in places:
        inside[a : a + n] = True
    assert torch.equal(flat[~inside], kept[~inside])


def test_other_layouts():
    base = some((40, 50, 6), F32, 9)
    check([base.permute(2, 0, 1), some((30, 20), BF16, 10).t()], 0.5)
    wide = some((64, 100), F32, 11)
    kept = wide.clone()
    check([wide[:, ::2], wide[:, 1:99:2], some((8,), F32, 12)], 0.5)  # (gaps: through a copy; elements beside each other, not shared)
    assert torch.equal(wide[:, 99], kept[:, 99])


def test_large_and_small_values():
    for scale in (1e25, 3e37, 1e-25, 1e-30):
        check([some((50_000,), F32, 13, scale), some((77,), F32, 14, scale)], 0.25 if scale > 1 else 2.0)
    g = some((1000,), F32, 15, 1e-12)  # the norm is near the 1e-6 of the denominator
    check([g], 0.5)
    zero = torch.zeros(5000, device="cuda")
    assert float(tb.clip_grad_norm_([zero], 1.0)) == 0.0 and not bool(zero.any())
    g = some((3000,), F32, 16)
    tb.clip_grad_norm_([g], 0.0)
    assert not bool(g.any())
    g = some((3000,), F32, 16)
    kept = g.clone()
    tb.clip_grad_norm_([g], math.inf)
    assert torch.equal(g, kept)


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_nan_and_infinity(norm_type):
    a, b = some((40_000,), F32, 17), some((100,), BF16, 18)
    a[31_000] = float("nan")
    assert math.isnan(float(tb.clip_grad_norm_([a, b], 1.0, norm_type=norm_type)))
    assert bool(a.isnan().all()) and bool(b.isnan().all())
    a, b = some((40_000,), F32, 17), some((100,), BF16, 18)
    a[31_000] = -math.inf
    assert float(tb.clip_grad_norm_([a, b], 1.0, norm_type=norm_type)) == math.inf
    assert bool(a[31_000].isnan()) and int(a.count_nonzero()) == 1 and not bool(b.any())


def test_agrees_with_torch():
    params = [torch.nn.Parameter(some((130, 70), F32, i)) for i in range(9)]
    for i, p in enumerate(params):
        p.grad = some((130, 70), F32, 20 + i)
    ours = [p.grad.clone() for p in params]
    theirs = torch.nn.utils.clip_grad_norm_(params, 2.5)
    norm = tb.clip_grad_norm_(ours, 2.5)
    assert abs(float(norm) - float(theirs)) <= 64 * U * float(theirs)
    for p, g in zip(params, ours):
        assert bool(((p.grad - g).abs() <= 128 * U * g.abs()).all())


def test_forms_of_the_argument():
    a, b = some((10,), F32, 1), some((11,), F32, 2)
    want = norm_of([a, b], 2)
    for form in ([a, b], (a, b), iter([a, None, b]), [a, b, None]):
        assert abs(float(tb.grad_norm(form)) - want) <= 8 * U * want
    assert abs(float(tb.grad_norm(a, norm_type=2)) - norm_of([a], 2)) <= 8 * U * want
    assert float(tb.clip_grad_norm_([], 1.0)) == 0.0 and float(tb.grad_norm([None])) == 0.0
    assert float(tb.grad_norm([torch.empty(0, device="cuda")])) == 0.0
    version = a._version
    tb.clip_grad_norm_([a], 1e-3)
    assert a._version > version
    p = torch.nn.Parameter(a.clone())
    assert float(tb.grad_norm([p])) > 0.0
    with pytest.raises(RuntimeError, match="inplace"):  # autograd learns that a saved tensor was changed
        y = (p * a).sum()
        tb.clip_grad_norm_([a], 1e-4)
        y.backward()


def test_streams_and_graphs():
    make = lambda: [some((n,), F32, n) for n in (5, 70_000, 300_001)]  # noqa: E731
    want = make()
    norm = tb.clip_grad_norm_(want, 3.0)
    got = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = tb.clip_grad_norm_(got, 3.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, other) and all(torch.equal(p, q) for p, q in zip(want, got))
    held = make()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other = tb.clip_grad_norm_(held, 3.0)
    for _ in range(3):
        for h, f in zip(held, make()):
            h.copy_(f)
        graph.replay()
        assert torch.equal(norm, other) and all(torch.equal(p, q) for p, q in zip(want, held))


def test_ops():
    a, b = some((1000,), F32, 1), some((500,), BF16, 2)
    torch.library.opcheck(torch.ops.triturus.clip_grad_norm_, ([a, b], 1.0, False), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.triturus.grad_norm, ([a, b], True), test_utils=("test_schema", "test_faketensor"))


def test_more_than_32_bits_count():
    big = torch.zeros(2**31 + 70_000, dtype=F16, device="cuda")
    big[-3:] = torch.tensor([3.0, 4.0, 12.0], dtype=F16, device="cuda")
    assert float(tb.clip_grad_norm_([big], 6.5)) == 13.0
    assert big[-4:].tolist() == [0.0, 1.5, 2.0, 6.0]


def test_refusals():
    a = some((12, 4), F32, 1)
    with pytest.raises(AssertionError):
        tb.clip_grad_norm_([a.double()], 1.0)
    with pytest.raises(AssertionError):
        tb.clip_grad_norm_([a, a.cpu()], 1.0)
    with pytest.raises(tb.NativeLibraryError, match="CUDA"):
        tb.clip_grad_norm_([a.cpu()], 1.0)
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            tb.clip_grad_norm_([a], limit)
    for norm_type in (1.0, 0.0, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            tb.clip_grad_norm_([a], 1.0, norm_type=norm_type)
        with pytest.raises(ValueError, match="norm_type"):
            tb.grad_norm([a], norm_type=norm_type)
    with pytest.raises(ValueError, match="share memory"):
        tb.clip_grad_norm_([a, a], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        tb.clip_grad_norm_([a[:7], a[6:]], 1.0)
    with pytest.raises(ValueError, match="expanded"):
        tb.clip_grad_norm_([a[:1].expand(5, 4)], 1.0)
    with pytest.raises(ValueError, match="requires a gradient"):
        tb.clip_grad_norm_([torch.nn.Parameter(a)], 1.0)
