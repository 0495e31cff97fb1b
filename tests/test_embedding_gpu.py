"""GPU: embedding and embedding_backward against their formulas in float64 on the CPU, elementwise.

Bounds.  u = 2^-24 is half the relative step of a 32-bit number.  Forward: one product (u) and one rounding to the result's type, half a step
(2^-8 of the value for bfloat16, 2^-11 for float16: finfo.eps / 2); a scale of 1 copies.  Gradient: n terms added in 32 bits, at most n u of
the sum of magnitudes, a product and the rounding.  The smallest steps are 2^-24 for float16 (half of it off), 2^-133 for bfloat16."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0**-24
KINDS = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]
HALF = {k: torch.finfo(k).eps / 2 for k in KINDS}
LEAST = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}


def check_forward(tokens, weight, scale):
    y = tb.embedding(tokens, weight, scale=scale)
    assert y.shape == (*tokens.shape, weight.shape[1]) and y.dtype == weight.dtype and y.is_contiguous()
    t, w = tokens.long().cpu(), weight.double().cpu()
    ok = (t >= 0) & (t < len(w))
    want = w[torch.where(ok, t, 0)] * scale
    got = y.double().cpu()
    if scale == 1.0:
        assert torch.equal(got[ok], want[ok])
    else:
        assert bool(((got - want)[ok].abs() <= ((HALF[y.dtype] + 2 * U) * want.abs() + LEAST[y.dtype])[ok]).all())
    assert bool(got[~ok].isnan().all())


def check_backward(dy, tokens, symbols, scale=1.0, padding=None):
    got = tb.embedding_backward(dy, tokens, symbols, scale=scale, padding_idx=padding)
    assert got.shape == (symbols, dy.shape[-1]) and got.dtype == dy.dtype and got.is_contiguous()
    t, d = tokens.long().cpu().reshape(-1), dy.double().cpu().reshape(-1, dy.shape[-1])
    keep = (t >= 0) & (t < symbols) & (t != (-1 if padding is None else padding))
    want, size = torch.zeros(symbols, d.shape[1], dtype=torch.float64), torch.zeros(symbols, d.shape[1], dtype=torch.float64)
    want.index_add_(0, t[keep], d[keep])
    size.index_add_(0, t[keep], d[keep].abs())
    n = torch.bincount(t[keep], minlength=symbols)[:, None]
    want, size = want * scale, size * abs(scale)
    bound = (n + 2) * U * size + HALF[dy.dtype] * want.abs() + LEAST[dy.dtype]
    out = got.double().cpu()
    assert bool(((out - want).abs() <= bound).all())
    assert bool((out[(n == 0).squeeze(1)] == 0).all())
    assert torch.equal(got, tb.embedding_backward(dy, tokens, symbols, scale=scale, padding_idx=padding))
    return got


def draw_tokens(count, symbols, seed=0):
    """Half of them the first few symbols."""
    g = torch.Generator().manual_seed(seed * 1009 + count)
    t = torch.randint(symbols, (count,), generator=g)
    few = torch.randint(min(3, symbols), (count,), generator=g)
    return torch.where(torch.rand(count, generator=g) < 0.5, few, t).cuda()


def rand(*shape, kind=torch.float32, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(kind).cuda()


SIZES = [(1, 1, 1), (1, 5, 3), (7, 3, 8), (31, 40, 17), (32, 40, 64), (33, 2, 100), (200, 513, 130), (1000, 50, 1001), (1025, 511, 33), (3000, 512, 24), (2100, 100_003, 40), (5000, 7, 1537), (40, 300_000, 8)]


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("count,symbols,width", SIZES)
def test_matches_definition(count, symbols, width, kind):
    tokens = draw_tokens(count, symbols)
    weight = rand(symbols, width, kind=kind)
    for scale in (1.0, -2.3):
        check_forward(tokens, weight, scale)
        check_backward(rand(count, width, kind=kind, seed=2), tokens, symbols, scale)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("count,symbols,width", [(2, 1, 520), (255, 3, 65), (256, 90, 511), (257, 90, 512), (513, 70_000, 264), (1023, 6, 256), (1024, 2000, 255)])
def test_few_positions(count, symbols, width, kind):
    """Numbers of positions, and of vectors of a row, at the borders of what the form without a sort takes at a time."""
    tokens = draw_tokens(count, symbols)
    dy = rand(count, width + 3, kind=kind)
    check_backward(dy[:, :width], tokens, symbols, 0.7)
    check_backward(dy[:, 1 : 1 + width], tokens.int(), symbols, padding=0)
    tokens[::3], tokens[1::7] = -1, symbols
    check_backward(dy[:, 3:], tokens, symbols)
    check_backward(dy[:, :width].contiguous(), torch.full_like(tokens, symbols - 1), symbols)
    assert not check_backward(dy[:, 3:], torch.full_like(tokens, symbols), symbols).any()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_one_symbol_everywhere(kind):
    """A run over all tiles."""
    for count in (32, 33, 64, 65, 700, 8192, 8193, 20_000, 65_537):
        tokens = torch.full((count,), 4, device="cuda")
        check_backward(rand(count, 72, kind=kind), tokens, 9)
        tokens[count // 2 :] = 8  # the last symbol, beside the mark of positions without a gradient
        check_backward(rand(count, 72, kind=kind), tokens, 9)


def test_every_symbol_once():
    g = torch.Generator().manual_seed(3)
    tokens = torch.randperm(4096, generator=g).cuda()
    got = check_backward(rand(4096, 40), tokens, 4096)
    assert torch.equal(got[tokens], rand(4096, 40))


def test_many_positions():
    """More than one subtile to a block of the sort, three of its passes, and tiles longer than the least."""
    tokens = draw_tokens(300_000, 300_000)
    check_backward(rand(300_000, 8), tokens, 300_000, padding=1)


@pytest.mark.parametrize("wide", [torch.int64, torch.int32])
def test_padding_and_symbols_outside(wide):
    tokens = draw_tokens(500, 40).to(wide)
    tokens[::7], tokens[3], tokens[11], tokens[12] = 5, 40, -1, torch.iinfo(wide).min
    tokens[13] = torch.iinfo(wide).max
    weight = rand(40, 50, kind=torch.bfloat16)
    check_forward(tokens, weight, 1.0)
    check_forward(tokens, weight, 2.0)
    dy = rand(500, 50, kind=torch.bfloat16)
    dy[tokens == 5] = float("nan")  # not looked at
    got = check_backward(torch.nan_to_num(dy), tokens, 40, padding=5)
    assert torch.equal(tb.embedding_backward(dy, tokens, 40, padding_idx=5), got)
    nothing = torch.full((100,), 5, dtype=wide, device="cuda")
    assert not tb.embedding_backward(dy[:100], nothing, 40, padding_idx=5).any()


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_strides(kind):
    """Views of rows at any distance and on any element; other views; and the memory around them stays as it was."""
    tokens = draw_tokens(77, 60).view(7, 11)
    big = rand(130, 120, kind=kind)
    for w in (big[3:63, 5:108], big[:120:2, 1:65], big.flip(0)[:60], big[0].expand(60, 120), big.t()[:60, :100], big[:60, ::2]):
        check_forward(tokens, w, 1.0)
        check_forward(tokens, w, 0.5)
    check_forward(tokens.t(), big[:60], 1.0)
    check_forward(torch.stack([tokens, tokens], -1)[..., 0], big[:60], 1.0)
    d = rand(14, 11, 200, kind=kind)
    for dy in (d[:7, :, 3:106], d[::2, :, :64], d[:7].transpose(1, 2)[:, :11, :11].transpose(1, 2), d[:1, :, :80].expand(7, 11, 80), d[:7, :, ::3]):
        check_backward(dy, tokens, 60)


def test_ends_of_memory():
    """Rows on odd elements at both ends of an allocation of their own."""
    for offset in range(1, 8):
        flat = rand(offset + 4 * 37, kind=torch.bfloat16)
        weight = flat[offset:].view(4, 37)
        check_forward(torch.tensor([0, 3, 1, 3], device="cuda"), weight, 1.0)
        check_backward(weight, torch.tensor([2, 0, 2, 1], device="cuda"), 3)


def test_no_positions():
    for shape in ((0,), (3, 0), (0, 5)):
        tokens = torch.empty(shape, dtype=torch.int64, device="cuda")
        assert tb.embedding(tokens, rand(5, 8)).shape == (*shape, 8)
        got = tb.embedding_backward(torch.empty(*shape, 8, device="cuda"), tokens, 5)
        assert got.shape == (5, 8) and not got.any()
    one = torch.tensor(3, device="cuda")  # no dimension: one symbol
    assert torch.equal(tb.embedding(one, rand(5, 8)), rand(5, 8)[3])
    assert torch.equal(tb.embedding_backward(rand(8), one, 5)[3], rand(8))


def test_non_finite_values():
    weight = rand(10, 40)
    weight[2, 3], weight[2, 4], weight[4, 1] = float("inf"), float("-inf"), float("nan")
    tokens = torch.tensor([2, 4, 2, 0], device="cuda")
    y = tb.embedding(tokens, weight, scale=2.0)
    assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(weight[tokens] * 2.0)) and bool(y[1, 1].isnan())
    dy = rand(4, 40)
    dy[1, 7], dy[0, 5] = float("nan"), float("inf")
    got = tb.embedding_backward(dy, tokens, 10)
    assert bool(got[4, 7].isnan()) and bool(got[2, 5].isinf()) and int((~got.isfinite()).sum()) == 2


def test_large_offsets():
    """A table beyond 2^31 elements: the last rows are read and written at 64-bit offsets."""
    symbols, width = 140_000, 16_384
    weight = torch.zeros(symbols, width, dtype=torch.bfloat16, device="cuda")
    weight[-2:] = rand(2, width, kind=torch.bfloat16)
    tokens = torch.tensor([symbols - 1, 0, symbols - 2], device="cuda")
    assert torch.equal(tb.embedding(tokens, weight), weight[tokens])
    dy = rand(3, width, kind=torch.bfloat16)
    got = tb.embedding_backward(dy, tokens, symbols)
    assert torch.equal(got[tokens], dy) and not got[1:-2].any()


def test_autograd():
    tokens = draw_tokens(300, 40).view(20, 15)
    weight = rand(40, 33).requires_grad_()
    y = tb.embedding(tokens, weight, scale=1.5, padding_idx=2)
    dy = rand(20, 15, 33, seed=5)
    y.backward(dy)
    assert torch.equal(weight.grad, tb.embedding_backward(dy, tokens, 40, scale=1.5, padding_idx=2))
    # against differences of a sum of squares, in the entries of two symbols (exact but for 32-bit rounding: it is quadratic)
    f = lambda w: float((tb.embedding(tokens, w, scale=1.5).double() ** 2).sum())  # noqa: E731
    (grad,) = torch.autograd.grad((tb.embedding(tokens, weight, scale=1.5) ** 2).sum(), weight)
    for v, c in ((0, 0), (7, 32)):
        up, down = weight.detach().clone(), weight.detach().clone()
        up[v, c] += 0.25
        down[v, c] -= 0.25
        assert abs((f(up) - f(down)) / 0.5 - float(grad[v, c])) <= 1e-4 * (1 + abs(float(grad[v, c])))
    # a gradient that is a broadcast view, and one that is no sum of rows in memory
    y = tb.embedding(tokens, weight)
    (grad,) = torch.autograd.grad(y.sum(), weight)
    assert torch.equal(grad[:, 0], torch.bincount(tokens.flatten(), minlength=40).float())


def test_streams_and_graphs():
    tokens, weight, dy = draw_tokens(3000, 200), rand(200, 64), rand(3000, 64)
    want = tb.embedding(tokens, weight, scale=3.0), tb.embedding_backward(dy, tokens, 200, padding_idx=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tb.embedding(tokens, weight, scale=3.0), tb.embedding_backward(dy, tokens, 200, padding_idx=1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = tb.embedding(tokens, weight, scale=3.0), tb.embedding_backward(dy, tokens, 200, padding_idx=1)
        graphs.append((graph, got))
    tokens.copy_(tokens.flip(0))
    dy.copy_(dy.flip(0).clone())
    for graph, got in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = tb.embedding(tokens, weight, scale=3.0), tb.embedding_backward(dy, tokens, 200, padding_idx=1)
    for _, got in graphs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_few_positions_in_graphs():
    """The form without a sort, captured twice and replayed in turn on other symbols and gradients, and beside itself on two streams."""
    tokens, dy = draw_tokens(300, 200), rand(300, 64)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = tb.embedding_backward(dy, tokens, 200, padding_idx=1)
        graphs.append((graph, got))
    tokens.copy_(tokens.flip(0))
    dy.copy_(dy.flip(0).clone())
    want = check_backward(dy, tokens, 200, padding=1)
    for graph, got in graphs + graphs:
        got.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for s in streams * 4:
        with torch.cuda.stream(s):
            out.append(tb.embedding_backward(dy, tokens, 200, padding_idx=1))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want) for a in out)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_strides_of_sorted_positions(kind):
    """Views of more rows than the form without a sort takes, at odd distances and elements, and at the ends of an allocation of their own."""
    tokens = draw_tokens(1100, 60)
    d = rand(2200, 120, kind=kind)
    for dy in (d[:1100, 3:106], d[::2, :64], d[1099:2199, 1:120], d[:1, :80].expand(1100, 80), d[:1100, ::3]):
        check_backward(dy, tokens, 60)
    for offset in (1, 3):
        check_backward(rand(offset + 1100 * 37, kind=kind)[offset:].view(1100, 37), tokens, 60)
