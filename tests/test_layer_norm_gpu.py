"""GPU: layer_norm and layer_norm_backward against their formulas in float64 on the CPU, elementwise.

Bounds.  u = 2^-24 is the rounding of a 32-bit operation.  Forward: the error of the mean is at most some 30 u of the mean of |x| (a tree of
sums, up to 16 terms in a thread and 10 levels), the variance's relative error as small again, so
|err y| <= 64 u (|h w| + |b| + rstd |w| max|x|).  Backward, for the same mean and rstd: each of the three terms of dx is off by at most the
same 64 u of what is added up in magnitude.  dweight and dbias add up to `rows` terms one by one: (rows + 64) u of the
sum of magnitudes.  16-bit results are rounded once more, by half a unit of their last place: 2^-9 (bfloat16) or 2^-12 of
the value, doubled here, and the smallest step of float16, 2^-25."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0**-24
KINDS = [torch.float32, torch.bfloat16, torch.float16]
LAST = {torch.float32: 2 * U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-24}


def definition(x, w, b, eps):
    x = x.double().cpu()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double().cpu()
    h = (x - mean) * rstd
    bound = 64 * U * ((h * w).abs() + b.abs() + rstd * w.abs() * x.abs().amax(-1, keepdim=True))
    return h * w + b, mean.squeeze(-1), rstd.squeeze(-1), bound


def check_forward(x, w, b, eps=1e-5):
    y, mean, rstd = tb.layer_norm(x, w, b, eps=eps, return_stats=True)
    want, m, r, bound = definition(x, w, b, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    assert mean.shape == rstd.shape == x.shape[:-1] and mean.dtype == rstd.dtype == torch.float32
    bound = bound + LAST[x.dtype] * want.abs() + LEAST[x.dtype]
    assert bool(((y.double().cpu() - want).abs() <= bound).all())
    top = x.double().cpu().abs().amax(-1) if x.shape[-1] else None
    assert bool(((mean.double().cpu() - m).abs() <= 64 * U * top + 1e-37).all())
    # the relative error of rstd: that of the variance, and of what the error of the mean adds to it
    assert bool(((rstd.double().cpu() - r).abs() <= r * 64 * U * (1 + r * top)).all())
    assert torch.equal(y, tb.layer_norm(x, w, b, eps=eps))
    return mean, rstd


def check_backward(dy, x, mean, rstd, w):
    dx, dw, db = tb.layer_norm_backward(dy, x, mean, rstd, w)
    d, f = dy.double().cpu(), x.double().cpu()
    m, r = mean.double().cpu().unsqueeze(-1), rstd.double().cpu().unsqueeze(-1)
    wf = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    h, g = (f - m) * r, d * wf
    want = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    bound = 64 * U * r * (g.abs() + g.abs().mean(-1, keepdim=True) + h.abs() * (g * h).abs().mean(-1, keepdim=True))
    assert dx.shape == x.shape and dx.dtype == x.dtype
    assert bool(((dx.double().cpu() - want).abs() <= bound + LAST[x.dtype] * want.abs() + LEAST[x.dtype]).all())
    kind = x.dtype if w is None else w.dtype
    n = mean.numel()
    for got, terms in ((dw, d * h), (db, d)):
        assert got.shape == x.shape[-1:] and got.dtype == kind
        terms = terms.reshape(-1, x.shape[-1])
        s = terms.sum(0)
        assert bool(((got.double().cpu() - s).abs() <= (n + 64) * U * terms.abs().sum(0) + LAST[kind] * s.abs() + LEAST[kind]).all())
    again = tb.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def inputs(rows, width, kind, weights):
    g = torch.Generator().manual_seed(rows * 100003 + width)
    x = (torch.randn(rows, width, generator=g) * torch.exp(torch.randn(width, generator=g)) + 2 * torch.randn(width, generator=g)).to(kind).cuda()
    dy = torch.randn(rows, width, generator=g).to(kind).cuda()
    w = b = None
    if weights:
        wk = kind if weights == "same" else torch.float32
        w, b = (1 + 0.2 * torch.randn(width, generator=g)).to(wk).cuda(), torch.randn(width, generator=g).to(wk).cuda()
    return x, dy, w, b


SIZES = [(1, 1), (3, 2), (4, 7), (1, 32), (5, 33), (300, 64), (9, 1000), (17, 513), (2, 1537), (600, 130), (33, 4096), (5, 8190), (3, 16384), (2, 16387), (3, 32768), (2, 40001)]


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,width", SIZES)
def test_matches_definition(rows, width, kind):
    for weights in ("same",) if kind == torch.float32 else ("same", "f32"):
        x, dy, w, b = inputs(rows, width, kind, weights)
        check_backward(dy, x, *check_forward(x, w, b), w)


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "bf16", "f16"])
def test_without_weight_or_bias(kind):
    x, dy, w, b = inputs(21, 200, kind, "same")
    check_backward(dy, x, *check_forward(x, None, None), None)
    check_forward(x, w, None)
    check_forward(x, None, b)
    mean, rstd = tb.layer_norm(x, return_stats=True)[1:]
    full = tb.layer_norm_backward(dy, x, mean, rstd, w)
    for want_w, want_b in ((True, False), (False, True), (False, False)):
        part = tb.layer_norm_backward(dy, x, mean, rstd, w, weight_grad=want_w, bias_grad=want_b)
        assert torch.equal(part[0], full[0])
        assert (part[1] is None) == (not want_w) and (part[2] is None) == (not want_b)
        assert part[1] is None or torch.equal(part[1], full[1])
        assert part[2] is None or torch.equal(part[2], full[2])


@pytest.mark.parametrize("kind", KINDS, ids=["f32", "bf16", "f16"])
def test_strides(kind):
    g = torch.Generator().manual_seed(5)
    base = torch.randn(40, 3, 1100, generator=g).to(kind).cuda()
    w = torch.randn(1000, generator=g).to(kind).cuda()
    # rows of a wider tensor at an odd offset, a transposed view, every other element, a middle dimension, one row for all
    for x in (base[:, 1, 3:1003], base[:, 0, 1:1001], base[0].t()[:1000].t(), base[:, 2, 50:1050], base[:, :, :1000], base[::2, 0, ::1][:, 7:1007],
              torch.randn(1000, 30, generator=g).to(kind).cuda().t(), torch.randn(20, 2000, generator=g).to(kind).cuda()[:, ::2],
              base[3, 1, :1000].expand(25, 1000)):  # fmt: skip
        mean, rstd = check_forward(x, w, None)
        dy = torch.randn(x.shape, generator=g).to(kind).cuda()
        check_backward(dy, x, mean, rstd, w)
        check_backward(dy[..., :1].expand(x.shape), x, mean, rstd, w)
    x = torch.randn(64, generator=g).to(kind).cuda()  # one row
    check_backward(x.flip(0), x, *check_forward(x, None, None), None)
    wide = torch.randn(2000, generator=g).to(kind).cuda()[::2]  # a weight that is a view
    check_forward(base[:, 1, :1000], wide, wide)


def test_no_rows():
    x = torch.empty(0, 48, device="cuda")
    y, mean, rstd = tb.layer_norm(x, return_stats=True)
    assert y.shape == (0, 48) and mean.shape == (0,)
    dx, dw, db = tb.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 48) and not bool(dw.any()) and not bool(db.any())


def test_hard_rows():
    """A constant row, rows far from zero, a row of the largest values, rows with NaN and infinity beside ordinary ones."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(8, 300, generator=g)
    x[0] = 3.5
    x[1] += 1e4
    x[2] *= 1e15
    x[3] *= 1e-20
    x = x.cuda()
    check_forward(x, None, None)
    y = tb.layer_norm(x)
    assert not bool(y[0].any())
    x[5, 17] = float("nan")
    x[6, 200] = float("inf")
    z = tb.layer_norm(x)
    assert bool(z[5].isnan().all()) and bool(z[6].isnan().all())
    keep = [0, 1, 2, 3, 4, 7]
    assert torch.equal(z[keep], y[keep])


@pytest.mark.parametrize("rows,width", [(6, 40), (3, 520)])
def test_gradient_against_differences(rows, width):
    """The derivative along a direction, from two evaluations a step of 1e-2 apart: its error is the third derivative's share, some
    1e-4 of the terms, and the rounding of y, 1e-7 / 1e-2 of them; 2e-3 of the sum of magnitudes bounds both."""
    g = torch.Generator().manual_seed(3)
    x, w, b = torch.randn(rows, width, generator=g), 1 + 0.3 * torch.randn(width, generator=g), torch.randn(width, generator=g)
    c, vx, vw, vb = (torch.randn(t.shape, generator=g) for t in (x, x, w, b))
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = tb.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, c.cuda())
    t = 5e-3
    for leaf, direction, grad in zip(range(3), (vx, vw, vb), grads):
        ends = []
        for s in (t, -t):
            moved = [a.clone() for a in (x, w, b)]
            moved[leaf] += s * direction
            ends.append((tb.layer_norm(*(a.cuda() for a in moved)).double().cpu() * c.double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * t)
        along = float((grad.double().cpu() * direction.double()).sum())
        assert abs(slope - along) <= 2e-3 * float(grad.abs().double().cpu().mul(direction.double().abs()).sum() + c.abs().sum())


def test_autograd_and_ops():
    x, dy, w, b = inputs(12, 96, torch.bfloat16, "f32")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y, mean, rstd = tb.layer_norm(*leaves, return_stats=True)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    grads = torch.autograd.grad(y, leaves, dy)
    want = tb.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(grads, want))
    with torch.no_grad():
        assert not tb.layer_norm(*leaves).requires_grad
    (only,) = torch.autograd.grad(tb.layer_norm(x, w, leaves[2]), leaves[2:], dy)
    assert torch.equal(only, want[2])
    # a 32-bit bias without a weight
    (only,) = torch.autograd.grad(tb.layer_norm(x, None, leaves[2]), leaves[2:], dy)
    assert only.dtype == torch.float32
    out = torch.ops.triturus.layer_norm(*leaves, 1e-5)
    assert torch.equal(out[0], y)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(out[0], leaves, dy), want))
    torch.library.opcheck(torch.ops.triturus.layer_norm, (x, w, b, 1e-5), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.triturus.layer_norm_backward, (dy, x, mean, rstd, w, True, False), test_utils=("test_schema", "test_faketensor"))


def test_streams_and_graphs():
    x, dy, w, b = inputs(500, 1536, torch.float32, "same")
    want = tb.layer_norm(x, w, b, return_stats=True)
    back = tb.layer_norm_backward(dy, x, want[1], want[2], w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tb.layer_norm(x, w, b, return_stats=True)
        got_back = tb.layer_norm_backward(dy, x, got[1], got[2], w)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip((*want, *back), (*got, *got_back)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tb.layer_norm(x, w, b, return_stats=True)
        out_back = tb.layer_norm_backward(dy, x, out[1], out[2], w)
    x.copy_(x.flip(0))
    dy.copy_(dy.flip(0))
    graph.replay()
    assert torch.equal(out[0], want[0].flip(0)) and torch.equal(out_back[0], back[0].flip(0))


def test_more_elements_than_32_bits_count():
    rows, width = 262_200, 8192
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(3, width, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    x[-3:] = tail
    y, mean, rstd = tb.layer_norm(x, return_stats=True)
    want = tb.layer_norm(tail, return_stats=True)
    assert torch.equal(y[-3:], want[0]) and torch.equal(mean[-3:], want[1])
    assert not bool(y[-4].any())
    dx = tb.layer_norm_backward(x, x, mean, rstd)[0]
    assert torch.equal(dx[-3:], tb.layer_norm_backward(tail, tail, *want[1:])[0])


def test_refusals():
    x, dy, w, b = inputs(4, 32, torch.float32, "same")
    _, mean, rstd = tb.layer_norm(x, return_stats=True)
    for call in (
        lambda: tb.layer_norm(x.double()),
        lambda: tb.layer_norm(x, w[:31]),
        lambda: tb.layer_norm(x, w.bfloat16()),
        lambda: tb.layer_norm(x, w, b.bfloat16()),
        lambda: tb.layer_norm(x.bfloat16(), w.half()),
        lambda: tb.layer_norm(x, w.cpu()),
        lambda: tb.layer_norm(x, w[None]),
        lambda: tb.layer_norm_backward(dy[:3], x, mean, rstd),
        lambda: tb.layer_norm_backward(dy.bfloat16(), x, mean, rstd),
        lambda: tb.layer_norm_backward(dy, x, mean[:3], rstd),
        lambda: tb.layer_norm_backward(dy, x, mean.double(), rstd),
        lambda: tb.layer_norm_backward(dy, x, mean.cpu(), rstd),
    ):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(ValueError, match="no elements"):
        tb.layer_norm(torch.empty(3, 0, device="cuda"))
    with pytest.raises(tb.NativeLibraryError, match="CUDA"):
        tb.layer_norm(x.cpu())
