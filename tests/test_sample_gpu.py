"""GPU: sample against its definition in float64 on the CPU.

Where two scores p / noise, or a sum of p and its limit, are closer than 1e-5 of themselves, 32 bits may decide otherwise: the definition is
evaluated with the limits moved by that to either side, and with the second-best symbol where its score is that close; the token has to be one of
those.  The logarithm's error: (x - max) / T has two roundings, 3 |x - max| / T u for the exponent, which is below 20 where p counts in a sum, the
exponential 4 u, a sum some 30 u: 100 u = 6e-6 for the sum, bounded here by 1e-5, and 8 u of the logarithm itself."""

import math

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0**-24
NEAR = 1e-5
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def definition(x, q, t, k, p, m):
    """[(token, logprob), ...] that a row may give."""
    x = x.double().clamp(max=torch.finfo(F32).max)
    if bool(x.isnan().any()):
        return [(-1, math.nan)]
    if float(x.max()) == -math.inf:
        return [(-1, -math.inf)]
    if not t > 0:
        return [(int(torch.nonzero(x == x.max())[0]), 0.0)]
    order = torch.sort(x, descending=True, stable=True).indices
    pr = torch.exp((x[order] - x.max()) / t)
    pr[x[order] == -math.inf] = 0.0
    n = int((x > -math.inf).sum())
    if k is not None and 1 <= k:
        n = min(n, k)
    found = []
    for move in (0.0, NEAR, -NEAR):
        keep = n
        if p is not None and p < 1:
            upto = torch.cumsum(pr[:n], 0)
            keep = min(n, 1 + int((upto < p * (1 + move) * upto[-1]).sum()))
        if m is not None and m > 0:
            keep = min(keep, max(1, int((pr >= min(m * (1 + move), 1.0)).sum())))
        score = pr[:keep] / q[order[:keep]].double()
        top = float(score.max())
        for i in torch.nonzero(score >= top * (1 - NEAR)).flatten().tolist():
            found.append((int(order[i]), math.log(float(pr[i])) - math.log(float(pr[:keep].sum())) if pr[i] > 0 else -math.inf))
            if score[i] == top:  # (of equal ones the lowest index stands first: all of the top are among them)
                found[0], found[-1] = found[-1], found[0]
    return found


def value(v, i):
    return v.flatten()[i].item() if isinstance(v, torch.Tensor) else v


def check(logits, noise, temperature=1.0, top_k=None, top_p=None, min_p=None):
    given = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    token, logprob = tb.sample(logits, noise, **given, return_logprob=True)
    assert token.shape == logprob.shape == logits.shape[:-1] and token.dtype == torch.int64 and logprob.dtype == F32
    assert torch.equal(token, tb.sample(logits, noise, **given))
    x, q = logits.float().cpu().reshape(-1, logits.shape[-1]), noise.cpu().reshape(-1, logits.shape[-1])
    for i in range(x.shape[0]):
        may = definition(x[i], q[i], *(value(v, i) for v in given.values()))
        tok, lp = int(token.flatten()[i]), float(logprob.flatten()[i])
        assert tok in [a for a, _ in may], (i, tok, may[:4])
        same = [b for a, b in may if a == tok]
        assert any(lp == b or (math.isnan(lp) and math.isnan(b)) or abs(lp - b) <= NEAR + 8 * U * abs(b) for b in same), (i, tok, lp, same)
    return token, logprob


def inputs(rows, symbols, kind=F32, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed * 1009 + symbols)
    x = torch.log_softmax(scale * torch.randn(rows, symbols, generator=g), -1)
    if symbols > 4:
        x[torch.rand(rows, symbols, generator=g) < 0.02] = -math.inf
    return x.to(kind).cuda(), torch.empty(rows, symbols).exponential_(generator=g).cuda()


FILTERS = [dict(), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=20, top_p=0.7, min_p=0.05, temperature=0.6),
           dict(top_k=3000, top_p=0.99, temperature=1.7), dict(top_p=0.999, temperature=3.0), dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0)]  # fmt: skip


@pytest.mark.parametrize("kind", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("symbols", [1, 2, 5, 31, 257, 1000, 4104, 10007, 32768, 50021, 131075])
def test_matches_definition(symbols, kind):
    for n, given in enumerate(FILTERS):
        check(*inputs(3, symbols, kind, n), **given)


@pytest.mark.parametrize("rows", [1, 40, 160])
def test_numbers_of_rows(rows):
    for given in FILTERS[:6]:
        check(*inputs(rows, 6001, F32, rows), **given)


@pytest.mark.parametrize("symbols", [300, 5000, 40_000, 140_000])
def test_equal_values(symbols):
    """Rows of one value, of two, of a few: the first by index are kept."""
    q = inputs(4, symbols, F32, 1)[1]
    x = torch.zeros(4, symbols)
    x[1, ::3] = 1.0
    x[2] = torch.arange(symbols) % 5
    x[3] = -7.25
    x[3, symbols // 2] = -math.inf
    x = x.cuda()
    for given in (dict(), dict(top_k=symbols // 2), dict(top_k=7), dict(top_p=0.5), dict(top_p=0.95, min_p=0.5), dict(top_k=symbols - 1),
                  dict(top_k=symbols // 3, top_p=0.9), dict(top_p=1e-6), dict(temperature=0.0)):  # fmt: skip
        check(x, q, **given)


def test_flat_rows_of_many_values():
    g = torch.Generator().manual_seed(4)
    for kind in (F32, BF16):
        x = (1e-2 * torch.randn(3, 60_000, generator=g)).to(kind).cuda()
        q = torch.empty(3, 60_000).exponential_(generator=g).cuda()
        for given in (dict(top_k=30_000), dict(top_p=0.6), dict(top_k=40_001, top_p=0.3), dict(top_p=0.95, temperature=0.01), dict(top_k=59_999, min_p=0.98)):
            check(x, q, **given)


def test_signs_zeros_and_wide_ranges():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(6, 7000, generator=g)
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3] = torch.where(torch.rand(7000, generator=g) < 0.5, -0.0, 0.0)
    x[4] = x[4].exp().reciprocal() * 1e4
    x[5] = torch.where(x[5] > 0, 3.4e38, -3.4e38)
    q = torch.empty(6, 7000).exponential_(generator=g)
    for given in (dict(), dict(top_k=3500), dict(top_k=4), dict(top_p=0.5), dict(top_p=0.9, temperature=1e-30), dict(top_k=6000, top_p=0.99, temperature=1e30)):
        check(x.cuda(), q.cuda(), **given)


@pytest.mark.parametrize("symbols", [9, 900, 20_000])
def test_rows_that_leave_nothing(symbols):
    x, q = inputs(7, symbols)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, symbols - 1] = -3e38  # the only possible one
    x[2, symbols // 2] = math.nan
    x[3] = math.nan
    x[4, 3] = math.inf
    x[5, 1:] = torch.finfo(F32).min
    for given in FILTERS:
        token, logprob = check(x, q, **given)
        assert token[0] == -1 and logprob[0] == -math.inf and token[2] == -1 and bool(logprob[2].isnan()) and token[4] == 3


def test_parameters_by_row():
    rows = 24
    x, q = inputs(rows, 9000)
    g = torch.Generator().manual_seed(2)
    t = (2 * torch.rand(rows, generator=g) - 0.2).cuda()
    k = torch.randint(-2, 60, (rows,), generator=g).to(torch.int32).cuda()
    p = (1.2 * torch.rand(rows, generator=g)).cuda()
    m = (0.3 * torch.rand(rows, generator=g) - 0.1).cuda()
    check(x, q, t, k, p, m)
    check(x, q, 0.9, k, 0.8, None)
    check(x, q, t, None, p, 0.02)
    check(x.view(4, 6, 9000), q.view(4, 6, 9000), t.view(4, 6), k.view(4, 6), p.view(4, 6), m.view(4, 6))
    every = torch.stack([t, t], 1)[:, 0]  # (not contiguous)
    check(x, q, every, k, p, m)


def test_strides():
    g = torch.Generator().manual_seed(8)
    for kind in (F32, BF16):
        wide = torch.randn(9, 3000, generator=g).to(kind).cuda()
        q = torch.empty(9, 3000).exponential_(generator=g).cuda()
        for given in (dict(), dict(top_k=30, top_p=0.8)):
            for a, b in ((1, 2), (3, 0), (7, 5), (0, 1)):
                check(wide[:, a : a + 2500], q[:, b : b + 2500], **given)
            check(wide[::2, ::3], q[1::2, ::3].contiguous()[[0, 1, 2, 3, 0]], **given)
            # the columns of a circuit's output [R, V, K]: one row per column
            out = torch.randn(2, 300, 5, generator=g).to(kind).cuda().transpose(1, 2)
            check(out, q.reshape(-1)[: 2 * 5 * 300].view(2, 5, 300), **given)
            check(wide[:1].expand(9, 3000), q, **given)
            check(wide[0], q[0], **given)


def test_symbols_beyond_shared_memory():
    g = torch.Generator().manual_seed(12)
    x = torch.randn(2, 8 * 48 * 1024 + 77, generator=g)
    q = torch.empty(x.shape).exponential_(generator=g)
    for kind in (F32, F16):
        for given in (dict(), dict(top_k=40), dict(top_p=0.9), dict(top_k=100_000, top_p=0.5), dict(min_p=0.3)):
            check(x.to(kind).cuda(), q.cuda(), **given)


def test_frequencies():
    """40000 rows of one distribution: chi square of 9 degrees of freedom, below 60 but for one in 10^9."""
    n = 40_000
    x = torch.log_softmax(torch.randn(10, generator=torch.Generator().manual_seed(3)), 0)
    q = torch.empty(n, 10, device="cuda").exponential_(generator=torch.Generator("cuda").manual_seed(3))
    token = tb.sample(x.cuda().expand(n, 10), q)
    want = n * x.double().exp()
    seen = torch.bincount(token.cpu(), minlength=10).double()
    assert float(((seen - want) ** 2 / want).sum()) < 60


def test_streams_graphs_and_ops():
    x, q = inputs(30, 33_000)
    given = dict(temperature=0.8, top_k=100, top_p=0.9)
    want = tb.sample(x, q, **given, return_logprob=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tb.sample(x, q, **given, return_logprob=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tb.sample(x, q, **given, return_logprob=True)
    x.copy_(x.flip(0))
    q.copy_(q.flip(0))
    graph.replay()
    assert all(torch.equal(a.flip(0), b) for a, b in zip(want, out))
    args = (x, q, None, 0.8, None, 100, None, 0.9, None, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(torch.ops.triturus.sample(*args), out))
    torch.library.opcheck(torch.ops.triturus.sample, args, test_utils=("test_schema", "test_faketensor"))
    assert tb.sample(torch.empty(0, 5, device="cuda"), torch.empty(0, 5, device="cuda")).shape == (0,)


def test_more_than_32_bits_count():
    rows, symbols = 70_000, 32_768
    x = torch.zeros(rows, symbols, dtype=BF16, device="cuda")
    tail, q = inputs(2, symbols, BF16, 5)
    x[-2:] = tail
    token = tb.sample(x, q[:1].expand(rows, symbols), top_k=40)
    assert torch.equal(token[-2:], tb.sample(tail, q[:1].expand(2, symbols), top_k=40))
    assert bool((token[:-2] == token[0]).all())


def test_refusals():
    x, q = inputs(4, 40)
    lead = torch.ones(4, device="cuda")
    for call in (
        lambda: tb.sample(x.double(), q),
        lambda: tb.sample(x, q.bfloat16()),
        lambda: tb.sample(x, q[:, :39]),
        lambda: tb.sample(x, q.cpu()),
        lambda: tb.sample(x, q, temperature=lead[:3]),
        lambda: tb.sample(x, q, temperature=lead.double()),
        lambda: tb.sample(x, q, top_k=lead),
        lambda: tb.sample(x, q, top_k=lead.long()),
        lambda: tb.sample(x, q, top_p=lead.cpu()),
        lambda: tb.sample(x, q, min_p=lead[:, None]),
    ):
        with pytest.raises(AssertionError):
            call()
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_k=0), dict(top_k=-1), dict(top_k=2.5),
                dict(top_p=-0.1), dict(top_p=1.01), dict(min_p=-0.1), dict(min_p=1.5), dict(top_p=math.nan)):  # fmt: skip
        with pytest.raises(ValueError, match="out of range"):
            tb.sample(x, q, **bad)
    with pytest.raises(ValueError, match="no symbols"):
        tb.sample(torch.empty(3, 0, device="cuda"), torch.empty(3, 0, device="cuda"))
    with pytest.raises(tb.NativeLibraryError, match="CUDA"):
        tb.sample(x.cpu(), q.cpu())
