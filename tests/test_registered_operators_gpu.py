"""GPU: the registered operators, called by themselves and compiled, check and do what the functions of the package do."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

OPS = torch.ops.triturus


def test_arguments_are_checked():
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    q, lead = torch.rand(4, 32, device="cuda"), torch.ones(4, device="cuda")
    for call in (
        lambda: OPS.layer_norm(x, w[:31], None, 1e-5),
        lambda: OPS.layer_norm(x.bfloat16(), w, w.bfloat16(), 1e-5),
        lambda: OPS.layer_norm(x, w.cpu(), None, 1e-5),
        lambda: OPS.layer_norm_backward(x, x, lead[:3], lead, None, True, True),
        lambda: OPS.layer_norm_backward(x[:, :31], x, lead, lead, None, True, True),
        lambda: OPS.grad_norm([x.double()], False),
        lambda: OPS.sample(x, q[:3], None, 1.0, None, 0, None, 1.0, None, 0.0),
        lambda: OPS.sample(x, q.half(), None, 1.0, None, 0, None, 1.0, None, 0.0),
        lambda: OPS.sample(x, q, lead[:2], 1.0, None, 0, None, 1.0, None, 0.0),
    ):
        with pytest.raises(AssertionError):
            call()
    for call, what in (
        (lambda: OPS.clip_grad_norm_([x, x[1:]], 1.0, False), "share memory"),
        (lambda: OPS.clip_grad_norm_([x[:1].expand(4, 32)], 1.0, False), "expanded"),
        (lambda: OPS.layer_norm(torch.empty(3, 0, device="cuda"), None, None, 1e-5), "no elements"),
    ):
        with pytest.raises(ValueError, match=what):
            call()


def test_compiled_calls():
    """Traced as a whole, with the same results."""
    compiled = lambda f: torch.compile(f, backend="aot_eager", fullgraph=True)  # noqa: E731
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(6, 200, generator=g).cuda(), torch.randn(200, generator=g).cuda()
    q = torch.empty(6, 200).exponential_(generator=g).cuda()
    y, mean, rstd = tb.layer_norm(x, w, return_stats=True)
    assert all(torch.equal(a, b) for a, b in zip(compiled(lambda t: tb.layer_norm(t, w, return_stats=True))(x), (y, mean, rstd)))
    got = compiled(lambda t: tb.layer_norm_backward(t, x, mean, rstd, w, bias_grad=False))(y)
    want = tb.layer_norm_backward(y, x, mean, rstd, w, bias_grad=False)
    assert got[2] is None and all(torch.equal(a, b) for a, b in zip(got[:2], want[:2]))
    assert torch.equal(compiled(lambda t: tb.grad_norm([t, w]))(x), tb.grad_norm([x, w]))
    mine, other = [x.clone(), w.clone()], [x.clone(), w.clone()]
    norm = compiled(lambda a, b: tb.clip_grad_norm_([a, b], 0.5))(*mine)
    assert torch.equal(norm, tb.clip_grad_norm_(other, 0.5)) and all(torch.equal(a, b) for a, b in zip(mine, other))
    given = dict(temperature=0.7, top_k=50, top_p=torch.full((6,), 0.9, device="cuda"), return_logprob=True)
    assert all(torch.equal(a, b) for a, b in zip(compiled(lambda t: tb.sample(t, q, **given))(x), tb.sample(x, q, **given)))
