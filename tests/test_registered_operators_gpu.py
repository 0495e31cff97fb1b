"""GPU: the registered operators, compiled, do what the functions of the package do."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu


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
