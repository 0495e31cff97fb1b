"""GPU: layer_norm under the modes of differentiation, and gradients in a type of their own."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0**-24


def test_forward_mode_is_refused():
    """There is no forward-mode derivative: a call that asks for one fails, and does not give a result without a tangent."""
    x, w, b = torch.randn(5, 24, device="cuda"), torch.ones(24, device="cuda"), torch.zeros(24, device="cuda")
    want = tb.layer_norm(x, w, b)
    with fw.dual_level():
        for i in range(3):
            for view in (False, True):
                given = [x, w, b]
                given[i] = fw.make_dual(given[i], torch.ones_like(given[i]))
                if view:
                    given[i] = given[i].view_as(given[i])
                with pytest.raises(NotImplementedError):
                    tb.layer_norm(*given)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    tb.layer_norm(*given, return_stats=True)
        assert torch.equal(tb.layer_norm(x, w, b), want)  # (in a dual level, with ordinary tensors)
    assert torch.equal(tb.layer_norm(x, w, b), want)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows,width", [(50, 200), (700, 33), (3, 20_000)])
def test_gradient_of_a_wide_bias_without_a_weight(rows, width, kind):
    """A bias in 32 bits has a gradient in 32 bits: a sum of `rows` terms one by one, (rows + 64) u of their magnitudes, and no rounding
    to the 16 bits of x."""
    g = torch.Generator().manual_seed(rows + width)
    x = torch.randn(rows, width, generator=g).to(kind).cuda()
    dy = torch.randn(rows, width, generator=g).to(kind).cuda()
    terms = dy.double().cpu()
    bound = (rows + 64) * U * terms.abs().sum(0) + 1e-37
    for call in (lambda bias: tb.layer_norm(x, None, bias), lambda bias: torch.ops.triturus.layer_norm(x, None, bias, 1e-5)[0]):
        bias = torch.randn(width, generator=g).cuda().requires_grad_()
        (grad,) = torch.autograd.grad(call(bias), bias, dy)
        assert grad.dtype == torch.float32
        assert bool(((grad.double().cpu() - terms.sum(0)).abs() <= bound).all())
    leaf = x.clone().requires_grad_()
    dx, db = torch.autograd.grad(tb.layer_norm(leaf, None, bias), (leaf, bias), dy)
    _, mean, rstd = tb.layer_norm(x, None, bias.detach(), return_stats=True)
    assert torch.equal(dx, tb.layer_norm_backward(dy, x, mean, rstd)[0]) and torch.equal(db, grad)


def test_statistics_have_no_gradient():
    """In the registered operator, and where it is compiled, as in the function: a loss of y and the statistics has y's gradient alone, and
    the statistics say so."""
    x = torch.randn(6, 40, device="cuda")
    dy = torch.randn(6, 40, device="cuda")

    def stats(t):
        return tb.layer_norm(t, return_stats=True)

    want = None
    for call in (stats, lambda t: torch.ops.triturus.layer_norm(t, None, None, 1e-5), torch.compile(stats, backend="aot_eager", fullgraph=True)):
        leaf = x.clone().requires_grad_()
        y, mean, rstd = call(leaf)
        assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
        (grad,) = torch.autograd.grad((y * dy).sum() + mean.sum() + rstd.sum(), leaf)
        want = grad if want is None else want
        assert torch.equal(grad, want)
