"""GPU: the gradients of embedding and linear_cross_entropy refuse tensors with a forward-mode tangent, which their results would lose."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import triturus_b200 as tb

pytestmark = pytest.mark.gpu


def given():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(50, 16, generator=g).cuda()
    x = torch.randn(20, 16, generator=g).cuda()
    t = torch.randint(50, (20,), generator=g).cuda()
    return x, w, t


def test_gradients_refuse_tangents():
    x, w, t = given()
    loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
    with fw.dual_level():
        dual = lambda y: fw.make_dual(y, torch.ones_like(y))  # noqa: E731
        calls = [lambda: tb.embedding_backward(dual(x), t, 50), lambda: torch.ops.triturus.embedding_backward(dual(x), t, 50, 1.0, None)]
        for i in range(4):
            args = [dual(y) if i == j else y for j, y in enumerate((torch.ones_like(loss), x, w, lse))]
            calls.append(lambda a=args: tb.linear_cross_entropy_backward(a[0], a[1], a[2], t, a[3]))
            calls.append(lambda a=args: torch.ops.triturus.linear_cross_entropy_backward(a[0], a[1], a[2], t, a[3], 1, -100, True, True))
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        tb.embedding_backward(x, t, 50)
        tb.linear_cross_entropy_backward(torch.ones_like(loss), x, w, t, lse)


def test_forward_over_reverse_is_refused():
    """A tangent that reaches the gradients through what is computed from the results."""
    x, w, t = given()
    leaf = w.clone().requires_grad_()
    with fw.dual_level():
        scale = fw.make_dual(torch.ones((), device="cuda"), torch.ones((), device="cuda"))
        for y in (tb.embedding(t, leaf), tb.linear_cross_entropy(x, leaf, t)):
            with pytest.raises(NotImplementedError):
                torch.autograd.grad((y * scale).sum(), leaf)
