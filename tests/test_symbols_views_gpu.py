"""GPU: embedding and linear_cross_entropy of tensors whose memory holds their negatives (the imaginary part of a conjugate, for one)."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu

neg = torch._neg_view


def given(width):
    g = torch.Generator().manual_seed(width)
    w = torch.randn(50, width, generator=g).cuda()
    x = torch.randn(20, width, generator=g).cuda()
    t = torch.randint(50, (20,), generator=g).cuda()
    return x, w, t


def same(got, want):
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("width", [1, 16])
def test_negative_views(width):
    x, w, t = given(width)
    y, d = tb.embedding(t, w, scale=0.5), tb.embedding_backward(x, t, 50)
    loss, lse = tb.linear_cross_entropy(x, w, t, return_lse=True)
    one = torch.full_like(loss, 3.0)
    grads = tb.linear_cross_entropy_backward(one, x, w, t, lse)
    assert neg(-w).is_neg() and neg(-w).is_contiguous()
    same([tb.embedding(t, neg(-w), scale=0.5), tb.embedding(neg(-t), w, scale=0.5)], [y, y])
    same([tb.embedding_backward(neg(-x), t, 50), tb.embedding_backward(x, neg(-t), 50)], [d, d])
    args = x, w, t
    for i in range(3):
        same(tb.linear_cross_entropy(*(neg(-a) if i == j else a for j, a in enumerate(args)), return_lse=True), (loss, lse))
    args = one, x, w, t, lse
    for i in range(5):
        same(tb.linear_cross_entropy_backward(*(neg(-a) if i == j else a for j, a in enumerate(args))), grads)
    leaf = w.clone().requires_grad_()
    (grad,) = torch.autograd.grad(tb.linear_cross_entropy(neg(-x), leaf, t), leaf)
    same([grad], [tb.linear_cross_entropy_backward(torch.ones_like(loss), x, w, t, lse)[1]])


@pytest.mark.parametrize("width", [1, 16])
def test_imaginary_parts_of_conjugates(width):
    x, w, t = given(width)
    a, b = (torch.complex(torch.zeros_like(y), -y).conj().imag for y in (x, w))
    assert a.is_neg() and torch.equal(a, x)
    same([tb.embedding(t, b), tb.embedding_backward(a, t, 50)], [tb.embedding(t, w), tb.embedding_backward(x, t, 50)])
    same(tb.linear_cross_entropy(a, b, t, return_lse=True), tb.linear_cross_entropy(x, w, t, return_lse=True))
