"""CPU: what the registered operators refuse and tell autograd, on tensors without storage."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import triturus_b200  # noqa: F401


def test_statistics_of_the_registered_layer_norm_have_no_gradient():
    """As in layer_norm itself: a loss of mean or rstd does not get a gradient without their terms."""
    with FakeTensorMode():
        x = torch.empty(4, 40, device="cuda", requires_grad=True)
        w = torch.empty(40, device="cuda", requires_grad=True)
        y, mean, rstd = torch.ops.triturus.layer_norm(x, w, None, 1e-5)
        assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad


def test_registered_operators_check_their_arguments():
    """Called by themselves, they refuse what the functions of the package refuse, before anything is read."""
    ops = torch.ops.triturus
    with FakeTensorMode():
        x, q = torch.empty(4, 32, device="cuda"), torch.empty(4, 32, device="cuda")
        half, w, lead = x.bfloat16(), torch.empty(32, device="cuda"), torch.empty(4, device="cuda")

        def sample(logits=x, noise=q, t=None, k=None, p=None, m=None):
            return ops.sample(logits, noise, t, 1.0, k, 0, p, 1.0, m, 0.0)

        for call in (
            lambda: ops.layer_norm(x.double(), None, None, 1e-5),
            lambda: ops.layer_norm(x, w[:31], None, 1e-5),
            lambda: ops.layer_norm(x, None, w[:31], 1e-5),
            lambda: ops.layer_norm(x, w.half(), None, 1e-5),
            lambda: ops.layer_norm(half, w, w.bfloat16(), 1e-5),
            lambda: ops.layer_norm_backward(x[:3], x, lead, lead, None, True, True),
            lambda: ops.layer_norm_backward(half, x, lead, lead, None, True, True),
            lambda: ops.layer_norm_backward(x, x, lead[:3], lead, None, True, True),
            lambda: ops.layer_norm_backward(x, x, lead, lead.double(), None, True, True),
            lambda: ops.layer_norm_backward(x, x, lead, lead, w[:31], True, True),
            lambda: ops.clip_grad_norm_([x, x.double()], 1.0, False),
            lambda: ops.grad_norm([x.double()], False),
            lambda: sample(x.double()),
            lambda: sample(noise=q[:, :31]),
            lambda: sample(noise=q.half()),
            lambda: sample(t=lead[:3]),
            lambda: sample(k=lead),
            lambda: sample(p=lead.double()),
            lambda: sample(m=lead[:, None]),
        ):
            with pytest.raises(AssertionError):
                call()
        empty = torch.empty(4, 0, device="cuda")
        for call, what in (
            (lambda: ops.layer_norm(empty, None, None, 1e-5), "no elements"),
            (lambda: sample(empty, empty), "no symbols"),
            (lambda: ops.clip_grad_norm_([x[:1].expand(5, 32)], 1.0, False), "expanded"),
        ):
            with pytest.raises(ValueError, match=what):
                call()
