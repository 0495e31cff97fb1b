"""CPU: what the registered operators tell autograd, on tensors without storage."""

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
