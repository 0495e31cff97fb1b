"""CPU: layer_norm, clip_grad_norm_ and sample refuse what they cannot take; nothing here launches a kernel."""

import ctypes
import math

import pytest
import torch

import triturus_b200 as tb
from triturus_b200 import _native

LIB = _native.LIB
NULL = None
HERE = 4096  # never read: every call below is refused, or has no rows


def test_layer_norm_codes():
    f = LIB.triturus_b200_layer_norm
    good = [HERE, NULL, NULL, HERE, NULL, NULL, 3, 8, 8, 0, 0, 1e-5, NULL]

    def call(**change):
        names = ["x", "weight", "bias", "y", "mean", "rstd", "rows", "width", "stride", "type", "weight_type", "eps", "stream"]
        return f(*[change.get(n, v) for n, v in zip(names, good)])

    assert call(rows=0) == 0
    assert call(x=NULL) == -1 and call(y=NULL) == -1
    assert call(rows=-1) == -1 and call(width=0) == -1 and call(width=1 << 31) == -1
    assert call(type=3) == -1 and call(type=-1) == -1
    assert call(type=1, weight_type=2) == -1 and call(type=0, weight_type=1) == -1
    assert call(x=HERE + 2) == -2 and call(y=HERE + 1) == -2 and call(mean=HERE + 2) == -2
    assert call(type=1, weight_type=1, x=HERE + 1) == -2 and call(weight=HERE + 2) == -2


def test_layer_norm_backward_codes():
    f = LIB.triturus_b200_layer_norm_backward
    need = LIB.triturus_b200_layer_norm_backward_workspace_bytes(5, 8, 0)
    assert need >= 2 * 8 * 4 and LIB.triturus_b200_layer_norm_backward_workspace_bytes(5, 0, 0) == 0
    names = ["dy", "x", "weight", "mean", "rstd", "dx", "dweight", "dbias", "rows", "width", "dy_stride", "x_stride", "type", "weight_type", "ws", "bytes", "stream"]
    good = [HERE, HERE, NULL, HERE, HERE, HERE, HERE, HERE, 5, 8, 8, 8, 0, 0, HERE, need, NULL]

    def call(**change):
        return f(*[change.get(n, v) for n, v in zip(names, good)])

    for name in ("dy", "x", "mean", "rstd", "dx", "ws"):
        assert call(**{name: NULL}) == -1
    assert call(rows=-2) == -1 and call(width=-1) == -1 and call(type=7) == -1
    assert call(bytes=need - 1) == -3
    assert call(dy=HERE + 2) == -2 and call(ws=HERE + 8) == -2 and call(dweight=HERE + 1) == -2
    assert call(rows=0, dweight=NULL, dbias=NULL) == 0


def test_clip_codes():
    f = LIB.triturus_b200_clip_grad_norm
    need = LIB.triturus_b200_clip_grad_norm_workspace_bytes(2)
    assert need > 0 and LIB.triturus_b200_clip_grad_norm_workspace_bytes(-1) == 0
    assert LIB.triturus_b200_clip_grad_norm_workspace_bytes(5000) > need

    def call(data=(HERE, HERE * 2), numels=(4, 4), types=(0, 1), count=2, limit=1.0, norm=HERE, ws=HERE, nbytes=need, arrays=True):
        n = len(data)
        a = ((ctypes.c_void_p * n)(*data), (ctypes.c_int64 * n)(*numels), (ctypes.c_int * n)(*types)) if arrays else (None, None, None)
        return f(*a, count, limit, 0, 1, norm, ws, nbytes, NULL)

    assert call(count=-1) == -1 and call(arrays=False) == -1
    assert call(norm=NULL) == -1 and call(ws=NULL) == -1
    assert call(limit=-1.0) == -1 and call(limit=math.nan) == -1
    assert call(numels=(4, -1)) == -1 and call(types=(0, 3)) == -1 and call(data=(HERE, NULL)) == -1
    assert call(data=(HERE + 2, HERE)) == -2 and call(data=(HERE, HERE + 1)) == -2 and call(norm=HERE + 2) == -2 and call(ws=HERE + 4) == -2
    assert call(nbytes=need - 8) == -3


def test_sample_codes():
    f = LIB.triturus_b200_sample
    names = ["logits", "noise", "token", "logprob", "rows", "symbols", "stride", "noise_stride", "type", "t", "t0", "k", "k0", "p", "p0", "m", "m0", "stream"]
    good = [HERE, HERE, HERE, HERE, 2, 10, 10, 10, 0, NULL, 1.0, NULL, 0, NULL, 1.0, NULL, 0.0, NULL]

    def call(**change):
        return f(*[change.get(n, v) for n, v in zip(names, good)])

    assert call(rows=0) == 0
    for name in ("logits", "noise", "token"):
        assert call(**{name: NULL}) == -1
    assert call(rows=-1) == -1 and call(symbols=0) == -1 and call(symbols=(1 << 30) + 1) == -1 and call(rows=1 << 28) == -1
    assert call(type=3) == -1
    assert call(logits=HERE + 2) == -2 and call(token=HERE + 4) == -2 and call(noise=HERE + 1) == -2
    for name in ("logprob", "t", "k", "p", "m"):
        assert call(**{name: HERE + 2}) == -2


def test_cpu_tensors_are_refused():
    x, q = torch.randn(3, 8), torch.rand(3, 8)
    stats = torch.ones(3)
    for call in (
        lambda: tb.layer_norm(x),
        lambda: tb.layer_norm(x.requires_grad_(), torch.ones(8)),
        lambda: tb.layer_norm_backward(q, q, stats, stats),
        lambda: tb.clip_grad_norm_([q], 1.0),
        lambda: tb.grad_norm([q]),
        lambda: tb.sample(q, q),
    ):
        with pytest.raises(tb.NativeLibraryError, match="CUDA"):
            call()


def test_arguments_are_checked_before_the_device():
    x = torch.randn(3, 8)
    with pytest.raises(AssertionError):
        tb.layer_norm(x.double())
    with pytest.raises(AssertionError):
        tb.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="no elements"):
        tb.layer_norm(torch.empty(3, 0))
    with pytest.raises(ValueError, match="max_norm"):
        tb.clip_grad_norm_([x], -0.5)
    with pytest.raises(ValueError, match="norm_type"):
        tb.clip_grad_norm_([x], 0.5, norm_type=3.0)
    for bad in (dict(temperature=-1.0), dict(top_k=0), dict(top_p=1.5), dict(min_p=-0.1)):
        with pytest.raises(ValueError, match="out of range"):
            tb.sample(x, x, **bad)
    with pytest.raises(AssertionError):
        tb.sample(x, x[:2])


def test_operators_trace_without_a_device():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(4, 6, 40, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(40, device="cuda")
        y, mean, rstd = torch.ops.triturus.layer_norm(x, w, None, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == (4, 6) and rstd.dtype == torch.float32
        dx, dw, db = torch.ops.triturus.layer_norm_backward(x, x, mean, rstd, w, True, False)
        assert dx.shape == x.shape and dw.shape == (40,) and dw.dtype == torch.float32 and db.shape == (0,)
        assert torch.ops.triturus.clip_grad_norm_([x, w], 1.0, False).shape == ()
        token, logprob = torch.ops.triturus.sample(x, torch.empty(4, 6, 40, device="cuda"), None, 1.0, None, 5, None, 1.0, None, 0.0)
        assert token.shape == logprob.shape == (4, 6) and token.dtype == torch.int64
