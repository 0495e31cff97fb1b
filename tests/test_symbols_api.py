"""CPU: embedding and linear_cross_entropy refuse what they cannot take; nothing here launches a kernel."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import triturus_b200 as tb
from triturus_b200 import _native

LIB = _native.LIB
NULL = None
HERE = 4096  # never read: every call below is refused, or has no rows


def test_embedding_codes():
    f = LIB.triturus_b200_embedding
    names = ["tokens", "bytes", "weight", "y", "count", "symbols", "width", "stride", "type", "scale", "stream"]
    good = [HERE, 8, HERE, HERE, 3, 5, 8, 8, 0, 1.0, NULL]

    def call(**change):
        return f(*[change.get(n, v) for n, v in zip(names, good)])

    assert call(count=0) == 0
    for name in ("tokens", "weight", "y"):
        assert call(**{name: NULL}) == -1
    assert call(count=-1) == -1 and call(count=(1 << 30) + 1) == -1 and call(symbols=0) == -1 and call(symbols=1 << 30) == -1
    assert call(width=0) == -1 and call(type=3) == -1 and call(bytes=2) == -1
    assert call(tokens=HERE + 4) == -2 and call(bytes=4, tokens=HERE + 2) == -2 and call(weight=HERE + 2) == -2 and call(y=HERE + 1) == -2


def test_embedding_backward_codes():
    size = LIB.triturus_b200_embedding_backward_workspace_bytes
    need = size(5, 7, 8, 0)
    assert need >= 5 * 16 and size(-1, 7, 8, 0) == 0 and size(5, 0, 8, 0) == 0 and size(5, 7, 8, 4) == 0 and size(0, 7, 8, 1) > 0
    f = LIB.triturus_b200_embedding_backward
    names = ["dy", "tokens", "token_bytes", "dweight", "count", "symbols", "width", "stride", "type", "scale", "padding", "ws", "bytes", "stream"]
    good = [HERE, HERE, 8, HERE, 5, 7, 8, 8, 0, 1.0, -1, HERE, need, NULL]

    def call(**change):
        return f(*[change.get(n, v) for n, v in zip(names, good)])

    for name in ("dy", "tokens", "dweight", "ws"):
        assert call(**{name: NULL}) == -1
    assert call(count=-2) == -1 and call(symbols=-1) == -1 and call(type=9) == -1 and call(token_bytes=1) == -1
    assert call(bytes=need - 1) == -3
    assert call(dy=HERE + 2) == -2 and call(ws=HERE + 8) == -2 and call(dweight=HERE + 1) == -2 and call(tokens=HERE + 1) == -2


NAMES = ["x", "weight", "target", "target_bytes", "loss", "lse", "rows", "symbols", "width", "xs", "ws", "type", "reduction", "ignore", "space", "bytes", "status", "stream"]


def test_linear_cross_entropy_codes():
    size = LIB.triturus_b200_linear_cross_entropy_workspace_bytes
    need = size(HERE, HERE, 5, 7, 8, 8, 8, 1)
    assert need > 0
    assert size(HERE, HERE, 5, 7, 8, 8, 8, 3) == size(HERE, HERE, -1, 7, 8, 8, 8, 1) == size(HERE, HERE, 5, 0, 8, 8, 8, 1) == size(HERE, HERE, 0, 7, 8, 8, 8, 1) == 0
    assert size(HERE + 2, HERE, 5, 7, 8, 8, 8, 1) > need  # a copy of what is off 16-byte boundaries
    f = LIB.triturus_b200_linear_cross_entropy
    good = [HERE, HERE, HERE, 8, HERE, HERE, 5, 7, 8, 8, 8, 1, 1, -100, HERE, need, NULL, NULL]

    def call(**change):
        return f(*[change.get(n, v) for n, v in zip(NAMES, good)])

    assert call(rows=0, reduction=0) == 0
    for name in ("x", "weight", "target", "loss", "lse", "space"):
        assert call(**{name: NULL}) == -1
    assert call(rows=-1) == -1 and call(rows=(1 << 30) + 1) == -1 and call(symbols=0) == -1 and call(width=0) == -1 and call(type=3) == -1
    assert call(reduction=3) == -1 and call(reduction=-1) == -1 and call(target_bytes=1) == -1 and call(rows=0, loss=NULL) == -1
    assert call(bytes=need - 1) == -3
    assert call(x=HERE + 1) == -2 and call(weight=HERE + 1) == -2 and call(target=HERE + 4) == -2 and call(loss=HERE + 2) == -2 and call(lse=HERE + 2) == -2
    assert call(space=HERE + 16) == -2 and call(rows=0, loss=HERE + 2) == -2


def test_linear_cross_entropy_backward_codes():
    need = LIB.triturus_b200_linear_cross_entropy_backward_workspace_bytes(HERE, HERE, 5, 7, 8, 8, 8, 2)
    f = LIB.triturus_b200_linear_cross_entropy_backward
    names = ["dloss", "x", "weight", "target", "target_bytes", "lse", "dx", "dweight", *NAMES[6:]]
    good = [HERE, HERE, HERE, HERE, 8, HERE, HERE, HERE, 5, 7, 8, 8, 8, 2, 1, -100, HERE, need, NULL, NULL]

    def call(**change):
        return f(*[change.get(n, v) for n, v in zip(names, good)])

    for name in ("dloss", "x", "weight", "target", "lse", "space"):
        assert call(**{name: NULL}) == -1
    assert call(dx=NULL, dweight=NULL) == 0 and call(rows=0, dweight=NULL) == 0
    assert call(rows=-1) == -1 and call(symbols=0) == -1 and call(width=-3) == -1 and call(type=-1) == -1 and call(reduction=9) == -1
    assert call(bytes=need - 1) == -3
    assert call(dx=HERE + 1) == -2 and call(dweight=HERE + 1) == -2 and call(dloss=HERE + 2) == -2 and call(space=HERE + 128) == -2
    # sizes up to the limits are planned without a division by zero or a negative size
    for rows in (1, 64, 65, 193, 4096, 1 << 20, 1 << 30):
        for symbols in (1, 255, 70_000, 1 << 30):
            for width in (1, 64, 513, 1 << 20):
                for kind in (0, 1, 2):
                    for size in (LIB.triturus_b200_linear_cross_entropy_workspace_bytes, LIB.triturus_b200_linear_cross_entropy_backward_workspace_bytes):
                        assert 0 < size(HERE, HERE, rows, symbols, width, width, width, kind) < 1 << 63


def test_cpu_tensors_are_refused():
    tokens, weight, x = torch.tensor([1, 2]), torch.randn(5, 8), torch.randn(2, 8)
    lse = torch.zeros(2)
    for call in (
        lambda: tb.embedding(tokens, weight),
        lambda: tb.embedding(tokens, weight.clone().requires_grad_()),
        lambda: tb.embedding_backward(x, tokens, 5),
        lambda: tb.linear_cross_entropy(x, weight, tokens),
        lambda: tb.linear_cross_entropy(x, weight.clone().requires_grad_(), tokens),
        lambda: tb.linear_cross_entropy_backward(torch.ones(()), x, weight, tokens, lse),
    ):
        with pytest.raises(tb.NativeLibraryError, match="CUDA"):
            call()


def test_arguments_are_checked_before_the_device():
    tokens, weight, x = torch.tensor([1, 2]), torch.randn(5, 8), torch.randn(2, 8)
    lse, one = torch.zeros(2), torch.ones(())
    for call in (
        lambda: tb.embedding(tokens.float(), weight),
        lambda: tb.embedding(tokens, weight.double()),
        lambda: tb.embedding(tokens, weight[0]),
        lambda: tb.embedding_backward(x, tokens[:1], 5),
        lambda: tb.embedding_backward(x.double(), tokens, 5),
        lambda: tb.linear_cross_entropy(x, weight[:, :7], tokens),
        lambda: tb.linear_cross_entropy(x, weight.bfloat16(), tokens),
        lambda: tb.linear_cross_entropy(x, weight, tokens[:1]),
        lambda: tb.linear_cross_entropy(x, weight, tokens.short()),
        lambda: tb.linear_cross_entropy_backward(one, x, weight, tokens, lse[:1]),
        lambda: tb.linear_cross_entropy_backward(lse, x, weight, tokens, lse),
        lambda: tb.linear_cross_entropy_backward(one, x, weight, tokens, lse, reduction="none"),
        lambda: tb.linear_cross_entropy_backward(one.double(), x, weight, tokens, lse),
    ):
        with pytest.raises(AssertionError):
            call()
    for call, what in (
        (lambda: tb.embedding(tokens, weight[:, :0]), "not supported"),
        (lambda: tb.embedding(tokens, weight[:0]), "not supported"),
        (lambda: tb.embedding(tokens, weight, scale=float("inf")), "scale"),
        (lambda: tb.embedding(tokens, weight, padding_idx=5), "padding_idx"),
        (lambda: tb.embedding_backward(x, tokens, 5, padding_idx=-1), "padding_idx"),
        (lambda: tb.embedding_backward(x, tokens, 0), "not supported"),
        (lambda: tb.linear_cross_entropy(x, weight, tokens, reduction="max"), "reduction"),
        (lambda: tb.linear_cross_entropy_backward(one, x, weight, tokens, lse, reduction=None), "reduction"),
        (lambda: tb.linear_cross_entropy(x[:, :0], weight[:, :0], tokens), "not supported"),
        (lambda: tb.linear_cross_entropy(x, weight, tokens, ignore_index=2**63), "ignore_index"),
    ):
        with pytest.raises(ValueError, match=what):
            call()


def test_operators_trace_and_check_without_a_device():
    ops = torch.ops.triturus
    with FakeTensorMode():
        tokens = torch.empty(4, 6, dtype=torch.int64, device="cuda")
        w = torch.empty(50, 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = ops.embedding(tokens, w, 2.0, None)
        assert y.shape == (4, 6, 16) and y.dtype == w.dtype and y.requires_grad
        assert ops.embedding_backward(y.detach(), tokens, 50, 1.0, 3).shape == (50, 16)
        loss, lse = ops.linear_cross_entropy(y, w, tokens, 1, -100)
        assert loss.shape == () and lse.shape == (4, 6) and loss.dtype == lse.dtype == torch.float32
        assert loss.requires_grad and not lse.requires_grad
        assert ops.linear_cross_entropy(y, w, tokens, 0, -100)[0].shape == (4, 6)
        dx, dw = ops.linear_cross_entropy_backward(loss.detach(), y.detach(), w.detach(), tokens, lse, 1, -100, True, False)
        assert dx.shape == y.shape and dw.shape == (0,)
        for call in (
            lambda: ops.embedding(tokens.float(), w, 1.0, None),
            lambda: ops.embedding(tokens, w[0], 1.0, None),
            lambda: ops.embedding_backward(y, tokens[:3], 50, 1.0, None),
            lambda: ops.linear_cross_entropy(y, w[:, :15], tokens, 1, -100),
            lambda: ops.linear_cross_entropy(y.float(), w, tokens, 1, -100),
            lambda: ops.linear_cross_entropy_backward(lse, y, w, tokens, lse, 1, -100, True, True),
        ):
            with pytest.raises(AssertionError):
                call()
        for call in (lambda: ops.embedding(tokens, w, 1.0, 50), lambda: ops.embedding(tokens, w, float("nan"), None), lambda: ops.linear_cross_entropy(y, w, tokens, 3, -100)):
            with pytest.raises(ValueError):
                call()
