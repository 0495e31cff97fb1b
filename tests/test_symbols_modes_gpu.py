"""GPU: embedding and linear_cross_entropy as registered operators, compiled, under the modes of differentiation, and their launches refused."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import triturus_b200 as tb
from triturus_b200 import _native

pytestmark = pytest.mark.gpu

OPS = torch.ops.triturus


def given():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(300, 40, generator=g).cuda()
    tokens = torch.randint(300, (7, 30), generator=g).cuda()
    target = torch.randint(300, (7, 30), generator=g).cuda()
    target[:, 25:] = -100
    return w, tokens, target


def test_compiled_calls():
    """Traced as a whole, with the same results and gradients."""
    compiled = lambda f: torch.compile(f, backend="aot_eager", fullgraph=True)  # noqa: E731
    w, tokens, target = given()

    def model(t):
        h = tb.embedding(tokens, t, scale=2.0, padding_idx=3)
        loss, lse = tb.linear_cross_entropy(h, t, target, return_lse=True)
        return loss, lse, h

    results = []
    for f in (model, compiled(model)):
        leaf = w.clone().requires_grad_()
        loss, lse, h = f(leaf)
        assert not lse.requires_grad
        results.append((loss.detach(), lse, h.detach(), *torch.autograd.grad(loss, leaf)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    h, (loss, lse) = results[0][2], results[0][:2]
    dy = torch.ones_like(h)
    assert torch.equal(compiled(lambda t: tb.embedding_backward(t, tokens, 300))(dy), tb.embedding_backward(dy, tokens, 300))
    got = compiled(lambda t: tb.linear_cross_entropy_backward(torch.ones_like(loss), t, w, target, lse, weight_grad=False))(h)
    want = tb.linear_cross_entropy_backward(torch.ones_like(loss), h, w, target, lse, weight_grad=False)
    assert torch.equal(got[0], want[0]) and got[1] is None and want[1] is None


def test_registered_operators():
    w, tokens, target = given()
    h = tb.embedding(tokens, w)
    assert torch.equal(OPS.embedding(tokens, w, 1.0, None), h)
    loss, lse = OPS.linear_cross_entropy(h, w, target, 1, -100)
    assert torch.equal(loss, tb.linear_cross_entropy(h, w, target))
    leaf = w.clone().requires_grad_()
    (grad,) = torch.autograd.grad(OPS.linear_cross_entropy(h, leaf, target, 1, -100)[0], leaf)
    assert torch.equal(grad, tb.linear_cross_entropy_backward(torch.ones_like(loss), h, w, target, lse, x_grad=False)[1])
    for call in (lambda: OPS.embedding(tokens, w.cpu(), 1.0, None), lambda: OPS.linear_cross_entropy(h, w.cpu(), target, 1, -100), lambda: OPS.linear_cross_entropy(h, w, target[:3], 1, -100)):
        with pytest.raises((AssertionError, NotImplementedError, RuntimeError)):
            call()


def test_the_two_ways_to_the_library_agree():
    """Calls through the extension, and those that it leaves to Python."""
    w, tokens, target = given()
    x = tb.embedding(tokens, w)
    loss, lse = tb.linear_cross_entropy(x, w, target, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(_native._linear_cross_entropy_impl(x, w, target, 1, -100), (loss, lse)))
    assert torch.equal(_native._embedding_impl(tokens, w, 1.0), x)
    g = torch.full((), 3.0, device="cuda")
    mine = tb.linear_cross_entropy_backward(g, x, w, target, lse)
    assert all(torch.equal(a, b) for a, b in zip(_native._linear_cross_entropy_backward_impl(g, x, w, target, lse, 1, -100, True, True), mine))
    assert torch.equal(_native._embedding_backward_impl(x, tokens, 300, 1.0, 3), tb.embedding_backward(x, tokens, 300, padding_idx=3))
    # arguments of other Python types
    assert torch.equal(tb.embedding(tokens, w, scale=2), tb.embedding(tokens, w, scale=2.0))
    as_bool, as_int = (tb.linear_cross_entropy(x, w, target, ignore_index=i, reduction="none") for i in (True, 1))
    assert torch.allclose(as_bool, as_int, rtol=0, atol=0, equal_nan=True)  # (the targets of -100 are no symbols then: NaN)
    with torch.inference_mode():
        assert torch.equal(tb.embedding(tokens, w), x) and torch.equal(tb.linear_cross_entropy(x, w, target), loss)


def test_forward_mode_is_refused():
    w, tokens, target = given()
    x = tb.embedding(tokens, w)
    with fw.dual_level():
        dual = fw.make_dual(w, torch.ones_like(w))
        for call in (lambda: tb.embedding(tokens, dual), lambda: tb.linear_cross_entropy(x, dual, target), lambda: tb.linear_cross_entropy(fw.make_dual(x, x), w, target)):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        assert torch.equal(tb.embedding(tokens, w), x)


def test_second_derivatives_are_refused():
    w, tokens, target = given()
    leaf = w.clone().requires_grad_()
    for y in (tb.embedding(tokens, leaf).square().sum(), tb.linear_cross_entropy(tb.embedding(tokens, w), leaf, target)):
        (grad,) = torch.autograd.grad(y, leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grad.sum(), leaf)


ELAUNCH = -5


def test_a_refused_launch_is_not_reported_again():
    """As for the other operators: a capture that was made invalid refuses every launch into it, on the host, and nothing of that is left for
    a call on an ordinary stream."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    lib = _native.LIB
    w, tokens, target = given()
    w16 = w.bfloat16()
    x = tb.embedding(tokens.flatten(), w)
    few, many = x[:60].contiguous(), torch.cat([x, x])
    t_few, t_many = target.flatten()[:60].contiguous(), torch.cat([target.flatten()] * 2)
    lse, one = torch.zeros(500, device="cuda"), torch.ones((), device="cuda")
    out, dw = torch.empty(500, 40, device="cuda"), torch.empty(300, 40, device="cuda")
    space = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    p = lambda t: t.data_ptr()  # noqa: E731
    n = space.numel()
    calls = [
        ("embedding", lambda s: lib.triturus_b200_embedding(p(tokens), 8, p(w), p(out), 210, 300, 40, 40, 0, 1.0, s)),
        ("embedding_backward", lambda s: lib.triturus_b200_embedding_backward(p(x), p(tokens), 8, p(dw), 210, 300, 40, 40, 0, 1.0, -1, p(space), n, s)),
        ("gradients of no rows", lambda s: lib.triturus_b200_embedding_backward(None, None, 8, p(dw), 0, 300, 40, 40, 0, 1.0, -1, None, 0, s)),
        ("few", lambda s: lib.triturus_b200_linear_cross_entropy(p(few), p(w), p(t_few), 8, p(one), p(lse), 60, 300, 40, 40, 40, 0, 2, -100, p(space), n, None, s)),
        ("many", lambda s: lib.triturus_b200_linear_cross_entropy(p(many), p(w), p(t_many), 8, p(one), p(lse), 420, 300, 40, 40, 40, 0, 2, -100, p(space), n, None, s)),
        ("none", lambda s: lib.triturus_b200_linear_cross_entropy(None, None, None, 8, p(one), None, 0, 300, 40, 40, 40, 0, 2, -100, None, 0, None, s)),
        ("few, gradients", lambda s: lib.triturus_b200_linear_cross_entropy_backward(
            p(one), p(few), p(w), p(t_few), 8, p(lse), p(out), p(dw), 60, 300, 40, 40, 40, 0, 2, -100, p(space), n, None, s)),
        ("many, gradients", lambda s: lib.triturus_b200_linear_cross_entropy_backward(
            p(one), p(many), p(w), p(t_many), 8, p(lse), p(out), p(dw), 420, 300, 40, 40, 40, 0, 2, -100, p(space), n, None, s)),
        ("16 bits", lambda s: lib.triturus_b200_linear_cross_entropy(
            p(w16), p(w16), p(t_many), 8, p(one), p(lse), 300, 300, 40, 40, 40, 1, 2, -100, p(space), n, None, s)),
    ]  # fmt: skip
    main = torch.cuda.current_stream().cuda_stream
    for name, call in calls:
        assert call(main) == 0, name
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    mode = runtime.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed
    for first, refused in calls:
        (err,) = runtime.cudaStreamBeginCapture(side.cuda_stream, mode)
        assert int(err) == 0
        (err,) = runtime.cudaStreamSynchronize(side.cuda_stream)  # not allowed in a capture: ends its validity
        assert int(err) != 0
        rc = refused(side.cuda_stream)
        err, _graph = runtime.cudaStreamEndCapture(side.cuda_stream)
        assert int(err) != 0
        runtime.cudaGetLastError()
        assert rc == ELAUNCH, first
        for name, call in calls:
            assert call(main) == 0, (first, name)
    torch.cuda.synchronize()
