"""GPU: a launch that CUDA refuses is reported by the call that made it, and by no later one."""

import pytest
import torch

from triturus_b200 import _native

pytestmark = pytest.mark.gpu

LIB = _native.LIB
ELAUNCH = -5


def _calls():
    """(name, call(stream)) of each entry point, on tensors that are kept with it."""
    x = torch.randn(40, 64, device="cuda")
    long = torch.randn(2, 20_000, device="cuda")
    stat, out = torch.ones(40, device="cuda"), torch.empty(4, 40, 20_000, device="cuda")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    token = torch.empty(40, dtype=torch.int64, device="cuda")
    p = [t.data_ptr() for t in (x, long, stat, out, ws, token)]
    y, mean, rstd, grad = (out[i].data_ptr() for i in range(4))
    one = (_native.c_void_p * 1)(p[0]), (_native.c_int64 * 1)(x.numel()), (_native.c_int * 1)(0)
    big = (_native.c_void_p * 1)(p[3]), (_native.c_int64 * 1)(out.numel()), (_native.c_int * 1)(0)
    n = len(ws)
    kept = (x, long, stat, out, ws, token)
    return [
        ("layer_norm", lambda s: LIB.triturus_b200_layer_norm(p[0], None, None, y, mean, rstd, 40, 64, 64, 0, 0, 1e-5, s)),
        ("layer_norm of long rows", lambda s: LIB.triturus_b200_layer_norm(p[1], None, None, y, mean, rstd, 2, 20_000, 20_000, 0, 0, 1e-5, s)),
        ("layer_norm_backward", lambda s: LIB.triturus_b200_layer_norm_backward(p[0], p[0], None, p[2], p[2], y, grad, grad, 40, 64, 64, 64, 0, 0, p[4], n, s)),
        ("layer_norm_backward of long rows",
         lambda s: LIB.triturus_b200_layer_norm_backward(p[1], p[1], None, p[2], p[2], y, grad, grad, 2, 20_000, 20_000, 20_000, 0, 0, p[4], n, s)),
        ("gradients of no rows", lambda s: LIB.triturus_b200_layer_norm_backward(None, None, None, None, None, None, grad, grad, 0, 64, 64, 64, 0, 0, p[4], n, s)),
        ("clip_grad_norm, small", lambda s: LIB.triturus_b200_clip_grad_norm(*one, 1, 1.0, 0, 1, rstd, p[4], n, s)),
        ("clip_grad_norm", lambda s: LIB.triturus_b200_clip_grad_norm(*big, 1, 1.0, 0, 1, p[2], p[4], n, s)),
        ("sample", lambda s: LIB.triturus_b200_sample(p[0], p[0], p[5], rstd, 40, 64, 64, 64, 0, None, 1.0, None, 0, None, 1.0, None, 0.0, s)),
    ], kept  # fmt: skip


def test_a_refused_launch_is_not_reported_again():
    """A capture that was made invalid refuses every launch into it, on the host.  None of those refusals is left behind for a
    call on an ordinary stream."""
    runtime = pytest.importorskip("cuda.bindings.runtime")
    calls, kept = _calls()
    main = torch.cuda.current_stream().cuda_stream
    for name, call in calls:
        assert call(main) == 0, name  # (and what a first call sets up is set up)
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
