"""GPU: clip_grad_norm_ and grad_norm while other threads change the list that they were given."""

import sys
import threading

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu


def test_lists_that_lose_their_tensors_meanwhile():
    """The interpreter's lock is free during the launches.  The tensors that the call began with are its own until it ends: those of a list
    that another thread empties and fills again all hold ones, and so does whatever takes their memory."""
    n, size = 8, 5000
    grads = [torch.ones(size, device="cuda") for _ in range(n)]
    want = float(tb.grad_norm(grads))
    stop = threading.Event()

    def change():
        while not stop.is_set():
            fresh = [torch.ones(size, device="cuda") for _ in range(n)]
            for i in range(n):
                grads[i] = fresh[i]

    switch = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    other = threading.Thread(target=change)
    other.start()
    try:
        norms = []
        for _ in range(1500):
            norms.append(tb.clip_grad_norm_(grads, 1e6))
            norms.append(tb.grad_norm(grads))
    finally:
        stop.set()
        other.join()
        sys.setswitchinterval(switch)
    assert bool((torch.stack(norms) == want).all())
    kept = [torch.full((size,), 2.0, device="cuda") for _ in range(n)]
    versions = [t._version for t in kept]
    tb.clip_grad_norm_(kept, 1e6)
    assert [t._version for t in kept] == [v + 1 for v in versions]
