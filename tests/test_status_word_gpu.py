"""GPU: the status word of a device, whatever mode the first call that needs it runs in; each in a process of its own."""

import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

START = """
import ctypes
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import triturus_b200 as tb
from triturus_b200 import _native

def given():
    return torch.ones(20, 16, device="cuda"), torch.ones(50, 16, device="cuda"), torch.ones(20, dtype=torch.int64, device="cuda")

def timed_out():
    # a wait that gives up after a moment leaves its code, which is reported once
    word = _native._status_word(torch.device("cuda", 0))
    assert type(word) is torch.Tensor and _native._status_address(given()[0]) == word.data_ptr() != 0
    assert _native.LIB.triturus_b200_selftest_wait_timeout(word.data_ptr(), 100000, torch.cuda.current_stream().cuda_stream) == 0
    try:
        tb.check_status()
    except tb.NativeLibraryError as e:
        assert "105" in str(e), e
    else:
        raise AssertionError("not reported")
    tb.check_status()
"""


def run(code):
    root = Path(__file__).resolve().parent.parent
    done = subprocess.run([sys.executable, "-c", START + textwrap.dedent(code)], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_after_inference_mode():
    run("""
    with torch.inference_mode():
        tb.linear_cross_entropy(*given())
    timed_out()
    """)


def test_after_fake_tensors():
    run("""
    with FakeTensorMode():
        try:
            tb.linear_cross_entropy(*given())
        except Exception:
            pass
        else:
            raise AssertionError("there is nothing to compute with")
    tb.linear_cross_entropy(*given())
    timed_out()
    """)
