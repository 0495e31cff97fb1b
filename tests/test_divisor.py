"""Division by a constant of the host (csrc/divisor.cuh), compiled for the CPU: around the multiples of small and large divisors, up to 2^31 - 1."""

import ctypes
import random
import shutil
import subprocess

import pytest

from triturus_b200 import build

MOST = 2**31 - 1


@pytest.fixture(scope="module")
def divide(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    tmp = tmp_path_factory.mktemp("divisor")
    src = tmp / "divisor.cpp"
    src.write_text(
        f'#include "{build.CSRC / "divisor.cuh"}"\n'
        'extern "C" long wrong(int d, const int* n, long count) {\n'
        "  const tb200::Divisor by(d);\n  long bad = 0;\n  for (long i = 0; i < count; ++i) bad += by(n[i]) != n[i] / d;\n  return bad;\n}\n"
    )
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(tmp / "divisor.so"), str(src)], check=True)
    lib = ctypes.CDLL(str(tmp / "divisor.so"))
    lib.wrong.restype = ctypes.c_long
    return lambda d, n: lib.wrong(d, (ctypes.c_int * len(n))(*n), ctypes.c_long(len(n)))


def test_quotients(divide):
    rng = random.Random(1)
    divisors = [*range(1, 300), *(2**k + e for k in range(8, 31) for e in (-1, 0, 1)), MOST - 1, MOST, *(rng.randrange(1, MOST) for _ in range(300))]
    for d in divisors:
        multiples = [d * k for k in (0, 1, 2, 3, MOST // d, rng.randrange(0, MOST // d + 1))]
        n = [x for m in multiples for x in (m - 1, m, m + 1) if 0 <= x <= MOST] + [MOST, MOST - 1, *(rng.randrange(0, MOST) for _ in range(50))]
        assert divide(d, n) == 0, d
