"""Radix selection's ranges of keys (csrc/key_range.cuh), compiled for the CPU: over all of the 32 bits, where the widths of the first bins reach
beyond either end."""

import ctypes
import random
import shutil
import struct
import subprocess

import pytest

from triturus_b200 import build

LEAST, MOST = -3.4028234663852886e38, 3.4028234663852886e38


@pytest.fixture(scope="module")
def keys(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    tmp = tmp_path_factory.mktemp("key_range")
    src = tmp / "key_range.cpp"
    src.write_text(
        f'#include "{build.CSRC / "key_range.cuh"}"\n'
        "using tb200::KeyRange;\n"
        'extern "C" int shift(uint32_t lo, uint32_t hi) { return KeyRange{lo, hi}.shift(); }\n'
        'extern "C" void bin(uint32_t lo, uint32_t hi, uint32_t b, int s, int up, uint32_t* out) {\n'
        "  const KeyRange r = up ? KeyRange{lo, hi}.bin_upwards(b, s) : KeyRange{lo, hi}.bin_downwards(b, s);\n  out[0] = r.lo, out[1] = r.hi;\n}\n"
        'extern "C" int rounds() { return tb200::kKeyRounds; }\n'
    )
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(tmp / "key_range.so"), str(src)], check=True)
    lib = ctypes.CDLL(str(tmp / "key_range.so"))
    lib.shift.argtypes = [ctypes.c_uint32] * 2
    lib.bin.argtypes = [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_uint32)]
    return lib


def key_of(x):
    """A 32-bit float's bits in the order of the values, as the kernel makes them."""
    u = struct.unpack("<I", struct.pack("<f", x))[0]
    return u ^ (0xFFFFFFFF if u >> 31 else 0x80000000)


def select(lib, values, rank, up):
    """The key of that rank (from the lowest, or from the highest downwards), by the kernel's rounds."""
    lo, hi = min(values), max(values)
    order = sorted(values, reverse=not up)
    out = (ctypes.c_uint32 * 2)()
    before = 0
    for _ in range(lib.rounds()):
        s = lib.shift(lo, hi)
        assert (hi - lo) >> s < 256 and (s == 0 or (hi - lo) >> (s - 1) >= 256)
        places = [((v - lo) if up else (hi - v)) >> s for v in values if lo <= v <= hi]
        assert places  # never an empty range
        for b in sorted(set(places)):
            if before + places.count(b) >= rank:
                break
            before += places.count(b)
        was = lo, hi
        lib.bin(lo, hi, b, s, int(up), out)
        lo, hi = out
        assert was[0] <= lo <= hi <= was[1] and hi - lo < 1 << s
        assert lo <= order[rank - 1] <= hi
        if s == 0:
            break
    assert lo == hi == order[rank - 1]


@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("first", [0.25, 1.0, 1.5, 4.0, 5.0, 7.0, 16.0, 30.0, 100.0, MOST, 1e-30])
@pytest.mark.parametrize("last", [LEAST, -1e38, -1.8e38, -1.0, 0.0])
def test_a_positive_value_and_one_at_the_other_end(keys, first, last, up):
    flip = 0xFFFFFFFF if up else 0  # (lists are ordered by falling values: the keys inverted)
    values = [key_of(first) ^ flip] * 10 + [key_of(last) ^ flip] * 290
    for rank in (1, 10, 11, 200, 300):
        select(keys, values, rank, up)


@pytest.mark.parametrize("up", [True, False])
def test_ranges_at_both_ends_of_the_keys(keys, up):
    rng = random.Random(5)
    for _ in range(300):
        spans = [rng.randrange(1 << rng.randrange(1, 33)) for _ in range(40)]
        values = [s if rng.random() < 0.5 else 0xFFFFFFFF - s for s in spans]
        if rng.random() < 0.3:
            values += [0, 0xFFFFFFFF]
        select(keys, values, rng.randrange(1, len(values) + 1), up)


def test_every_bin_of_the_widest_ranges(keys):
    out = (ctypes.c_uint32 * 2)()
    for lo, hi in ((0, 0xFFFFFFFF), (1, 0xFFFFFFFF), (0, 0xFFFFFFFE), (0x3F5FFFFF, 0xFF7FFFFF), (0x00800000, 0xC0A00000), (0xFFFFFF00, 0xFFFFFFFF), (0, 255), (7, 7)):
        s = keys.shift(lo, hi)
        for up in (1, 0):
            at = lo if up else hi
            for b in range(((hi - lo) >> s) + 1):
                keys.bin(lo, hi, b, s, up, out)
                assert (out[0] if up else out[1]) == at and lo <= out[0] <= out[1] <= hi
                at = out[1] + 1 if up else out[0] - 1
            assert at == (hi + 1 if up else lo - 1)
