"""CPU: the registers that the warps of entropy_kernel hand to each other are those that its blocks are launched with; a kernel compiled to another number is refused
by a code that says so."""

import re

from triturus_b200 import _native, build


def test_shares_add_up():
    kernel = (build.CSRC / "entropy_kernel.cuh").read_text()
    host = (build.CSRC / "linear_cross_entropy.cu").read_text()
    (less,) = re.findall(r"setmaxnreg\.dec\.sync\.aligned\.u32 (\d+);", kernel)
    (more,) = re.findall(r"setmaxnreg\.inc\.sync\.aligned\.u32 (\d+);", kernel)
    (launched,) = re.findall(r"numRegs != (\d+)\) return TRITURUS_B200_EREGISTERS", host)
    (epilogue,) = re.findall(r"int EPI_WARPS = (\d+);", kernel)
    less, more, launched, epilogue = int(less), int(more), int(launched), int(epilogue)
    assert 4 * less + epilogue * more <= (4 + epilogue) * launched <= 65536 // 32
    assert less % 8 == more % 8 == 0


def test_the_code_gives_the_reason():
    assert "registers" in _native.strerror(-8) and "168" in _native.strerror(-8)
