"""Operands of linear_cross_entropy whose rows overlap (windows that slide over a signal): copied, since a tensor map describes rows that lie one behind the other."""

import pytest
import torch

import triturus_b200 as tb
from triturus_b200 import _native

HERE = 4096  # never read


@pytest.mark.parametrize("kind,size", [(0, 4), (1, 2), (2, 2)])
def test_room_for_a_copy(kind, size):
    rows, symbols, width = 40, 70, 128
    need = _native.LIB.triturus_b200_linear_cross_entropy_workspace_bytes
    for which, count in (("x", rows), ("weight", symbols)):
        if kind == 0 and which == "x":
            continue  # (copied in any case)
        apart = {"x": width, "weight": width}
        whole = need(HERE, HERE, rows, symbols, width, apart["x"], apart["weight"], kind)
        for step in (32, 64, width - 64):
            apart[which] = step
            assert need(HERE, HERE, rows, symbols, width, apart["x"], apart["weight"], kind) == whole + count * width * size


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [40, 300, 2500])
def test_sliding_windows(n, kind):
    g = torch.Generator().manual_seed(n)
    signal = torch.randn(32 * n + 200, generator=g).to(kind).cuda()
    table = (0.1 * torch.randn(32 * 90 + 200, generator=g)).to(kind).cuda()
    t = torch.randint(90, (n,), generator=g).cuda()
    for width in (64, 130):
        x, w = signal.unfold(0, width, 32)[:n], table.unfold(0, width, 32)[:90]
        results = []
        for a, b in ((x, w), (x.contiguous(), w.contiguous())):
            loss, lse = tb.linear_cross_entropy(a, b, t, return_lse=True)
            results.append((loss, lse, *tb.linear_cross_entropy_backward(torch.ones_like(loss), a, b, t, lse)))
        assert all(torch.equal(a, b) for a, b in zip(*results))
    tb.check_status()
