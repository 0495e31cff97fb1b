"""GPU: rows of the table's gradient beyond what one launch covers."""

import pytest
import torch

import triturus_b200 as tb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("extra", [0, 1, 5])
def test_very_wide_rows(extra):
    """Rows of more than 65535 x 128 vectors of 16 bytes.  Small whole numbers: the sums are exact in every type."""
    width = 65535 * 128 * 8 + extra
    dy = (torch.arange(3 * width, device="cuda") % 251 - 125).to(torch.float16).view(3, width)
    tokens = torch.tensor([2, 0, 2], device="cuda")
    want = torch.zeros(3, width, dtype=torch.float16, device="cuda")
    want[2], want[0] = dy[0] + dy[2], dy[1]
    got = tb.embedding_backward(dy, tokens, 3)
    assert torch.equal(got, want)
    assert torch.equal(tb.embedding(tokens, got), want[tokens])
    tokens = torch.full((130,), 1, device="cuda")  # more than one tile of positions: its parts are joined
    got = tb.embedding_backward(dy[:1].expand(130, width), tokens, 3)
    assert torch.equal(got[1], dy[0] * 130) and not got[0].any() and not got[2].any()
