"""The norms around a block without columns: sums over nothing are zero."""

import pytest
import torch

from evograd_amd.pairs import block_norm as pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16, torch.float32))
@pytest.mark.parametrize("gate", ("none", "channel", "row", "element"))
@pytest.mark.parametrize("rows", (0, 1, 700))
def test_no_columns(rows, gate, dtype):
    x, w = torch.empty(rows, 0, dtype=dtype, device="cuda"), torch.empty(0, dtype=dtype, device="cuda")
    g = {"none": None, "channel": w, "row": torch.ones(rows, 1, dtype=dtype, device="cuda"),
         "element": x}[gate]
    out, saved = pair.block_norm_forward_with_saved(x, x, w, g, w)
    assert out.shape == (2, rows, 0)
    # what the allocator hands out next holds ones
    held = [torch.ones(max(rows, 1), 1, dtype=dtype, device="cuda") for _ in range(8)]
    del held
    dx, dh, dpost, dgate, dpre = pair.block_norm_backward_from_saved(out, saved)
    assert dx.shape == dh.shape == (rows, 0) and dpost.shape == dpre.shape == (0,)
    if gate == "none":
        assert dgate is None
    else:
        assert dgate.shape == g.shape and int(torch.count_nonzero(dgate)) == 0
