"""Limits of the packed-batch operators' arguments that the entry points and their wrappers share,
and what their autograd nodes refuse (CPU)."""

import ctypes
import os

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.pairs._util import MAX_HEAD_STRIDE, MAX_TOKEN_STRIDE, head_rows

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
P = 1 << 20  # an address no refused call reads


@built
@pytest.mark.parametrize("at,most", ((0, MAX_TOKEN_STRIDE), (1, MAX_HEAD_STRIDE)))
@pytest.mark.parametrize("which", (0, 2))
def test_rotary_takes_every_step_that_the_wrappers_pass_on(which, at, most):
    """Steps that head_rows leaves as they are (calls without tokens: checked, nothing launched)."""
    def turn(step):
        steps = [64, 64, 64, 64]
        steps[which + at] = step
        _lib.call("eg_rotary", P, P, P, P, P, 0, P, 0, 2, 2, 64, 32, (ctypes.c_int64 * 4)(*steps), 1.0,
                  0, 0, _lib.EG_F32, None)

    turn(most)
    with pytest.raises(RuntimeError, match="strides must"):
        turn((1 << 40) + 1)
    with pytest.raises(RuntimeError, match="strides must"):
        turn(-1)


def test_head_rows_keeps_steps_up_to_the_limits():
    def view(tokens, heads, dim, token, head):
        t = torch.empty((tokens - 1) * token + (heads - 1) * head + dim, device="meta")
        return t.as_strided((tokens, heads, dim), (token, head, 1))

    for token, head in ((64, 1 << 33), (64, MAX_HEAD_STRIDE), (MAX_TOKEN_STRIDE, 64)):
        t = view(2, 2, 64, token, head)
        assert head_rows(t) is t
    for token, head in ((MAX_TOKEN_STRIDE + 1, 64), (64, MAX_HEAD_STRIDE + 1), (63, 64), (0, 64)):
        t = view(2, 2, 64, token, head)
        assert head_rows(t) is not t and head_rows(t).is_contiguous()
