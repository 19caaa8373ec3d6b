"""Limits of the packed-batch operators' arguments that the entry points and their wrappers share,
and what their autograd nodes refuse (CPU)."""

import ctypes
import os

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.pairs._util import MAX_HEAD_STRIDE, MAX_TOKEN_STRIDE, head_rows
from evograd_amd.pairs.block_norm import BlockNorm
from evograd_amd.pairs.rotary import RotaryQK

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


@pytest.fixture
def no_kernels(monkeypatch):
    """The pairs on CPU tensors with every launch left out (results are not looked at)."""
    for name in ("require_gpu", "call_on"):
        monkeypatch.setattr(_lib, name, lambda *a: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "query", lambda *a: 16)


def test_gradients_of_gradients_are_refused(no_kernels):
    """The backward kernels have no backward of their own: a second differentiation through the
    nodes raises, where it would leave their part out."""
    def leaf(*shape):
        return torch.zeros(shape, requires_grad=True)

    x, h, w1, w2 = leaf(4, 8), leaf(4, 8), leaf(8), leaf(8)
    s, y = BlockNorm.apply(x, h, w1, None, w2, 1.0, 1e-6)
    norm_grads = torch.autograd.grad((s * s).sum() + (y * y).sum(), (x, h), create_graph=True)
    q, k = leaf(4, 2, 8), leaf(4, 1, 8)
    a, b = RotaryQK.apply(q, k, torch.arange(4), torch.ones(4, dtype=torch.float64))
    turn_grads = torch.autograd.grad((a * a).sum() + (b * b).sum(), (q, k), create_graph=True)
    for g, other in ((norm_grads[0], x), (norm_grads[1], h), (turn_grads[0], q), (turn_grads[1], k)):
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (g.sum() + other.sum()).backward(retain_graph=True)


def test_first_gradients_need_no_second(no_kernels):
    x, h, w1, w2 = (torch.zeros(s, requires_grad=True) for s in ((4, 8), (4, 8), 8, 8))
    s, _ = BlockNorm.apply(x, h, w1, None, w2, 1.0, 1e-6)
    s.sum().backward()
    assert all(t.grad is not None and t.grad.shape == t.shape for t in (x, h, w1, w2))
