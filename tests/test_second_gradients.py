"""What a graph of the backward pass holds of gradients that kernels wrote (CPU, no launches)."""

import pytest
import torch

from evograd_amd import _lib, decls
from evograd_amd.bind import bind
from evograd_amd.pairs import (block_norm, cross_entropy, embedding, layernorm, norm_rotary, rmsnorm,
                               rope, rotary, softmax, topk_distillation)
from tests import stub_pairs


@pytest.fixture
def no_kernels(monkeypatch):
    """The pairs on CPU tensors with every launch left out (results are not looked at)."""
    for name in ("require_gpu", "call_on", "call"):
        monkeypatch.setattr(_lib, name, lambda *a: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "query", lambda *a: 16)


POS, FREQ = torch.arange(4, dtype=torch.int32), torch.ones(4, dtype=torch.float64)
IDS, TARGET, T = (torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4, dtype=torch.int64),
                  torch.zeros(4, 3))
# declaration, pair, shapes of the leaves, the other arguments
CASES = {
    "embedding": (decls.EMBEDDING, embedding, ((6, 8),), (POS,)),
    "norm_rotary": (decls.NORM_ROTARY, norm_rotary, ((4, 2, 8), (8,)), (POS, FREQ)),
    "topk_distillation": (decls.TOPK_DISTILLATION, topk_distillation, ((4, 9),), (TARGET, T, IDS)),
    "rotary": (decls.ROTARY, rotary, ((4, 2, 8),), (POS, FREQ)),
    "rmsnorm": (decls.RMSNORM, rmsnorm, ((4, 8), (8,)), ()),
    "layernorm": (decls.LAYERNORM, layernorm, ((4, 8), (8,), (8,)), ()),
    "softmax": (decls.SOFTMAX, softmax, ((4, 8),), ()),
    "cross_entropy": (decls.CROSS_ENTROPY, cross_entropy, ((4, 9),), (TARGET,)),
}
LINEAR = ("embedding", "rotary")  # whose gradients do not depend on their leaves


def bound(name, strided=False):
    op, module, shapes, rest = CASES[name]
    leaves = [torch.zeros(s, requires_grad=True) for s in shapes]
    # every second column: saved as a contiguous copy
    args = [t.repeat_interleave(2, -1)[..., ::2] for t in leaves] if strided else leaves
    return leaves, bind(op, module)(*args, *rest)


@pytest.mark.parametrize("strided", (False, True))
@pytest.mark.parametrize("name", CASES)
def test_a_penalty_on_a_gradient_is_refused(no_kernels, name, strided):
    leaves, y = bound(name, strided)
    assert y.requires_grad and not isinstance(y, tuple)
    grads = torch.autograd.grad((y * y).sum(), leaves, create_graph=True)
    for g, leaf in zip(grads, leaves):
        assert g.requires_grad and (strided or not g._is_view())
        with pytest.raises(RuntimeError, match=f"{name}.*differentiate twice"):
            (g.sum() + leaf.sum()).backward(retain_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(g.sum() + leaf.sum(), leaf, retain_graph=True)


@pytest.mark.parametrize("strided", (False, True))
@pytest.mark.parametrize("name", CASES)
def test_so_is_one_with_constant_upstream_gradients(no_kernels, name, strided):
    """A sum's gradient is ones: the graph leads back through the saved tensors alone."""
    leaves, y = bound(name, strided)
    grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    if name in LINEAR:  # constants indeed
        assert not any(g.requires_grad for g in grads) or strided
        return
    for g in grads:
        with pytest.raises(RuntimeError, match="differentiate twice"):
            torch.autograd.grad(g.sum() + leaves[0].sum(), leaves[0], retain_graph=True)


@pytest.mark.parametrize("name", CASES)
def test_first_gradients_are_plain(no_kernels, name):
    leaves, y = bound(name)
    y.sum().backward()
    for leaf in leaves:
        assert leaf.grad.shape == leaf.shape and not leaf.grad.requires_grad
    leaves, y = bound(name)
    y.sum().backward(create_graph=True)  # gradients that nobody differentiates
    for leaf in leaves:
        leaf.grad.detach_().zero_()
        leaf.grad = None


def test_other_parts_of_a_graph_are_differentiated_as_ever(no_kernels):
    x, scale = torch.randn(4, 8, requires_grad=True), torch.tensor(2.0, requires_grad=True)
    y = bind(decls.SOFTMAX, softmax)(x)
    grad, = torch.autograd.grad((scale ** 3 * 5.0) + 0.0 * y.sum(), scale, create_graph=True)
    again, = torch.autograd.grad(grad, scale)
    assert grad.item() == 60.0 and again.item() == 60.0


def test_pairs_of_torch_operations_keep_their_graph():
    """A pair that is differentiable itself is differentiated again, not refused."""
    x = torch.randn(3, 5, dtype=torch.float32, requires_grad=True)
    way, up = torch.randn(3, 5), torch.randn(3, 5)

    def twice(fn):
        g, = torch.autograd.grad(fn(x), x, up, create_graph=True)
        return torch.autograd.grad((g * way).sum(), x)[0]

    got, want = twice(bind(decls.SOFTMAX, stub_pairs)), twice(lambda t: torch.softmax(t, -1))
    assert torch.allclose(got, want, atol=1e-6)


def test_a_tie_holds_no_argument(no_kernels):
    """A strided argument saved as its copy is itself not kept for the backward."""
    import weakref

    x = torch.zeros(4, 16, requires_grad=True)
    part = (x * 1.0)[:, ::2]
    kept = weakref.ref(part)
    y = bind(decls.LAYERNORM, layernorm)(part, torch.ones(8), torch.zeros(8))
    del part
    assert kept() is None and y.requires_grad


def node(name, strided):
    """Leaves, and a joint node's two outputs (RopeQK, RotaryQK, NormRotaryQK, BlockNorm)."""
    shapes = {"BlockNorm": ((4, 8), (4, 8), (8,), (8,), (8,)),
              "NormRotaryQK": ((4, 2, 8), (4, 1, 8), (8,), (8,)),
              "RotaryQK": ((4, 2, 8), (4, 1, 8)), "RopeQK": ((1, 2, 4, 8), (1, 1, 4, 8))}[name]
    leaves = [torch.zeros(s, requires_grad=True) for s in shapes]
    args = [t.repeat_interleave(2, -1)[..., ::2] for t in leaves] if strided else leaves
    if name == "BlockNorm":
        return leaves, block_norm.BlockNorm.apply(*args, 1.0, 1e-6)
    if name == "RopeQK":
        return leaves, rope.RopeQK.apply(*args, torch.ones(4, 8), torch.ones(4, 8))
    return leaves, getattr(norm_rotary if name[0] == "N" else rotary, name).apply(*args, POS, FREQ)


@pytest.mark.parametrize("strided", (False, True))
@pytest.mark.parametrize("name", ("BlockNorm", "NormRotaryQK", "RotaryQK", "RopeQK"))
def test_joint_nodes_refuse_the_same(no_kernels, name, strided):
    leaves, out = node(name, strided)
    assert len(out) == 2
    for constant in (False, True):  # upstream gradients
        loss = sum((t if constant else t * t).sum() for t in out)
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        if constant and name in ("RotaryQK", "RopeQK"):  # linear: their gradients are constants
            assert strided or not any(g.requires_grad for g in grads)
            continue
        for g in grads:
            with pytest.raises(RuntimeError, match=f"{name}.*differentiate twice"):
                torch.autograd.grad(g.sum() + leaves[0].sum(), leaves[0], retain_graph=True)
            with pytest.raises(RuntimeError, match="differentiate twice"):
                (g.sum() + leaves[0].sum()).backward(retain_graph=True)
    leaves, out = node(name, strided)
    (out[0].sum() + out[1].sum()).backward()
    assert all(t.grad.shape == t.shape and not t.grad.requires_grad for t in leaves)


def test_what_a_pair_returns_is_what_a_call_returns():
    """Also a pair's tuple of outputs, which no declaration has, without gradients."""
    import types
    both = types.SimpleNamespace(forward_with_saved=lambda x: ((x + 1, x + 2), (x,)),
                                 backward_from_saved=lambda dy, saved: dy)
    with torch.no_grad():
        out = bind(decls.SOFTMAX, both)(torch.zeros(3))
    assert isinstance(out, tuple) and out[0].tolist() == [1.0] * 3 and out[1].tolist() == [2.0] * 3
