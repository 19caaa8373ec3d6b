"""Bound operators whose nodes hold a tie (once.py): on another stream and in captured graphs."""

import pytest
import torch

from evograd_amd import decls
from evograd_amd.bind import bind
from evograd_amd.pairs import embedding, layernorm, norm_rotary, rotary

pytestmark = pytest.mark.gpu


def leaf(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").requires_grad_(True)


def grads_of(x, w, b, dy):
    # every second column: saved as a contiguous copy, which hides x
    y = bind(decls.LAYERNORM, layernorm)(x[:, ::2], w, b)
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))


def test_a_node_with_a_tie_on_another_stream_and_captured():
    x, w, b, dy = leaf(64, 256), leaf(128, seed=1), leaf(128, seed=2), leaf(64, 128, seed=3).detach()
    want = [t.clone() for t in grads_of(x, w, b, dy)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = grads_of(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(stream)
    for a, c in zip(other, want):
        assert torch.equal(a, c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads_of(x, w, b, dy)
    for seed in range(3):
        with torch.no_grad():
            x.copy_(leaf(64, 256, seed=10 + seed))
            dy.copy_(leaf(64, 128, seed=20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, c in zip(got, grads_of(x, w, b, dy)):
            assert torch.equal(a, c)


def test_joint_nodes_with_strided_columns():
    x = leaf(37, 6, 128)
    q, k = x[:, :4, ::2], x[:, 4:, ::2]
    qw, kw = leaf(64, seed=1), leaf(64, seed=2)
    pos = torch.arange(37, dtype=torch.int32, device="cuda")
    freqs = rotary.rotary_frequencies(64, 500000.0, device="cuda")
    out = norm_rotary.NormRotaryQK.apply(q, k, qw, kw, pos, freqs)
    ups = [torch.randn_like(t) for t in out]
    got = torch.autograd.grad(out, (x, qw, kw), ups)
    args = [t.detach().contiguous().requires_grad_(True) for t in (q, k, qw, kw)]
    plain = norm_rotary.NormRotaryQK.apply(*args, pos, freqs)
    dq, dk, dqw, dkw = torch.autograd.grad(plain, args, ups)
    assert torch.equal(out[0], plain[0]) and torch.equal(out[1], plain[1])
    assert torch.equal(got[0][..., ::2], torch.cat((dq, dk), 1)) and not bool(got[0][..., 1::2].any())
    assert torch.equal(got[1], dqw) and torch.equal(got[2], dkw)


def test_a_penalty_on_a_gradient_is_refused():
    table, ids = leaf(50, 64), torch.arange(20, dtype=torch.int32, device="cuda")
    y = bind(decls.EMBEDDING, embedding)(table, ids)
    grad, = torch.autograd.grad((y * y).sum(), table, create_graph=True)
    assert torch.equal(grad.detach()[:20], 2 * table.detach()[:20])
    with pytest.raises(RuntimeError, match="embedding.*differentiate twice"):
        (grad.square().sum() + table.sum()).backward()


def test_a_gradient_added_in_place_moves_its_version():
    table, dout = leaf(50, 64).detach(), leaf(20, 64, seed=1).detach()
    ids = torch.arange(20, dtype=torch.int32, device="cuda")
    y = torch.ones(50, 64, device="cuda", requires_grad=True) * table
    embedding.embedding_backward_into(table, dout, (ids, 50, 64, torch.float32))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
