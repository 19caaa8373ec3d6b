"""The packed-batch operators' oracle functions, pinned to the ones that test_oracle_pins.py
pins, to closed forms and to fp64 finite differences (CPU)."""

import math

import pytest
import torch

from evograd_amd import decls
from evograd_amd.inputs import make_case_inputs
from oracle import forward_refs as fr
from oracle.oracle import oracle


def _normal(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g, dtype=torch.float64)


def test_packed_attention_is_each_sequence_by_itself():
    q, k, v = _normal(14, 4, 6), _normal(14, 2, 6, seed=1), _normal(14, 2, 6, seed=2)
    cu = torch.tensor([0, 5, 5, 6, 12], dtype=torch.int32)
    o = fr.packed_attention_forward_ref(q, k, v, cu)
    for a, b in ((0, 5), (5, 6), (6, 12)):
        want = fr.causal_attention_gqa_forward_ref(
            *(t[a:b].transpose(0, 1)[None] for t in (q, k, v)))[0].transpose(0, 1)
        assert torch.allclose(o[a:b], want, atol=1e-6)
    assert int(torch.count_nonzero(o[12:])) == 0
    # a sequence of one row is its value row, shared by the group
    assert torch.allclose(o[5], v[5].repeat_interleave(2, 0), atol=1e-12)


def test_packed_attention_brute_force():
    q, k, v = _normal(3, 1, 2), _normal(3, 1, 2, seed=1), _normal(3, 1, 2, seed=2)
    o = fr.packed_attention_forward_ref(q, k, v, torch.tensor([0, 3], dtype=torch.int32))
    for i in range(3):
        w = [math.exp(float(q[i, 0] @ k[j, 0]) / math.sqrt(2)) for j in range(i + 1)]
        want = sum(w[j] * v[j, 0] for j in range(i + 1)) / sum(w)
        assert torch.allclose(o[i, 0], want, atol=1e-12)


def test_rotary_half_layout_is_rope_by_its_tables():
    x = _normal(9, 3, 8)
    freqs = 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4)
    angle = torch.arange(9, dtype=torch.float64)[:, None] * freqs
    angle = torch.cat((angle, angle), -1)
    want = fr.rope_forward_ref(x.transpose(0, 1)[None].float(), angle.cos().float(),
                               angle.sin().float())[0].transpose(0, 1)
    got = fr.rotary_forward_ref(x, torch.arange(9), freqs)
    assert torch.allclose(got.float(), want, atol=1e-5)


@pytest.mark.parametrize("interleaved", (0, 1))
def test_rotary_is_a_complex_product(interleaved):
    x = _normal(5, 2, 10, seed=3)
    freqs = torch.tensor([1.0, 0.25, 0.01], dtype=torch.float64)
    pos = torch.tensor([0, 3, -7, 100000, 1 << 40])
    y = fr.rotary_forward_ref(x, pos, freqs, 1.5, interleaved)
    turn = torch.polar(torch.full((5, 3), 1.5, dtype=torch.float64), pos.double()[:, None] * freqs)
    a, b = (x[..., 0:6:2], x[..., 1:6:2]) if interleaved else (x[..., :3], x[..., 3:6])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn[:, None]
    ya, yb = (y[..., 0:6:2], y[..., 1:6:2]) if interleaved else (y[..., :3], y[..., 3:6])
    assert torch.allclose(ya, z.real, atol=1e-12) and torch.allclose(yb, z.imag, atol=1e-12)
    assert torch.equal(y[..., 6:], x[..., 6:])
    assert torch.allclose(y[0, :, :6], 1.5 * x[0, :, :6])  # position 0


def test_block_norm_is_two_norms_and_a_residual():
    x, h, gate = _normal(6, 16), _normal(6, 16, seed=1), _normal(6, 1, seed=2)
    w1, w2 = _normal(16, seed=3), _normal(16, seed=4)
    s, y = fr.block_norm_forward_ref(x, h, w1, gate, w2, 0.5, 1e-6)
    n = fr.rmsnorm_forward_ref(h, w1, 1e-6).double()  # fp32 inside
    assert torch.allclose(s, x + 0.5 * gate * n, atol=1e-5)
    assert torch.allclose(y, fr.rmsnorm_forward_ref(s, w2, 1e-6).double(), atol=1e-5)
    same = fr.block_norm_forward_ref(x, h, w1, torch.ones(16, dtype=torch.float64), w2)
    assert torch.equal(same, fr.block_norm_forward_ref(x, h, w1, None, w2))
    # a zero gate leaves the residual stream
    assert torch.equal(fr.block_norm_forward_ref(x, h, w1, 0 * gate, w2)[0], x)


def _difference(fn, args, i, dout, e=1e-6):
    d = _normal(*args[i].shape, seed=11)
    up, down = list(args), list(args)
    up[i], down[i] = args[i] + e * d, args[i] - e * d
    return float(((fn(*up) - fn(*down)) * dout).sum()) / (2 * e), d


@pytest.mark.parametrize("name", ("packed_attention", "rotary", "block_norm"))
def test_oracle_gradients_against_differences(name):
    op = decls.get_op(name)
    for w in op.correctness:
        if w.dtype != "float32":
            continue
        inputs = make_case_inputs(op, w, "cpu")
        inputs = {k: t.double() if torch.is_tensor(t) and t.is_floating_point() else t
                  for k, t in inputs.items()}
        _, grads = oracle(op, inputs, use_reference_dtype=False)
        fn = getattr(fr, f"{name}_forward_ref")
        args = [inputs[a.name] for a in op.args]
        for i, arg in enumerate(op.args):
            if getattr(arg, "grad_name", None) in grads:
                want, d = _difference(fn, args, i, inputs[op.upstream_grad_name])
                got = float((grads[arg.grad_name] * d).sum())
                assert got == pytest.approx(want, rel=1e-5, abs=1e-6)
