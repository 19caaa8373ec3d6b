"""The oracle functions of a distillation step's operators, pinned to other ones, to closed forms
and to fp64 finite differences (CPU)."""

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


def test_embedding_is_a_product_with_one_hot_rows():
    w = _normal(7, 5)
    ids = torch.tensor([3, 0, 6, 3])
    assert torch.allclose(fr.embedding_forward_ref(w, ids, 1.5),
                          1.5 * torch.nn.functional.one_hot(ids, 7).double() @ w)
    out = fr.embedding_forward_ref(w, torch.tensor([-100, 7, -1, 2]), 2.0)
    assert int(torch.count_nonzero(out[0])) == 0 and bool(out[1:3].isnan().all())
    assert torch.equal(out[3], 2.0 * w[2])
    assert int(torch.count_nonzero(fr.embedding_forward_ref(w, torch.tensor([2]), 1.0, 2))) == 0


def test_norm_rotary_is_the_norm_then_the_rotation():
    x, w = _normal(5, 3, 8), _normal(8, seed=1)
    pos, freqs = torch.tensor([0, 3, -7, 1000, 1 << 30]), torch.tensor([1.0, 0.1, 0.01], dtype=torch.float64)
    n = fr.rmsnorm_forward_ref(x.view(-1, 8), w, 1e-6).double().view(5, 3, 8)
    got = fr.norm_rotary_forward_ref(x, w, pos, freqs, 1e-6, 1.5, 1)
    assert torch.allclose(got, fr.rotary_forward_ref(n, pos, freqs, 1.5, 1), atol=1e-5)
    # lengths of a head's unturned norms are kept by the rotation
    turned = fr.norm_rotary_forward_ref(x, torch.ones(8, dtype=torch.float64), pos, freqs, 0.0)
    assert torch.allclose(turned.pow(2).sum(-1), torch.full((5, 3), 8.0, dtype=torch.float64))


def test_distillation_by_hand():
    z = torch.tensor([[0.0, math.log(2.0), math.log(5.0)]], dtype=torch.float64)
    t, i = torch.tensor([[math.log(3.0), 0.0]], dtype=torch.float64), torch.tensor([[2, 0]])
    p, q = (0.75, 0.25), (5 / 8, 1 / 8)
    want = sum(a * math.log(a / b) for a, b in zip(p, q))
    got = fr.topk_distillation_forward_ref(z, torch.tensor([1]), t, i)
    assert float(got) == pytest.approx(want, rel=1e-12)
    got = fr.topk_distillation_forward_ref(z, torch.tensor([1]), t, i, 1.0, 0.5, 2.0)
    assert float(got) == pytest.approx(0.5 * want + 2.0 * math.log(4.0), rel=1e-12)
    # at temperature 2 the odds are square roots
    r = [math.sqrt(v) for v in (1, 2, 5, 3)]
    p, q = (r[3] / (r[3] + 1), 1 / (r[3] + 1)), (r[2] / sum(r[:3]), r[0] / sum(r[:3]))
    want = 4 * sum(a * math.log(a / b) for a, b in zip(p, q))
    assert float(fr.topk_distillation_forward_ref(z, torch.tensor([1]), t, i, 2.0)) == pytest.approx(want)


def test_distillation_of_its_own_distribution_is_zero():
    z, target = _normal(4, 9), torch.zeros(4, dtype=torch.int64)
    ids = torch.arange(9).expand(4, 9)
    assert abs(float(fr.topk_distillation_forward_ref(z, target, z + 3.0, ids, 2.0))) < 1e-14


def test_distillation_rows_and_entries_left_out():
    z, t = _normal(4, 9), _normal(4, 3, seed=1)
    ids = torch.tensor([[1, 2, 3], [4, -1, 6], [-1, -1, -1], [0, 1, 2]])
    target = torch.tensor([0, 5, 7, -100])
    rows = [float(fr.topk_distillation_forward_ref(z[r:r + 1], target[r:r + 1], t[r:r + 1], ids[r:r + 1],
                                                   1.5, 0.5, 0.25)) for r in range(3)]
    assert float(fr.topk_distillation_forward_ref(z, target, t, ids, 1.5, 0.5, 0.25)) == pytest.approx(
        sum(rows) / 3, rel=1e-12)
    short = fr.topk_distillation_forward_ref(z[1:2], target[1:2], t[1:2, [0, 2]], ids[1:2, [0, 2]], 1.5,
                                             0.5, 0.25)
    assert float(short) == pytest.approx(rows[1], rel=1e-12)
    hard = fr.cross_entropy_forward_ref(z[2:3], target[2:3])
    assert 0.25 * float(hard) == pytest.approx(rows[2], rel=1e-6)  # fp32 inside
    twice = fr.topk_distillation_forward_ref(z[:1], target[:1], t[:1, :2], torch.tensor([[5, 5]]))
    once = -float(torch.log_softmax(z[0], 0)[5])
    p = torch.softmax(t[0, :2], 0)
    assert float(twice) == pytest.approx(once + float((p * p.log()).sum()), rel=1e-12)


def _difference(fn, args, i, dout, e=1e-6):
    d = _normal(*args[i].shape, seed=11)
    up, down = list(args), list(args)
    up[i], down[i] = args[i] + e * d, args[i] - e * d
    return float(((fn(*up) - fn(*down)) * dout).sum()) / (2 * e), d


@pytest.mark.parametrize("name", ("embedding", "norm_rotary", "topk_distillation"))
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
