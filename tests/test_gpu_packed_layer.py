"""The packed-batch operators together, as a training step runs them: the norms around the
block, one projection to q, k and v, rotary positions that restart with every sequence, packed
attention on the projection's own column ranges, the output projection, and the next norms."""

import pytest
import torch

from evograd_amd.decls import PACKED_ATTENTION
from evograd_amd.bind import bind
from evograd_amd.pairs import packed_attention, rotary
from evograd_amd.pairs.block_norm import BlockNorm

pytestmark = pytest.mark.gpu

EPS = 1e-6


def attention64(q, k, v, lengths):
    out, a = [], 0
    for n in lengths:
        qs, ks, vs = (t[a:a + n].transpose(0, 1) for t in (q, k, v))
        group = q.shape[1] // k.shape[1]
        ks, vs = ks.repeat_interleave(group, 0), vs.repeat_interleave(group, 0)
        s = qs @ ks.transpose(1, 2) / q.shape[2] ** 0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -float("inf"))
        out.append((torch.softmax(s, -1) @ vs).transpose(0, 1))
        a += n
    return torch.cat(out)


def turn64(x, positions, freqs):
    angle = positions.double()[:, None, None] * freqs
    x1, x2 = x.chunk(2, -1)
    return torch.cat((x1 * angle.cos() - x2 * angle.sin(), x2 * angle.cos() + x1 * angle.sin()), -1)


def norms64(x, h, w1, gate, w2, scale):
    def norm(a, w):
        return a * torch.rsqrt(a.pow(2).mean(-1, keepdim=True) + EPS) * w

    s = x + scale * gate * norm(h, w1)
    return s, norm(s, w2)


def sub_layer(ops, p, x, h, positions, freqs, cu, H, KVH, D):
    norms, turn, attend = ops
    s, y = norms(x, h, p["post1"], p["gate1"], p["pre1"])
    T = x.shape[0]
    qkv = y @ p["wqkv"].T
    q, k, v = qkv.view(T, H + 2 * KVH, D).split((H, KVH, KVH), 1)
    q, k = turn(q, k)
    o = attend(q, k, v).reshape(T, H * D) @ p["wo"].T
    return norms(s, o, p["post2"], p["gate2"], p["pre2"])


@pytest.mark.parametrize("dtype,D,tol", (
    # fp32: ten composed operators, the longest sums 256 terms of the projections' (2^-24 * 256
    # each way), against gradients of order one
    (torch.float32, 32, 2e-4),
    # bf16: each of about 20 stored tensors on the way is rounded to 2^-8 of its value; the
    # errors add as independent ones, 2^-8 * sqrt(20) = 0.017 of a tensor's norm, twice for the
    # way back
    (torch.bfloat16, 64, 0.035)))
def test_a_packed_sub_layer_steps_like_its_definition(dtype, D, tol):
    H, KVH, lengths = 4, 2, [37, 1, 90, 5]
    T, C = sum(lengths), 256
    g = torch.Generator(device="cuda").manual_seed(0)

    def normal(scale, *shape):
        return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    p = {"wqkv": normal(C ** -0.5, (H + 2 * KVH) * D, C), "wo": normal((H * D) ** -0.5, C, H * D)}
    for i in "12":
        p["post" + i], p["pre" + i] = 1 + normal(0.1, C), 1 + normal(0.1, C)
        p["gate" + i] = 1 + normal(0.1, C)
    x, h, ds, dy = (normal(1.0, T, C) for _ in range(4))
    positions = torch.cat([torch.arange(n) for n in lengths]).to("cuda", torch.int32)
    freqs = rotary.rotary_frequencies(D, device="cuda")
    cu = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")

    attend = bind(PACKED_ATTENTION, packed_attention)
    mine = (lambda *a: BlockNorm.apply(*a, 0.5, EPS),
            lambda q, k: rotary.RotaryQK.apply(q, k, positions, freqs),
            lambda q, k, v: attend(q, k, v, cu))
    true = (lambda *a: norms64(*a, 0.5),
            lambda q, k: (turn64(q, positions, freqs), turn64(k, positions, freqs)),
            lambda q, k, v: attention64(q, k, v, lengths))

    def step(ops, dt):
        leaf = {n: t.detach().clone().to(dt).requires_grad_(True) for n, t in {**p, "x": x, "h": h}.items()}
        weights = {n: leaf[n] for n in p}
        s, y = sub_layer(ops, weights, leaf["x"], leaf["h"], positions, freqs, cu, H, KVH, D)
        torch.autograd.backward((s, y), (ds.to(dt), dy.to(dt)))
        return {"s": s.detach(), "y": y.detach(), **{"d" + n: t.grad for n, t in leaf.items()}}

    got, want = step(mine, dtype), step(true, torch.float64)
    for name, value in want.items():
        error = float((got[name].double() - value).norm() / value.norm())
        assert error <= tol, (name, error)
