"""Norms per head with the rotation behind them against 64 bits (tests/step_refs.py)."""

import pytest
import torch

from evograd_amd.bind import bind
from evograd_amd.decls import NORM_ROTARY
from evograd_amd.pairs import norm_rotary as pair
from evograd_amd.pairs import rotary
from tests.packed_refs import assert_within
from tests.step_refs import norm_rotary64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def make(*shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def gain(D, dtype, seed):
    return (1 + 0.1 * make(D, dtype=F32, seed=seed)).to(dtype)


def spots(T, far, seed=0, dtype=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(100 + seed)
    return torch.randint(0, far, (T,), generator=g, device="cuda").to(dtype)


def turns(pairs):
    return (rotary.rotary_frequencies(2 * pairs, 500000.0, device="cuda") if pairs
            else torch.empty(0, dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
@pytest.mark.parametrize("T,H,KVH,D,pairs", (
    (1, 1, 1, 2, 1), (1, 32, 8, 128, 64), (3, 5, 1, 64, 32), (67, 4, 4, 80, 40), (33, 6, 2, 96, 24),
    (129, 9, 3, 128, 16), (20, 3, 7, 10, 3), (5, 2, 1, 7, 2), (300, 16, 16, 256, 64), (4, 1, 1, 8, 0),
    (3000, 2, 1, 64, 32), (11, 70, 5, 128, 64), (6, 130, 2, 256, 128), (9, 2, 2, 1, 0),
    (40, 3, 2, 200, 33), (7, 2, 1, 514, 257), (3, 1, 2, 1024, 512)))
def test_q_and_k_both_ways(T, H, KVH, D, pairs, interleaved, dtype):
    print(f"\n[gpu-norm-rotary] {T} {H}/{KVH} D={D} pairs={pairs} {interleaved} {dtype}", flush=True)
    q, k, dq, dk = (make(T, h, D, dtype=dtype, seed=i) for i, h in enumerate((H, KVH, H, KVH)))
    qw, kw = gain(D, dtype, 7), gain(D, dtype, 8)
    pos, freqs = spots(T, 131072), turns(pairs)
    outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs, EPS, 1.25, interleaved)
    grads = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.25, interleaved)
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        want = norm_rotary64(x, w, pos, freqs, EPS, 1.25, interleaved, dy)
        got = {"y": outs[i], "dx": grads[i], "dweight": grads[2 + i]}
        for name, (value, bound) in want.items():
            assert got[name].dtype == dtype and got[name].is_contiguous()
            assert_within(f"{'qk'[i]} {name}", got[name], value, bound)
    again = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.25, interleaved)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)
    y, s = pair.norm_rotary_forward_with_saved(k, kw, pos, freqs, EPS, 1.25, interleaved)
    dx, dw = pair.norm_rotary_backward_from_saved(dk, s, EPS, 1.25, interleaved)
    assert torch.equal(y, outs[1]) and torch.equal(dx, grads[1])
    value, bound = want["dweight"]
    assert_within("dweight alone", dw, value, bound)


@pytest.mark.parametrize("positions", (
    torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 20, 12345678], dtype=torch.int32),
    torch.tensor([0, -1, 2 ** 40, -(2 ** 33), 2 ** 31], dtype=torch.int64)))
def test_far_positions_of_both_types(positions):
    x, dy, w = make(5, 3, 128, dtype=F32), make(5, 3, 128, dtype=F32, seed=1), gain(128, F32, 2)
    positions, freqs = positions.cuda(), turns(64)
    y, saved = pair.norm_rotary_forward_with_saved(x, w, positions, freqs)
    dx, dw = pair.norm_rotary_backward_from_saved(dy, saved)
    want = norm_rotary64(x, w, positions, freqs, EPS, 1.0, 0, dy)
    for name, got in (("y", y), ("dx", dx), ("dweight", dw)):
        assert_within(name, got, *want[name])


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
def test_strided_and_unaligned_inputs(dtype, interleaved):
    T, H, KVH, D = 50, 6, 2, 64
    qkv, dqkv = make(T, H + 2 * KVH, D, dtype=dtype), make(T, H + 2 * KVH, D, dtype=dtype, seed=1)
    q, k, dq, dk = qkv[:, :H], qkv[:, H:H + KVH], dqkv[:, :H], dqkv[:, H:H + KVH]
    qw, kw, pos, freqs = gain(D, dtype, 3), gain(D, dtype, 4), spots(T, 5000), turns(24)

    def run(q, k, dq, dk, qw=qw):
        outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs, EPS, 1.0,
                                                             interleaved)
        return (*outs, *pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.0, interleaved))

    want = run(*(t.contiguous() for t in (q, k, dq, dk)))
    columns = q.transpose(1, 2).contiguous().transpose(1, 2)  # a head's columns apart: copied
    heads = dq.transpose(0, 1).contiguous().transpose(0, 1)
    for got in (run(q, k, dq, dk), run(columns, k, heads, dk)):
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    # an element off 16 bytes: narrower packs, whose sums take another order
    room = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")
    odd = room[1:].view(q.shape)
    odd.copy_(q)
    wide = torch.empty(D + 1, dtype=dtype, device="cuda")
    shifted = wide[1:]
    shifted.copy_(qw)
    for dqs in (dq, odd):  # odd holds q's values
        got = run(odd, k, dqs, dk, shifted)
        for i, (x, w, d) in enumerate(((q, qw, dqs), (k, kw, dk))):
            expect = norm_rotary64(x, w, pos, freqs, EPS, 1.0, interleaved, d)
            for j, name in enumerate(("y", "dx", "dweight")):
                assert_within(f"{'qk'[i]} {name}", got[2 * j + i], *expect[name])
    shared = q[:1].expand(T, H, D)
    for a, b in zip(run(shared, k, dq[:1].expand(T, H, D), dk),
                    run(shared.contiguous(), k, dq[:1].expand(T, H, D).contiguous(), dk)):
        assert torch.equal(a, b)


def test_no_tokens_and_no_heads():
    freqs, w = turns(4), gain(8, BF16, 1)
    for T, H in ((0, 4), (3, 0)):
        x = make(T, H, 8, dtype=BF16)
        y, saved = pair.norm_rotary_forward_with_saved(x, w, spots(T, 10), freqs)
        dx, dw = pair.norm_rotary_backward_from_saved(x, saved)
        assert y.shape == dx.shape == (T, H, 8) and int(torch.count_nonzero(dw)) == 0
    q, k = make(5, 2, 8, dtype=F32), make(5, 0, 8, dtype=F32)
    w = gain(8, F32, 1)
    outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, w, w, spots(5, 10), freqs)
    grads = pair.norm_rotary_qk_backward_from_saved((q, k), saved)
    assert outs[1].shape == grads[1].shape == (5, 0, 8) and int(torch.count_nonzero(grads[3])) == 0
    assert_within("dq", grads[0], *norm_rotary64(q, w, saved[4], freqs, EPS, 1.0, 0, q)["dx"])


def test_a_non_finite_value_stays_in_its_head():
    x, w, pos, freqs = make(9, 2, 16, dtype=F32), gain(16, F32, 1), spots(9, 100), turns(8)
    dy = make(9, 2, 16, dtype=F32, seed=3)
    clean, saved = pair.norm_rotary_forward_with_saved(x, w, pos, freqs)
    dclean, _ = pair.norm_rotary_backward_from_saved(dy, saved)
    x = x.clone()
    x[4, 1, 3] = float("nan")
    y, saved = pair.norm_rotary_forward_with_saved(x, w, pos, freqs)
    dx, dw = pair.norm_rotary_backward_from_saved(dy, saved)
    assert bool(y[4, 1].isnan().all()) and bool(dx[4, 1].isnan().all()) and bool(dw.isnan().all())
    y[4, 1], dx[4, 1] = clean[4, 1], dclean[4, 1]
    assert torch.equal(y, clean) and torch.equal(dx, dclean)


def test_a_head_of_zeros():
    x = torch.zeros(3, 2, 64, dtype=F32, device="cuda")
    dy, w, pos, freqs = make(3, 2, 64, dtype=F32), gain(64, F32, 1), spots(3, 10), turns(32)
    y, saved = pair.norm_rotary_forward_with_saved(x, w, pos, freqs)
    dx, dw = pair.norm_rotary_backward_from_saved(dy, saved)
    assert int(torch.count_nonzero(y)) == 0 and int(torch.count_nonzero(dw)) == 0
    assert_within("dx", dx, *norm_rotary64(x, w, pos, freqs, EPS, 1.0, 0, dy)["dx"])


def test_gradients_against_differences():
    """d(sum(y dy))/dx along a direction, from y in 64 bits on either side of x."""
    x, w, dy = make(6, 3, 32, dtype=F32), gain(32, F32, 1), make(6, 3, 32, dtype=F32, seed=2)
    pos, freqs = spots(6, 1000), turns(10)
    _, saved = pair.norm_rotary_forward_with_saved(x, w, pos, freqs, EPS, 0.7, 1)
    dx, dw = pair.norm_rotary_backward_from_saved(dy, saved, EPS, 0.7, 1)
    e, dirx, dirw = 1e-4, make(6, 3, 32, dtype=F32, seed=4).double(), make(32, dtype=F32, seed=5).double()

    def f(s):
        x64, w64 = x.double() + s * e * dirx, w.double() + s * e * dirw
        n = x64 * (x64.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w64
        angle = pos.double()[:, None, None] * freqs
        a, b = n[..., 0:20:2], n[..., 1:20:2]
        ya, yb = 0.7 * (a * angle.cos() - b * angle.sin()), 0.7 * (b * angle.cos() + a * angle.sin())
        d = dy.double()
        return float((ya * d[..., 0:20:2] + yb * d[..., 1:20:2]).sum() + (n[..., 20:] * d[..., 20:]).sum())

    slope = (f(1) - f(-1)) / (2 * e)
    got = float((dx.double() * dirx).sum() + (dw.double() * dirw).sum())
    # the difference is off by e^2 times third derivatives (order 1 a head), the kernel by fp32
    # roundings of 576 terms of order 1: 600 * 2^-24 * 50
    assert abs(got - slope) < 18 * 32 * e * e * 10 + 600 * 2.0 ** -24 * 50


def test_autograd_nodes_match_the_pair():
    q, k = make(21, 4, 64, dtype=BF16, seed=1), make(21, 2, 64, dtype=BF16, seed=2)
    dq, dk = make(21, 4, 64, dtype=BF16, seed=3), make(21, 2, 64, dtype=BF16, seed=4)
    qw, kw, pos, freqs = gain(64, BF16, 5), gain(64, BF16, 6), spots(21, 1000), turns(32)
    outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs, EPS, 1.5, 1)
    want = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.5, 1)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, qw, kw)]
    y = pair.NormRotaryQK.apply(*leaves, pos, freqs, EPS, 1.5, 1)
    assert torch.equal(y[0], outs[0]) and torch.equal(y[1], outs[1])
    torch.autograd.backward(y, (dq, dk))
    for leaf, grad in zip(leaves, want):
        assert torch.equal(leaf.grad, grad)
    a, w = q.clone().requires_grad_(True), qw.clone().requires_grad_(True)
    bind(NORM_ROTARY, pair)(a, w, pos, freqs, eps=EPS, amplitude=1.5, interleaved=1).backward(dq)
    assert torch.equal(a.grad, want[0])


def test_two_streams_and_a_captured_graph():
    q, k, qw, kw = make(64, 8, 128, dtype=BF16, seed=1), make(64, 2, 128, dtype=BF16, seed=2), \
        gain(128, BF16, 3), gain(128, BF16, 4)
    dq, dk = make(64, 8, 128, dtype=BF16, seed=5), make(64, 2, 128, dtype=BF16, seed=6)
    pos, freqs = spots(64, 1000), turns(64)

    def step():
        outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs)
        return (*outs, *pair.norm_rotary_qk_backward_from_saved((dq, dk), saved))

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(step())
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(r, want):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        pos.copy_(spots(64, 100000, seed))
        q.copy_(make(64, 8, 128, dtype=BF16, seed=10 + seed))
        dq.copy_(make(64, 8, 128, dtype=BF16, seed=20 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


def test_tensors_past_32_bit_offsets():
    """The last tokens of q and k of 2.5e9 elements, against a call on those tokens alone."""
    T, H, KVH, D = 480000, 32, 8, 128
    q, k = (torch.zeros(T, h, D, dtype=BF16, device="cuda") for h in (H, KVH))
    n = 7
    tail = [make(n, h, D, dtype=BF16, seed=i) for i, h in enumerate((H, KVH, H, KVH))]
    q[-n:], k[-n:] = tail[0], tail[1]
    qw, kw, freqs = gain(D, BF16, 3), gain(D, BF16, 4), turns(64)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs)
    want, s = pair.norm_rotary_qk_forward_with_saved(*tail[:2], qw, kw, pos[-n:], freqs)
    assert torch.equal(outs[0][-n:], want[0]) and torch.equal(outs[1][-n:], want[1])
    assert not bool(outs[0][:-n].any()) and not bool(outs[1][:-n].any())
    del outs
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    dq[-n:], dk[-n:] = tail[2], tail[3]
    grads = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved)
    wants = pair.norm_rotary_qk_backward_from_saved(tail[2:], s)
    for got, w in zip(grads[:2], wants[:2]):
        assert torch.equal(got[-n:], w) and not bool(got[:-n].any())
    for i, (x, w, d) in enumerate(((tail[0], qw, tail[2]), (tail[1], kw, tail[3]))):
        assert_within("dweight", grads[2 + i],
                      *norm_rotary64(x, w, pos[-n:], freqs, EPS, 1.0, 0, d)["dweight"])


def test_two_graphs_with_a_workspace_each():
    """Two captured backward passes, replayed one over the other."""
    q, w, pos, freqs = make(700, 5, 64, dtype=BF16), gain(64, BF16, 1), spots(700, 1000), turns(32)
    grads = [make(700, 5, 64, dtype=BF16, seed=s) for s in (2, 3)]
    _, saved = pair.norm_rotary_forward_with_saved(q, w, pos, freqs)
    want = [pair.norm_rotary_backward_from_saved(d, saved) for d in grads]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for d in grads:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pair.norm_rotary_backward_from_saved(d, saved))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("T,H,KVH,D,pairs", ((3, 2, 1, 8192, 4096), (2, 1, 1, 8191, 4095),
                                             (2, 65536, 1, 2, 1), (2, 300, 65536, 16, 4)))
def test_the_widest_and_the_most_heads(T, H, KVH, D, pairs, dtype):
    print(f"\n[gpu-norm-rotary] largest {T} {H}/{KVH} D={D} {dtype}", flush=True)
    q, k, dq, dk = (make(T, h, D, dtype=dtype, seed=i) for i, h in enumerate((H, KVH, H, KVH)))
    qw, kw = gain(D, dtype, 7), gain(D, dtype, 8)
    pos, freqs = spots(T, 5000), turns(pairs)
    for interleaved in (0, 1):
        outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs, EPS, 1.0,
                                                             interleaved)
        grads = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.0, interleaved)
        for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
            want = norm_rotary64(x, w, pos, freqs, EPS, 1.0, interleaved, dy)
            for name, got in (("y", outs[i]), ("dx", grads[i]), ("dweight", grads[2 + i])):
                assert_within(f"{'qk'[i]} {name}", got, *want[name])


# Shapes whose walk takes several steps: tokens past those that the resident workgroups hold at once.
@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
@pytest.mark.parametrize("T,H,KVH,D,pairs", (
    (40001, 4, 1, 64, 32),    # 8 or 16 tokens a workgroup
    (4001, 16, 16, 128, 64),  # a token, 3 steps forward and 8 backward
    (20003, 3, 2, 96, 24),    # columns that are not turned, lanes without columns
    (40001, 12, 2, 64, 32),   # more than 64 MB: the streaming form
    (70001, 1, 1, 10, 3),     # single columns
    (9001, 40, 9, 64, 16),    # tokens that share workgroups of no whole number of them
    (3001, 300, 2, 32, 8)))   # several workgroups a token
def test_walks_of_several_steps(T, H, KVH, D, pairs, interleaved, dtype):
    print(f"\n[gpu-norm-rotary] walk {T} {H}/{KVH} D={D} pairs={pairs} {interleaved} {dtype}", flush=True)
    q, k, dq, dk = (make(T, h, D, dtype=dtype, seed=i) for i, h in enumerate((H, KVH, H, KVH)))
    qw, kw = gain(D, dtype, 7), gain(D, dtype, 8)
    pos, freqs = spots(T, 131072), turns(pairs)
    outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs, EPS, 1.25, interleaved)
    grads = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.25, interleaved)
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        want = norm_rotary64(x, w, pos, freqs, EPS, 1.25, interleaved, dy)
        for name, got in (("y", outs[i]), ("dx", grads[i]), ("dweight", grads[2 + i])):
            assert_within(f"{'qk'[i]} {name}", got, *want[name])
    again = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 1.25, interleaved)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
@pytest.mark.parametrize("T,H,KVH,D,pairs", ((2100, 2, 1, 514, 257), (3000, 1, 2, 130, 65),
                                             (1500, 2, 3, 259, 65)))
def test_a_wave_with_several_heads(T, H, KVH, D, pairs, interleaved, dtype):
    """Heads of more than 64 lanes, more of them than the 2048 waves: q's and k's in one wave."""
    print(f"\n[gpu-norm-rotary] wide {T} {H}/{KVH} D={D} pairs={pairs} {interleaved} {dtype}", flush=True)
    q, k, dq, dk = (make(T, h, D, dtype=dtype, seed=i) for i, h in enumerate((H, KVH, H, KVH)))
    qw, kw = gain(D, dtype, 7), gain(D, dtype, 8)
    pos, freqs = spots(T, 131072), turns(pairs)
    outs, saved = pair.norm_rotary_qk_forward_with_saved(q, k, qw, kw, pos, freqs, EPS, 0.75, interleaved)
    grads = pair.norm_rotary_qk_backward_from_saved((dq, dk), saved, EPS, 0.75, interleaved)
    for i, (x, w, dy) in enumerate(((q, qw, dq), (k, kw, dk))):
        want = norm_rotary64(x, w, pos, freqs, EPS, 0.75, interleaved, dy)
        for name, got in (("y", outs[i]), ("dx", grads[i]), ("dweight", grads[2 + i])):
            assert_within(f"{'qk'[i]} {name}", got, *want[name])
