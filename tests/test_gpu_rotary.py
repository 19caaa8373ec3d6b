"""Rotary positions per token against the rotation in 64 bits (tests/packed_refs.py)."""

import pytest
import torch

from evograd_amd.bind import bind
from evograd_amd.decls import ROTARY
from evograd_amd.pairs import rotary as pair
from tests.packed_refs import assert_within, rotary64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(T, H, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, H, D, generator=g, device="cuda").to(dtype)


def spots(T, far, seed=0, dtype=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(100 + seed)
    return torch.randint(0, far, (T,), generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
@pytest.mark.parametrize("T,H,KVH,D,pairs", (
    (1, 1, 1, 2, 1), (1, 32, 8, 128, 64), (3, 5, 1, 64, 32), (67, 4, 4, 80, 40), (33, 6, 2, 96, 24),
    (129, 9, 3, 128, 16), (20, 3, 7, 10, 3), (5, 2, 1, 7, 2), (300, 16, 16, 256, 64), (4, 1, 1, 8, 0)))
def test_q_and_k_both_ways(T, H, KVH, D, pairs, interleaved, dtype):
    print(f"\n[gpu-rotary] {T} {H}/{KVH} D={D} pairs={pairs} {interleaved} {dtype}", flush=True)
    q, k, dq, dk = (make(T, h, D, dtype, i) for i, h in enumerate((H, KVH, H, KVH)))
    pos = spots(T, 131072)
    freqs = (pair.rotary_frequencies(2 * pairs, 500000.0, device="cuda") if pairs
             else torch.empty(0, dtype=torch.float64, device="cuda"))
    outs, saved = pair.rotary_qk_forward_with_saved(q, k, pos, freqs, 1.25, interleaved)
    grads = pair.rotary_qk_backward_from_saved((dq, dk), saved, 1.25, interleaved)
    for name, x, y, inverse in (("q", q, outs[0], False), ("k", k, outs[1], False),
                                ("dq", dq, grads[0], True), ("dk", dk, grads[1], True)):
        assert y.dtype == dtype and y.is_contiguous()
        assert_within(name, y, *rotary64(x, pos, freqs, 1.25, interleaved, inverse))
        alone, s = pair.rotary_forward_with_saved(x, pos, freqs, 1.25, interleaved)
        if inverse:
            alone = pair.rotary_backward_from_saved(x, s, 1.25, interleaved)
        assert torch.equal(alone, y)


@pytest.mark.parametrize("positions", (
    torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 20, 12345678], dtype=torch.int32),
    torch.tensor([0, -1, 2 ** 40, -(2 ** 33), 2 ** 31], dtype=torch.int64)))
@pytest.mark.parametrize("dtype", (F32, BF16))
def test_far_positions_of_both_types(positions, dtype):
    x = make(5, 3, 128, dtype)
    positions = positions.cuda()
    freqs = pair.rotary_frequencies(128, 10000.0, device="cuda")
    y, saved = pair.rotary_forward_with_saved(x, positions, freqs)
    assert_within("y", y, *rotary64(x, positions, freqs, 1.0, 0))
    if dtype == F32:  # fp32 angles would be off by whole turns out here
        at = (x.double()[..., :64] - rotary64(y, positions, freqs, 1.0, 0, True)[0][..., :64]).abs()
        # both turns are formed from fp64 products: position p's angle (freqs[0] = 1) is off by up
        # to 2^-52 p for each, here and there, which moves a pair by its length (below 8)
        far = positions.double().abs().max()
        assert float(at.max()) < 1e-5 + 8 * float(far) * 2.0 ** -51


@pytest.mark.parametrize("scaling", (
    None, {"kind": "linear", "factor": 8.0}, {"kind": "base", "factor": 8.0},
    {"kind": "bands", "factor": 8.0, "context": 8192, "low": 1.0, "high": 4.0}))
def test_scaled_frequencies(scaling):
    x, pos = make(40, 2, 64, F32), spots(40, 100000)
    freqs = pair.rotary_frequencies(64, 500000.0, scaling, device="cuda")
    y, _ = pair.rotary_forward_with_saved(x, pos, freqs)
    assert_within("y", y, *rotary64(x, pos, freqs, 1.0, 0))


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
def test_strided_and_unaligned_inputs_give_the_contiguous_run_s_bits(dtype, interleaved):
    T, H, KVH, D = 50, 6, 2, 64
    qkv = make(T, H + 2 * KVH, D, dtype)
    q, k = qkv[:, :H], qkv[:, H:H + KVH]
    pos, freqs = spots(T, 5000), pair.rotary_frequencies(48, device="cuda")
    want, _ = pair.rotary_qk_forward_with_saved(q.contiguous(), k.contiguous(), pos, freqs, 1.0,
                                                interleaved)
    got, _ = pair.rotary_qk_forward_with_saved(q, k, pos, freqs, 1.0, interleaved)
    outside, _ = pair.rotary_qk_forward_with_saved(
        q.transpose(0, 1).contiguous().transpose(0, 1), k, pos, freqs, 1.0, interleaved)
    room = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")
    odd = room[1:].view(q.shape)
    odd.copy_(q)
    shifted, _ = pair.rotary_qk_forward_with_saved(odd, k, pos[::1], freqs, 1.0, interleaved)
    columns = q.transpose(1, 2).contiguous().transpose(1, 2)  # a head's columns apart: copied
    copied, _ = pair.rotary_qk_forward_with_saved(columns, k, pos, freqs, 1.0, interleaved)
    shared, _ = pair.rotary_forward_with_saved(q[:1].expand(T, H, D), pos, freqs, 1.0, interleaved)
    alone, _ = pair.rotary_forward_with_saved(q[:1].expand(T, H, D).contiguous(), pos, freqs, 1.0,
                                              interleaved)
    assert torch.equal(shared, alone)
    for x in (got, outside, shifted, copied):
        assert torch.equal(x[0], want[0]) and torch.equal(x[1], want[1])


def test_no_tokens_and_no_heads():
    freqs = pair.rotary_frequencies(8, device="cuda")
    for T, H in ((0, 4), (3, 0)):
        y, saved = pair.rotary_forward_with_saved(make(T, H, 8, BF16), spots(T, 10), freqs)
        assert y.shape == (T, H, 8)
        assert pair.rotary_backward_from_saved(y, saved).shape == (T, H, 8)


def test_a_non_finite_value_stays_in_its_pair():
    x = make(9, 2, 16, F32)
    pos, freqs = spots(9, 100), pair.rotary_frequencies(16, device="cuda")
    clean, _ = pair.rotary_forward_with_saved(x, pos, freqs)
    x[4, 1, 3] = float("nan")
    y, _ = pair.rotary_forward_with_saved(x, pos, freqs)
    assert bool(torch.isnan(y[4, 1, [3, 11]]).all())
    y[4, 1, [3, 11]] = clean[4, 1, [3, 11]]
    assert torch.equal(y, clean)


def test_the_backward_is_the_transpose():
    """<rotate(x), d> = <x, back(d)>: each side within its bounds' sum."""
    x, d = make(30, 4, 64, F32, 1), make(30, 4, 64, F32, 2)
    pos, freqs = spots(30, 100000), pair.rotary_frequencies(32, device="cuda")
    y, saved = pair.rotary_forward_with_saved(x, pos, freqs, 0.7, 1)
    back = pair.rotary_backward_from_saved(d, saved, 0.7, 1)
    left = float((y.double() * d.double()).sum())
    right = float((x.double() * back.double()).sum())
    slack = float((rotary64(x, pos, freqs, 0.7, 1)[1] * d.double().abs()).sum()
                  + (rotary64(d, pos, freqs, 0.7, 1, True)[1] * x.double().abs()).sum())
    assert abs(left - right) <= slack


def test_autograd_nodes_match_the_pair():
    q, k = make(21, 4, 64, BF16, 1), make(21, 2, 64, BF16, 2)
    dq, dk = make(21, 4, 64, BF16, 3), make(21, 2, 64, BF16, 4)
    pos, freqs = spots(21, 1000), pair.rotary_frequencies(64, device="cuda")
    outs, saved = pair.rotary_qk_forward_with_saved(q, k, pos, freqs, 1.5, 1)
    want = pair.rotary_qk_backward_from_saved((dq, dk), saved, 1.5, 1)
    a, b = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    y = pair.RotaryQK.apply(a, b, pos, freqs, 1.5, 1)
    assert torch.equal(y[0], outs[0]) and torch.equal(y[1], outs[1])
    torch.autograd.backward(y, (dq, dk))
    assert torch.equal(a.grad, want[0]) and torch.equal(b.grad, want[1])
    a = q.clone().requires_grad_(True)
    fn = bind(ROTARY, pair)
    fn(a, pos, freqs, amplitude=1.5, interleaved=1).backward(dq)
    assert torch.equal(a.grad, want[0])


def test_a_captured_graph_replays_with_other_positions():
    q, k = make(64, 8, 128, BF16, 1), make(64, 2, 128, BF16, 2)
    pos, freqs = spots(64, 1000), pair.rotary_frequencies(128, device="cuda")
    pair.rotary_qk_forward_with_saved(q, k, pos, freqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = pair.rotary_qk_forward_with_saved(q, k, pos, freqs)
    for seed in range(4):
        pos.copy_(spots(64, 100000, seed))
        q.copy_(make(64, 8, 128, BF16, 10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for x, y in zip(got, pair.rotary_qk_forward_with_saved(q, k, pos, freqs)[0]):
            assert torch.equal(x, y)
