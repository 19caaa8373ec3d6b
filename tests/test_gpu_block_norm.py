"""The norms around a block against their definition in 64 bits (tests/packed_refs.py)."""

import pytest
import torch

from evograd_amd.bind import bind
from evograd_amd.decls import BLOCK_NORM
from evograd_amd.pairs import block_norm as pair
from tests.packed_refs import assert_within, block_norm64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def make(rows, cols, gate, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def around(mean, spread, *shape):
        return (mean + spread * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    shape = {"none": None, "channel": (cols,), "row": (rows, 1), "element": (rows, cols)}[gate]
    return dict(x=around(0, 1, rows, cols), h=around(0, 2, rows, cols), w1=around(1, 0.1, cols),
                gate=None if shape is None else around(0.3, 0.5, *shape), w2=around(1, 0.1, cols),
                ds=around(0, 1, rows, cols), dy=around(0, 1, rows, cols))


def run(t, alpha, split=False):
    out, saved = pair.block_norm_forward_with_saved(t["x"], t["h"], t["w1"], t["gate"], t["w2"],
                                                    alpha, EPS)
    dout = (t["ds"], t["dy"]) if split else torch.stack((t["ds"], t["dy"]))
    return (out[0], out[1], *pair.block_norm_backward_from_saved(dout, saved, alpha))


NAMES = ("s", "y", "dx", "dh", "dpost_weight", "dgate", "dpre_weight")


def check(rows, cols, gate, dtype, alpha=0.7, seed=0):
    print(f"\n[gpu-block-norm] {rows}x{cols} {gate} {dtype}", flush=True)
    t = make(rows, cols, gate, dtype, seed)
    want = block_norm64(t["x"], t["h"], t["w1"], t["gate"], t["w2"], alpha, EPS, t["ds"], t["dy"])
    for name, x in zip(NAMES, run(t, alpha)):
        if name == "dgate" and t["gate"] is None:
            assert x is None
            continue
        assert x.dtype == dtype
        assert_within(name, x, *want[name])


GATES = ("none", "channel", "row", "element")


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("rows,cols", (
    (1, 1), (3, 5), (1, 8), (7, 9), (4, 511), (5, 512), (2, 520), (1, 2048), (3, 2051), (2, 4096),
    (3, 4100), (2, 8191), (1, 8192), (2, 8200), (2, 16389), (70, 768), (1100, 65)))
def test_widths_of_every_kernel(rows, cols, gate, dtype):
    if gate == "row" and cols == 1:
        pytest.skip("[rows, 1] is the element shape too")
    check(rows, cols, gate, dtype)


@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("rows,cols,dtype", ((2500, 1024, BF16), (1500, 8192, F16), (600, 12296, BF16),
                                             (1300, 4096, F32), (40000, 64, F32)))
def test_more_rows_than_workgroups(rows, cols, gate, dtype):
    check(rows, cols, gate, dtype)


@pytest.mark.parametrize("alpha", (1.0, 0.0, -0.5, 8.0))
def test_residual_scales(alpha):
    check(33, 256, "channel", F32, alpha)


def test_two_upstream_tensors_are_the_stacked_one():
    t = make(40, 768, "row", BF16)
    for x, y in zip(run(t, 0.5), run(t, 0.5, split=True)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("gate", ("channel", "element"))
def test_strided_and_unaligned_inputs_are_taken(gate, dtype):
    t = make(20, 1024, gate, dtype)
    want = run(t, 0.5)
    other = {}
    for name, x in t.items():
        if name in ("x", "ds") or x.dim() == 1:  # one element off a 16-byte boundary
            room = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
            other[name] = room[1:].view(x.shape)
            other[name].copy_(x)
        else:  # every second column of a wider matrix
            room = torch.empty(x.shape[0], 2 * x.shape[1], dtype=dtype, device="cuda")
            other[name] = room[:, ::2]
            other[name].copy_(x)
    t64 = block_norm64(t["x"], t["h"], t["w1"], t["gate"], t["w2"], 0.5, EPS, t["ds"], t["dy"])
    for name, x, y in zip(NAMES, run(other, 0.5, split=True), want):
        assert_within(name, x, *t64[name])
        assert_within(name, y, *t64[name])


@pytest.mark.parametrize("rows", (0,))
def test_no_rows(rows):
    for gate in GATES:
        t = make(rows, 128, gate, BF16)
        got = dict(zip(NAMES, run(t, 1.0)))
        assert got["s"].shape == got["dx"].shape == (0, 128)
        for name in ("dpost_weight", "dpre_weight"):
            assert got[name].shape == (128,) and int(torch.count_nonzero(got[name])) == 0
        if gate == "channel":
            assert int(torch.count_nonzero(got["dgate"])) == 0


def test_zero_rows_and_non_finite_rows_keep_to_themselves():
    t = make(12, 512, "element", F32)
    clean = dict(zip(NAMES, run(t, 1.0)))
    t["h"][3] = 0.0  # a block that put out nothing: rstd = eps^-1/2
    t["x"][7, 100] = float("nan")
    t["h"][9, 5] = float("inf")
    got = dict(zip(NAMES, run(t, 1.0)))
    assert torch.equal(got["s"][3], t["x"][3])
    assert bool(torch.isfinite(got["dh"][3]).all())
    keep = [r for r in range(12) if r not in (3, 7, 9)]
    for name in ("s", "y", "dx", "dh", "dgate"):
        assert torch.equal(got[name][keep], clean[name][keep])
        assert bool(torch.isnan(got[name][[7, 9]]).any())


def test_same_bits_on_every_run_and_on_another_stream():
    t = make(3000, 2048, "channel", BF16)
    a = run(t, 0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(t, 0.9)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("gate", GATES)
def test_gradient_against_differences_of_the_definition(gate):
    t = make(6, 48, gate, F32)
    grads = dict(zip(NAMES, run(t, 0.7)))
    args = ("x", "h", "w1", "gate", "w2")
    slots = dict(zip(args, ("dx", "dh", "dpost_weight", "dgate", "dpre_weight")))
    limits = block_norm64(*(t[n] for n in args), 0.7, EPS, t["ds"], t["dy"])
    gen = torch.Generator(device="cuda").manual_seed(3)
    for name in args:
        if t[name] is None:
            continue
        d = torch.randn(t[name].shape, generator=gen, device="cuda", dtype=torch.float64)
        d /= d.norm()
        e, loss = 1e-5, []
        for sign in (1, -1):
            moved = {n: None if t[n] is None else t[n].double() for n in args}
            moved[name] = moved[name] + sign * e * d
            out = block_norm64(*(moved[n] for n in args), 0.7, EPS, t["ds"].double(),
                               t["dy"].double())
            loss.append(float((out["s"][0] * t["ds"].double()).sum()
                              + (out["y"][0] * t["dy"].double()).sum()))
        want = (loss[0] - loss[1]) / (2 * e)
        got = float((grads[slots[name]].double() * d).sum())
        slack = float((limits[slots[name]][1] * d.abs()).sum())
        # e^2 times third derivatives of order 10, and 2^-52 of a loss of order 100 over e
        assert abs(got - want) <= slack + 1e-8, (name, got, want, slack)


def test_autograd_nodes_match_the_pair():
    for gate in GATES:
        t = make(50, 256, gate, BF16)
        want = run(t, 0.6)
        names = [n for n in ("x", "h", "w1", "gate", "w2") if t[n] is not None]
        leaf = {n: t[n].clone().requires_grad_(True) for n in names}
        s, y = pair.BlockNorm.apply(leaf["x"], leaf["h"], leaf["w1"], leaf.get("gate"), leaf["w2"],
                                    0.6, EPS)
        assert torch.equal(s, want[0]) and torch.equal(y, want[1])
        torch.autograd.backward((s, y), (t["ds"], t["dy"]))
        fn = bind(BLOCK_NORM, pair)
        again = {n: t[n].clone().requires_grad_(True) for n in names}
        out = fn(again["x"], again["h"], again["w1"], again.get("gate"), again["w2"], 0.6, EPS)
        out.backward(torch.stack((t["ds"], t["dy"])))
        grads = [g for g in want[2:] if g is not None]
        for n, g in zip(names, grads):
            assert torch.equal(leaf[n].grad, g) and torch.equal(again[n].grad, g)
    # only the residual stream is used downstream
    t = make(10, 256, "none", F32)
    x = t["x"].clone().requires_grad_(True)
    s, _ = pair.BlockNorm.apply(x, t["h"], t["w1"], None, t["w2"], 1.0, EPS)
    s.backward(t["ds"])
    assert torch.equal(x.grad, t["ds"])


def test_a_captured_graph_replays_beside_an_eager_graph():
    """Forward and backward captured while an eager autograd graph of the same tensors lives."""
    t = make(700, 1024, "channel", BF16)
    leaves = [t[n].clone().requires_grad_(True) for n in ("x", "h", "w1", "gate", "w2")]
    eager = pair.BlockNorm.apply(*leaves, 0.5, EPS)
    run(t, 0.5, split=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(t, 0.5, split=True)
    for seed in range(4):
        fresh = make(700, 1024, "channel", BF16, seed)
        for n in t:
            t[n].copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for x, y in zip(got, run(fresh, 0.5, split=True)):
            assert torch.equal(x, y)
    first = make(700, 1024, "channel", BF16)
    torch.autograd.backward(eager, (first["ds"], first["dy"]))
    for leaf, want in zip(leaves, run(first, 0.5, split=True)[2:]):
        assert torch.equal(leaf.grad, want)


def test_offsets_past_32_bits():
    rows, cols = (1 << 31) // 4096 + 3, 4096
    print(f"\n[gpu-block-norm] {rows} rows of {cols}", flush=True)
    tail = make(3, cols, "row", BF16, seed=5)
    t = {n: torch.full((rows, cols), 0.5, dtype=BF16, device="cuda") for n in ("x", "h", "ds", "dy")}
    t["gate"] = torch.full((rows, 1), 0.25, dtype=BF16, device="cuda")
    for n in t:
        t[n][-3:] = tail[n]
    t["w1"], t["w2"] = tail["w1"], tail["w2"]
    got = dict(zip(NAMES, run(t, 1.0, split=True)))
    want = block_norm64(*(tail[n] for n in ("x", "h", "w1", "gate", "w2")), 1.0, EPS, tail["ds"],
                        tail["dy"])
    for name in ("s", "y", "dx", "dh", "dgate"):
        assert_within(name, got[name][-3:], *want[name])
    del t, got
    torch.cuda.empty_cache()
