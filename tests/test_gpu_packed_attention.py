"""Packed causal attention against its definition in 64 bits, with the bounds that the kernels'
roundings allow (tests/packed_refs.py)."""

import sys

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.bind import bind
from evograd_amd.decls import PACKED_ATTENTION
from evograd_amd.pairs import packed_attention as pair
from evograd_amd.pairs._util import strides_arg
from tests.packed_refs import assert_within, attention64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def bounds(lengths, device="cuda"):
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths, dtype=torch.int32).cumsum(0)
    return cu.to(device)


def make(lengths, H, KVH, D, dtype, pad=0, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lengths) + pad
    shapes = ((T, H, D), (T, KVH, D), (T, KVH, D), (T, H, D))
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(dtype) for s in shapes]


def run(q, k, v, do, cu):
    o, saved = pair.packed_attention_forward_with_saved(q, k, v, cu)
    return (o, *pair.packed_attention_backward_from_saved(do, saved))


def takes_mfma(q, k, v):
    return q.dtype != F32 and q.shape[2] in (64, 128)


def check(lengths, H, KVH, D, dtype, pad=0, seed=0, scale=1.0):
    print(f"\n[gpu-packed] {lengths[:8]}x{len(lengths)} {H}/{KVH} D={D} {dtype} pad={pad}",
          flush=True)
    q, k, v, do = make(lengths, H, KVH, D, dtype, pad, seed, scale)
    got = run(q, k, v, do, bounds(lengths))
    want = attention64(q, k, v, do, lengths, takes_mfma(q, k, v))
    for name, x, (value, bound) in zip(("o", "dq", "dk", "dv"), got, want):
        assert x.dtype == dtype
        assert_within(name, x, value, bound)
    n = sum(lengths)
    for x in got:
        assert int(torch.count_nonzero(x[n:])) == 0


# One sequence of each length: a single row, both sides of the 16-, 64- and 128-row tiles.
@pytest.mark.parametrize("n", (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 300))
@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (64, F32)))
def test_one_sequence_of_every_tile_edge(n, D, dtype):
    check([n], 4, 2, D, dtype, seed=n)


LENGTHS = {
    "equal": [64, 64, 64],
    "ragged": [5, 130, 1, 77, 64, 3],
    "empty": [0, 40, 0, 0, 129, 0],
    "ones": [1] * 40,
    "long_and_short": [700, 1, 2, 3, 90],
    "past_a_wave": [3, 0, 17] * 23 + [140],
    "past_its_registers": [2, 0, 5, 1] * 70 + [150, 33],
}


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("H,KVH,D,dtype", (
    (8, 2, 128, BF16), (3, 1, 64, BF16), (4, 4, 128, F16), (4, 1, 64, F16),
    (2, 1, 64, F32), (2, 2, 128, F32), (4, 2, 18, F32), (4, 2, 96, BF16), (2, 1, 32, F16),
    (1, 1, 2, BF16)))
def test_batches(name, H, KVH, D, dtype):
    check(LENGTHS[name], H, KVH, D, dtype, pad=7 if name != "equal" else 0)


@pytest.mark.parametrize("dtype,D", ((BF16, 128), (F16, 64), (F32, 32)))
def test_thousands_of_sequences(dtype, D):
    """Empty, one-token and longer ones, ordered by a plan on the GPU."""
    check([1, 0, 3] * 500 + [200] + [17, 2] * 30 + [0, 0, 70], 2, 1, D, dtype, pad=11)


@pytest.mark.parametrize("dtype,D", ((BF16, 128), (BF16, 64), (F32, 64)))
@pytest.mark.parametrize("lengths,H,KVH", (
    ([1500], 8, 1), ([1200, 30, 600], 8, 8), ([2100, 100], 2, 1), ([900, 800, 20], 32, 8)))
def test_long_walks(lengths, H, KVH, dtype, D):
    """Grids small and large: walks cut into pieces and whole ones, key groups taken by turns."""
    if dtype == F32 and H == 32:
        H, KVH = 8, 2
    check(lengths, H, KVH, D, dtype, pad=3)


@pytest.mark.parametrize("dtype,D", ((BF16, 128), (F16, 64), (F32, 32)))
def test_large_scores(dtype, D):
    """Scores spread over hundreds: one key takes each row, the running maximum moves often."""
    check([150, 70], 4, 2, D, dtype, seed=5, scale=6.0)


def test_all_sequences_empty_or_none():
    q, k, v, do = make([], 4, 2, 64, BF16, pad=33)
    for cu in (torch.zeros(1, dtype=torch.int32, device="cuda"), bounds([0, 0, 0])):
        for x in run(q.fill_(float("nan")), k, v, do, cu):
            assert int(torch.count_nonzero(x)) == 0
    q, k, v, do = make([], 4, 2, 64, BF16)
    for x in run(q, k, v, do, bounds([0])):
        assert x.numel() == 0


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (32, F32), (80, BF16)))
def test_strided_inputs_give_the_contiguous_run_s_bits(D, dtype):
    lengths, H, KVH = [70, 1, 130], 4, 2
    T = sum(lengths) + 4
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(T, (H + 2 * KVH) * D, generator=g, device="cuda").to(dtype)
    q = qkv[:, :H * D].view(T, H, D)
    k = qkv[:, H * D:(H + KVH) * D].view(T, KVH, D)
    v = qkv[:, (H + KVH) * D:].view(T, KVH, D)
    do = torch.randn(T, H, D, generator=g, device="cuda").to(dtype)
    cu = bounds(lengths)
    a = run(q, k, v, do, cu)
    b = run(q.contiguous(), k.contiguous(), v.contiguous(), do, cu)
    # heads outside tokens, a transposed do, and one value row shared by every token
    c = run(q.transpose(0, 1).contiguous().transpose(0, 1), k, v,
            do.transpose(0, 1).contiguous().transpose(0, 1), cu)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    shared = v[:1].expand(T, KVH, D)
    for x, y in zip(run(q, k, shared, do, cu), run(q, k, shared.contiguous(), do, cu)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
def test_rows_at_any_alignment(dtype):
    """Views one element off a 16-byte boundary."""
    lengths, H, KVH, D = [66, 20], 2, 1, 64
    parts = make(lengths, H, KVH, D, dtype, seed=3)
    off = []
    for t in parts[:3]:
        room = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        view = room[1:].view(t.shape)
        view.copy_(t)
        off.append(view)
    got = run(*off, parts[3], bounds(lengths))
    want = attention64(*parts, lengths, False)
    wide = attention64(*parts, lengths, True)
    for name, x, (value, bound), (_, loose) in zip(("o", "dq", "dk", "dv"), got, want, wide):
        assert_within(name, x, value, torch.maximum(bound, loose))


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (64, F32)))
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), float("-inf")))
def test_values_behind_the_last_sequence_are_read_into_nothing(D, dtype, bad):
    lengths = [61, 5, 66]
    clean = make(lengths, 4, 2, D, dtype, pad=40)
    a = run(*clean, bounds(lengths))
    dirty = [t.clone() for t in clean]
    for t in dirty:
        t[sum(lengths):] = bad
    b = run(*dirty, bounds(lengths))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def reaches_only_the_rows_that_see_it(lengths, row, bad, H, KVH, D, dtype):
    """A value of `row` of the second sequence's k, v, q and do is `bad`: everything that does
    not depend on it is what it is without it."""
    first, own_end, T = lengths[0], sum(lengths[:2]), sum(lengths)
    at = first + row
    clean = make(lengths, H, KVH, D, dtype, seed=2)
    cu = bounds(lengths)
    o_, dq_, dk_, dv_ = attention64(*clean, lengths, takes_mfma(*clean[:3]))
    before, own, after = slice(first, at), slice(at, own_end), slice(at + 1, own_end)
    others = torch.cat((torch.arange(first), torch.arange(own_end, T))).cuda()

    def clean_values(name, x, want, rows, cols=slice(None)):
        assert_within(name, x[rows][..., cols], want[0][rows][..., cols], want[1][rows][..., cols])

    # k, then v, of the row: rows before it and other sequences
    for which in (1, 2):
        t = [x.clone() for x in clean]
        t[which][at, :, 5] = bad
        o, dq, dk, dv = run(*t, cu)
        for rows in (before, others):
            clean_values("o", o, o_, rows)
            clean_values("dq", dq, dq_, rows)
        clean_values("dk", dk, dk_, others)
        clean_values("dv", dv, dv_, others)
        if which == 2:
            assert not bool(torch.isfinite(o[own, :, 5]).any())
            clean_values("o", o, o_, own, slice(6, None))
    # q of the row: every other row, and the keys after it
    t = [x.clone() for x in clean]
    t[0][at, :, 5] = bad
    o, dq, dk, dv = run(*t, cu)
    for rows in (before, after, others):
        clean_values("o", o, o_, rows)
        clean_values("dq", dq, dq_, rows)
    for rows in (after, others):
        clean_values("dk", dk, dk_, rows)
        clean_values("dv", dv, dv_, rows)
    assert bool(torch.isnan(dk[before]).all()) and bool(torch.isnan(dq[at]).any())
    # do of the row
    t = [x.clone() for x in clean]
    t[3][at, :, 5] = bad
    o, dq, dk, dv = run(*t, cu)
    clean_values("o", o, o_, slice(None))
    for rows in (before, after, others):
        clean_values("dq", dq, dq_, rows)
    for rows in (after, others):
        clean_values("dk", dk, dk_, rows)
        clean_values("dv", dv, dv_, rows)


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (64, F32)))
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), float("-inf")))
@pytest.mark.parametrize("row", (0, 3, 70, 129))
def test_a_non_finite_row_reaches_only_the_rows_that_see_it(D, dtype, bad, row):
    reaches_only_the_rows_that_see_it([40, 130, 9], row, bad, 4, 2, D, dtype)


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, BF16), (64, F32)))
@pytest.mark.parametrize("bad", (float("nan"), float("inf")))
@pytest.mark.parametrize("H,KVH", ((4, 1), (3, 3), (48, 12)))
def test_a_non_finite_row_of_long_sequences(H, KVH, bad, D, dtype):
    """Two key groups, whole and cut walks, groups of four heads and none."""
    reaches_only_the_rows_that_see_it([350, 900, 20], 333, bad, H, KVH, D, dtype)


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (32, F32)))
def test_same_bits_on_every_run_and_on_another_stream(D, dtype):
    lengths = [300, 7, 450, 0, 64]
    t = make(lengths, 8, 2, D, dtype, pad=5)
    cu = bounds(lengths)
    a = run(*t, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(*t, cu)
        c = run(*t, cu)
    torch.cuda.current_stream().wait_stream(side)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F32)))
@pytest.mark.parametrize("many", (False, True))
def test_a_captured_graph_replays_with_other_lengths(many, D, dtype):
    sets = ([100, 60, 40], [1, 199, 0], [0, 0, 150], [64, 64, 72])
    if many:  # past what the kernels search themselves
        sets = ([1] * 150 + [0] * 150, [0] * 299 + [200], [0, 1] * 100 + [99] + [0] * 99,
                [150] + [0, 0] * 149 + [50])
    T = 200
    t = make([T], 4, 2, D, dtype)
    cu = bounds(sets[0])
    run(*t, cu)  # warm up outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*t, cu)
    for seed, lengths in enumerate(sets * 2):
        fresh = make([T], 4, 2, D, dtype, seed=seed)
        for x, y in zip(t, fresh):
            x.copy_(y)
        cu.copy_(bounds(lengths))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        for x, y in zip(got, run(*fresh, bounds(lengths))):
            assert torch.equal(x, y)


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (64, F32)))
@pytest.mark.parametrize("many", (False, True))
def test_bounds_that_are_no_sequences_stay_inside_the_tensors(many, D, dtype):
    """Decreasing, negative, overlapping and far bounds give undefined rows; every tensor lies
    between guards, which stay as they were, and a sound call on the same memory afterwards is
    right."""
    H, KVH, guard = 8, 2, 4096
    lengths = [1] * 260 + [140] if many else [100, 0, 60, 40]
    T = sum(lengths)
    n = len(lengths)
    held = []

    def guarded(shape, dt):
        count = torch.Size(shape).numel()
        whole = torch.full((count + 2 * guard,), 7.0, device="cuda", dtype=dt)
        held.append((whole, count))
        return whole[guard:guard + count].view(shape)

    src = make([T], H, KVH, D, dtype)
    q, k, v, do = [guarded(t.shape, dtype).copy_(t) for t in src]
    o, dq = guarded(q.shape, dtype), guarded(q.shape, dtype)
    dk, dv = guarded(k.shape, dtype), guarded(k.shape, dtype)
    lse = guarded((H, T), F32)
    fwd_bytes = _lib.query("eg_packed_attn_fwd_workspace_bytes", n)
    bwd_bytes = _lib.query("eg_packed_attn_workspace_bytes", T, n, H, KVH, D, _lib.dtype_tag(dtype))
    fws, bws = guarded((fwd_bytes // 4 + 1,), F32), guarded((bwd_bytes // 4 + 1,), F32)
    steps = strides_arg(q, k, v)
    common = (T, n, H, KVH, D, steps, D ** -0.5, _lib.dtype_tag(dtype), _lib.stream_of(q))

    def step(cu):
        _lib.call("eg_packed_attn_fwd", *map(_lib.ptr, (q, k, v, cu, o, lse, fws)), *common)
        _lib.call("eg_packed_attn_bwd",
                  *map(_lib.ptr, (do, q, k, v, cu, o, lse, dq, dk, dv, bws)), *common)
        torch.cuda.synchronize()

    far = (1 << 31) - 1
    g = torch.Generator().manual_seed(3)
    for bad in ([T, 0] * n, [0, T] * n, [-5, far] * n, [far] * (2 * n), [-far] * (2 * n),
                torch.randint(-T, 3 * T, (2 * n,), generator=g).tolist()):
        cu = torch.tensor(bad[:n + 1], dtype=torch.int32, device="cuda")
        print(f"\n[gpu-packed] bad bounds {bad[:4]} x {n} D={D} {dtype}", flush=True)
        step(cu)
        for whole, count in held:
            assert bool((whole[:guard] == 7).all()) and bool((whole[guard + count:] == 7).all())
        for x, y in zip((q, k, v, do), src):
            assert torch.equal(x, y)
    cu = bounds(lengths)
    step(cu)
    for x, y in zip((o, dq, dk, dv), run(*src, cu)):
        assert torch.equal(x, y)


def test_gradient_against_differences_of_the_definition():
    """<gradient, d> against (L(t + e d) - L(t - e d)) / 2e of the 64-bit forward, L = <o, do>:
    the differences are off by e^2 times third derivatives (of order one here: 1e-8) and by
    2^-52 / e, the gradients by their own bounds."""
    lengths, H, KVH, D = [19, 1, 40], 4, 2, 32
    q, k, v, do = make(lengths, H, KVH, D, F32, scale=0.5)
    grads = run(q, k, v, do, bounds(lengths))[1:]
    limits = [b for _, b in attention64(q, k, v, do, lengths, False)][1:]
    g = torch.Generator(device="cuda").manual_seed(9)
    for i, t in enumerate((q, k, v)):
        d = torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64)
        d /= d.norm()
        e, loss = 1e-4, []
        for sign in (1, -1):
            moved = [x.double() for x in (q, k, v)]
            moved[i] = moved[i] + sign * e * d
            o = attention64(*moved, do.double(), lengths, False)[0][0]
            loss.append(float((o * do.double()).sum()))
        want = (loss[0] - loss[1]) / (2 * e)
        got = float((grads[i].double() * d).sum())
        slack = float((limits[i] * d.abs()).sum())
        assert abs(got - want) <= slack + 1e-6, (i, got, want, slack)


def test_bound_callable_matches_the_pair():
    lengths = [30, 45]
    q, k, v, do = make(lengths, 4, 2, 64, BF16)
    cu = bounds(lengths)
    fn = bind(PACKED_ATTENTION, pair)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o = fn(*leaves, cu)
    o.backward(do)
    want = run(q, k, v, do, cu)
    assert torch.equal(o.detach(), want[0])
    for leaf, w in zip(leaves, want[1:]):
        assert torch.equal(leaf.grad, w)


def test_offsets_past_32_bits():
    """2^31 elements of q in front of the last sequences: their results are the ones they have
    by themselves."""
    H, KVH, D, n = 64, 8, 128, 128
    T = (1 << 31) // (H * D) + 2 * n
    lengths = [n] * (T // n)
    print(f"\n[gpu-packed] {T} tokens x {H} heads x {D}", flush=True)
    sys.stdout.flush()
    q = torch.empty(T, H, D, device="cuda", dtype=BF16)
    k = torch.empty(T, KVH, D, device="cuda", dtype=BF16)
    v, do = torch.empty_like(k), torch.empty_like(q)
    for t in (q, k, v, do):
        t.fill_(0.25)
    tail = make([n, n], H, KVH, D, BF16, seed=4)
    for t, x in zip((q, k, v, do), tail):
        t[-2 * n:] = x
    got = run(q, k, v, do, bounds(lengths))
    want = run(*tail, bounds([n, n]))
    value = attention64(*tail, [n, n], True)
    for name, x, y, (ref, bound) in zip(("o", "dq", "dk", "dv"), got, want, value):
        assert_within(name, x[-2 * n:], ref, bound)
        assert_within(name, y, ref, bound)
    del q, k, v, do, got
    torch.cuda.empty_cache()
