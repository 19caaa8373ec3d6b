"""Embedding lookup and its gradient against sums in 64 bits (tests/step_refs.py)."""

import pytest
import torch

from evograd_amd.bind import bind
from evograd_amd.decls import EMBEDDING
from evograd_amd.pairs import embedding as pair
from tests.packed_refs import assert_within
from tests.step_refs import embedding64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(*shape, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def tokens(T, V, how="flat", seed=0, dtype=torch.int32):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (T,), generator=g)
    if how == "low":  # frequencies that fall with the id
        ids = (V ** torch.rand(T, generator=g, dtype=torch.float64)).long().clamp(1, V) - 1
    elif how == "same":
        ids = torch.full((T,), V - 1)
    elif how == "mixed":
        ids[torch.rand(T, generator=g) < 0.4] = V // 2
        ids[torch.rand(T, generator=g) < 0.1] = -100
    return ids.to("cuda", dtype)


def assert_rows(name, got, value, bound):
    """assert_within, where a NaN value asks for a NaN."""
    nan = value.isnan()
    assert torch.equal(got.isnan(), nan), name
    assert_within(name, got.masked_fill(nan, 0), value.masked_fill(nan, 0), bound.masked_fill(nan, 0))


def both_ways(weight, ids, dout, scale=1.0, ignore_index=-100):
    out, saved = pair.embedding_forward_with_saved(weight, ids, scale, ignore_index)
    return out, pair.embedding_backward_from_saved(dout, saved, scale, ignore_index)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("T,V,H,how", (
    (1, 1, 1, "flat"), (1, 300, 64, "flat"), (31, 7, 3, "flat"), (32, 50, 8, "flat"),
    (33, 50, 136, "flat"), (64, 2, 24, "flat"), (65, 1, 40, "flat"), (257, 1000, 127, "mixed"),
    (1000, 255, 512, "low"), (1000, 256, 520, "same"), (1024, 257, 64, "mixed"),
    (1025, 4096, 65, "low"), (3000, 70000, 100, "low"), (5000, 300, 2056, "mixed"),
    (2100, 3, 4100, "flat"), (900, 262144, 8, "low"), (9000, 262145, 9, "mixed"),
    (70, 2500000, 16, "flat"), (17000, 5000, 33, "low"), (40000, 600, 20, "mixed")))
def test_against_64_bits(T, V, H, how, dtype):
    print(f"\n[gpu-embedding] {T} {V}x{H} {how} {dtype}", flush=True)
    weight, dout, ids = normal(V, H, dtype=dtype), normal(T, H, dtype=dtype, seed=1), tokens(T, V, how)
    out, grad = both_ways(weight, ids, dout, 1.75)
    want, wgrad = embedding64(weight, ids, 1.75, -100, dout)
    assert out.dtype == dtype and grad.dtype == dtype and grad.shape == weight.shape
    assert_within("out", out, *want)
    assert_within("dweight", grad, *wgrad)
    again = both_ways(weight, ids, dout, 1.75)
    assert torch.equal(out, again[0]) and torch.equal(grad, again[1])


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("index", (torch.int32, torch.int64))
def test_tokens_outside_the_table(index, dtype):
    V, H = 40, 48
    ids = torch.tensor([3, -1, 40, 39, 7, 3, -100, 2 ** 31 - 1, -(2 ** 31), 0], dtype=index, device="cuda")
    if index == torch.int64:
        ids[7], ids[8] = 2 ** 40 + 3, -(2 ** 40) + 3  # whose low words are ids of the table
    weight, dout = normal(V, H, dtype=dtype), normal(10, H, dtype=dtype, seed=1)
    dout[[1, 2, 6, 7, 8]] = float("nan")  # of tokens that have no gradient
    for ignore in (-100, 7, -1):
        out, grad = both_ways(weight, ids, dout, 1.0, ignore)
        clean = dout.clone()
        clean[[1, 2, 6, 7, 8]] = 0
        want, wgrad = embedding64(weight, ids, 1.0, ignore, clean)
        assert_rows("out", out, *want)
        assert_within("dweight", grad, *wgrad)


def test_a_scale_of_one_copies_bits():
    for dtype in (BF16, F16, F32):
        weight, ids = normal(99, 130, dtype=dtype), tokens(50, 99)
        out, _ = pair.embedding_forward_with_saved(weight, ids)
        assert torch.equal(out, weight[ids.long()])


def test_ids_of_one_bucket_and_a_run_over_many_pieces():
    """Ids a power of two apart share a bucket; then one id takes every token but a few."""
    V, H = 70000, 24
    weight, dout = normal(V, H, dtype=F32), normal(20000, H, dtype=F32, seed=1)
    strided = (tokens(20000, 270).long() * 256 + 5).to(torch.int32)
    alone = torch.full((20000,), 4100, dtype=torch.int32, device="cuda")
    alone[[0, 7, 31, 32, 9999, 19999]] = torch.tensor([1, 4099, 4101, 69999, 0, 2], dtype=torch.int32,
                                                      device="cuda")
    for ids in (strided, alone):
        _, grad = both_ways(weight, ids, dout)
        assert_within("dweight", grad, *embedding64(weight, ids, 1.0, -100, dout)[1])


def test_no_tokens_and_empty_tables():
    for T, V, H in ((0, 5, 8), (3, 5, 0), (0, 0, 8)):
        weight, ids = normal(V, H, dtype=BF16), torch.zeros(T, dtype=torch.int64, device="cuda")
        out, grad = both_ways(weight, ids, normal(T, H, dtype=BF16))
        assert out.shape == (T, H) and grad.shape == (V, H)
        assert int(torch.count_nonzero(grad)) == 0
    out, grad = both_ways(normal(0, 8, dtype=F32), tokens(4, 1), normal(4, 8, dtype=F32))
    assert bool(out.isnan().all()) and grad.shape == (0, 8)


def test_every_token_ignored():
    weight = normal(30, 64, dtype=F16)
    ids = torch.full((100,), -100, dtype=torch.int32, device="cuda")
    out, grad = both_ways(weight, ids, torch.full((100, 64), float("inf"), dtype=F16, device="cuda"))
    assert int(torch.count_nonzero(out)) == 0 and int(torch.count_nonzero(grad)) == 0


@pytest.mark.parametrize("dtype", (BF16, F32))
def test_shapes_of_ids_and_strided_or_unaligned_tensors(dtype):
    V, H = 60, 72
    room = normal(V * H + 1, dtype=dtype)
    weight = room[1:].view(V, H)  # not 16-byte aligned
    ids = tokens(12 * 20, V).view(12, 20)
    dout = normal(12, 20, H, dtype=dtype, seed=2)
    want = both_ways(weight.clone(), ids.flatten(), dout.view(-1, H))
    out, grad = both_ways(weight, ids, dout)
    assert out.shape == (12, 20, H)
    assert torch.equal(out.view(-1, H), want[0]) and torch.equal(grad, want[1])
    turned = both_ways(weight.t().contiguous().t(), ids.t().contiguous().t(),
                       dout.transpose(0, 2).contiguous().transpose(0, 2))
    assert torch.equal(turned[0], out) and torch.equal(turned[1], grad)
    wide = torch.cat((dout, dout), -1)[..., :H]
    assert torch.equal(both_ways(weight, ids, wide)[1], grad)
    odd = normal(dout.numel() + 1, dtype=dtype)[1:].view(dout.shape)
    odd.copy_(dout)
    assert torch.equal(both_ways(weight, ids, odd)[1], grad)
    one = both_ways(weight, ids[0, 0], dout[0, 0])
    assert one[0].shape == (H,) and torch.equal(one[0], out[0, 0])


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("H", (64, 77))
def test_added_into_a_gradient(dtype, H):
    T, V = 700, 500
    weight, dout, ids = normal(V, H, dtype=dtype), normal(T, H, dtype=dtype, seed=1), tokens(T, V, "mixed")
    ids[ids == 3] = 4
    _, saved = pair.embedding_forward_with_saved(weight, ids)
    old = normal(V, H, dtype=dtype, seed=5)
    old[3] = float("nan")  # of no token: neither read nor written
    got = old.clone()
    assert pair.embedding_backward_into(got, dout, saved, 0.5) is got
    _, (grad, bound) = embedding64(weight, ids, 0.5, -100, dout)
    used = torch.zeros(V, dtype=torch.bool, device="cuda")
    used[ids[ids >= 0].long()] = True
    assert torch.equal(got[~used].nan_to_num(7.0), old[~used].nan_to_num(7.0))
    total = old.double() + grad
    room = bound + (2.0 ** -24 + torch.finfo(dtype).eps / 2) * total.abs()
    assert_within("dweight", got[used], total[used], room[used])


def test_a_non_finite_row_stays_in_its_token_s_row():
    weight, dout, ids = normal(50, 64, dtype=BF16), normal(400, 64, dtype=BF16, seed=1), tokens(400, 50)
    clean = both_ways(weight, ids, dout)[1]
    dout[17, 5], dout[100, 6] = float("nan"), float("inf")
    grad = both_ways(weight, ids, dout)[1]
    a, b = int(ids[17]), int(ids[100])
    assert bool(grad[a, 5].isnan()) and not bool(grad[b, 6].isfinite())
    grad[a, 5], grad[b, 6] = clean[a, 5], clean[b, 6]
    assert torch.equal(grad, clean)


def test_tables_past_32_bit_offsets():
    V, H = 540000, 4096  # 2.2e9 elements
    weight = torch.zeros(V, H, dtype=BF16, device="cuda")
    ids = torch.tensor([V - 1, 0, 525000, V - 1, 3], dtype=torch.int32, device="cuda")
    rows = normal(5, H, dtype=BF16)
    weight[ids.long()] = rows  # of the two rows for one token either may be there
    rows = torch.stack([weight[int(i)] for i in ids])
    dout = normal(5, H, dtype=BF16, seed=1)
    out, saved = pair.embedding_forward_with_saved(weight, ids)
    assert torch.equal(out, rows)
    del weight
    grad = pair.embedding_backward_from_saved(dout, saved)
    assert torch.equal(grad[V - 1], (dout[0].float() + dout[3].float()).to(BF16))
    for t in (1, 2, 4):
        assert torch.equal(grad[int(ids[t])], dout[t])
    assert int(torch.count_nonzero(grad)) == sum(
        int(torch.count_nonzero(grad[v])) for v in (V - 1, 0, 525000, 3))


def test_autograd_node_and_another_stream():
    weight, dout, ids = normal(80, 96, dtype=BF16), normal(60, 96, dtype=BF16, seed=1), tokens(60, 80)
    want = both_ways(weight, ids, dout, 2.0)
    leaf = weight.clone().requires_grad_(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = bind(EMBEDDING, pair)(leaf, ids, scale=2.0)
        out.backward(dout)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out, want[0]) and torch.equal(leaf.grad, want[1])


def test_a_captured_graph_replays_with_other_tokens():
    T, V, H = 300, 128, 64
    weight, dout, ids = normal(V, H, dtype=BF16), normal(T, H, dtype=BF16, seed=1), tokens(T, V)
    both_ways(weight, ids, dout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = both_ways(weight, ids, dout)
    for seed, how in enumerate(("flat", "same", "mixed", "low")):
        ids.copy_(tokens(T, V, how, seed))
        dout.copy_(normal(T, H, dtype=BF16, seed=10 + seed))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), grad.clone()
        for x, y in zip(got, both_ways(weight, ids, dout)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("T", (1, 2, 9, 64, 255, 256, 257))
def test_few_tokens(T, dtype):
    """Around the limit of the single launch: runs over its pieces, buckets of many tokens."""
    for V, H, how in ((1, 520, "flat"), (2, 2056, "flat"), (300, 33, "mixed"), (5000, 1100, "low"),
                      (70000, 24, "strided"), (262144, 40, "flat"), (262145, 40, "low")):
        print(f"\n[gpu-embedding] few {T} {V}x{H} {how} {dtype}", flush=True)
        strided = how == "strided"  # in one bucket, whatever their number below 256 is
        ids = tokens(T, 6).long() * 256 + 3 if strided else tokens(T, V, how, dtype=torch.int64)
        weight, dout = normal(V, H, dtype=dtype), normal(T, H, dtype=dtype, seed=1)
        _, grad = both_ways(weight, ids, dout, 0.75)
        want, bound = embedding64(weight, ids, 0.75, -100, dout)[1]
        assert_within("dweight", grad, want, bound)
        assert torch.equal(grad, both_ways(weight, ids.int(), dout, 0.75)[1])
        old = normal(V, H, dtype=dtype, seed=4)
        _, saved = pair.embedding_forward_with_saved(weight, ids)
        got = pair.embedding_backward_into(old.clone(), dout, saved, 0.75)
        total = old.double() + want
        room = bound + (2.0 ** -24 + torch.finfo(dtype).eps / 2) * total.abs()
        used = torch.zeros(V, dtype=torch.bool, device="cuda")
        used[ids[ids >= 0]] = True
        assert_within("into", got[used], total[used], room[used])
        assert torch.equal(got[~used], old[~used])


def test_few_tokens_added_past_32_bit_offsets():
    V, H = 540000, 4096  # 2.2e9 elements
    grad = torch.zeros(V, H, dtype=BF16, device="cuda")
    ids = torch.tensor([V - 1, 0, 525000, V - 1, 3], dtype=torch.int32, device="cuda")
    dout = normal(5, H, dtype=BF16, seed=1)
    saved = (ids, V, H, BF16)
    pair.embedding_backward_into(grad, dout, saved)
    assert torch.equal(grad[V - 1], (dout[0].float() + dout[3].float()).to(BF16))
    for t in (1, 2, 4):
        assert torch.equal(grad[int(ids[t])], dout[t])
    assert int(torch.count_nonzero(grad)) == sum(
        int(torch.count_nonzero(grad[v])) for v in (V - 1, 0, 525000, 3))


def test_a_captured_graph_of_few_tokens():
    T, V, H = 200, 128, 72
    dout, ids, table = normal(T, H, dtype=BF16, seed=1), tokens(T, V), normal(V, H, dtype=BF16)
    saved, into = (ids, V, H, BF16), table.clone()
    pair.embedding_backward_into(into, dout, saved)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = pair.embedding_backward_from_saved(dout, saved)
        pair.embedding_backward_into(into, dout, saved)
    for seed, how in enumerate(("flat", "same", "mixed", "low")):
        ids.copy_(tokens(T, V, how, seed))
        dout.copy_(normal(T, H, dtype=BF16, seed=10 + seed))
        into.copy_(table)
        graph.replay()
        torch.cuda.synchronize()
        got = grad.clone(), into.clone()
        assert torch.equal(got[0], pair.embedding_backward_from_saved(dout, saved))
        assert torch.equal(got[1], pair.embedding_backward_into(table.clone(), dout, saved))


@pytest.mark.parametrize("T,V,H", ((3, 5, 2 ** 20), (300, 5, 2 ** 20), (2, 3, 2 ** 20 - 1)))
def test_the_widest_rows(T, V, H):
    print(f"\n[gpu-embedding] widest {T} {V}x{H}", flush=True)
    weight, dout, ids = normal(V, H, dtype=BF16), normal(T, H, dtype=BF16, seed=1), tokens(T, V - 1)
    out, grad = both_ways(weight, ids, dout, 0.5)
    (value, bound), (gvalue, gbound) = embedding64(weight, ids, 0.5, -100, dout)
    assert_within("out", out, value, bound)
    assert_within("dweight", grad, gvalue, gbound)
