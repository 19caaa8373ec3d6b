"""The embedding's gradient by each of its ways: few tokens in one launch and more of them in three,
into tables of any alignment, with tokens that have no row."""

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.bind import bind
from evograd_amd.decls import EMBEDDING
from evograd_amd.pairs import embedding as pair
from evograd_amd.pairs._util import workspace
from tests.packed_refs import assert_within
from tests.step_refs import embedding64
from tests.test_gpu_embedding import assert_rows, both_ways, normal, tokens

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# up to 256 tokens: one launch; past 8192 the order reads the ids a second time
COUNTS = (10, 256, 257, 600, 8192, 9001)


def used_rows(ids, V, ignore=-100):
    ids = ids.long().flatten()
    used = torch.zeros(V, dtype=torch.bool, device="cuda")
    used[ids[(ids >= 0) & (ids < V) & (ids != ignore)]] = True
    return used


def assert_added(got, old, ids, grad, bound, ignore=-100):
    """``got``: the gradient added to ``old``, in the rows with tokens alone."""
    used = used_rows(ids, old.shape[0], ignore)
    total = old.double() + grad
    room = bound + (2.0 ** -24 + torch.finfo(old.dtype).eps / 2) * total.abs()
    assert_within("added", got[used], total[used], room[used])
    assert torch.equal(got[~used].nan_to_num(7.0), old[~used].nan_to_num(7.0))


@pytest.mark.parametrize("H", (48, 50))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("index", (torch.int32, torch.int64))
@pytest.mark.parametrize("T", COUNTS)
def test_tokens_without_a_row(T, index, dtype, H):
    V = 400
    print(f"\n[gpu-embedding] without a row {T} {index} {dtype} {H}", flush=True)
    ids = tokens(T, V, "low", dtype=torch.int64)
    ids[::11] = 7
    bad = [-1, V, V + 256, -100, 2 ** 31 - 1, -(2 ** 31)]
    if index == torch.int64:  # the low words of these are ids of the table
        bad += [2 ** 40 + 3, -(2 ** 40) + 3, (1 << 32) + 7, -(2 ** 63)]
    for i, b in enumerate(bad):
        if i < T:
            ids[torch.arange(i, T, 17)] = b
    ids = ids.to(index)
    weight = normal(V, H, dtype=dtype)
    for ignore in (-100, 7, -1, V):
        out_of = (ids < 0) | (ids >= V) | (ids == ignore)
        dout = normal(T, H, dtype=dtype, seed=1)
        clean = dout.masked_fill(out_of[:, None], 0)
        dout[out_of] = float("nan")  # of tokens that have no gradient
        out, grad = both_ways(weight, ids, dout, 1.0, ignore)
        want, (value, bound) = embedding64(weight, ids, 1.0, ignore, clean)
        assert_rows("out", out, *want)
        assert_within("dweight", grad, value, bound)
        old = normal(V, H, dtype=dtype, seed=5)
        got = pair.embedding_backward_into(old.clone(), dout, (ids, V, H, dtype), 1.0, ignore)
        assert_added(got, old, ids, value, bound, ignore)


@pytest.mark.parametrize("T", COUNTS)
def test_no_token_has_a_row(T):
    V, H = 300, 64
    for ids in (torch.full((T,), -100, device="cuda"), torch.full((T,), V, device="cuda"),
                torch.full((T,), 2 ** 32, device="cuda")):
        dout = torch.full((T, H), float("inf"), dtype=F16, device="cuda")
        dirt = torch.full((V, H), float("nan"), dtype=F16, device="cuda")
        del dirt
        grad = pair.embedding_backward_from_saved(dout, (ids, V, H, F16))
        assert int(torch.count_nonzero(grad)) == 0
        old = normal(V, H, dtype=F16)
        assert torch.equal(pair.embedding_backward_into(old.clone(), dout, (ids, V, H, F16)), old)


@pytest.mark.parametrize("V,H", ((300000, 8), (60000, 1024), (40000, 1001)))
def test_no_tokens_of_a_large_table(V, H):
    """Past the single launch's limits: ids, bytes, and bytes of ragged rows."""
    dirt = torch.full((V, H), float("nan"), dtype=BF16, device="cuda")
    del dirt
    ids = torch.zeros(0, dtype=torch.int32, device="cuda")
    grad = pair.embedding_backward_from_saved(torch.zeros(0, H, dtype=BF16, device="cuda"),
                                              (ids, V, H, BF16))
    assert grad.shape == (V, H) and int(torch.count_nonzero(grad)) == 0


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("T", (240, 600, 9000))
def test_strided_or_unaligned_gradients(T, dtype):
    """Also of several dimensions, and through the autograd node on another stream."""
    V, H = 60, 72
    weight, ids = normal(V, H, dtype=dtype), tokens(T, V, "mixed").view(12, -1)
    dout = normal(12, T // 12, H, dtype=dtype, seed=2)
    want = both_ways(weight, ids.flatten(), dout.view(-1, H), 3.0)
    odd = normal(dout.numel() + 1, dtype=dtype)[1:].view(dout.shape)
    odd.copy_(dout)
    wide = torch.cat((dout, dout), -1)[..., :H]
    for d in (dout, odd, wide):
        assert torch.equal(both_ways(weight, ids, d, 3.0)[1], want[1])
    leaf = weight.clone().requires_grad_(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = bind(EMBEDDING, pair)(leaf, ids, scale=3.0)
        out.backward(odd)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(out.view(-1, H), want[0]) and torch.equal(leaf.grad, want[1])


def room_for(V, H, dtype, off):
    """Memory of NaN around a [V, H] table that begins ``off`` elements behind 16 bytes, and it."""
    room = torch.full((off + V * H + 64,), float("nan"), dtype=dtype, device="cuda")
    return room, room[off:off + V * H].view(V, H)


def assert_around(room, V, H, off):
    assert bool(room[:off].isnan().all()) and bool(room[off + V * H:].isnan().all())


@pytest.mark.parametrize("off", (0, 1, 4))
@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("V,H", ((50, 64), (300, 66), (2000, 7), (900, 1), (41, 1032), (400, 2)))
@pytest.mark.parametrize("T", (5, 200, 256, 257, 600, 9000))
def test_a_table_within_a_buffer(T, V, H, dtype, off):
    """As a view of a flat gradient buffer: added to, and written by the entry point."""
    print(f"\n[gpu-embedding] within a buffer {T} {V}x{H} {dtype} {off}", flush=True)
    ids, dout = tokens(T, V, "mixed"), normal(T, H, dtype=dtype, seed=1)
    _, (value, bound) = embedding64(normal(V, H, dtype=dtype), ids, 0.75, -100, dout)
    room, table = room_for(V, H, dtype, off)
    old = normal(V, H, dtype=dtype, seed=5)
    table.copy_(old)
    assert pair.embedding_backward_into(table, dout, (ids, V, H, dtype), 0.75) is table
    assert_added(table, old, ids, value, bound)
    assert_around(room, V, H, off)

    room, table = room_for(V, H, dtype, off)
    ws = workspace(_lib.query("eg_embedding_workspace_bytes", T, V, H), "cuda")
    _lib.call("eg_embedding_bwd", dout.data_ptr(), ids.data_ptr(), 0, table.data_ptr(), ws.data_ptr(),
              T, V, H, 0.75, -100, 0, _lib.dtype_tag(dtype), _lib.stream_of(dout))
    assert_within("written", table, value, bound)
    assert_around(room, V, H, off)
    plain = pair.embedding_backward_from_saved(dout, (ids, V, H, dtype), 0.75)
    assert_within("written at 16 bytes", plain, value, bound)


@pytest.mark.parametrize("off", (0, 1))
@pytest.mark.parametrize("V,H,dtype", ((300000, 8, F32), (33000, 1024, BF16), (60000, 640, BF16)))
def test_a_large_table_within_a_buffer(V, H, dtype, off):
    """Past the single launch's limits, without tokens and with few."""
    for T in (0, 3, 200):
        ids, dout = tokens(T, V, "low"), normal(T, H, dtype=dtype, seed=1)
        value = bound = torch.zeros(V, H, dtype=torch.float64, device="cuda")
        if T:
            weight = torch.zeros(V, H, dtype=dtype, device="cuda")
            _, (value, bound) = embedding64(weight, ids, 1.0, -100, dout)
        room, table = room_for(V, H, dtype, off)
        ws = workspace(_lib.query("eg_embedding_workspace_bytes", T, V, H), "cuda")
        _lib.call("eg_embedding_bwd", dout.data_ptr() or None, ids.data_ptr() or None, 0,
                  table.data_ptr(), ws.data_ptr(), T, V, H, 1.0, -100, 0, _lib.dtype_tag(dtype),
                  _lib.stream_of(room))
        assert_within("written", table, value, bound)
        assert_around(room, V, H, off)
