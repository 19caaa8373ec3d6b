"""Packed attention where its arithmetic has an edge: scores of -inf, values that no row sees,
rows of few keys, upstream gradients past fp16's range, rows that share their memory. Against
the definition in 64 bits (tests/packed_edge_refs.py)."""

import pytest
import torch

from evograd_amd.pairs import packed_attention as pair
from tests.packed_edge_refs import attention64
from tests.packed_refs import assert_within

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FAR = 1.0e4  # a finite stand-in for inf: its scores weigh exp(-FAR / sqrt(D)), which is zero


def bounds(lengths):
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths, dtype=torch.int32).cumsum(0)
    return cu.cuda()


def make(lengths, H, KVH, D, dtype, seed=0, scale=1.0):
    print(f"\n[gpu-packed-edges] {lengths[:6]}x{len(lengths)} {H}/{KVH} D={D} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lengths)
    shapes = ((T, H, D), (T, KVH, D), (T, KVH, D), (T, H, D))
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(dtype) for s in shapes]


def run(q, k, v, do, cu):
    o, saved = pair.packed_attention_forward_with_saved(q, k, v, cu)
    dq, dk, dv = pair.packed_attention_backward_from_saved(do, saved)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv, "lse": saved[4]}


KINDS = ((128, BF16), (64, BF16), (64, F16), (64, F32), (96, BF16))


# ------------------------------------------------------------- rows of few keys
@pytest.mark.parametrize("scale", (1.0, 2.0))
@pytest.mark.parametrize("lengths", ([2], [4] * 9, [1, 3, 16, 7, 12], [26] * 3, [64, 63, 33]))
@pytest.mark.parametrize("H,KVH,D,dtype", (
    (8, 2, 128, BF16), (3, 1, 64, BF16), (4, 4, 128, F16), (4, 2, 64, F16), (2, 1, 64, F32),
    (4, 2, 96, BF16), (2, 1, 80, F16), (4, 2, 32, F16)))
def test_rows_of_few_keys_have_delta_in_32_bits(H, KVH, D, dtype, lengths, scale):
    """Where a row's keys fit one tile, delta = sum p dp takes no rounding of o in, which for peaked
    rows would be most of the error of dq and dk."""
    q, k, v, do = make(lengths, H, KVH, D, dtype, seed=3, scale=scale)
    want, _ = attention64(q, k, v, do, lengths)
    got = run(q, k, v, do, bounds(lengths))
    for name in got:
        assert_within(name, got[name], *want[name])


@pytest.mark.parametrize("H,KVH,D,dtype", ((8, 2, 128, BF16), (4, 4, 64, F16), (2, 1, 64, BF16)))
@pytest.mark.parametrize("lengths", ([700, 300], [66, 90, 70] * 4))
def test_the_first_rows_of_longer_sequences(lengths, H, KVH, D, dtype):
    q, k, v, do = make(lengths, H, KVH, D, dtype, seed=4, scale=2.0)
    want, _ = attention64(q, k, v, do, lengths)
    got = run(q, k, v, do, bounds(lengths))
    first = torch.cat([torch.arange(64) + sum(lengths[:i]) for i in range(len(lengths))]).cuda()
    assert_within("dq", got["dq"][first], *(x[first] for x in want["dq"]))


@pytest.mark.parametrize("D,dtype", KINDS)
def test_a_row_of_one_key_has_no_gradient_through_its_weight(D, dtype):
    """p is one whatever the score, so dS is zero: exactly, not to rounding."""
    lengths = [1] * 20
    q, k, v, do = make(lengths, 4, 2, D, dtype, seed=5, scale=3.0)
    got = run(q, k, v, do, bounds(lengths))
    for name in ("dq", "dk"):
        assert int(torch.count_nonzero(got[name])) == 0, name


# ------------------------------------------------------------------ scores of -inf
@pytest.mark.parametrize("D,dtype", KINDS)
@pytest.mark.parametrize("lengths,H,KVH", (([200], 2, 1), ([200], 4, 1), ([150, 1, 1, 1, 9], 4, 2)))
@pytest.mark.parametrize("first,last", ((64, 65), (0, 64)))
@pytest.mark.parametrize("spoilt", (None, 70))
def test_a_first_tile_of_hidden_and_infinitely_low_scores(spoilt, first, last, lengths, H, KVH, D,
                                                          dtype):
    """Keys first .. last - 1 score -inf against every row, and a row whose keys so far all do has
    no maximum yet: its later (or other group's) keys alone decide it, whether or not another row
    of its workgroup is NaN."""
    q, k, v, do = make(lengths, H, KVH, D, dtype, seed=1)
    q[..., 5] = -1.0
    k[first:last, :, 5] = FAR
    want, _ = attention64(q, k, v, do, lengths)
    k[first:last, :, 5] = float("inf")
    n = lengths[0]
    rows = torch.arange(last if first == 0 else 0, n, device="cuda")
    if spoilt is not None:
        q[spoilt, :, 5] = 1.0  # its scores against those keys are +inf: the row is NaN
        rows = rows[rows != spoilt]
    got = run(q, k, v, do, bounds(lengths))
    assert_within("o", got["o"][rows], *(x[rows] for x in want["o"]))
    assert_within("lse", got["lse"][:, rows], *(x[:, rows] for x in want["lse"]))
    if first > 0:  # dq's column 5 is 0 times inf
        keep = [i for i in range(D) if i != 5]
        assert_within("dq", got["dq"][rows][..., keep], *(x[rows][..., keep] for x in want["dq"]))
    else:  # the first rows see nothing else
        assert bool(torch.isnan(got["o"][:last]).all())


# ------------------------------------------------- rows past the end see no key
@pytest.mark.parametrize("D,dtype", KINDS)
@pytest.mark.parametrize("n", (64, 65, 95, 130, 450))
@pytest.mark.parametrize("H,KVH", ((2, 2), (8, 2)))
def test_an_infinite_key_that_weighs_nothing_has_the_gradients_of_one(H, KVH, n, D, dtype):
    """The last key of a sequence scores -inf against its only row. What a tile holds past the
    sequence's end takes no part in its gradients, whether or not the tile is full."""
    lengths = [n, 40]
    q, k, v, do = make(lengths, H, KVH, D, dtype, seed=n)
    q[n - 1, :, 5] = -1.0
    k[n - 1, :, 5] = FAR
    want, _ = attention64(q, k, v, do, lengths)
    k[n - 1, :, 5] = float("inf")
    got = run(q, k, v, do, bounds(lengths))
    for name in ("o", "dk", "dv"):
        assert_within(name, got[name], *want[name])
    keep = [i for i in range(D) if i != 5]  # of that row, dq's column 5 is 0 times inf
    assert_within("dq", got["dq"][..., keep], *(x[..., keep] for x in want["dq"]))


# -------------------------------------------------------------- fp16's range of dS
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("lengths,H,KVH", (([2, 3, 5, 9, 1], 2, 2), ([40, 64, 17], 4, 4),
                                           ([300, 5], 2, 2), ([2] * 300, 2, 1)))
@pytest.mark.parametrize("spoilt", (None, 1))
def test_gradients_whose_products_pass_the_half_range(spoilt, lengths, H, KVH, D):
    """Upstream gradients of a scaled loss: dS passes 65504 where dq and dk are well inside it."""
    q, k, v, do = make(lengths, H, KVH, D, F16, seed=6)
    q, k = (0.25 * q.float()).half(), (0.25 * k.float()).half()
    v = (3.0 * v.float()).half()
    do = (1.2e4 * torch.sign(do.float())).half()
    want, largest = attention64(q, k, v, do, lengths, half_range=True)
    assert largest > 65504 and all(float(x.abs().max()) < 60000 for x, _ in want.values())
    keep = torch.ones(sum(lengths), dtype=torch.bool, device="cuda")
    if spoilt is not None:  # a NaN row of the first sequence: the others are what they were
        q[spoilt] = float("nan")
        keep[:lengths[0]] = False
    got = run(q, k, v, do, bounds(lengths))
    for name in ("o", "dq", "dk", "dv"):
        assert_within(name, got[name][keep], *(x[keep] for x in want[name]))


@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("lengths,row", (([50, 30], 20), ([200], 100)))
def test_a_row_past_the_half_range_leaves_its_neighbours_theirs(lengths, row, D):
    """Upstream gradients of one row far above the others', whose dS are small normal numbers."""
    q, k, v, do = make(lengths, 2, 2, D, F16, seed=7)
    v = (8.0 * v.float()).half()
    do = (1e-5 * do.float()).half()
    want, _ = attention64(q, k, v, do, lengths)
    others = torch.arange(sum(lengths), device="cuda") != row
    later = torch.arange(sum(lengths), device="cuda") > row  # keys that the row does not see
    do[row] = 6e4
    got = run(q, k, v, do, bounds(lengths))
    assert_within("dq", got["dq"][others], *(x[others] for x in want["dq"]))
    for name in ("dk", "dv"):
        assert_within(name, got[name][later], *(x[later] for x in want[name]))
