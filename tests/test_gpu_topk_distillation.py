"""Distillation from a teacher's top logits against 64 bits (tests/step_refs.py)."""

import pytest
import torch

from evograd_amd.bind import bind
from evograd_amd.decls import TOPK_DISTILLATION
from evograd_amd.pairs import cross_entropy
from evograd_amd.pairs import topk_distillation as pair
from tests.packed_refs import assert_within
from tests.step_refs import distill64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(rows, cols, K, dtype, seed=0, spread=2.0, ignore=0.2, cut=True, index=torch.int32,
         teacher_dtype=F32):
    """Student logits, targets (some ignored), teacher values at K distinct columns a row in no
    order, of which only some are kept with ``cut``, none in every fifth row."""
    g = torch.Generator().manual_seed(seed)
    logits = (spread * torch.randn(rows, cols, generator=g)).to(dtype)
    ids = torch.randint(0, cols - K + 1, (rows, K), generator=g).sort(1).values + torch.arange(K)
    ids = ids.gather(1, torch.rand(rows, K, generator=g).argsort(1))
    teacher = (8 + 2 * torch.randn(rows, K, generator=g)).to(teacher_dtype)
    if cut and K:
        kept = torch.randint(1, K + 1, (rows, 1), generator=g)
        kept[3::5] = 0
        # any places of the row, not its end alone
        ids[torch.rand(rows, K, generator=g).argsort(1) >= kept] = -1
    target = torch.randint(0, cols, (rows,), generator=g)
    target[torch.rand(rows, generator=g) < ignore] = -100
    target[rows - 1] = cols - 1
    return [t.cuda() for t in (logits, target, teacher, ids.to(index))]


def step(logits, target, teacher, ids, tau=1.0, soft=1.0, hard=0.0, ignore=-100, dloss=1.0):
    loss, saved = pair.topk_distillation_forward_with_saved(logits, target, teacher, ids, tau, soft,
                                                            hard, ignore)
    d = torch.full((), dloss, device="cuda")
    return loss, pair.topk_distillation_backward_from_saved(d, saved, tau, soft, hard, ignore)


def check(args, tau=1.0, soft=1.0, hard=0.0, ignore=-100, dloss=1.0):
    got = step(*args, tau, soft, hard, ignore, dloss)
    want = distill64(*args, tau, soft, hard, ignore, dloss)
    assert got[0].dtype == F32 and got[0].shape == () and got[1].dtype == args[0].dtype
    assert_within("loss", got[0], *want[0])
    assert_within("dlogits", got[1], *want[1])
    again = step(*args, tau, soft, hard, ignore, dloss)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    return got


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("tau,soft,hard", (
    (1.0, 1.0, 0.0), (2.0, 0.7, 0.3), (1.0, 0.5, 0.5), (0.5, 1.0, 0.0), (3.0, 0.0, 1.0)))
@pytest.mark.parametrize("rows,cols,K", (
    (1, 1, 1), (2, 3, 2), (5, 7, 7), (9, 64, 5), (33, 100, 100), (700, 40, 3), (17, 1000, 64),
    (3, 8192, 16), (6, 8200, 300), (12, 20001, 33), (2, 70000, 1000)))
def test_against_64_bits(rows, cols, K, tau, soft, hard, dtype):
    print(f"\n[gpu-distill] {rows}x{cols} K={K} tau={tau} {soft}/{hard} {dtype}", flush=True)
    check(make(rows, cols, K, dtype, seed=rows), tau, soft, hard, dloss=1024.0)


def test_rows_in_many_and_in_one_part():
    """The same rows alone (their columns dealt to several workgroups) and among many."""
    logits, target, teacher, ids = make(600, 17000, 20, F32, ignore=0.0)
    for r in (slice(0, 1), slice(4, 9), slice(0, 600)):
        check([t[r].contiguous() for t in (logits, target, teacher, ids)], 2.0, 0.5, 0.5, dloss=100.0)


@pytest.mark.parametrize("index", (torch.int32, torch.int64))
@pytest.mark.parametrize("teacher_dtype", (BF16, F16, F32))
def test_types_of_the_teacher(index, teacher_dtype):
    check(make(20, 500, 16, BF16, index=index, teacher_dtype=teacher_dtype), 1.5, 1.0, 0.25)


def test_entries_of_one_token_add_up():
    logits, target, teacher, ids = make(40, 300, 24, F32, cut=False, ignore=0.0)
    ids[:, 5:9] = ids[:, 1:2]  # five entries of one column, in places apart
    ids[:, 20] = ids[:, 19]
    ids[7] = 299  # all of them
    check((logits, target, teacher, ids), 2.0, 1.0, 0.5, dloss=100.0)
    teacher[:, 1] = -1e4  # the first of the five has no weight
    check((logits, target, teacher, ids), 2.0, 1.0, 0.5, dloss=100.0)


def test_no_entries_at_all():
    logits, target, teacher, ids = make(12, 333, 4, BF16)
    none = torch.full_like(ids, -1)
    loss, grad = check((logits, target, teacher, none))
    assert float(loss) == 0.0 and int(torch.count_nonzero(grad)) == 0
    empty = teacher[:, :0], ids[:, :0]
    loss, grad = step(logits, target, *empty, 2.0, 1.0, 0.5)
    want = step(logits, target, teacher, none, 2.0, 1.0, 0.5)
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
    # -inf leaves an entry out as a negative id does
    gone = step(logits, target, torch.full_like(teacher, -float("inf")), ids.clamp(min=0), 2.0, 1.0, 0.5)
    assert torch.equal(loss, gone[0]) and torch.equal(grad, gone[1])


def test_hard_labels_alone_are_cross_entropy():
    logits, target, teacher, ids = make(50, 4099, 8, F32)
    loss, grad = step(logits, target, teacher, ids, 2.0, 0.0, 1.0)
    other, saved = cross_entropy.cross_entropy_forward_with_saved(logits, target)
    dother = cross_entropy.cross_entropy_backward_from_saved(torch.ones((), device="cuda"), saved)
    want = distill64(logits, target, teacher, ids, 2.0, 0.0, 1.0, -100, 1.0)
    assert abs(float(loss) - float(other)) <= 2 * float(want[0][1])
    # the other takes its exponents from the rounded logsumexp, of about 12
    assert bool(((grad - dother).abs().double() <= 2 * want[1][1] + 2.0 ** -24 * 20 * dother.abs()).all())


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("cols", (96, 20000))
def test_masked_logits_and_far_values(cols, dtype):
    logits, target, teacher, ids = make(10, cols, 6, dtype, ignore=0.0, cut=False)
    seen = torch.zeros(10, cols, dtype=torch.bool, device="cuda").scatter_(1, ids.long(), True)
    seen.scatter_(1, target[:, None], True)
    mask = ~seen & (torch.arange(cols, device="cuda") % 3 == 0)
    masked = logits.masked_fill(mask, -float("inf"))
    lowest = logits.masked_fill(mask, torch.finfo(dtype).min)
    for soft, hard in ((1.0, 0.0), (0.5, 0.5)):
        got = step(masked, target, teacher, ids, 2.0, soft, hard)
        low = step(lowest, target, teacher, ids, 2.0, soft, hard)
        assert torch.equal(got[0], low[0]) and torch.equal(got[1], low[1])
        assert bool(got[0].isfinite()) and bool(got[1].isfinite().all())
        assert int(torch.count_nonzero(got[1][mask])) == 0
        # the rows without their masked columns
        keep = masked.double().masked_fill(mask, -1e4)
        want = distill64(keep, target, teacher, ids, 2.0, soft, hard, -100, 1.0)[1][0]
        assert float((got[1].double() - want).norm() / want.norm()) <= torch.finfo(dtype).eps
    # shifted far off: in fp32 differences to the row's maximum stay exact
    far = (logits.float() * 4).round() + 1e6
    near = (logits.float() * 4).round()
    a, b = (step(x, target, teacher, ids, 2.0, 0.5, 0.5) for x in (far, near))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # a teacher's token that the student's mask forbids
    logits[2, int(ids[2, 0])] = -float("inf")
    assert float(step(logits, target, teacher, ids)[0]) == float("inf")


def test_ignored_rows_are_not_read():
    logits, target, teacher, ids = make(30, 900, 9, BF16, ignore=0.5)
    gone = target == -100
    want = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)
    logits[gone], teacher[gone] = float("nan"), float("inf")
    ids[gone] = 900
    got = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert int(torch.count_nonzero(got[1][gone])) == 0
    target.fill_(-100)
    loss, grad = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)
    assert bool(loss.isnan()) and int(torch.count_nonzero(grad)) == 0
    target.fill_(7)
    loss, grad = step(logits, target, teacher, ids, 2.0, 0.5, 0.5, ignore=7)
    assert bool(loss.isnan()) and int(torch.count_nonzero(grad)) == 0


@pytest.mark.parametrize("cols", (60, 30000))
def test_tokens_outside_the_vocabulary(cols):
    logits, target, teacher, ids = make(8, cols, 5, F32, ignore=0.0, cut=False)
    clean = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)[1]
    for bad in (cols, 2 ** 31 - 1):
        wrong = ids.clone()
        wrong[3, 2] = bad
        loss, grad = step(logits, target, teacher, wrong, 2.0, 0.5, 0.5)
        assert bool(loss.isnan()) and bool(grad[3].isnan().all())
        grad[3] = clean[3]
        assert torch.equal(grad, clean)
    for bad in (cols, -1, 2 ** 40):
        wrong = target.clone()
        wrong[5] = bad
        loss, grad = step(logits, wrong, teacher, ids, 2.0, 0.5, 0.5)
        assert bool(loss.isnan()) and bool(grad[5].isnan().all())
        grad[5] = clean[5]
        assert torch.equal(grad, clean)
        # without a hard label a target only says whether its row counts
        assert bool(step(logits, wrong, teacher, ids)[0].isfinite())


def test_a_non_finite_row_stays_in_its_row():
    for what in (float("nan"), float("inf")):
        logits, target, teacher, ids = make(30, 700, 9, BF16, ignore=0.0, cut=False)
        clean = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)[1]
        logits[4, 33] = what
        teacher[9, 2] = what
        loss, grad = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)
        assert not bool(loss.isfinite()) and not bool(grad[4].isfinite().all())
        assert bool(grad[9].isnan().all())
        grad[4], grad[9] = clean[4], clean[9]
        assert torch.equal(grad, clean)


def test_parts_with_no_weight_are_not_looked_at():
    logits, target, teacher, ids = make(10, 300, 5, BF16, ignore=0.0)
    want = step(logits, target, teacher, ids, 2.0, 0.0, 1.0)
    got = step(logits, target, torch.full_like(teacher, float("nan")), torch.full_like(ids, 300), 2.0,
               0.0, 1.0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool(want[0].isfinite())
    nothing = step(logits, target, teacher, ids, 2.0, 0.0, 0.0)
    assert float(nothing[0]) == 0.0 and int(torch.count_nonzero(nothing[1])) == 0


def test_no_rows():
    logits, target, teacher, ids = (t[:0] for t in make(3, 50, 4, BF16))
    loss, grad = step(logits, target, teacher, ids)
    assert bool(loss.isnan()) and grad.shape == (0, 50)


def test_strided_and_unaligned_inputs():
    logits, target, teacher, ids = make(20, 128, 6, BF16)
    want = step(logits, target, teacher, ids, 2.0, 0.5, 0.5)
    wide = torch.cat((logits, logits), 1)[:, :128]
    got = step(wide, torch.stack((target, target), 1)[:, 0], teacher.t().contiguous().t(),
               ids.t().contiguous().t(), 2.0, 0.5, 0.5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    room = torch.empty(logits.numel() + 1, dtype=BF16, device="cuda")
    odd = room[1:].view(logits.shape)
    odd.copy_(logits)
    check((odd, target, teacher, ids), 2.0, 0.5, 0.5)


def test_gradient_against_differences():
    logits, target, teacher, ids = make(6, 50, 8, F32, ignore=0.0)
    _, grad = step(logits, target, teacher, ids, 1.5, 0.6, 0.4)
    way = torch.randn(6, 50, generator=torch.Generator().manual_seed(9)).cuda().double()
    e = 1e-4

    def f(s):
        return float(distill64(logits.double() + s * e * way, target, teacher, ids, 1.5, 0.6, 0.4,
                               -100, 1.0)[0][0])

    # e^2 times third derivatives of a mean of order 1; the gradient's fp32 roundings
    assert abs(float((grad.double() * way).sum()) - (f(1) - f(-1)) / (2 * e)) < 20 * e * e + 1e-5


def test_autograd_node_and_another_stream():
    logits, target, teacher, ids = make(20, 1000, 6, BF16)
    want = step(logits, target, teacher, ids, 2.0, 0.5, 0.5, dloss=3.0)
    leaf = logits.clone().requires_grad_(True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        loss = bind(TOPK_DISTILLATION, pair)(leaf, target, teacher, ids, temperature=2.0,
                                             soft_weight=0.5, hard_weight=0.5)
        (3.0 * loss).backward()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(loss, want[0]) and torch.equal(leaf.grad, want[1])


@pytest.mark.parametrize("rows,cols", ((24, 513), (4, 40000)))
def test_a_captured_graph_replays_with_other_batches(rows, cols):
    args = make(rows, cols, 7, BF16)
    step(*args, 2.0, 0.5, 0.5)
    torch.cuda.synchronize()
    d = torch.ones((), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, saved = pair.topk_distillation_forward_with_saved(*args, 2.0, 0.5, 0.5)
        grad = pair.topk_distillation_backward_from_saved(d, saved, 2.0, 0.5, 0.5)
    for seed in range(4):
        for old, new in zip(args, make(rows, cols, 7, BF16, seed=50 + seed)):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = loss.clone(), grad.clone()
        for x, y in zip(got, step(*args, 2.0, 0.5, 0.5)):
            assert torch.equal(x, y)


def test_logits_past_32_bit_offsets():
    rows, cols = 36000, 60008  # 2.16e9 elements
    logits = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    target = torch.full((rows,), -100, device="cuda")
    logits[rows - 1, 5::7], logits[rows - 2, cols - 1] = 2.0, 3.0
    target[rows - 2:] = torch.tensor([cols - 1, 5])
    ids = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
    ids[rows - 2:] = torch.tensor([[3, cols - 1], [12, 0]], dtype=torch.int32)
    teacher = torch.ones(rows, 2, device="cuda")
    loss, grad = step(logits, target, teacher, ids, 2.0, 0.5, 0.5, dloss=1e4)
    tail = [t[rows - 2:].contiguous() for t in (logits, target, teacher, ids)]
    want = distill64(*tail, 2.0, 0.5, 0.5, -100, 1e4)
    assert_within("loss", loss, *want[0])
    assert_within("dlogits", grad[rows - 2:], *want[1])
    assert not bool(grad[:rows - 2].any())


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("tau,soft,hard", ((1.5, 0.7, 0.3), (4.0, 1.0, 0.5), (0.5, 0.25, 1.0)))
@pytest.mark.parametrize("rows,cols,K", (
    (1, 1, 1), (2, 3, 2), (9, 64, 5), (33, 100, 100), (700, 40, 3), (17, 1000, 64), (3, 8192, 16),
    (6, 8200, 300), (12, 20001, 33), (2, 70000, 1000), (1100, 8192, 9), (300, 4097, 40)))
def test_two_exponentials_a_logit(rows, cols, K, tau, soft, hard, dtype):
    """Temperatures other than 1 and 2 with hard labels: whole and ragged rows, in one part and in
    several, of less than a workgroup and more."""
    print(f"\n[gpu-distill] two {rows}x{cols} K={K} tau={tau} {soft}/{hard} {dtype}", flush=True)
    check(make(rows, cols, K, dtype, seed=rows), tau, soft, hard, dloss=1024.0)


@pytest.mark.parametrize("tau", (2.0 ** -100, 1e-6, 1e6, 2.0 ** 60))
def test_the_ends_of_the_temperatures(tau):
    """Nothing overflows on the way to the loss or its gradient."""
    logits, target, teacher, ids = make(9, 200, 9, F32, ignore=0.0, cut=False)
    loss, grad = step(logits, target, teacher, ids, tau, 1.0, 0.5)
    assert bool(loss.isfinite()) and bool(grad.isfinite().all())
