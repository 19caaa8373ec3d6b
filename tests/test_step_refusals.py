"""What the pairs of a distillation step and their C entry points refuse, before any launch (CPU)."""

import ctypes
import os

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.pairs import embedding, norm_rotary, topk_distillation

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
P = 1 << 20  # an address no refused call reads


@pytest.fixture
def no_device_check(monkeypatch):
    """The pairs' own checks on CPU tensors (the device check comes first)."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *a: None)


@pytest.fixture
def no_kernels(monkeypatch):
    """The pairs on CPU tensors with every launch left out (results are not looked at)."""
    for name in ("require_gpu", "call_on"):
        monkeypatch.setattr(_lib, name, lambda *a: None)
    monkeypatch.setattr(_lib, "stream_of", lambda t: 0)
    monkeypatch.setattr(_lib, "query", lambda *a: 16)


W, IDS = torch.zeros(6, 8), torch.zeros(4, dtype=torch.int32)
POS, FREQ = torch.arange(4, dtype=torch.int32), torch.ones(4, dtype=torch.float64)
Z, TARGET, T, TI = (torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64), torch.zeros(4, 3),
                    torch.zeros(4, 3, dtype=torch.int32))


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding.embedding_forward_with_saved(W, IDS)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding.embedding_backward_into(W, torch.zeros(4, 8), (IDS, 6, 8, torch.float32))
    with pytest.raises(RuntimeError, match="GPU"):
        norm_rotary.norm_rotary_forward_with_saved(x, torch.ones(8), POS, FREQ)
    with pytest.raises(RuntimeError, match="GPU"):
        topk_distillation.topk_distillation_forward_with_saved(Z, TARGET, T, TI)


def test_embedding_arguments(no_device_check):
    call = embedding.embedding_forward_with_saved
    with pytest.raises(ValueError, match=r"\[vocab, hidden\]"):
        call(W[0], IDS)
    with pytest.raises(TypeError, match="int32 or int64"):
        call(W, IDS.float())
    with pytest.raises(TypeError, match="int32 or int64"):
        call(W, IDS.to(torch.int16))
    with pytest.raises(TypeError, match="unsupported dtype"):
        call(W.double(), IDS)
    back, into = embedding.embedding_backward_from_saved, embedding.embedding_backward_into
    saved = (IDS, 6, 8, torch.float32)
    for bad in (torch.zeros(8), torch.zeros(3, 8), torch.zeros(4, 7), torch.zeros(2, 2, 8),
                torch.zeros(4, 8).half(), torch.zeros(4, 8).double()):
        with pytest.raises(ValueError, match="dout must be"):
            back(bad, saved)
    for bad in (torch.zeros(5, 8), torch.zeros(6, 7), torch.zeros(6, 8).half()):
        with pytest.raises(ValueError, match="dweight must be"):
            into(bad, torch.zeros(4, 8), saved)
    with pytest.raises(ValueError, match="contiguous"):
        into(torch.zeros(8, 6).t(), torch.zeros(4, 8), saved)


@pytest.mark.parametrize("x,w,pos,freqs,error,words", (
    (torch.zeros(4, 8), torch.ones(8), POS, FREQ, ValueError, "tokens, heads, head_dim"),
    (torch.zeros(4, 2, 8), torch.ones(7), POS, FREQ, ValueError, "weight must be"),
    (torch.zeros(4, 2, 8), torch.ones(1, 8), POS, FREQ, ValueError, "weight must be"),
    (torch.zeros(4, 2, 8), torch.ones(8).half(), POS, FREQ, TypeError, "mismatch"),
    (torch.zeros(4, 2, 8), torch.ones(8), POS[:3], FREQ, ValueError, "positions must be"),
    (torch.zeros(4, 2, 8), torch.ones(8), POS.float(), FREQ, TypeError, "int32 or int64"),
    (torch.zeros(4, 2, 8), torch.ones(8), POS, FREQ.float(), TypeError, "float64"),
    (torch.zeros(4, 2, 6), torch.ones(6), POS, FREQ, ValueError, "at most head_dim"),
    (torch.zeros(4, 2, 8).double(), torch.ones(8).double(), POS, FREQ, TypeError, "unsupported dtype"),
))
def test_norm_rotary_arguments(no_device_check, x, w, pos, freqs, error, words):
    with pytest.raises(error, match=words):
        norm_rotary.norm_rotary_forward_with_saved(x, w, pos, freqs)


def test_norm_rotary_q_and_k_must_agree(no_device_check):
    x, w = torch.zeros(4, 2, 8), torch.ones(8)
    call, back = norm_rotary.norm_rotary_qk_forward_with_saved, norm_rotary.norm_rotary_qk_backward_from_saved
    with pytest.raises(ValueError, match="share head_dim"):
        call(x, torch.zeros(4, 2, 10), w, torch.ones(10), POS, FREQ)
    with pytest.raises(ValueError, match="share head_dim"):
        call(x, x.half(), w, w.half(), POS, FREQ)
    with pytest.raises(ValueError, match="positions must be"):
        call(x, torch.zeros(5, 2, 8), w, w, POS, FREQ)
    saved = (x, x, w, w, POS, FREQ)
    for bad in ((x, x[:, :1]), (x[:3], x), (x, x.half())):
        with pytest.raises(ValueError, match="upstream gradients"):
            back(bad, saved)
    with pytest.raises(ValueError, match="upstream gradients"):
        norm_rotary.norm_rotary_backward_from_saved(x[:, :1], (x, w, POS, FREQ))


@pytest.mark.parametrize("z,target,t,ids,error,words", (
    (Z[0], TARGET, T, TI, ValueError, r"\[rows, cols\]"),
    (Z, TARGET[:3], T, TI, ValueError, "target must be"),
    (Z, TARGET[:, None], T, TI, ValueError, "target must be"),
    (Z, TARGET.int(), T, TI, TypeError, "int64"),
    (Z, TARGET, T, TI[:3], ValueError, "teacher_ids must be"),
    (Z, TARGET, T, TI[:, 0], ValueError, "teacher_ids must be"),
    (Z, TARGET, T, TI.float(), TypeError, "int32 or int64"),
    (Z, TARGET, T[:, :2], TI, ValueError, "same shape"),
    (Z.double(), TARGET, T, TI, TypeError, "unsupported dtype"),
    (Z, TARGET, T.double(), TI, TypeError, "unsupported dtype"),
))
def test_distillation_arguments(no_device_check, z, target, t, ids, error, words):
    with pytest.raises(error, match=words):
        topk_distillation.topk_distillation_forward_with_saved(z, target, t, ids)


def test_distillation_gradient_arguments(no_device_check):
    back = topk_distillation.topk_distillation_backward_from_saved
    saved = (Z, TARGET, TI, torch.zeros(4 * 7 + 1))
    with pytest.raises(ValueError, match="saved state"):
        back(torch.ones(()), (Z, TARGET, TI, torch.zeros(4 * 7)))
    for bad in (torch.ones(2), torch.ones((), dtype=torch.float64), torch.ones(()).half()):
        with pytest.raises(ValueError, match="one float32"):
            back(bad, saved)


@built
def test_entry_points_check_their_arguments():
    def embed(tokens=4, vocab=6, hidden=8, weight=P, dtype=_lib.EG_F32):
        _lib.call("eg_embedding_fwd", weight, P, 0, P, tokens, vocab, hidden, 1.0, -100, dtype, None)

    for words, kw in (("negative", dict(tokens=-1)), ("negative", dict(vocab=-1)),
                      ("out of range", dict(tokens=1 << 31)), ("out of range", dict(vocab=1 << 31)),
                      ("out of range", dict(hidden=1 << 21)), ("null pointer", dict(weight=None)),
                      ("dtype", dict(dtype=9)), ("grid too large", dict(tokens=1 << 30, hidden=4096))):
        with pytest.raises(RuntimeError, match=words):
            embed(**kw)
    embed(tokens=0, weight=None)  # nothing to do is no error

    def scatter(tokens=4, vocab=6, hidden=8, dweight=P, ws=P, dtype=_lib.EG_F32):
        _lib.call("eg_embedding_bwd", P, P, 0, dweight, ws, tokens, vocab, hidden, 1.0, -100, 0, dtype,
                  None)

    for words, kw in (("negative", dict(tokens=-1)), ("out of range", dict(hidden=1 << 21)),
                      ("null pointer", dict(dweight=None)), ("null pointer", dict(ws=None)),
                      ("16-byte aligned", dict(ws=P + 4)), ("dtype", dict(dtype=9)),
                      ("grid too large", dict(vocab=1 << 30, hidden=1 << 20))):
        with pytest.raises(RuntimeError, match=words):
            scatter(**kw)
    scatter(vocab=0, dweight=None)

    steps = (ctypes.c_int64 * 8)(16, 8, 16, 8, 16, 8, 16, 8)

    def turn(tokens=4, hq=2, hk=2, dim=8, pairs=4, strides=steps, dtype=_lib.EG_F32, q=P):
        _lib.call("eg_norm_rotary_fwd", q, P, P, P, P, P, P, 0, P, tokens, hq, hk, dim, pairs, strides,
                  1e-6, 1.0, 0, dtype, None)

    def back(tokens=4, hq=2, hk=2, dim=8, pairs=4, strides=steps, dtype=_lib.EG_F32, q=P):
        _lib.call("eg_norm_rotary_bwd", P, P, q, P, P, P, P, 0, P, P, P, P, P, P, tokens, hq, hk, dim,
                  pairs, strides, 1e-6, 1.0, 0, dtype, None)

    for fn in (turn, back):
        for words, kw in (("negative", dict(tokens=-1)), ("do not fit", dict(pairs=5)),
                          ("do not fit", dict(pairs=-1)), ("out of range", dict(hq=1 << 17)),
                          ("out of range", dict(dim=1 << 14, pairs=1)),
                          ("null strides", dict(strides=None)), ("null pointer", dict(q=None)),
                          ("strides must", dict(strides=(ctypes.c_int64 * 8)(-1, *[8] * 7))),
                          ("strides must", dict(strides=(ctypes.c_int64 * 8)(8, 8, 1 << 33, *[8] * 5))),
                          ("dtype", dict(dtype=9))):
            with pytest.raises(RuntimeError, match=words):
                fn(**kw)
    with pytest.raises(RuntimeError, match="strides must"):
        back(strides=(ctypes.c_int64 * 8)(*[8] * 7, 1 << 41))
    for fn in (turn, back):  # the walk's grid does not grow with the tokens
        with pytest.raises(RuntimeError, match="out of range"):
            fn(tokens=(1 << 32) + 1, hq=1, hk=1)
    turn(tokens=0, q=None)

    def distill(rows=4, cols=9, k=3, tau=1.0, z=P, dtype=_lib.EG_F32, teacher=_lib.EG_F32):
        _lib.call("eg_topk_distill_fwd", z, P, P, teacher, P, 0, P, P, P, P, P, rows, cols, k, tau, 1.0,
                  0.0, -100, dtype, None)

    def distill_back(rows=4, cols=9, k=3, tau=1.0, z=P, dtype=_lib.EG_F32):
        _lib.call("eg_topk_distill_bwd", P, z, P, P, 0, P, P, P, P, rows, cols, k, tau, 1.0, 0.0, -100,
                  dtype, None)

    for fn in (distill, distill_back):
        for words, kw in (("negative", dict(rows=-1)), ("negative", dict(k=-1)),
                          ("zero classes", dict(cols=0)), ("out of range", dict(rows=1 << 23)),
                          ("out of range", dict(k=1025)), ("temperature", dict(tau=0.0)),
                          ("temperature", dict(tau=-1.0)), ("temperature", dict(tau=float("nan"))),
                          ("temperature", dict(tau=float("inf"))), ("null pointer", dict(z=None)),
                          ("grid too large", dict(rows=1 << 22, cols=1 << 30)),
                          ("dtype", dict(dtype=9))):
            with pytest.raises(RuntimeError, match=words):
                fn(**kw)
    with pytest.raises(RuntimeError, match="dtype"):
        distill(teacher=9)
    distill_back(rows=0, z=None)


@built
def test_workspaces():
    al = lambda n: (n + 255) // 256 * 256  # noqa: E731
    q = _lib.query
    assert q("eg_embedding_workspace_bytes", 100, 0, 8) == 0
    # one piece of 8 tokens: the order, its ids and 256 buckets of 4 ids' bounds
    assert q("eg_embedding_workspace_bytes", 8, 1000, 8) == 2 * al(8 * 4) + al((256 * 4 + 1) * 4)
    assert (q("eg_embedding_workspace_bytes", 9, 1000, 8)
            == 2 * al(9 * 4) + al((256 * 4 + 1) * 4) + 2 * 2 * 8 * 4)
    assert (q("eg_embedding_workspace_bytes", 16384, 128256, 4096)
            == 2 * 16384 * 4 + al((256 * 501 + 1) * 4) + 512 * 2 * 4096 * 4)
    assert q("eg_norm_rotary_workspace_bytes", 0, 8, 2, 64) == 0
    assert q("eg_norm_rotary_workspace_bytes", 5, 8, 2, 64) == 2048 * 2 * 64 * 4
    assert q("eg_topk_distill_workspace_bytes", 0, 100, 3) == 0
    assert q("eg_topk_distill_workspace_bytes", 8192, 128256, 64) == 8192 * (4 + 64) * 4
    assert q("eg_topk_distill_workspace_bytes", 4, 128256, 0) == 4 * (1 + 3 * 31) * 4
    assert q("eg_topk_distill_workspace_bytes", 300, 128256, 9) == 300 * (1 + 3 * 3 + 9) * 4


def test_gradients_of_gradients_are_refused(no_kernels):
    q, k = (torch.zeros(s, requires_grad=True) for s in ((4, 2, 8), (4, 1, 8)))
    qw, kw = (torch.ones(8, requires_grad=True) for _ in range(2))
    a, b = norm_rotary.NormRotaryQK.apply(q, k, qw, kw, POS, FREQ)
    grads = torch.autograd.grad((a * a).sum() + (b * b).sum(), (q, k, qw, kw), create_graph=True)
    for g, other in zip(grads, (q, k, qw, kw)):
        with pytest.raises(RuntimeError, match="differentiate twice"):
            (g.sum() + other.sum()).backward(retain_graph=True)


def test_the_embedding_keeps_no_table(no_kernels):
    _, saved = embedding.embedding_forward_with_saved(W, IDS)
    assert saved[0] is IDS and saved[1:] == (6, 8, torch.float32)


def test_a_gradient_added_in_place_is_a_change_that_autograd_sees(no_kernels):
    """A node that saved the tensor before notices, and so does one that saved a view of it."""
    dout, saved = torch.zeros(4, 8), (IDS, 6, 8, torch.float32)
    flat = torch.zeros(48)
    for held, target in ((flat, flat.view(6, 8)), (flat.view(6, 8), flat.view(6, 8))):
        version = held._version
        y = torch.zeros(held.shape, requires_grad=True) * held
        assert embedding.embedding_backward_into(target, dout, saved) is target
        assert held._version == version + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    version = dout._version
    embedding.embedding_backward_from_saved(dout, saved)
    assert dout._version == version


def test_a_gradient_is_not_added_to_what_requires_gradients(no_kernels):
    leaf, dout, saved = torch.zeros(6, 8, requires_grad=True), torch.zeros(4, 8), (IDS, 6, 8, torch.float32)
    into = embedding.embedding_backward_into
    for bad in (leaf, leaf * 1.0):
        with pytest.raises(RuntimeError, match="requires gradients"):
            into(bad, dout, saved)
    with torch.no_grad():
        assert into(leaf, dout, saved) is leaf
    leaf.grad = torch.zeros(6, 8)
    into(leaf.grad, dout, saved)
    with torch.inference_mode():
        into(torch.zeros(6, 8), dout, saved)


def _short_form_cases():
    """Tensors [4, 2, 8] of many steps, and broken ones, as norm_rotary may be given them."""
    base = torch.zeros(4096)
    for token in (0, 1, 8, 15, 16, 40, 1 << 22, (1 << 22) + 1):
        for head in (0, 4, 8, 32, 1 << 40, (1 << 40) + 1):
            for column in (1, 2):
                yield torch.empty(3 * token + head + 7 * column + 1,
                                  device="meta").as_strided((4, 2, 8), (token, head, column))
    for shape in ((1, 2, 8), (4, 1, 8), (1, 1, 8), (4, 2, 1), (0, 2, 8), (4, 0, 8), (1, 1, 1)):
        n = shape[0] * shape[1] * shape[2]
        yield base[:n].view(shape)
        if n:
            for steps in ((0, 0, 0), (1, 1, 1), (3, 5, 7), (200, 30, 1), (1, 30, 1)):
                yield base.as_strided(shape, steps)


def test_norm_rotary_steps_are_those_of_the_strided_pairs():
    """Its shorter form says what head_rows and strides_arg say, for every tensor."""
    from evograd_amd.pairs._util import head_rows, strides_arg
    for t in _short_form_cases():
        (got, other), steps = norm_rotary._steps(t, t)
        want = head_rows(t)
        assert (got is t) == (want is t), (t.shape, t.stride())
        assert got.stride() == want.stride() and got.shape == want.shape
        assert steps == strides_arg(want, want), (t.shape, t.stride())


def test_norm_rotary_takes_what_its_checks_take():
    """The short look at the arguments never passes what the full one refuses, or the reverse."""
    floats = (torch.float32, torch.float16, torch.bfloat16, torch.float64, torch.int32)
    seen = set()
    for shape in ((4, 2, 8), (4, 2, 7), (4, 8), (4, 2, 8, 1), (0, 2, 8)):
        for dtype in floats:
            x = torch.zeros(shape, dtype=dtype)
            for weight in (torch.zeros(8, dtype=dtype), torch.zeros(7, dtype=dtype), torch.zeros(1, 8, dtype=dtype),
                           torch.zeros(8, dtype=torch.float16)):
                for pos in (POS, POS.long(), POS.float(), POS[:3], POS[:0], POS[:, None]):
                    for freqs in (FREQ, FREQ.float(), FREQ[:3], FREQ[:0], FREQ[None], torch.ones(5).double()):
                        try:
                            norm_rotary._check("norm_rotary", x, weight, pos, freqs)
                            _lib.dtype_tag(x.dtype)
                            good = True
                        except (TypeError, ValueError):
                            good = False
                        assert norm_rotary._fits(x, weight, pos, freqs) == good, (
                            x.shape, dtype, weight.shape, weight.dtype, pos.shape, pos.dtype, freqs.shape)
                        seen.add(good)
    assert seen == {True, False}


@built
@pytest.mark.parametrize("tau", (2.0 ** -101, 2.0 ** -149, 2.0 ** 61, 2.0 ** 127))
def test_temperatures_whose_square_or_quotients_leave_fp32(tau):
    """Refused before soft labels become NaN, whose factors grow infinite, or 0 times infinite."""
    with pytest.raises(RuntimeError, match="temperature"):
        _lib.call("eg_topk_distill_fwd", P, P, P, _lib.EG_F32, P, 0, P, P, P, P, P, 4, 9, 3, tau, 1.0, 0.0,
                  -100, _lib.EG_F32, None)
    with pytest.raises(RuntimeError, match="temperature"):
        _lib.call("eg_topk_distill_bwd", P, P, P, P, 0, P, P, P, P, 4, 9, 3, tau, 1.0, 0.0, -100,
                  _lib.EG_F32, None)
