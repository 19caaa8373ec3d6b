"""What the packed-batch pairs and their C entry points refuse, before any launch."""

import ctypes
import math
import os

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.pairs import block_norm, packed_attention, rotary

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="library not built")
P = 1 << 20  # an address no refused call reads


@pytest.fixture
def no_device_check(monkeypatch):
    """The pairs' own checks on CPU tensors (the device check comes first)."""
    monkeypatch.setattr(_lib, "require_gpu", lambda *a: None)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        packed_attention.packed_attention_forward_with_saved(x, x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU"):
        rotary.rotary_forward_with_saved(x, torch.zeros(4, dtype=torch.int32),
                                         torch.zeros(4, dtype=torch.float64))
    w = torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU"):
        block_norm.block_norm_forward_with_saved(x[:, 0], x[:, 0], w, None, w)


CU = torch.tensor([0, 4], dtype=torch.int32)


@pytest.mark.parametrize("q,k,v,cu,error,words", (
    ((4, 8), (4, 8), (4, 8), CU, ValueError, "tokens, heads, head_dim"),
    ((4, 4, 8), (4, 3, 8), (4, 3, 8), CU, ValueError, "not a multiple"),
    ((4, 4, 8), (4, 0, 8), (4, 0, 8), CU, ValueError, "not a multiple"),
    ((4, 0, 8), (4, 2, 8), (4, 2, 8), CU, ValueError, "not a multiple"),
    ((4, 4, 8), (5, 2, 8), (5, 2, 8), CU, ValueError, "matching q"),
    ((4, 4, 8), (4, 2, 8), (4, 4, 8), CU, ValueError, "matching q"),
    ((4, 4, 9), (4, 2, 9), (4, 2, 9), CU, ValueError, "even"),
    ((4, 4, 130), (4, 2, 130), (4, 2, 130), CU, ValueError, "at most 128"),
    ((4, 4, 8), (4, 2, 8), (4, 2, 8), CU.long(), TypeError, "int32"),
    ((4, 4, 8), (4, 2, 8), (4, 2, 8), CU[:0], ValueError, r"sequences \+ 1"),
    ((4, 4, 8), (4, 2, 8), (4, 2, 8), CU[None], ValueError, r"sequences \+ 1"),
))
def test_packed_attention_shapes(no_device_check, q, k, v, cu, error, words):
    with pytest.raises(error, match=words):
        packed_attention.packed_attention_forward_with_saved(
            torch.zeros(q), torch.zeros(k), torch.zeros(v), cu)


def test_packed_attention_types(no_device_check):
    x = torch.zeros(4, 2, 8)
    with pytest.raises(TypeError, match="mismatch"):
        packed_attention.packed_attention_forward_with_saved(x, x.half(), x, CU)
    with pytest.raises(TypeError, match="unsupported dtype"):
        packed_attention.packed_attention_forward_with_saved(x.double(), x.double(), x.double(), CU)
    saved = (x, x, x, x, torch.zeros(2, 4), CU)
    with pytest.raises(ValueError, match="do must match"):
        packed_attention.packed_attention_backward_from_saved(torch.zeros(4, 2, 6), saved)
    with pytest.raises(ValueError, match="do must match"):
        packed_attention.packed_attention_backward_from_saved(x.half(), saved)


POS, FREQ = torch.arange(4, dtype=torch.int32), torch.ones(4, dtype=torch.float64)


@pytest.mark.parametrize("x,pos,freqs,error,words", (
    (torch.zeros(4, 8), POS, FREQ, ValueError, "tokens, heads, head_dim"),
    (torch.zeros(4, 2, 8), POS[:3], FREQ, ValueError, "positions must be"),
    (torch.zeros(4, 2, 8), POS.float(), FREQ, TypeError, "int32 or int64"),
    (torch.zeros(4, 2, 8), POS, FREQ.float(), TypeError, "float64"),
    (torch.zeros(4, 2, 6), POS, FREQ, ValueError, "at most head_dim"),
    (torch.zeros(4, 2, 8).double(), POS, FREQ, TypeError, "unsupported dtype"),
))
def test_rotary_arguments(no_device_check, x, pos, freqs, error, words):
    with pytest.raises(error, match=words):
        rotary.rotary_forward_with_saved(x, pos, freqs)


def test_rotary_q_and_k_must_agree(no_device_check):
    x = torch.zeros(4, 2, 8)
    with pytest.raises(ValueError, match="share head_dim"):
        rotary.rotary_qk_forward_with_saved(x, torch.zeros(4, 2, 10), POS, FREQ)
    with pytest.raises(ValueError, match="share head_dim"):
        rotary.rotary_qk_forward_with_saved(x, x.half(), POS, FREQ)
    with pytest.raises(ValueError, match="positions must be"):
        rotary.rotary_qk_forward_with_saved(x, torch.zeros(5, 2, 8), POS, FREQ)


@pytest.mark.parametrize("dim,theta,scaling,words", (
    (7, 1e4, None, "even"), (0, 1e4, None, "even"), (8, 0.0, None, "theta"),
    (8, 1e4, {"kind": "cubic", "factor": 2.0}, "unknown scaling"),
    (8, 1e4, {"kind": "linear"}, "takes"),
    (8, 1e4, {"kind": "linear", "factor": 2.0, "low": 1.0}, "takes"),
    (8, 1e4, {"kind": "linear", "factor": 0.0}, "factor"),
    (2, 1e4, {"kind": "base", "factor": 2.0}, "above 2"),
    (8, 1e4, {"kind": "bands", "factor": 2.0, "context": 10, "low": 4.0, "high": 4.0}, "low < high"),
))
def test_frequency_arguments(dim, theta, scaling, words):
    with pytest.raises(ValueError, match=words):
        rotary.rotary_frequencies(dim, theta, scaling)


def test_frequencies_by_their_formulas():
    f = rotary.rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64
    assert f.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    lin = rotary.rotary_frequencies(8, 10000.0, {"kind": "linear", "factor": 4.0})
    assert lin.tolist() == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-14)
    # base: the highest frequency stays, the lowest is divided by the factor
    base = rotary.rotary_frequencies(8, 10000.0, {"kind": "base", "factor": 4.0})
    assert base[0] == 1.0 and float(base[-1]) == pytest.approx(0.001 / 4, rel=1e-13)
    # bands over a context of 2 pi * 100 positions: 100, 10, 1 and 0.1 turns
    bands = rotary.rotary_frequencies(8, 10000.0, {"kind": "bands", "factor": 4.0, "low": 1.0,
                                                   "high": 19.0, "context": 200 * math.pi})
    half = (10 - 1) / 18
    assert bands.tolist() == pytest.approx(
        [1.0, half * 0.1 + (1 - half) * 0.025, 0.01 / 4, 0.001 / 4], rel=1e-13)


def test_block_norm_arguments(no_device_check):
    x, w = torch.zeros(4, 8), torch.ones(8)
    call = block_norm.block_norm_forward_with_saved
    with pytest.raises(ValueError, match=r"\[rows, cols\]"):
        call(x[0], x[0], w, None, w)
    with pytest.raises(ValueError, match="x's shape"):
        call(x, x[:3], w, None, w)
    with pytest.raises(ValueError, match="length cols"):
        call(x, x, w[:7], None, w)
    with pytest.raises(ValueError, match="length cols"):
        call(x, x, w, None, torch.ones(8, 1))
    with pytest.raises(TypeError, match="mismatch"):
        call(x, x.half(), w, None, w)
    with pytest.raises(TypeError, match="mismatch"):
        call(x, x, w, w.half(), w)
    with pytest.raises(TypeError, match="unsupported dtype"):
        call(x.double(), x.double(), w.double(), None, w.double())
    for shape in ((4,), (1, 8), (8, 4), (4, 8, 1), ()):
        with pytest.raises(ValueError, match="gate must be"):
            call(x, x, w, torch.ones(shape), w)
    saved = (x, x, w, None, w, torch.ones(2, 4))
    for bad in (torch.zeros(4, 8), torch.zeros(2, 4, 7), (x, x[:3]), (x, x.half())):
        with pytest.raises(ValueError, match="block_norm"):
            block_norm.block_norm_backward_from_saved(bad, saved)


@built
def test_entry_points_check_their_arguments():
    steps = (ctypes.c_int64 * 6)(16, 8, 16, 8, 16, 8)

    def attention(tokens=4, seqs=1, heads=2, kv=2, dim=8, strides=steps, dtype=_lib.EG_F32, q=P,
                  ws=None):
        _lib.call("eg_packed_attn_fwd", q, P, P, P, P, P, ws, tokens, seqs, heads, kv, dim, strides,
                  1.0, dtype, None)

    for words, kw in (("negative", dict(tokens=-1)), ("negative", dict(seqs=-1)),
                      ("multiple", dict(kv=0)), ("multiple", dict(heads=3)),
                      ("even", dict(dim=7)), ("at most 128", dict(dim=256)),
                      ("dtype", dict(dtype=9)), ("null strides", dict(strides=None)),
                      ("strides must", dict(strides=(ctypes.c_int64 * 6)(-1, 8, 16, 8, 16, 8))),
                      ("strides must", dict(strides=(ctypes.c_int64 * 6)(16, 8, 1 << 23, 8, 16, 8))),
                      ("strides must", dict(strides=(ctypes.c_int64 * 6)(16, 8, 16, 8, 16, 1 << 41))),
                      ("out of range", dict(tokens=1 << 29)),
                      ("out of range", dict(seqs=1 << 25)),
                      ("out of range", dict(heads=8192, kv=1)),
                      ("out of range", dict(tokens=1 << 28, heads=128, kv=128)),
                      ("null pointer", dict(q=None)),
                      ("null pointer", dict(tokens=400, seqs=257))):
        with pytest.raises(RuntimeError, match=words):
            attention(**kw)
    attention(tokens=0, q=None)  # nothing to do is no error
    with pytest.raises(RuntimeError, match="null pointer"):
        _lib.call("eg_packed_attn_bwd", P, P, P, P, P, P, P, P, P, P, None, 4, 1, 2, 2, 8, steps,
                  1.0, _lib.EG_F32, None)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        _lib.call("eg_packed_attn_bwd", P, P, P, P, P, P, P, P, P, P, P + 4, 4, 1, 2, 2, 8, steps,
                  1.0, _lib.EG_F32, None)
    with pytest.raises(RuntimeError, match="positive multiple"):
        attention(heads=0)

    def turn(tokens=4, hq=2, hk=2, dim=8, pairs=4, strides=steps, dtype=_lib.EG_F32, q=P):
        _lib.call("eg_rotary", q, P, P, P, P, 0, P, tokens, hq, hk, dim, pairs, strides, 1.0, 0, 0,
                  dtype, None)

    for words, kw in (("negative", dict(tokens=-1)), ("do not fit", dict(pairs=5)),
                      ("do not fit", dict(pairs=-1)), ("out of range", dict(hq=1 << 17)),
                      ("null strides", dict(strides=None)), ("null pointer", dict(q=None)),
                      ("strides must", dict(strides=(ctypes.c_int64 * 4)(-1, 8, 16, 8))),
                      ("dtype", dict(dtype=9))):
        with pytest.raises(RuntimeError, match=words):
            turn(**kw)
    turn(tokens=0, q=None)

    def norm(rows=4, cols=8, kind=0, gate=None, x=P, dtype=_lib.EG_F32):
        _lib.call("eg_block_norm_fwd", x, P, P, gate, P, P, P, P, rows, cols, kind, 1.0, 1e-6,
                  dtype, None)

    for words, kw in (("negative", dict(rows=-1)), ("gate kind", dict(kind=4)),
                      ("gate kind", dict(kind=-1)), ("null pointer", dict(kind=1)),
                      ("null pointer", dict(x=None)), ("out of range", dict(cols=1 << 25)),
                      ("dtype", dict(dtype=9))):
        with pytest.raises(RuntimeError, match=words):
            norm(**kw)
    norm(rows=0, x=None)
    with pytest.raises(RuntimeError, match="null pointer"):
        _lib.call("eg_block_norm_bwd", P, P, P, P, P, None, P, P, P, P, P, None, P, None, 4, 8, 0,
                  1.0, _lib.EG_F32, None)


@built
def test_grids_past_32_bits_are_refused():
    """Sizes within every other limit whose grid would have 2^32 threads or more."""
    steps = (ctypes.c_int64 * 6)(1 << 14, 256, 1 << 14, 256, 1 << 14, 256)
    many = 1 << 24
    for dim, dtype in ((8, _lib.EG_F32), (128, _lib.EG_BF16)):
        with pytest.raises(RuntimeError, match="grid too large"):
            _lib.call("eg_packed_attn_fwd", P, P, P, P, P, P, P, 4, many, 64, 64, dim, steps, 1.0,
                      dtype, None)
        with pytest.raises(RuntimeError, match="grid too large"):
            _lib.call("eg_packed_attn_bwd", P, P, P, P, P, P, P, P, P, P, P, 4, many, 64, 64, dim,
                      steps, 1.0, dtype, None)
    with pytest.raises(RuntimeError, match="grid too large"):
        _lib.call("eg_rotary", P, P, P, P, P, 0, P, 1 << 32, 1, 1, 8, 4,
                  (ctypes.c_int64 * 4)(8, 8, 8, 8), 1.0, 0, 0, _lib.EG_F32, None)
    with pytest.raises(RuntimeError, match="grid too large"):
        _lib.call("eg_block_norm_fwd", P, P, P, None, P, P, P, P, 1 << 30, 64, 0, 1.0, 1e-6,
                  _lib.EG_BF16, None)
    with pytest.raises(RuntimeError, match="grid too large"):
        _lib.call("eg_block_norm_fwd", P, P, P, None, P, P, P, P, 1 << 26, 40000, 0, 1.0, 1e-6,
                  _lib.EG_BF16, None)


@built
def test_workspaces():
    al = lambda n: (n + 255) // 256 * 256
    assert _lib.query("eg_packed_attn_workspace_bytes", 0, 1, 2, 2, 64, _lib.EG_F32) == 0
    # fp32, 2 kv heads: the slabs (16 keys) of 512 cut pieces at most, or of every piece there is
    got = _lib.query("eg_packed_attn_workspace_bytes", 1600, 3, 8, 2, 32, _lib.EG_F32)
    assert got == al(1600 * 8 * 4) + 2 * min((1600 + 3 * 15) // 16 + 1 + 256, 513) * 2 * 16 * 32 * 4
    # bf16 on MFMA (128 keys): does not grow with the tokens but for delta
    mfma = lambda T: _lib.query("eg_packed_attn_workspace_bytes", T, 7, 32, 8, 128, _lib.EG_BF16)
    assert mfma(1 << 20) - mfma(1 << 17) == ((1 << 20) - (1 << 17)) * 32 * 4
    assert mfma(1 << 17) - al((1 << 17) * 32 * 4) == 8 * 129 * 2 * 128 * 128 * 4
    # no tile of index 8 (fp32, groups of 4 heads) or 1 (bf16 on MFMA): nothing to cut
    assert _lib.query("eg_packed_attn_workspace_bytes", 128, 3, 8, 2, 32, _lib.EG_F32) == 128 * 8 * 4
    assert _lib.query("eg_packed_attn_workspace_bytes", 128, 1, 8, 2, 128, _lib.EG_BF16) == 128 * 8 * 4
    # past 256 sequences: tables of their order, and no pieces
    assert _lib.query("eg_packed_attn_fwd_workspace_bytes", 256) == 0
    assert _lib.query("eg_packed_attn_fwd_workspace_bytes", 257) == al(4 * 515)
    many = _lib.query("eg_packed_attn_workspace_bytes", 9000, 300, 8, 2, 128, _lib.EG_BF16)
    assert many == al(9000 * 8 * 4) + 2 * al(4 * 601)
    assert _lib.query("eg_block_norm_workspace_bytes", 0, 64) == 0
    assert _lib.query("eg_block_norm_workspace_bytes", 3, 64) == 3 * 2 * 64 * 4
