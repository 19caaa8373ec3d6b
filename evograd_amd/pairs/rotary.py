"""Rotary positions by a position per token, as a pair on gfx950.

x is [tokens, heads, head_dim] and ``positions`` [tokens] gives each token's own position, so
packed sequences restart theirs and single tokens of many requests bring each its own. The
first 2 * len(freqs) columns of a head rotate, the others pass through:

    angle = position * freqs[i]
    (x1, x2) -> amplitude * (x1 cos - x2 sin, x2 cos + x1 sin)

over the pairs (i, i + len(freqs)), or (2i, 2i + 1) with ``interleaved``. The backward is the
transpose. ``freqs`` is fp64, radians per position (``rotary_frequencies`` builds it, scaled
for long contexts if asked): angles are formed and reduced in fp64, which far positions need.
Saved state: ``(positions, freqs)``, the caller's tensors.

``rotary_qk_forward_with_saved`` / ``rotary_qk_backward_from_saved`` rotate the query and key
tensors of a layer in one launch each way. x, q and k may be strided as long as a head's
columns are contiguous; the results are contiguous.
"""

from __future__ import annotations

if not __package__:
    # Loaded from this file's path as a top-level candidate module (evograd's verify
    # and bench commands load a program that way): put the package root on sys.path.
    import pathlib as _pathlib
    import sys as _sys

    _ROOT = str(_pathlib.Path(__file__).resolve().parents[2])
    if _ROOT not in _sys.path:
        _sys.path.insert(0, _ROOT)

import math

import torch

from evograd_amd import _lib
from evograd_amd.once import once
from evograd_amd.pairs._util import as_contiguous, contiguous_like, head_rows, strides_arg, tag


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: dict | None = None,
                       device=None) -> torch.Tensor:
    """Radians per position of each of rotary_dim / 2 pairs, fp64: theta ** (-2i / rotary_dim),
    scaled for contexts longer than the trained one by ``scaling``:

    * ``{"kind": "linear", "factor": f}``: every frequency divided by f;
    * ``{"kind": "base", "factor": f}``: theta times f ** (rotary_dim / (rotary_dim - 2)), which
      divides the lowest frequency by f and leaves the highest as it is;
    * ``{"kind": "bands", "factor": f, "context": n, "low": a, "high": b}``: frequencies that turn
      at least b times over the trained context of n positions stay, those that turn at most a
      times are divided by f, and between them the two are blended linearly in the turns.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim must be even and positive, got {rotary_dim}")
    if not theta > 0:
        raise ValueError(f"rotary_frequencies: theta must be positive, got {theta}")
    wanted = {"linear": {"factor"}, "base": {"factor"},
              "bands": {"factor", "context", "low", "high"}}
    kind = None if scaling is None else scaling.get("kind")
    if scaling is not None:
        if kind not in wanted:
            raise ValueError(f"rotary_frequencies: unknown scaling kind {kind!r}; known: "
                             f"{sorted(wanted)}")
        if set(scaling) - {"kind"} != wanted[kind]:
            raise ValueError(f"rotary_frequencies: scaling {kind!r} takes {sorted(wanted[kind])}, "
                             f"got {sorted(set(scaling) - {'kind'})}")
        if not scaling["factor"] > 0:
            raise ValueError("rotary_frequencies: factor must be positive")
    if kind == "base":
        if rotary_dim == 2:
            raise ValueError("rotary_frequencies: base scaling needs a rotary_dim above 2")
        theta = theta * scaling["factor"] ** (rotary_dim / (rotary_dim - 2))
    freqs = [theta ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if kind == "linear":
        freqs = [f / scaling["factor"] for f in freqs]
    elif kind == "bands":
        low, high = scaling["low"], scaling["high"]
        if not (0 <= low < high and scaling["context"] > 0):
            raise ValueError("rotary_frequencies: bands need 0 <= low < high and a positive context")
        keep = [min(1.0, max(0.0, (scaling["context"] * f / (2 * math.pi) - low) / (high - low)))
                for f in freqs]
        freqs = [k * f + (1 - k) * f / scaling["factor"] for k, f in zip(keep, freqs)]
    return torch.tensor(freqs, dtype=torch.float64, device=device)


def _check(name, x, positions, freqs):
    if x.dim() != 3:
        raise ValueError(f"{name}: expected [tokens, heads, head_dim], got {tuple(x.shape)}")
    tag(x.dtype)
    if positions.dim() != 1 or positions.shape[0] != x.shape[0]:
        raise ValueError(f"{name}: positions must be [tokens]={x.shape[0]}, got "
                         f"{tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: positions must be int32 or int64, got {positions.dtype}")
    if freqs.dtype != torch.float64:
        raise TypeError(f"{name}: freqs must be float64, got {freqs.dtype}")
    if freqs.dim() != 1 or 2 * freqs.shape[0] > x.shape[2]:
        raise ValueError(f"{name}: freqs {tuple(freqs.shape)} must be [pairs] with 2 * pairs at "
                         f"most head_dim {x.shape[2]}")


def _turn(name, q, k, positions, freqs, amplitude, interleaved, inverse):
    """q, and k unless it is None, rotated."""
    if k is None:
        _lib.require_gpu(name, q, positions, freqs)
        _check(name, q, positions, freqs)
    else:
        _lib.require_gpu(name, q, k, positions, freqs)
        _check(name, q, positions, freqs)
        _check(name, k, positions, freqs)
        if k.shape[2] != q.shape[2] or k.dtype != q.dtype:
            raise ValueError(f"{name}: q and k must share head_dim and dtype")
        k = head_rows(k)
        ko = contiguous_like(k)
    q = head_rows(q)
    qo = contiguous_like(q)
    positions, freqs = as_contiguous("positions", positions), as_contiguous("freqs", freqs)
    T, H, D = q.shape
    _lib.call_on(q, "eg_rotary", q.data_ptr(), _lib.ptr(k), qo.data_ptr(),
                 None if k is None else ko.data_ptr(), positions.data_ptr(),
                 positions.dtype == torch.int64, freqs.data_ptr(), T, H,
                 0 if k is None else k.shape[1], D, freqs.shape[0],
                 strides_arg(q, q if k is None else k), amplitude, bool(interleaved), inverse,
                 tag(q.dtype), _lib.stream_of(q))
    return (qo,) if k is None else (qo, ko), (positions, freqs)


def rotary_forward_with_saved(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor,
                              amplitude: float = 1.0, interleaved: int = 0):
    (y,), saved = _turn("rotary_forward_with_saved", x, None, positions, freqs, amplitude,
                        interleaved, False)
    return y, saved


def rotary_backward_from_saved(dy: torch.Tensor, saved, amplitude: float = 1.0,
                               interleaved: int = 0):
    (dx,), _ = _turn("rotary_backward_from_saved", dy, None, *saved, amplitude, interleaved, True)
    return dx


def rotary_qk_forward_with_saved(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                                 freqs: torch.Tensor, amplitude: float = 1.0,
                                 interleaved: int = 0):
    return _turn("rotary_qk_forward_with_saved", q, k, positions, freqs, amplitude, interleaved,
                 False)


def rotary_qk_backward_from_saved(grads, saved, amplitude: float = 1.0, interleaved: int = 0):
    dq_out, dk_out = grads
    (dq, dk), _ = _turn("rotary_qk_backward_from_saved", dq_out, dk_out, *saved, amplitude,
                        interleaved, True)
    return dq, dk


class RotaryQK(torch.autograd.Function):
    """The joint q/k pair as an autograd node: ``RotaryQK.apply(q, k, positions, freqs,
    amplitude, interleaved)`` -> ``(q', k')``; positions and frequencies get no gradient, and
    the node can be differentiated once."""

    @staticmethod
    def forward(ctx, q, k, positions, freqs, amplitude=1.0, interleaved=0):
        out, saved = rotary_qk_forward_with_saved(q, k, positions, freqs, amplitude, interleaved)
        ctx.save_for_backward(*saved)
        ctx.scalars = (amplitude, interleaved)
        return out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        grads = rotary_qk_backward_from_saved((dq_out, dk_out), ctx.saved_tensors, *ctx.scalars)
        return (*once("RotaryQK", grads, (dq_out, dk_out)), None, None, None, None)
