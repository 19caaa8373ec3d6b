"""Norms of queries and keys for each head with the position rotation behind them, on gfx950.

x is [tokens, heads, head_dim], ``weight`` [head_dim] and ``positions`` [tokens] each token's own
position. Per head, in one pass:

    n = x * rsqrt(mean(x^2) + eps) * weight
    y = n rotated by position * freqs over the first 2 * len(freqs) columns

with the rotation, pairs and ``freqs`` of the ``rotary`` pair (fp64, from
``rotary.rotary_frequencies``), whose ``amplitude`` scales the rotated columns alone. Sums and
angles as there; y is rounded once. Saved state: ``(x, weight, positions, freqs)``, the caller's
tensors: the backward forms the norms again from x, which it reads anyway, and so takes eps.

``norm_rotary_qk_forward_with_saved`` / ``norm_rotary_qk_backward_from_saved`` take the query and
key tensors of a layer, each with its weight, in one launch. x, q, k and the upstream gradients may
be strided as long as a head's columns are contiguous; the results are contiguous.
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

import struct

import torch

from evograd_amd import _lib
from evograd_amd.once import needs_tie, once, tie
from evograd_amd.pairs._util import (MAX_HEAD_STRIDE, MAX_TOKEN_STRIDE, as_contiguous, check_same,
                                     head_rows, tag, workspace)
from evograd_amd.pairs.rotary import _check as _check_positions

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _check(name, x, weight, positions, freqs):
    _check_positions(name, x, positions, freqs)
    if weight.dim() != 1 or weight.shape[0] != x.shape[2]:
        raise ValueError(f"{name}: the weight must be [head_dim]={x.shape[2]}, got "
                         f"{tuple(weight.shape)}")
    check_same(name, x, weight)


def _fits(x, weight, positions, freqs):
    """Whether _check has nothing to say, in a few lookups (small calls are bound by the host)."""
    shape, dtype = x.shape, x.dtype
    return (len(shape) == 3 and dtype in _FLOATS and weight.dtype is dtype
            and weight.shape == shape[2:] and positions.shape == shape[:1]
            and positions.dtype in (torch.int32, torch.int64) and freqs.dtype is torch.float64
            and freqs.dim() == 1 and 2 * freqs.shape[0] <= shape[2])


_PACKERS = {n: struct.Struct(f"{n}q").pack for n in (2, 4, 8)}


def _steps(*tensors):
    """[tokens, heads, head_dim] tensors as the kernels take them (head_rows), and their token and
    head steps as a C array of int64."""
    out, steps = [], []
    for t in tensors:
        tokens, heads, dim = t.shape
        token, head, column = t.stride()
        # an axis of one element has the step of a contiguous tensor, whatever torch notes for it
        if tokens <= 1:
            token = heads * dim
        if heads <= 1:
            head = dim
        if not (column == 1 and dim <= token <= MAX_TOKEN_STRIDE and head <= MAX_HEAD_STRIDE):
            t = head_rows(t)
            if t.is_contiguous():
                token, head = heads * dim, dim
        out.append(t)
        steps.append(token)
        steps.append(head)
    return out, _PACKERS[len(steps)](*steps)


def _forward(name, q, k, q_weight, k_weight, positions, freqs, eps, amplitude, interleaved):
    """y of q, and of k unless it is None, and the tensors as the kernels take them."""
    if k is None:
        _lib.require_gpu(name, q, q_weight, positions, freqs)
    else:
        _lib.require_gpu(name, q, k, q_weight, k_weight, positions, freqs)
        if not _fits(k, k_weight, positions, freqs):
            _check(name, k, k_weight, positions, freqs)
    if not _fits(q, q_weight, positions, freqs):
        _check(name, q, q_weight, positions, freqs)
    T, H, D = q.shape
    positions, freqs = as_contiguous("positions", positions), as_contiguous("freqs", freqs)
    q_weight, qo = as_contiguous("q_weight", q_weight), q.new_empty((T, H, D))
    if k is None:
        (q,), steps = _steps(q)
        steps, ko, heads_k = steps + steps, None, 0
    else:
        heads_k = k.shape[1]
        if k.shape[2] != D or k.dtype is not q.dtype:
            raise ValueError(f"{name}: q and k must share head_dim and dtype")
        (q, k), steps = _steps(q, k)
        k_weight, ko = as_contiguous("k_weight", k_weight), k.new_empty((T, heads_k, D))
    _lib.call_on(q, "eg_norm_rotary_fwd", q.data_ptr(), _lib.ptr(k), q_weight.data_ptr(),
                 _lib.ptr(k_weight), qo.data_ptr(), _lib.ptr(ko), positions.data_ptr(),
                 positions.dtype is torch.int64, freqs.data_ptr(), T, H, heads_k, D, freqs.shape[0],
                 steps, eps, amplitude, interleaved != 0, tag(q.dtype), _lib.stream_of(q))
    return qo, ko, (q, k, q_weight, k_weight, positions, freqs)


def _backward(name, dq_out, dk_out, saved, eps, amplitude, interleaved):
    """Gradients of the saved tensors, which are as _forward leaves them."""
    q, k, q_weight, k_weight, positions, freqs = saved
    _lib.require_gpu(name, *(t for t in (dq_out, dk_out, *saved) if t is not None))
    for d, x in ((dq_out, q), (dk_out, k)):
        if x is not None and (d.shape != x.shape or d.dtype is not x.dtype):
            raise ValueError(f"{name}: the upstream gradients must match q and k in shape and dtype")
    T, H, D = q.shape
    dq, dqw, dk, dkw, heads_k = q.new_empty((T, H, D)), torch.empty_like(q_weight), None, None, 0
    if k is None:
        (q, dq_out), steps = _steps(q, dq_out)
        steps = steps[:16] * 2 + steps[16:] * 2
    else:
        heads_k = k.shape[1]
        dk, dkw = k.new_empty((T, heads_k, D)), torch.empty_like(k_weight)
        (q, k, dq_out, dk_out), steps = _steps(q, k, dq_out, dk_out)
    ws = workspace(_lib.query("eg_norm_rotary_workspace_bytes", T, H, heads_k, D), q.device)
    _lib.call_on(q, "eg_norm_rotary_bwd", dq_out.data_ptr(), _lib.ptr(dk_out), q.data_ptr(),
                 _lib.ptr(k), q_weight.data_ptr(), _lib.ptr(k_weight), positions.data_ptr(),
                 positions.dtype is torch.int64, freqs.data_ptr(), dq.data_ptr(), _lib.ptr(dk),
                 dqw.data_ptr(), _lib.ptr(dkw), ws.data_ptr(), T, H, heads_k, D, freqs.shape[0],
                 steps, eps, amplitude, interleaved != 0, tag(q.dtype), _lib.stream_of(q))
    return dq, dk, dqw, dkw


def norm_rotary_forward_with_saved(x: torch.Tensor, weight: torch.Tensor, positions: torch.Tensor,
                                   freqs: torch.Tensor, eps: float = 1e-6, amplitude: float = 1.0,
                                   interleaved: int = 0):
    y, _, saved = _forward("norm_rotary_forward_with_saved", x, None, weight, None, positions,
                           freqs, eps, amplitude, interleaved)
    return y, (saved[0], saved[2], *saved[4:])


def norm_rotary_backward_from_saved(dy: torch.Tensor, saved, eps: float = 1e-6,
                                    amplitude: float = 1.0, interleaved: int = 0):
    x, weight, positions, freqs = saved
    dx, _, dweight, _ = _backward("norm_rotary_backward_from_saved", dy, None,
                                  (x, None, weight, None, positions, freqs), eps, amplitude,
                                  interleaved)
    return dx, dweight


def norm_rotary_qk_forward_with_saved(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                                      k_weight: torch.Tensor, positions: torch.Tensor,
                                      freqs: torch.Tensor, eps: float = 1e-6,
                                      amplitude: float = 1.0, interleaved: int = 0):
    qo, ko, saved = _forward("norm_rotary_qk_forward_with_saved", q, k, q_weight, k_weight,
                             positions, freqs, eps, amplitude, interleaved)
    return (qo, ko), saved


def norm_rotary_qk_backward_from_saved(grads, saved, eps: float = 1e-6, amplitude: float = 1.0,
                                       interleaved: int = 0):
    """``(dq, dk, dq_weight, dk_weight)`` from the pair of upstream gradients."""
    dq_out, dk_out = grads
    return _backward("norm_rotary_qk_backward_from_saved", dq_out, dk_out, saved, eps, amplitude,
                     interleaved)


class NormRotaryQK(torch.autograd.Function):
    """The joint q/k pair as an autograd node: ``NormRotaryQK.apply(q, k, q_weight, k_weight,
    positions, freqs, eps, amplitude, interleaved)`` -> ``(q', k')``; positions and frequencies
    get no gradient, and the node can be differentiated once."""

    @classmethod
    def apply(cls, *args):
        return super().apply(*args)[:2]

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, freqs, eps=1e-6, amplitude=1.0,
                interleaved=0):
        out, saved = norm_rotary_qk_forward_with_saved(q, k, q_weight, k_weight, positions, freqs,
                                                       eps, amplitude, interleaved)
        ties = (tie(),) if needs_tie((q, k, q_weight, k_weight), saved, out) else ()
        ctx.save_for_backward(*saved, *ties)
        ctx.scalars = (eps, amplitude, interleaved)
        return (*out, *ties)

    @staticmethod
    def backward(ctx, dq_out, dk_out, *_):
        kept = ctx.saved_tensors
        grads = norm_rotary_qk_backward_from_saved((dq_out, dk_out), kept[:6], *ctx.scalars)
        return (*once("NormRotaryQK", grads, (dq_out, dk_out, *kept)), None, None, None, None, None)
