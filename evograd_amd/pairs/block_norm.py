"""The norms around a block, fused with its gate, residual scale and residual, on gfx950.

Between one block (attention, MLP) and the next, a layer with a norm behind each block and
one before it computes, for the block's output h and the residual stream x:

    n = rmsnorm(h) * post_weight
    s = x + scale * gate * n            (the new residual stream)
    y = rmsnorm(s) * pre_weight         (the next block's input)

as one pair with ``out[0] = s`` and ``out[1] = y`` ([2, rows, cols]). ``gate`` is a learned
factor per channel [cols], per row [rows, 1] or per element [rows, cols], or None (a factor
of one, whose gradient slot is None). Statistics and sums are fp32; s and y are rounded once,
y from the unrounded s. Saved state: ``(x, h, post_weight, gate, pre_weight, rstd)``, the
inputs plus fp32 rstd [2, rows]; the backward forms s again from x and h, which moves the same
bytes as reading a saved s.

The backward takes ``dout`` as a [2, rows, cols] tensor or as the pair ``(ds, dy)``.
``BlockNorm.apply(x, h, post_weight, gate, pre_weight, scale, eps)`` -> ``(s, y)`` is the same
pair as an autograd node with two outputs, whose gradients arrive separately; it can be
differentiated once.
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

import torch

from evograd_amd import _lib
from evograd_amd.once import needs_tie, once, tie
from evograd_amd.pairs._util import as_contiguous, check_same, tag, workspace

_NONE, _CHANNEL, _ROW, _ELEMENT = range(4)


def _gate_kind(gate, rows: int, cols: int) -> int:
    if gate is None:
        return _NONE
    shape = tuple(gate.shape)
    for kind, want in ((_CHANNEL, (cols,)), (_ROW, (rows, 1)), (_ELEMENT, (rows, cols))):
        if shape == want:
            return kind
    raise ValueError(f"block_norm: gate must be [cols], [rows, 1] or [rows, cols] of "
                     f"[{rows}, {cols}], got {shape}")


def _check(x, h, post_weight, gate, pre_weight):
    if x.dim() != 2:
        raise ValueError(f"block_norm expects x [rows, cols], got {tuple(x.shape)}")
    if h.shape != x.shape:
        raise ValueError("block_norm: h must have x's shape")
    for weight in (post_weight, pre_weight):
        if weight.dim() != 1 or weight.shape[0] != x.shape[1]:
            raise ValueError("block_norm: the weights must be 1D with length cols")
    check_same("block_norm", x, h, post_weight, pre_weight)
    tag(x.dtype)
    if gate is not None:
        check_same("block_norm", x, gate)
    _gate_kind(gate, *x.shape)


def _forward(s, y, x, h, post_weight, gate, pre_weight, scale, eps):
    rows, cols = x.shape
    kind = _gate_kind(gate, rows, cols)
    rstd = x.new_empty((2, rows), dtype=torch.float32)
    _lib.call_on(x, "eg_block_norm_fwd", _lib.ptr(x), _lib.ptr(h), _lib.ptr(post_weight),
                 _lib.ptr(gate), _lib.ptr(pre_weight), _lib.ptr(s), _lib.ptr(y), _lib.ptr(rstd),
                 rows, cols, kind, float(scale), float(eps), tag(x.dtype), _lib.stream_of(x))
    return x, h, post_weight, gate, pre_weight, rstd


def _prepare(name, x, h, post_weight, gate, pre_weight):
    given = [t for t in (x, h, post_weight, gate, pre_weight) if t is not None]
    _lib.require_gpu(name, *given)
    _check(x, h, post_weight, gate, pre_weight)
    return tuple(None if t is None else as_contiguous(n, t) for n, t in
                 (("x", x), ("h", h), ("post_weight", post_weight), ("gate", gate),
                  ("pre_weight", pre_weight)))


def block_norm_forward_with_saved(x: torch.Tensor, h: torch.Tensor, post_weight: torch.Tensor,
                                  gate: torch.Tensor | None, pre_weight: torch.Tensor,
                                  scale: float = 1.0, eps: float = 1e-6):
    args = _prepare("block_norm_forward_with_saved", x, h, post_weight, gate, pre_weight)
    out = x.new_empty((2, *x.shape))
    return out, _forward(out[0], out[1], *args, scale, eps)


def block_norm_backward_from_saved(dout, saved, scale: float = 1.0):
    x, h, post_weight, gate, pre_weight, rstd = saved
    rows, cols = x.shape
    if torch.is_tensor(dout):
        if tuple(dout.shape) != (2, rows, cols):
            raise ValueError(f"block_norm: dout must be [2, {rows}, {cols}] or two tensors, got "
                             f"{tuple(dout.shape)}")
        dout = (dout[0], dout[1])
    ds, dy = dout
    _lib.require_gpu("block_norm_backward_from_saved", ds, dy, x, h)
    for d in (ds, dy):
        if d.shape != x.shape or d.dtype != x.dtype:
            raise ValueError("block_norm: ds and dy must match x in shape and dtype")
    ds, dy = as_contiguous("ds", ds), as_contiguous("dy", dy)
    dx, dh = torch.empty_like(x), torch.empty_like(h)
    dpost, dpre = torch.empty_like(post_weight), torch.empty_like(pre_weight)
    dgate = None if gate is None else torch.empty_like(gate)
    ws = workspace(_lib.query("eg_block_norm_workspace_bytes", rows, cols), x.device)
    _lib.call_on(x, "eg_block_norm_bwd", _lib.ptr(ds), _lib.ptr(dy), _lib.ptr(x), _lib.ptr(h),
                 _lib.ptr(post_weight), _lib.ptr(gate), _lib.ptr(pre_weight), _lib.ptr(rstd),
                 _lib.ptr(dx), _lib.ptr(dh), _lib.ptr(dpost), _lib.ptr(dgate), _lib.ptr(dpre),
                 _lib.ptr(ws), rows, cols, _gate_kind(gate, rows, cols), float(scale), tag(x.dtype),
                 _lib.stream_of(x))
    return dx, dh, dpost, dgate, dpre


class BlockNorm(torch.autograd.Function):
    """``BlockNorm.apply(x, h, post_weight, gate, pre_weight, scale, eps)`` -> ``(s, y)``."""

    @classmethod
    def apply(cls, *args):
        return super().apply(*args)[:2]

    @staticmethod
    def forward(ctx, x, h, post_weight, gate, pre_weight, scale=1.0, eps=1e-6):
        args = _prepare("BlockNorm", x, h, post_weight, gate, pre_weight)
        s, y = torch.empty_like(args[0]), torch.empty_like(args[0])
        saved = [t for t in _forward(s, y, *args, scale, eps) if t is not None]
        ties = (tie(),) if needs_tie((x, h, post_weight, gate, pre_weight), saved, (s, y)) else ()
        ctx.has_gate = gate is not None
        ctx.save_for_backward(*saved, *ties)
        ctx.scale = scale
        return (s, y, *ties)

    @staticmethod
    def backward(ctx, ds, dy, *_):
        kept = ctx.saved_tensors
        saved = kept[:6] if ctx.has_gate else (*kept[:3], None, *kept[3:5])
        grads = block_norm_backward_from_saved((ds, dy), saved, ctx.scale)
        return (*once("BlockNorm", grads, (ds, dy, *kept)), None, None)
