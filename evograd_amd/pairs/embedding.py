"""Embedding lookup with scaling, and its gradient by sorted tokens, on gfx950.

    out[t] = scale * weight[ids[t]]
    dweight[v] = scale * sum of dout[t] over the tokens t with ids[t] == v

``weight`` is [vocab, hidden], ``ids`` int32 or int64 of any shape, ``out`` [*ids.shape, hidden].
Sums are fp32, a token's rows piece by piece and then the pieces, in an order that the call fixes
(the same bits every run); each result is rounded once. A token equal to ``ignore_index`` gives a
row of zeros; any other one outside [0, vocab) gives a row of NaN. Neither has a gradient. Saved
state: ``(ids, vocab, hidden, dtype)``, and not the table.

``embedding_backward_into(dweight, dout, saved, ...)`` adds the gradient to one that is there, of the
table's shape and type (a table shared with the output projection): only the rows of the batch's
own tokens are read and written, each rounded once.
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
from evograd_amd.pairs._util import as_contiguous, tag, workspace


def _check_ids(name: str, ids: torch.Tensor) -> None:
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: ids must be int32 or int64, got {ids.dtype}")


def embedding_forward_with_saved(weight: torch.Tensor, ids: torch.Tensor, scale: float = 1.0,
                                 ignore_index: int = -100):
    _lib.require_gpu("embedding_forward_with_saved", weight, ids)
    if weight.dim() != 2:
        raise ValueError(f"embedding expects weight [vocab, hidden], got {tuple(weight.shape)}")
    _check_ids("embedding", ids)
    dtype = tag(weight.dtype)
    vocab, hidden = weight.shape
    weight, ids = as_contiguous("weight", weight), as_contiguous("ids", ids)
    out = weight.new_empty((*ids.shape, hidden))
    _lib.call_on(weight, "eg_embedding_fwd", weight.data_ptr(), ids.data_ptr(),
                 ids.dtype == torch.int64, out.data_ptr(), ids.numel(), vocab, hidden, scale,
                 ignore_index, dtype, _lib.stream_of(weight))
    return out, (ids, vocab, hidden, weight.dtype)


def _backward(name, dweight, dout, saved, scale, ignore_index):
    """Writes dweight, or adds to it if there is one."""
    ids, vocab, hidden, kind = saved
    _lib.require_gpu(name, dout, ids)
    _check_ids(name, ids)
    if dout.shape != (*ids.shape, hidden) or dout.dtype is not kind:
        raise ValueError(f"{name}: dout must be {[*ids.shape, hidden]} of {kind}, got "
                         f"{tuple(dout.shape)} of {dout.dtype}")
    dtype = tag(kind)
    add = dweight is not None
    if add:
        _lib.require_gpu(name, dout, dweight)
        if dweight.shape != (vocab, hidden) or dweight.dtype is not kind:
            raise ValueError(f"{name}: dweight must be [{vocab}, {hidden}] of {kind}, got "
                             f"{tuple(dweight.shape)} of {dweight.dtype}")
        if not dweight.is_contiguous():
            raise ValueError(f"{name}: dweight must be contiguous")
        if dweight.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name}: dweight requires gradients, and what is added in place has "
                               "none; use torch.no_grad()")
    else:
        dweight = dout.new_empty((vocab, hidden))
    dout, ids = as_contiguous("dout", dout), as_contiguous("ids", ids)
    ws = workspace(_lib.query("eg_embedding_workspace_bytes", ids.numel(), vocab, hidden),
                   dout.device)
    _lib.call_on(dout, "eg_embedding_bwd", dout.data_ptr(), ids.data_ptr(),
                 ids.dtype == torch.int64, dweight.data_ptr(), ws.data_ptr(), ids.numel(), vocab,
                 hidden, scale, ignore_index, add, dtype, _lib.stream_of(dout))
    if add:  # autograd sees a change through a pointer no other way
        torch.autograd.graph.increment_version(dweight)
    return dweight


def embedding_backward_from_saved(dout: torch.Tensor, saved, scale: float = 1.0,
                                  ignore_index: int = -100):
    return _backward("embedding_backward_from_saved", None, dout, saved, scale, ignore_index)


def embedding_backward_into(dweight: torch.Tensor, dout: torch.Tensor, saved, scale: float = 1.0,
                            ignore_index: int = -100):
    """``dweight += `` the gradient, in place; returns dweight, whose version moves on as in any
    in-place operation. dweight overlaps neither dout nor the ids, and where gradients are
    recorded it may not require any."""
    _lib.require_gpu("embedding_backward_into", dweight)
    return _backward("embedding_backward_into", dweight, dout, saved, scale, ignore_index)
