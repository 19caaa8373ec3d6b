"""Distillation from a teacher's top logits, beside the hard-label cross entropy, on gfx950.

``logits`` [rows, cols] are the student's, ``teacher_logits`` [rows, entries] the values a teacher
gave its top tokens and ``teacher_ids`` [rows, entries] those tokens. Per row, at a temperature (from
2^-100 to 2^60):

    p = softmax(teacher_logits / temperature) over the row's entries
    q = softmax(logits / temperature) over the whole vocabulary
    soft = temperature^2 * sum p (log p - log q[teacher_ids])
    hard = logsumexp(logits) - logits[target]

and ``loss`` (fp32, one element) is the mean of ``soft_weight * soft + hard_weight * hard`` over
the rows whose ``target`` (int64 [rows]) is not ``ignore_index``; the others are not read and get
a zero gradient. Other targets are used by a hard label alone: with ``hard_weight`` 0 any of them
will do.

An entry with a negative id is none (a nucleus of fewer tokens), nor is one of value -inf at a
column; entries of the same token add up; a row without entries has a soft part of 0. An id of cols
or more, whatever its value, or a value of NaN or +inf makes the loss and the row's gradient NaN, and
so does, with a hard label, a target outside [0, cols); neither is used as an index. With
``soft_weight`` 0 the entries are not looked at. Only the logits have a gradient:

    dlogits = dloss / n * (hard_weight * (softmax(logits) - onehot(target))
                           + soft_weight * temperature * (q - sum of p at their tokens))

Saved state: ``(logits, target, teacher_ids, state)``: the inputs and one fp32 tensor that holds
[rows, 4] row statistics, [rows, entries] probabilities and the count of rows.
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


def _check(name, logits, target, teacher_ids):
    if logits.dim() != 2:
        raise ValueError(f"{name}: expected logits [rows, cols], got {tuple(logits.shape)}")
    rows = logits.shape[0]
    if target.dim() != 1 or target.shape[0] != rows:
        raise ValueError(f"{name}: target must be [rows]={rows}, got {tuple(target.shape)}")
    if target.dtype != torch.int64:
        raise TypeError(f"{name}: target must be int64, got {target.dtype}")
    if teacher_ids.dim() != 2 or teacher_ids.shape[0] != rows:
        raise ValueError(f"{name}: teacher_ids must be [rows={rows}, entries], got "
                         f"{tuple(teacher_ids.shape)}")
    if teacher_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: teacher_ids must be int32 or int64, got {teacher_ids.dtype}")


def _parts(state: torch.Tensor, rows: int, entries: int):
    """Addresses of the state's statistics, probabilities and count."""
    at = state.data_ptr()
    return at, at + 16 * rows, at + 4 * rows * (4 + entries)


def topk_distillation_forward_with_saved(logits: torch.Tensor, target: torch.Tensor,
                                         teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                                         temperature: float = 1.0, soft_weight: float = 1.0,
                                         hard_weight: float = 0.0, ignore_index: int = -100):
    name = "topk_distillation"
    _lib.require_gpu("topk_distillation_forward_with_saved", logits, target, teacher_logits,
                     teacher_ids)
    _check(name, logits, target, teacher_ids)
    if teacher_logits.shape != teacher_ids.shape:
        raise ValueError(f"{name}: teacher_logits {tuple(teacher_logits.shape)} and teacher_ids "
                         f"{tuple(teacher_ids.shape)} must have the same shape")
    dtype, teacher_dtype = tag(logits.dtype), tag(teacher_logits.dtype)
    rows, cols = logits.shape
    entries = teacher_ids.shape[1]
    logits, target = as_contiguous("logits", logits), as_contiguous("target", target)
    teacher_logits = as_contiguous("teacher_logits", teacher_logits)
    teacher_ids = as_contiguous("teacher_ids", teacher_ids)
    loss = torch.empty((), dtype=torch.float32, device=logits.device)
    state = torch.empty(rows * (4 + entries) + 1, dtype=torch.float32, device=logits.device)
    ws = workspace(_lib.query("eg_topk_distill_workspace_bytes", rows, cols, entries), logits.device)
    _lib.call_on(logits, "eg_topk_distill_fwd", logits.data_ptr(), target.data_ptr(),
                 teacher_logits.data_ptr(), teacher_dtype, teacher_ids.data_ptr(),
                 teacher_ids.dtype is torch.int64, loss.data_ptr(), *_parts(state, rows, entries),
                 ws.data_ptr(), rows, cols, entries, temperature, soft_weight, hard_weight,
                 ignore_index, dtype, _lib.stream_of(logits))
    return loss, (logits, target, teacher_ids, state)


def topk_distillation_backward_from_saved(dloss: torch.Tensor, saved, temperature: float = 1.0,
                                          soft_weight: float = 1.0, hard_weight: float = 0.0,
                                          ignore_index: int = -100):
    name = "topk_distillation_backward_from_saved"
    logits, target, teacher_ids, state = saved
    _lib.require_gpu(name, dloss, logits, target, teacher_ids, state)
    if dloss.numel() != 1 or dloss.dtype is not torch.float32:
        raise ValueError(f"{name}: dloss must be one float32 element, got {tuple(dloss.shape)} of "
                         f"{dloss.dtype}")
    rows, cols = logits.shape
    entries = teacher_ids.shape[1]
    if state.shape != (rows * (4 + entries) + 1,):
        raise ValueError(f"{name}: the saved state is not of [{rows}, {entries}] entries")
    dlogits = torch.empty_like(logits)
    _lib.call_on(logits, "eg_topk_distill_bwd", dloss.data_ptr(), logits.data_ptr(),
                 target.data_ptr(), teacher_ids.data_ptr(), teacher_ids.dtype is torch.int64,
                 *_parts(state, rows, entries), dlogits.data_ptr(), rows, cols, entries, temperature,
                 soft_weight, hard_weight, ignore_index, tag(logits.dtype), _lib.stream_of(logits))
    return dlogits
