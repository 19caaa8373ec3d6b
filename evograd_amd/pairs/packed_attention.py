"""Causal grouped-query attention over packed sequences, as a pair on gfx950.

Sequences of different lengths lie one behind the other along the token axis: q is
[tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], and sequence s holds the
rows ``cu_seqlens[s] .. cu_seqlens[s + 1] - 1``. Every row attends to the rows of its own
sequence up to itself, query head h with kv head h // (heads // kv_heads):

    o_i = softmax_j<=i(q_i . k_j / sqrt(head_dim)) v_j

``cu_seqlens`` is int32 on the tensors' GPU, starts at 0 and does not decrease; empty
sequences are allowed. Rows from ``cu_seqlens[-1]`` on belong to no sequence: their o and
gradients are zero, and whatever their q, k, v and do hold is not read into any result. The
bounds are read on the GPU alone (no synchronisation, so a captured graph replays with new
lengths); bounds that break the rules give undefined values, but no access outside the tensors.

q, k and v may be strided (column ranges of one fused projection's rows, say) as long as a
head's columns are contiguous; o and the gradients come back contiguous. Saved state:
``(q, k, v, o, lse, cu_seqlens)``, lse fp32 [heads, tokens]. dk and dv are summed over each
query group in a fixed order (no atomics, bitwise repeatable).
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
from evograd_amd.pairs._util import (as_contiguous, check_same, contiguous_like, head_rows,
                                     strides_arg, tag, workspace)


def _check(q, k, v, cu_seqlens):
    name = "packed_attention"
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError(f"{name}: q, k and v must be [tokens, heads, head_dim], got "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    check_same(name, q, k, v)
    tag(q.dtype)
    T, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"{name}: k and v must be [tokens, kv_heads, head_dim] matching q "
                         f"{tuple(q.shape)}; got {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape[1] == 0 or H == 0 or H % k.shape[1]:
        raise ValueError(f"{name}: {H} query heads are not a multiple of {k.shape[1]} kv heads")
    if D < 2 or D > 128 or D % 2:
        raise ValueError(f"{name}: head_dim must be even and at most 128, got {D}")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError(f"{name}: cu_seqlens must be [sequences + 1], got "
                         f"{tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype != torch.int32:
        raise TypeError(f"{name}: cu_seqlens must be int32, got {cu_seqlens.dtype}")


def packed_attention_forward_with_saved(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                        cu_seqlens: torch.Tensor):
    _lib.require_gpu("packed_attention_forward_with_saved", q, k, v, cu_seqlens)
    _check(q, k, v, cu_seqlens)
    q, k, v = head_rows(q), head_rows(k), head_rows(v)
    cu_seqlens = as_contiguous("cu_seqlens", cu_seqlens)
    T, H, D = q.shape
    N = cu_seqlens.shape[0] - 1
    nbytes = _lib.query("eg_packed_attn_fwd_workspace_bytes", N)
    ws = workspace(nbytes, q.device) if nbytes else None
    o = contiguous_like(q)
    lse = q.new_empty((H, T), dtype=torch.float32)
    _lib.call_on(q, "eg_packed_attn_fwd", _lib.ptr(q), _lib.ptr(k), _lib.ptr(v),
                 _lib.ptr(cu_seqlens), _lib.ptr(o), _lib.ptr(lse), _lib.ptr(ws), T, N, H, k.shape[1],
                 D, strides_arg(q, k, v), 1.0 / math.sqrt(D), tag(q.dtype), _lib.stream_of(q))
    return o, (q, k, v, o, lse, cu_seqlens)


def packed_attention_backward_from_saved(do: torch.Tensor, saved):
    q, k, v, o, lse, cu_seqlens = saved
    _lib.require_gpu("packed_attention_backward_from_saved", do, q, k, v, o, lse, cu_seqlens)
    if do.shape != o.shape or do.dtype != o.dtype:
        raise ValueError("packed_attention: do must match o in shape and dtype")
    do = as_contiguous("do", do)
    T, H, D = q.shape
    KVH, N = k.shape[1], cu_seqlens.shape[0] - 1
    dq, dk, dv = contiguous_like(q), contiguous_like(k), contiguous_like(v)
    ws = workspace(_lib.query("eg_packed_attn_workspace_bytes", T, N, H, KVH, D, tag(q.dtype)),
                   q.device)
    _lib.call_on(q, "eg_packed_attn_bwd", _lib.ptr(do), _lib.ptr(q), _lib.ptr(k), _lib.ptr(v),
                 _lib.ptr(cu_seqlens), _lib.ptr(o), _lib.ptr(lse), _lib.ptr(dq), _lib.ptr(dk),
                 _lib.ptr(dv), _lib.ptr(ws), T, N, H, KVH, D, strides_arg(q, k, v),
                 1.0 / math.sqrt(D), tag(q.dtype), _lib.stream_of(q))
    return dq, dk, dv
