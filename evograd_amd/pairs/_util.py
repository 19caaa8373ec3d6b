"""Argument checks shared by the pair modules."""

from __future__ import annotations

import struct

import torch

from evograd_amd import _lib


def as_contiguous(name: str, t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def check_same(name: str, ref: torch.Tensor, *others: torch.Tensor) -> None:
    for o in others:
        if o.dtype != ref.dtype:
            raise TypeError(f"{name}: dtype mismatch {ref.dtype} vs {o.dtype}")


def workspace(nbytes: int, device) -> torch.Tensor:
    """Scratch bytes from torch's caching allocator (the library never allocates)."""
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


tag = _lib.dtype_tag


# The widest steps between tokens, whose rows the strided kernels address with 32-bit offsets
# inside a tile, and between heads.
MAX_TOKEN_STRIDE, MAX_HEAD_STRIDE = 1 << 22, 1 << 40


def head_rows(t: torch.Tensor) -> torch.Tensor:
    """A [tokens, heads, head_dim] tensor as the strided kernels take it: itself when a head's
    columns are contiguous, its rows do not overlap and its steps are in range, else a
    contiguous copy."""
    tokens, heads, dim = t.shape
    if ((dim == 1 or t.stride(2) == 1)
            and (tokens <= 1 or dim <= t.stride(0) <= MAX_TOKEN_STRIDE)
            and (heads <= 1 or t.stride(1) <= MAX_HEAD_STRIDE)):
        return t
    return t.contiguous()


def strides_arg(*tensors: torch.Tensor) -> bytes:
    """Token and head strides of [tokens, heads, head_dim] tensors as a C array of int64; an axis
    of one element has the step of a contiguous tensor, whatever torch notes for it."""
    steps = []
    for t in tensors:
        tokens, heads, dim = t.shape
        token, head, _ = t.stride()
        steps += (token if tokens > 1 else heads * dim, head if heads > 1 else dim)
    return struct.pack(f"{len(steps)}q", *steps)


def contiguous_like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of t's shape, dtype and device (empty_like would keep
    a strided tensor's order of axes)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)
