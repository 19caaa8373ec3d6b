"""Packed attention and rotary on tensors whose rows share their memory or lie far apart."""

import pytest
import torch

from evograd_amd import _lib
from evograd_amd.pairs import packed_attention, rotary
from evograd_amd.pairs._util import strides_arg
from tests.packed_refs import assert_within, attention64, rotary64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(dtype, *shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def bounds(lengths):
    cu = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    cu[1:] = torch.tensor(lengths, dtype=torch.int32).cumsum(0)
    return cu.cuda()


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (64, F32), (80, BF16)))
@pytest.mark.parametrize("shared", ("q", "k", "v", "qkv"))
def test_attention_over_one_row_shared_by_every_token(shared, D, dtype):
    """A token step of zero at the entry points (the wrappers copy such a tensor first)."""
    lengths, H, KVH = [70, 1, 33], 4, 2
    T = sum(lengths) + 3
    print(f"\n[gpu-packed-strides] {shared} D={D} {dtype}", flush=True)
    t = {n: normal(dtype, T, h, D, seed=i) for i, (n, h) in enumerate((("q", H), ("k", KVH), ("v", KVH)))}
    for n in shared:
        t[n] = t[n][:1].expand(T, -1, D)
        assert t[n].stride(0) == 0
    do, cu = normal(dtype, T, H, D, seed=9), bounds(lengths)
    o, dq = torch.empty_like(do), torch.empty_like(do)
    dk, dv = (torch.empty(T, KVH, D, dtype=dtype, device="cuda") for _ in range(2))
    lse = torch.empty(H, T, device="cuda")
    ws = torch.empty(_lib.query("eg_packed_attn_workspace_bytes", T, len(lengths), H, KVH, D,
                                _lib.dtype_tag(dtype)), dtype=torch.uint8, device="cuda")
    qkv = (t["q"], t["k"], t["v"])
    common = (T, len(lengths), H, KVH, D, strides_arg(*qkv), D ** -0.5, _lib.dtype_tag(dtype),
              _lib.stream_of(do))
    _lib.call("eg_packed_attn_fwd", *map(_lib.ptr, (*qkv, cu, o, lse, None)), *common)
    _lib.call("eg_packed_attn_bwd", *map(_lib.ptr, (do, *qkv, cu, o, lse, dq, dk, dv, ws)), *common)
    # rows that 16-byte loads may not take run without the rounding of P and dS
    narrow = attention64(*qkv, do, lengths, False)
    wide = attention64(*qkv, do, lengths, dtype != F32 and D in (64, 128))
    for name, x, (value, bound), (_, loose) in zip(("o", "dq", "dk", "dv"), (o, dq, dk, dv), narrow,
                                                   wide):
        assert_within(name, x, value, torch.maximum(bound, loose))


@pytest.mark.parametrize("D,dtype", ((128, BF16), (64, F16), (64, F32), (80, BF16)))
def test_attention_over_heads_that_share_their_rows(D, dtype):
    lengths, H, KVH = [70, 1, 133], 4, 2
    T = sum(lengths)
    q, k, v = (normal(dtype, T, 1, D, seed=i).expand(T, h, D) for i, h in enumerate((H, KVH, KVH)))
    do, cu = normal(dtype, T, H, D, seed=9), bounds(lengths)

    def run(*qkv):
        o, saved = packed_attention.packed_attention_forward_with_saved(*qkv, cu)
        assert all(a.data_ptr() == b.data_ptr() for a, b in zip(saved, qkv))  # taken as they are
        return (o, *packed_attention.packed_attention_backward_from_saved(do, saved))

    for x, y in zip(run(q, k, v), run(q.contiguous(), k.contiguous(), v.contiguous())):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", (BF16, F32))
@pytest.mark.parametrize("interleaved", (0, 1))
@pytest.mark.parametrize("steps", ((0, 64), (0, 0), (64, 0)))
def test_rotary_over_rows_that_share_their_memory(steps, interleaved, dtype):
    T, H, D = 37, 3, 64
    row = normal(dtype, 1 if steps[0] == 0 else T, 1 if steps[1] == 0 else H, D)
    x = row.expand(T, H, D)
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 17
    freqs = rotary.rotary_frequencies(48, device="cuda")
    y = torch.empty(T, H, D, dtype=dtype, device="cuda")
    _lib.call("eg_rotary", x.data_ptr(), None, y.data_ptr(), None, pos.data_ptr(), 0,
              freqs.data_ptr(), T, H, 0, D, 24, strides_arg(x, x), 1.0, interleaved, 0,
              _lib.dtype_tag(dtype), _lib.stream_of(x))
    assert_within("y", y, *rotary64(x, pos, freqs, 1.0, interleaved))
    want, _ = rotary.rotary_forward_with_saved(x.contiguous(), pos, freqs, 1.0, interleaved)
    assert torch.equal(y, want)


def test_rotary_of_heads_past_32_bits_apart():
    T, D, step = 3, 64, (1 << 32) + 64
    print(f"\n[gpu-packed-strides] heads {step} elements apart", flush=True)
    room = torch.empty(step + T * D, dtype=BF16, device="cuda")
    x = room.as_strided((T, 2, D), (D, step, 1))
    x.copy_(normal(BF16, T, 2, D))
    pos = torch.tensor([5, 70, 1 << 20], dtype=torch.int32, device="cuda")
    freqs = rotary.rotary_frequencies(D, device="cuda")
    small = x.contiguous()
    for call in (rotary.rotary_forward_with_saved,
                 lambda a, *rest: (rotary.rotary_backward_from_saved(a, rest), None)):
        y, _ = call(x, pos, freqs)
        assert torch.equal(y, call(small, pos, freqs)[0])
    del room, x
    torch.cuda.empty_cache()
