// Causal (grouped-query) attention for the shapes the 16-bit MFMA kernels do not take:
// fp32 tensors, and head sizes other than 64 and 128 in any dtype.
//
// Same contract as attention.hip (F.scaled_dot_product_attention(q, k, v,
// is_causal=True) as called by src/evograd/ops/level3/llama3_decoder_layer/
// forward_ref.py:107, with the kv head of query head h being h / (H / Hkv), the
// repeat_interleave of :101-105): o = softmax(q k^T * scale + causal mask) v, lse =
// logsumexp of the scaled, masked scores (natural log, fp32), and the backward
// dq, dk, dv with P recomputed from lse and delta = rowsum(do * o). The reference's
// decoder layer gates its algebra at fp32 with head_dim 32 and 16
// (src/evograd/ops/level3/llama3_decoder_layer/__init__.py:55-65).
//
// Every product runs in fp32 on v_mfma_f32_16x16x4_f32 (16-bit tensors are widened as
// they are loaded), whose operands are one value per lane: A holds row l%16, k = l/16;
// B column l%16, k = l/16; the 16 x 16 result has column l%16 in lane l and row
// 4(l/16) + r in register r. Two register layouts of a 16-row tile feed them:
//   rows (load_rows): lane l holds columns 16j + 4(l/16) + e of row l%16: MFMA step
//     4j + e takes those of each lane as its four k, for A and B alike;
//   columns (load_cols): lane l holds, of row 4(l/16) + r, the columns dcol(l%16, t),
//     the A operand of a product over the tile's rows. Its k order (row 4(l/16) + r in
//     step r) is the order in which a result tile already holds its rows, so a tile of
//     P or dS is the B operand of the next product as it stands.
// So no product needs a shuffle or LDS: operands come from global memory (L2) in
// 16-byte loads, each tile's loads issued one product ahead of their use.
//
// What bounds it: with few heads the work is one long chain per row block, so the walk
// over the other side is cut over the kGenWaves waves of a workgroup (tile t to wave
// t % kGenWaves), which add their parts through LDS in wave order; the dK/dV walk is
// also cut over `parts` workgroups whose fp32 slabs attn_gen_reduce_kernel adds in
// order. At fp32 [1, 8 / 2 kv, 1024, 64] a kernel trace has 21.1 us (forward), 32.2 (dQ) and
// 41.7 + 4.7 (dK/dV and its reduction), with the matrix cores busy for 38% of the cycles of
// each, against 6031, 6316 and 30931 us for one wave per
// 64 rows on VALU FMAs (128 waves on the chip's 1024 SIMDs, about 6 us per key of the
// longest row: one dependent chain with its operands broadcast from LDS).
// No atomics: every sum has a fixed order.
//
// A masked score's weight is an exact 0, but 0 times an infinite or NaN value is NaN:
// the tiles that hold masked pairs look for such values in the operand that meets the
// zeros and, where there is one, add their products pair by pair (add_pairs).
#include "attn_generic_kernel.hpp"

#include <algorithm>

namespace eg {
namespace {

// Row blocks lie along y and, past what y can hold, z (gen_grid).
constexpr int64_t kGenGridY = 32768;
__device__ __forceinline__ int block_index() { return blockIdx.z * gridDim.y + blockIdx.y; }
inline dim3 gen_grid(int64_t x, int64_t blocks) {
  const int64_t y = blocks < kGenGridY ? blocks : kGenGridY;
  return dim3((unsigned)x, (unsigned)y, (unsigned)((blocks + y - 1) / y));
}

// Order in which the blocks of a triangle are taken, 0 = the longest walk. Longest first,
// so that what a CU takes last is short. PAIR, for kernels with two workgroups on a CU:
// where the whole grid is resident at once (kGenTarget), nothing is taken last and the
// second workgroup of each CU comes shortest first, so that every CU holds a long and a
// short walk. fp32 calls, longest first against paired: [1, 8 / 2 kv, 1024, 64] forward 26.2 ->
// 22.1 us, backward 91.5 -> 77.0 (the longest CU had 1.5 times the mean work), [1, 8 / 2,
// 1000, 128] forward 45.9 -> 36.9; the backward there has registers for one workgroup on
// a CU and would go 176.6 -> 189.9.
template <bool PAIR>
__device__ __forceinline__ int walk_order(int blk, int n) {
  const int first = kGenTarget / 2 / gridDim.x;  // blocks of the first workgroup on each CU
  return PAIR && (int64_t)gridDim.x * n <= kGenTarget && blk >= first ? n - 1 - (blk - first)
                                                                      : blk;
}

// Forward: workgroup = 16 query rows of one head. The workgroups with the most keys come
// first.
template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, 2) void attn_gen_fwd_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v, T* __restrict__ o,
    float* __restrict__ lse, int S, int D, int nqb, int group, float scale_log2) {
  const int bh = blockIdx.x, blk = block_index();
  if (blk >= nqb) return;
  const int q0 = (nqb - 1 - walk_order<true>(blk, nqb)) * 16;
  const int64_t slice = (int64_t)S * D, own = bh * slice, kv = (bh / group) * slice;
  attn_gen_fwd_rows<T, DM, VEC>(q + own, D, k + kv, D, v + kv, D, o + own, D,
                                lse + (int64_t)bh * S, S, D, q0, scale_log2);
}

template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, DM > 64 ? 1 : 2) void attn_gen_dq_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ dout, const T* __restrict__ o, const float* __restrict__ lse,
    float* __restrict__ delta, T* __restrict__ dq, int S, int D, int nqb, int group,
    float scale) {
  const int bh = blockIdx.x, blk = block_index();
  if (blk >= nqb) return;
  const int q0 = (nqb - 1 - walk_order<(DM <= 64)>(blk, nqb)) * 16;
  const int64_t slice = (int64_t)S * D, own = bh * slice, kv = (bh / group) * slice;
  attn_gen_dq_rows<T, DM, VEC, false>(q + own, D, k + kv, D, v + kv, D, dout + own, D, o + own, D,
                                      lse + (int64_t)bh * S, delta + (int64_t)bh * S, dq + own, D,
                                      S, D, q0, scale);
}

// dK, dV: workgroup = 16 keys of one kv head, part pi of `parts`. With parts > 1 the sums go
// to fp32 slabs, part[pi] for dK and part[parts + pi] for dV ([BHkv][S][D] each).
template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, DM > 64 ? 1 : 2) void attn_gen_dkdv_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
    const T* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ delta,
    T* __restrict__ dk, T* __restrict__ dv, int S, int D, int BHkv, int group, float scale,
    int parts, float* __restrict__ part) {
  __shared__ float buf[kGenWaves][16][DM + 4];
  const int bhk = blockIdx.x % BHkv, pi = blockIdx.x / BHkv;
  const int nkb = (S + 15) / 16, blk = block_index();
  if (blk >= nkb) return;
  const int k0 = walk_order<(DM <= 64)>(blk, nkb) * 16;
  const int64_t slice = (int64_t)S * D, own = bhk * slice, heads = own * group;
  const int64_t rows = (int64_t)bhk * group * S;
  f32x4 adk[DM / 16], adv[DM / 16];
  attn_gen_dkdv_keys<T, DM, VEC>(q + heads, D, slice, k + own, D, v + own, D, dout + heads, D,
                                 slice, lse + rows, delta + rows, S, S, D, group, k0, parts, pi,
                                 scale, adk, adv);
  if (parts > 1) {
    const int64_t slab = (int64_t)BHkv * slice;
    store_sum<float, DM>(buf, adk, part + pi * slab + own, D, k0, S, D, scale);
    store_sum<float, DM>(buf, adv, part + (parts + pi) * slab + own, D, k0, S, D, 1.f);
  } else {
    store_sum<T, DM>(buf, adk, dk + own, D, k0, S, D, scale);
    store_sum<T, DM>(buf, adv, dv + own, D, k0, S, D, 1.f);
  }
}

// dK (blockIdx.y = 0) and dV (1) of a cut walk: the parts' slabs in order, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void attn_gen_reduce_kernel(const float* __restrict__ part,
                                                              int parts, int64_t n,
                                                              T* __restrict__ dk,
                                                              T* __restrict__ dv) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float* p = part + blockIdx.y * parts * n + i;
  float s = p[0];
  for (int j = 1; j < parts; ++j) s += p[j * n];
  (blockIdx.y ? dv : dk)[i] = from_f32<T>(s);
}

// Parts of the dK/dV walk: at least kGenTarget workgroups (two per CU), while the
// longest walk still gives every wave kGenMinSteps steps. From the shape only.
constexpr int64_t kGenMaxParts = 8, kGenMinSteps = 2;
int64_t gen_parts(int64_t BHkv, int64_t group, int64_t S) {
  const int64_t nkb = (S + 15) / 16;
  const int64_t want = (kGenTarget + BHkv * nkb - 1) / (BHkv * nkb);
  const int64_t most = group * nkb / (kGenWaves * kGenMinSteps);
  return std::max<int64_t>(1, std::min({want, most, kGenMaxParts}));
}

}  // namespace

size_t attn_generic_part_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D) {
  const int64_t parts = gen_parts(B * Hkv, H / Hkv, S);
  return parts > 1 ? (size_t)2 * parts * B * Hkv * S * D * sizeof(float) : 0;
}

int attn_generic_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int64_t B,
                     int64_t H, int64_t Hkv, int64_t S, int64_t D, float scale, int dtype,
                     hipStream_t st) {
  const int64_t nqb = (S + 15) / 16;
  const int group = (int)(H / Hkv);
  return gen_dispatch(dtype, D, {q, k, v}, "eg_attn_fwd", [&](auto tag, auto dm, auto vec) {
    using T = decltype(tag);
    EG_LAUNCH((attn_gen_fwd_kernel<T, decltype(dm)::value, decltype(vec)::value>),
              gen_grid(B * H, nqb), dim3(kGenThreads), 0, st, (const T*)q, (const T*)k,
              (const T*)v, (T*)o, lse, (int)S, (int)D, (int)nqb, group, scale * kGenLog2e);
    return check_launch("eg_attn_fwd(generic)");
  });
}

int attn_generic_bwd(const void* dout, const void* q, const void* k, const void* v,
                     const void* o, const float* lse, void* dq, void* dk, void* dv, float* delta,
                     float* part, int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D,
                     float scale, int dtype, hipStream_t st) {
  const int64_t nb = (S + 15) / 16;
  const int group = (int)(H / Hkv);
  const int parts = (int)gen_parts(B * Hkv, group, S);
  return gen_dispatch(dtype, D, {dout, q, k, v, o}, "eg_attn_bwd", [&](auto tag, auto dm,
                                                                       auto vec) {
    using T = decltype(tag);
    constexpr int DM = decltype(dm)::value;
    constexpr bool VEC = decltype(vec)::value;
    EG_LAUNCH((attn_gen_dq_kernel<T, DM, VEC>), gen_grid(B * H, nb), dim3(kGenThreads), 0, st,
              (const T*)q, (const T*)k, (const T*)v, (const T*)dout, (const T*)o, lse, delta,
              (T*)dq, (int)S, (int)D, (int)nb, group, scale);
    if (int e = check_launch("eg_attn_bwd(generic dq)")) return e;
    EG_LAUNCH((attn_gen_dkdv_kernel<T, DM, VEC>), gen_grid(B * Hkv * parts, nb),
              dim3(kGenThreads), 0, st, (const T*)q, (const T*)k, (const T*)v, (const T*)dout, lse,
              delta, (T*)dk, (T*)dv, (int)S, (int)D, (int)(B * Hkv), group, scale, parts, part);
    if (int e = check_launch("eg_attn_bwd(generic dkdv)")) return e;
    if (parts == 1) return 0;
    const int64_t n = B * Hkv * S * D;
    EG_LAUNCH((attn_gen_reduce_kernel<T>), dim3((unsigned)((n + 255) / 256), 2u), dim3(256), 0, st,
              (const float*)part, parts, n, (T*)dk, (T*)dv);
    return check_launch("eg_attn_bwd(generic dkdv reduce)");
  });
}

}  // namespace eg
