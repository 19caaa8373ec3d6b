// Causal scaled-dot-product attention forward/backward for gfx950 (bf16/fp16
// operands, fp32 accumulation on MFMA).
//
// Semantics: F.scaled_dot_product_attention(q, k, v, is_causal=True) as used by
// src/evograd/ops/level3/llama3_decoder_layer/forward_ref.py:107:
//   o = softmax(q k^T * scale + causal mask) v,   lse = logsumexp(q k^T * scale + mask)
// Backward recomputes P = exp(q k^T * scale - lse) and, with delta = rowsum(do * o):
//   dv = P^T do,  dS = P * (dP - delta) with dP = do v^T,  dq = scale * dS k,
//   dk = scale * dS^T q.
//
// Layout: q, o, do, dq are [B, H, S, D] row-major (D contiguous); k, v, dk, dv
// are [B, Hkv, S, D] with H a multiple of Hkv (grouped-query attention: query
// head h reads kv head h / (H / Hkv), the repeat_interleave of
// src/evograd/ops/level3/llama3_decoder_layer/forward_ref.py:101-105 without the
// copy; Hkv = H is ordinary multi-head attention); lse and delta are fp32 [B, H, S].
//
// MFMA: v_mfma_f32_32x32x16_{bf16,f16}. Lane l of a wave holds, for an M x K
// operand A, row l%32 and k = 8*(l/32) .. +7; for B (K x N), column l%32 and the
// same k; the 32 x 32 fp32 result C gives lane l column l%32 and, in register r,
// row (r/4)*8 + (l/32)*4 + r%4. Every product is arranged so that its result is
// the B operand of the next one without a shuffle: the k order of that product is
// permuted to C's register order (rows 8j + 4*(l/32) + i), and its A operand is
// read from LDS in the same order.
//
// LDS tiles are row-major ([rows][D], 16-byte chunks XOR-swizzled per row) and
// are filled by direct buffer->LDS loads (no VGPR staging). One tile serves both
// operand shapes:
//   rows as A (k along D): one 16-byte ds_read_b128 per lane;
//   transposed as A (rows = D index, k along the tile's rows): two
//   ds_read_b64_tr_b16, each giving a lane 4 consecutive tile rows of one column.
// gfx950 LDS serves 256 bytes per cycle; the swizzle 4*(r%4) + (r/4)%4 puts the
// 16 rows of a b128 read in 16 distinct bank groups and the 4 rows of a
// transpose read in 4 distinct 64-byte quarters (conflict-free at D = 128).
//
// Kernels (all deterministic, no atomics):
//   attn_fwd:   workgroup = 8 waves x 32 query rows (4 waves on grids of fewer than
//               512 8-wave workgroups; 2 x 4 waves cutting the keys between them on
//               small grids of long rows, split_keys); double-buffered 64-key K and
//               V tiles; online softmax in the log2 domain against a running
//               reference max, refreshed only when a P term could exceed 2^8 (a
//               lane's sum of P terms bounds each term, so no per-tile max is
//               formed; exact: the reference point cancels in o = sum / l);
//               S^T = K Q^T, O^T += V^T P^T.
//   attn_dq:    (runs first) workgroup = 4 waves x 32 query rows (or 2 x 4 waves, as
//               above); also computes
//               delta = rowsum(do * o) for its rows into the workspace;
//               double-buffered 64-key K, V tiles; S^T = K Q^T, dP^T = V dO^T,
//               dQ^T += K^T dS^T.
//   attn_dkdv:  workgroup = NW waves x 32 keys (K in registers, the workgroup's V
//               in LDS); double-buffered 32-row Q and dO tiles from the diagonal
//               down; S = Q K^T, dP = dO V^T, dV^T += dO^T P, dK^T += Q^T dS.
// The dQ pass recomputes S and dP (7 products executed where the causal
// FLOP convention counts 5) so that no atomics are needed.
//
// Workgroup order: workgroup i runs on XCD i % 8 and every block of one (b, h)
// is mapped to the same XCD, so K/V (or Q/dO) tiles of a head are shared in
// that XCD's L2; the blocks with the most work are dispatched first.
#include "attention_kernel.hpp"

#include <initializer_list>
#include <type_traits>

namespace eg {
namespace {

// Workgroup i -> (head, block index): XCD i % 8 holds heads xcd, xcd + 8, ...;
// block index 0 is dispatched first for every head.
__device__ __forceinline__ void block_coords(int BH, int& bh, int& blk) {
  const int i = blockIdx.x;
  const int xcd = i % 8, rest = i / 8;
  const int groups = (BH + 7) / 8;
  bh = xcd + 8 * (rest % groups);
  blk = rest / groups;
}

// Grouped-query attention: query head `bh_q` (flat over batch x heads) reads key/
// value head bh_q / group. A virtual head index v (the one block_coords spreads
// over the XCDs) maps to bh_q = (v % BHkv) * group + v / BHkv, so the `group`
// query heads that share a kv head have the same v % 8, i.e. the same XCD and L2,
// whenever BHkv is a multiple of 8. With group = 1 this is the identity.
__device__ __forceinline__ int query_head(int v, int BHkv, int group) {
  return (v % BHkv) * group + v / BHkv;
}

template <typename T, int D, int NW, int KG, bool ROPE>
__global__ __launch_bounds__(NW * KG * 64, 2) void attn_fwd_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
    const uint16_t* __restrict__ v, uint16_t* __restrict__ o, float* __restrict__ lse, int S,
    float scale_log2, int nqb, int BH, int group, const float* __restrict__ rope_cos,
    const float* __restrict__ rope_sin) {
  int vh, blk;
  block_coords(BH, vh, blk);
  if (vh >= BH) return;
  const int bh = query_head(vh, BH / group, group);
  const int q0 = (nqb - 1 - blk) * (32 * NW);  // longest rows first
  const int64_t own = (int64_t)bh * S * D, kv = (int64_t)(bh / group) * S * D;
  attn_fwd_rows<T, D, NW, KG, 1, ROPE, false>(q + own, D, 0, k + kv, D, v + kv, D, o + own, D, 0,
                                              lse + (int64_t)bh * S, 0, S, scale_log2, q0,
                                              rope_cos, rope_sin);
}

// Workgroup (kv head, part of the walk, key block); with parts > 1 the walk is cut into
// `parts` ranges of steps, each summed into its own fp32 slab of `part`
// (attn_dkdv_reduce_kernel adds the slabs in order). The parts of a kv head share its XCD
// when BHkv is a multiple of 8.
template <typename T, int D, int NW, int BQ, bool ROPE>
__global__ __launch_bounds__(NW * 64, 2) void attn_dkdv_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
    const uint16_t* __restrict__ v, const uint16_t* __restrict__ dout,
    const float* __restrict__ lse, const float* __restrict__ delta, uint16_t* __restrict__ dk,
    uint16_t* __restrict__ dv, int S, float scale, float scale_log2, int BHkv, int group,
    const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, int parts,
    float* __restrict__ part) {
  int vh, kb;
  block_coords(BHkv * parts, vh, kb);  // kb = 0 (the longest walk) first
  if (vh >= BHkv * parts) return;
  const int kvh = vh % BHkv, pi = vh / BHkv;
  const int64_t slice = (int64_t)S * D, own = kvh * slice, heads = own * group;
  const int64_t rows = (int64_t)kvh * group * S, slab = BHkv * slice;
  attn_dkdv_keys<T, D, NW, BQ, ROPE, false>(
      q + heads, D, slice, k + own, D, v + own, D, dout + heads, D, slice, lse + rows, delta + rows,
      S, dk + own, dv + own, D, S, scale, scale_log2, kb * 32 * NW, group, rope_cos, rope_sin,
      parts, pi, part ? part + pi * slab + own : nullptr,
      part ? part + (parts + pi) * slab + own : nullptr, D);
}

// dK, dV of a split walk: the parts' fp32 slabs ([2][parts][BHkv][S][D], dK slabs
// first) added in part order and rounded once; 4 consecutive elements of each per
// thread (D is a multiple of 4).
template <typename T>
__global__ __launch_bounds__(256) void attn_dkdv_reduce_kernel(const float* __restrict__ part,
                                                               int parts, int64_t n,
                                                               uint16_t* __restrict__ dk,
                                                               uint16_t* __restrict__ dv) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 a = *reinterpret_cast<const float4*>(part + i);
  float4 b = *reinterpret_cast<const float4*>(part + parts * n + i);
  for (int p = 1; p < parts; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(part + p * n + i);
    const float4 y = *reinterpret_cast<const float4*>(part + (parts + p) * n + i);
    a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
    b.x += y.x, b.y += y.y, b.z += y.z, b.w += y.w;
  }
  uint2 u;
  u.x = MM<T>::pack2(a.x, a.y);
  u.y = MM<T>::pack2(a.z, a.w);
  *reinterpret_cast<uint2*>(dk + i) = u;
  u.x = MM<T>::pack2(b.x, b.y);
  u.y = MM<T>::pack2(b.z, b.w);
  *reinterpret_cast<uint2*>(dv + i) = u;
}

template <typename T, int D, int NW, int KG, bool ROPE>
__global__ __launch_bounds__(NW * KG * 64, 2) void attn_dq_kernel(
    const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
    const uint16_t* __restrict__ v, const uint16_t* __restrict__ dout,
    const uint16_t* __restrict__ o, const float* __restrict__ lse, float* __restrict__ delta,
    uint16_t* __restrict__ dq, int S, float scale, float scale_log2, int nqb, int BH,
    int group, const float* __restrict__ rope_cos, const float* __restrict__ rope_sin) {
  int vh, blk;
  block_coords(BH, vh, blk);
  if (vh >= BH) return;
  const int bh = query_head(vh, BH / group, group);
  const int64_t own = (int64_t)bh * S * D, kv = (int64_t)(bh / group) * S * D;
  const int64_t row = (int64_t)bh * S;
  attn_dq_rows<T, D, NW, KG, 1, ROPE, false>(q + own, D, 0, k + kv, D, v + kv, D, dout + own,
                                             o + own, dq + own, D, 0, lse + row, delta + row, 0, S,
                                             scale, scale_log2, (nqb - 1 - blk) * (32 * NW),
                                             rope_cos, rope_sin);
}

// --------------------------------------------------------------- launchers
// Forward workgroup width: 8 waves (256 query rows), two per SIMD, each K/V tile
// serving 256 rows (interleaved at [4, 32, 4096, 128]: 590-597 us with 4 waves,
// 565-571 us with 8). dQ keeps 4 waves (8: 3.5% slower).
constexpr int kFwdWaves = 8;
// Forward grids of fewer than two 8-wave workgroups per CU (few heads or short
// sequences: the decoder layer's B = 1, 32 heads at T <= 2048) take 4-wave workgroups
// instead, twice as many of them; the rows each wave computes are the same, so the
// results are identical.
constexpr int kFwdSmallWaves = 4, kFwdFullGrid = 512;
constexpr int kDqWaves = 4;
constexpr int kDkdvRows = 32;
// dK/dV workgroup width: 4 waves (128 keys), one per SIMD, so that two workgroups
// share a CU and one's barrier waits overlap the other's work (at D = 128, 8-wave
// workgroups of 256 keys are 3-4% slower).
template <int D> constexpr int dkdv_waves() { return 4; }

// Split walk of the dK/dV kernel: with fewer than kDkdvTarget workgroups (kv heads
// x key blocks of 128 keys: small batches, few kv heads, short sequences), each key
// block's walk over the query tiles of its group is cut into `parts` (at most
// kDkdvMaxParts) whose fp32 sums go to workspace slabs, added in part order by
// attn_dkdv_reduce_kernel. The choice depends on the shape only, so results are
// the same on every run and device.
constexpr int kDkdvTarget = 1024, kDkdvMaxParts = 8;
int dkdv_parts(int64_t BHkv, int64_t S, int64_t D) {
  if (D != 64 && D != 128) return 1;
  const int64_t nkb = (S + 32 * dkdv_waves<128>() - 1) / (32 * dkdv_waves<128>());
  const int64_t wgs = BHkv * nkb;
  if (wgs <= 0 || wgs >= kDkdvTarget) return 1;
  return (int)std::min<int64_t>(kDkdvMaxParts, (kDkdvTarget + wgs - 1) / wgs);
}
// Parts to take, up to that bound: each shortens the longest
// walk until the chip is full (two workgroups per CU) and costs its slabs' write and read.
// In us, 1.1 (D = 128) or 0.9 (64) per 32-row step, 1.6 per million elements of dK and
// part, and 5 for the reduction: fitted over 48 shapes timed at every number of parts; the
// backward at the bound against at the choice: bf16 [2, 12, 1000, 64] 54.7 -> 46.4 us (6 parts,
// 3), [4, 8, 512, 128] 72.1 -> 44.4 (8, 1), [1, 8, 2048, 128] 107.7 -> 92.2 (8, 5), [8, 16, 256, 64]
// 40.9 -> 22.0 (4, 1); [1, 32 / 8, 512, 128] stays at 8 parts, [1, 4, 8192, 64] at 4.
int dkdv_split(int64_t BHkv, int64_t group, int64_t S, int64_t D) {
  const int most = dkdv_parts(BHkv, S, D);
  const double step = D == 128 ? 1.1 : 0.9;
  const double steps = (double)group * (double)((S + 31) / 32);  // the longest walk
  const double wgs = (double)BHkv * (double)((S + 127) / 128);
  const double full = wgs * steps / 2 / 512, slab = 1.6e-6 * (double)BHkv * (double)(S * D);
  int best = 1;
  double least = 0;
  for (int p = 1; p <= most; ++p) {
    const double c = step * std::max(steps / p, full) + (p > 1 ? slab * p + 5.0 : 0.0);
    if (p == 1 || c < least) least = c, best = p;
  }
  return best;
}
// Backward workspace after delta (fp32 [BH, S], rounded up to 256 bytes): the split
// walk's slabs, 2 x parts x BHkv x S x D fp32 (none without a split).
size_t attn_delta_bytes(int64_t BH, int64_t S) { return ((size_t)(BH * S) * 4 + 255) / 256 * 256; }
size_t attn_part_bytes(int64_t BHkv, int64_t group, int64_t S, int64_t D) {
  const int parts = dkdv_split(BHkv, group, S, D);
  return parts > 1 ? (size_t)2 * parts * BHkv * S * D * 4 : 0;
}

// The MFMA kernels take 16-bit tensors with head_dim 64 or 128; everything else
// (fp32, other even head sizes up to 128) runs on the generic kernels
// (attn_generic.hip).
bool mfma_shape(int64_t D, int dtype) {
  return (D == 64 || D == 128) && (dtype == EG_BF16 || dtype == EG_F16);
}

int check_attn(const char* what, int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D,
               int dtype, bool mfma_only = false) {
  if (B < 0 || H < 0 || S < 0) { set_error("%s: negative size", what); return 1; }
  if (H > 0 && (Hkv <= 0 || H % Hkv != 0)) {
    set_error("%s: heads (%lld) must be a positive multiple of kv_heads (%lld)", what,
              (long long)H, (long long)Hkv);
    return 1;
  }
  if (mfma_only) {
    if (D != 64 && D != 128) { set_error("%s: head_dim must be 64 or 128, got %lld", what, (long long)D); return 1; }
    if (dtype != EG_BF16 && dtype != EG_F16) { set_error("%s: dtype must be bf16 or fp16", what); return 1; }
  } else {
    if (D < 2 || D > 128 || D % 2) { set_error("%s: head_dim must be even and at most 128, got %lld", what, (long long)D); return 1; }
    if (dtype != EG_BF16 && dtype != EG_F16 && dtype != EG_F32) { set_error("%s: dtype must be fp32, bf16 or fp16", what); return 1; }
  }
  // One (b, h) slice is addressed with 32-bit buffer offsets: S * D * 2 < 2^31.
  if (S > ((int64_t)1 << 22) || B * H > ((int64_t)1 << 24)) {
    set_error("%s: size out of range (seq <= 4194304, batch*heads <= 16777216)", what);
    return 1;
  }
  return 0;
}

inline unsigned grid_for(int64_t BH, int nblocks) {
  return (unsigned)(((BH + 7) / 8) * 8 * nblocks);
}

// Two key groups per workgroup (KG = 2) in the forward and dQ: for grids of at most 512
// 128-row workgroups, where the chain of key tiles of the last rows sets the time, from
// 768 positions (12 tiles) on. bf16 forward / backward, one group against two: [1, 16 / 4,
// 2000, 128] 38.0 / 114.4 -> 30.7 / 108.5 us, [1, 4, 900, 128] 19.7 / 51.3 -> 17.7 / 50.7, [1, 8,
// 768, 64] 13.0 / 33.9 -> 12.0 / 34.0; shorter rows only pay for the exchange ([1, 2 / 1, 200,
// 128] 8.2 -> 9.0 us, [4, 8, 512, 128] 12.8 -> 13.3).
// A CU holds one workgroup of two groups or two of one, so past 256 workgroups the second
// round has to be won back by longer rows. Forward: at D = 128 from 2048 positions ([1, 64 / 8,
// 1000] 28.0 -> 30.1, [1, 32 / 8, 2048] 47.8 -> 44.5), at 64 always ([1, 64 / 8, 800] 16.2 -> 15.8,
// [1, 40 / 8, 1152] 19.5 -> 17.9). dQ, backward: up to 384 workgroups at 128 from 2048 ([1, 24 /
// 8, 2048] 150.4 -> 144.4, [1, 16 / 4, 2500] 146.3 -> 135.5, [1, 48 / 12, 903] 90.5 -> 97.0), at 64
// from 1152 ([3, 16, 900] 50.4 -> 53.8, [2, 24, 780] 44.3 -> 47.3, [1, 40 / 8, 1152] 60.7 -> 60.6,
// [1, 24 / 8, 2048] 86.0 -> 81.8); up to 512 from 4096 ([1, 32 / 8, 2048, 128] 173.4 -> 171.7 but
// 178.1 -> 180.9 on another card, [1, 16 / 4, 4096, 128] 287.6 -> 273.5).
// A head's result is a sum in the order its grid takes, so it may differ in its last bits
// between calls with few and with many heads.
constexpr int64_t kSplitKeysGrid = 512, kSplitKeysSeq = 768;
inline bool split_keys(int64_t BH, int64_t S, int64_t D, bool dq) {
  const int64_t grid = grid_for(BH, (int)((S + 127) / 128));
  if (S < kSplitKeysSeq || grid > kSplitKeysGrid) return false;
  if (grid <= 256) return true;
  if (!dq) return D == 64 || S >= 2048;
  return S >= 4096 || (grid <= 384 && S >= (D == 64 ? 1152 : 2048));
}

// With ROPE, q is rotated in registers by the fp32 tables rc/rs [S, D] as it is
// loaded (k must already be rotated).
template <typename T, int D, bool ROPE = false>
int attn_fwd_launch(const void* q, const void* k, const void* v, void* o, float* lse, int64_t BH,
                    int64_t S, int group, float scale, hipStream_t st,
                    const float* rc = nullptr, const float* rs = nullptr) {
  auto go = [&](auto nwc, auto kgc) {
    constexpr int NW = decltype(nwc)::value, KG = decltype(kgc)::value;
    const int nqb = (int)((S + 32 * NW - 1) / (32 * NW));
    EG_LAUNCH((attn_fwd_kernel<T, D, NW, KG, ROPE>), dim3(grid_for(BH, nqb)), dim3(NW * KG * 64), 0, st,
              (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)o, lse,
              (int)S, scale * kLog2e, nqb, (int)BH, group, rc, rs);
    return check_launch("eg_attn_fwd");
  };
  const int nqb_full = (int)((S + 32 * kFwdWaves - 1) / (32 * kFwdWaves));
  using One = std::integral_constant<int, 1>;
  if (split_keys(BH, S, D, false))
    return go(std::integral_constant<int, kFwdSmallWaves>{}, std::integral_constant<int, 2>{});
  if (grid_for(BH, nqb_full) < (unsigned)kFwdFullGrid)
    return go(std::integral_constant<int, kFwdSmallWaves>{}, One{});
  return go(std::integral_constant<int, kFwdWaves>{}, One{});
}

// BH counts query heads (x batch); the key/value tensors hold BH / group heads.
// With ROPE, q and k are the rotated tensors and dq, dk are written for the
// pre-rotation ones (the rotation's transpose applied to the results in registers).
template <typename T, int D, bool ROPE = false>
int attn_bwd_launch(const void* dout, const void* q, const void* k, const void* v, const void* o,
                    const float* lse, void* dq, void* dk, void* dv, float* delta, int64_t BH,
                    int64_t S, int group, float scale, hipStream_t st,
                    const float* rc = nullptr, const float* rs = nullptr) {
  // The split walk's slabs follow delta in the workspace.
  float* part = (float*)((char*)delta + attn_delta_bytes(BH, S));
  // dQ first: it also computes delta = rowsum(do * o) for its rows, which the
  // dK/dV kernel reads.
  constexpr int NQ = kDqWaves;
  const int nqb = (int)((S + 32 * NQ - 1) / (32 * NQ));
  auto run_dq = [&](auto kgc) {
    constexpr int KG = decltype(kgc)::value;
    EG_LAUNCH((attn_dq_kernel<T, D, NQ, KG, ROPE>), dim3(grid_for(BH, nqb)), dim3(NQ * KG * 64), 0,
              st, (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v,
              (const uint16_t*)dout, (const uint16_t*)o, lse, delta, (uint16_t*)dq, (int)S, scale,
              scale * kLog2e, nqb, (int)BH, group, rc, rs);
  };
  if (split_keys(BH, S, D, true)) run_dq(std::integral_constant<int, 2>{});
  else run_dq(std::integral_constant<int, 1>{});
  if (int rc = check_launch("eg_attn_bwd(dq)")) return rc;
  constexpr int NK = dkdv_waves<D>();
  const int nkb = (int)((S + 32 * NK - 1) / (32 * NK));
  const int64_t BHkv = BH / group;
  static_assert(NK == dkdv_waves<128>(), "dkdv_parts assumes one key-block width");
  const int parts = dkdv_split(BHkv, group, S, D);
  EG_LAUNCH((attn_dkdv_kernel<T, D, NK, kDkdvRows, ROPE>), dim3(grid_for(BHkv * parts, nkb)),
            dim3(NK * 64), 0, st, (const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v,
            (const uint16_t*)dout, lse, delta, (uint16_t*)dk, (uint16_t*)dv, (int)S, scale,
            scale * kLog2e, (int)BHkv, group, rc, rs, parts, parts > 1 ? part : nullptr);
  if (int e = check_launch("eg_attn_bwd(dkdv)")) return e;
  if (parts == 1) return 0;
  const int64_t n = BHkv * S * D;
  EG_LAUNCH((attn_dkdv_reduce_kernel<T>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, st,
            (const float*)part, parts, n, (uint16_t*)dk, (uint16_t*)dv);
  return check_launch("eg_attn_bwd(dkdv reduce)");
}

// Explicit instantiations: hip-clang leaves some implicitly instantiated kernel
// templates without a host launch stub (undefined symbol at load time); naming
// every kernel here makes the stubs certain.
#define EG_ATTN_INSTANTIATE(T, D, R)                                                         \
  template __global__ void attn_fwd_kernel<T, D, kFwdWaves, 1, R>(                           \
      const uint16_t*, const uint16_t*, const uint16_t*, uint16_t*, float*, int, float, int,   \
      int, int, const float*, const float*);                                                 \
  template __global__ void attn_fwd_kernel<T, D, kFwdSmallWaves, 1, R>(                      \
      const uint16_t*, const uint16_t*, const uint16_t*, uint16_t*, float*, int, float, int,   \
      int, int, const float*, const float*);                                                 \
  template __global__ void attn_fwd_kernel<T, D, kFwdSmallWaves, 2, R>(                      \
      const uint16_t*, const uint16_t*, const uint16_t*, uint16_t*, float*, int, float, int,   \
      int, int, const float*, const float*);                                                 \
  template __global__ void attn_dkdv_kernel<T, D, dkdv_waves<D>(), kDkdvRows, R>(            \
      const uint16_t*, const uint16_t*, const uint16_t*, const uint16_t*, const float*,        \
      const float*, uint16_t*, uint16_t*, int, float, float, int, int, const float*,           \
      const float*, int, float*);                                                            \
  template __global__ void attn_dq_kernel<T, D, kDqWaves, 1, R>(                                \
      const uint16_t*, const uint16_t*, const uint16_t*, const uint16_t*, const uint16_t*,     \
      const float*, float*, uint16_t*, int, float, float, int, int, int, const float*,         \
      const float*);                                                                      \
  template __global__ void attn_dq_kernel<T, D, kDqWaves, 2, R>(                                \
      const uint16_t*, const uint16_t*, const uint16_t*, const uint16_t*, const uint16_t*,     \
      const float*, float*, uint16_t*, int, float, float, int, int, int, const float*,         \
      const float*);
EG_ATTN_INSTANTIATE(bf16_t, 128, false)
EG_ATTN_INSTANTIATE(bf16_t, 64, false)
EG_ATTN_INSTANTIATE(f16_t, 128, false)
EG_ATTN_INSTANTIATE(f16_t, 64, false)
EG_ATTN_INSTANTIATE(bf16_t, 128, true)
EG_ATTN_INSTANTIATE(bf16_t, 64, true)
EG_ATTN_INSTANTIATE(f16_t, 128, true)
EG_ATTN_INSTANTIATE(f16_t, 64, true)
#undef EG_ATTN_INSTANTIATE

bool attn_aligned(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  return true;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" size_t eg_attn_gqa_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads,
                                              int64_t seq, int64_t head_dim) {
  if (batch <= 0 || heads <= 0 || seq <= 0 || kv_heads <= 0) return 0;
  // the dtype is not known here: the larger of the MFMA and the generic kernels' slabs
  return attn_delta_bytes(batch * heads, seq) +
         std::max(attn_part_bytes(batch * kv_heads, heads / kv_heads, seq, head_dim),
                  attn_generic_part_bytes(batch, heads, kv_heads, seq, head_dim));
}

extern "C" size_t eg_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t seq,
                                          int64_t head_dim) {
  return eg_attn_gqa_workspace_bytes(batch, heads, heads, seq, head_dim);
}

extern "C" int eg_attn_gqa_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                               int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq,
                               int64_t head_dim, float scale, int dtype, void* stream) {
  clear_error();
  if (check_attn("eg_attn_fwd", batch, heads, kv_heads, seq, head_dim, dtype)) return 1;
  if (batch == 0 || heads == 0 || seq == 0) return 0;
  if (!q || !k || !v || !o || !lse) { set_error("eg_attn_fwd: null pointer"); return 1; }
  hipStream_t st = as_stream(stream);
  if (!mfma_shape(head_dim, dtype))
    return attn_generic_fwd(q, k, v, o, lse, batch, heads, kv_heads, seq, head_dim, scale, dtype,
                            st);
  if (!attn_aligned({q, k, v, o})) { set_error("eg_attn_fwd: tensors must be 16-byte aligned"); return 1; }
  const int64_t BH = batch * heads;
  const int group = (int)(heads / kv_heads);
  if (dtype == EG_BF16)
    return head_dim == 128 ? attn_fwd_launch<bf16_t, 128>(q, k, v, o, lse, BH, seq, group, scale, st)
                           : attn_fwd_launch<bf16_t, 64>(q, k, v, o, lse, BH, seq, group, scale, st);
  return head_dim == 128 ? attn_fwd_launch<f16_t, 128>(q, k, v, o, lse, BH, seq, group, scale, st)
                         : attn_fwd_launch<f16_t, 64>(q, k, v, o, lse, BH, seq, group, scale, st);
}

extern "C" int eg_attn_gqa_bwd(const void* dout, const void* q, const void* k, const void* v,
                               const void* o, const float* lse, void* dq, void* dk, void* dv,
                               void* workspace, int64_t batch, int64_t heads, int64_t kv_heads,
                               int64_t seq, int64_t head_dim, float scale, int dtype,
                               void* stream) {
  clear_error();
  if (check_attn("eg_attn_bwd", batch, heads, kv_heads, seq, head_dim, dtype)) return 1;
  if (batch == 0 || heads == 0 || seq == 0) return 0;
  if (!dout || !q || !k || !v || !o || !lse || !dq || !dk || !dv || !workspace) {
    set_error("eg_attn_bwd: null pointer");
    return 1;
  }
  hipStream_t st = as_stream(stream);
  float* delta = (float*)workspace;
  if (!mfma_shape(head_dim, dtype))
    return attn_generic_bwd(dout, q, k, v, o, lse, dq, dk, dv, delta,
                            (float*)((char*)delta + attn_delta_bytes(batch * heads, seq)), batch,
                            heads, kv_heads, seq, head_dim, scale, dtype, st);
  if (!attn_aligned({dout, q, k, v, o, dq, dk, dv})) {
    set_error("eg_attn_bwd: tensors must be 16-byte aligned");
    return 1;
  }
  const int64_t BH = batch * heads;
  const int group = (int)(heads / kv_heads);
  if (dtype == EG_BF16)
    return head_dim == 128
               ? attn_bwd_launch<bf16_t, 128>(dout, q, k, v, o, lse, dq, dk, dv, delta, BH, seq, group, scale, st)
               : attn_bwd_launch<bf16_t, 64>(dout, q, k, v, o, lse, dq, dk, dv, delta, BH, seq, group, scale, st);
  return head_dim == 128
             ? attn_bwd_launch<f16_t, 128>(dout, q, k, v, o, lse, dq, dk, dv, delta, BH, seq, group, scale, st)
             : attn_bwd_launch<f16_t, 64>(dout, q, k, v, o, lse, dq, dk, dv, delta, BH, seq, group, scale, st);
}

extern "C" int eg_attn_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                           int64_t batch, int64_t heads, int64_t seq, int64_t head_dim,
                           float scale, int dtype, void* stream) {
  return eg_attn_gqa_fwd(q, k, v, o, lse, batch, heads, heads, seq, head_dim, scale, dtype, stream);
}

extern "C" int eg_attn_bwd(const void* dout, const void* q, const void* k, const void* v,
                           const void* o, const float* lse, void* dq, void* dk, void* dv,
                           void* workspace, int64_t batch, int64_t heads, int64_t seq,
                           int64_t head_dim, float scale, int dtype, void* stream) {
  return eg_attn_gqa_bwd(dout, q, k, v, o, lse, dq, dk, dv, workspace, batch, heads, heads, seq,
                         head_dim, scale, dtype, stream);
}

// ----------------------------------------- RoPE(q, k) -> grouped causal attention
// The attention half of the Llama-3 decoder layer
// (src/evograd/ops/level3/llama3_decoder_layer/forward_ref.py:93-107): q and k
// rotated by fp32 tables cos/sin [S, D], then causal GQA attention. The forward
// rotates k into the workspace (one small pass over the kv heads) and q in the
// attention kernel's registers as it loads them; the backward rotates q and k into
// the workspace again (the saved state holds the pre-rotation inputs only) and
// applies the rotation's transpose to dq and dk in the kernels' registers before
// the stores. Backward workspace: q_r [B, H, S, D], k_r [B, Hkv, S, D] (dtype),
// delta [B, H, S] fp32, in that order; the forward's holds only its k_r.
static size_t llama3_ws_qr(int64_t B, int64_t H, int64_t S, int64_t D) { return (size_t)(B * H * S * D) * 2; }
static size_t llama3_ws_kr(int64_t B, int64_t Hkv, int64_t S, int64_t D) { return (size_t)(B * Hkv * S * D) * 2; }

extern "C" size_t eg_llama3_attn_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads,
                                                 int64_t seq, int64_t head_dim) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || seq <= 0 || head_dim <= 0) return 0;
  return llama3_ws_qr(batch, heads, seq, head_dim) + llama3_ws_kr(batch, kv_heads, seq, head_dim) +
         attn_delta_bytes(batch * heads, seq) +
         attn_part_bytes(batch * kv_heads, heads / kv_heads, seq, head_dim);
}

template <typename F>
static int llama3_dispatch(int dtype, int64_t head_dim, F&& f) {
  if (dtype == EG_BF16)
    return head_dim == 128 ? f(bf16_t{}, std::integral_constant<int, 128>{})
                           : f(bf16_t{}, std::integral_constant<int, 64>{});
  return head_dim == 128 ? f(f16_t{}, std::integral_constant<int, 128>{})
                         : f(f16_t{}, std::integral_constant<int, 64>{});
}

extern "C" int eg_llama3_attn_fwd(const void* q, const void* k, const void* v, const float* cos,
                                  const float* sin, void* o, float* lse, void* workspace,
                                  int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq,
                                  int64_t head_dim, float scale, int dtype, void* stream) {
  static const char* name = "eg_llama3_attn_fwd";
  clear_error();
  if (check_attn(name, batch, heads, kv_heads, seq, head_dim, dtype, true)) return 1;
  if (batch == 0 || heads == 0 || seq == 0) return 0;
  if (!q || !k || !v || !cos || !sin || !o || !lse || !workspace) {
    set_error("%s: null pointer", name);
    return 1;
  }
  if (!attn_aligned({q, k, v, o, cos, sin, workspace})) {
    set_error("%s: tensors, tables and workspace must be 16-byte aligned", name);
    return 1;
  }
  hipStream_t st = as_stream(stream);
  void* k_r = workspace;
  if (int rc = rope_apply(nullptr, k, nullptr, k_r, cos, sin, batch, 0, kv_heads, seq, head_dim,
                          dtype, EG_F32, false, st))
    return rc;
  const int64_t BH = batch * heads;
  const int group = (int)(heads / kv_heads);
  return llama3_dispatch(dtype, head_dim, [&](auto tc, auto dc) {
    using T = decltype(tc);
    return attn_fwd_launch<T, decltype(dc)::value, true>(q, k_r, v, o, lse, BH, seq, group, scale,
                                                         st, cos, sin);
  });
}

extern "C" int eg_llama3_attn_bwd(const void* dout, const void* q, const void* k, const void* v,
                                  const void* o, const float* lse, const float* cos,
                                  const float* sin, void* dq, void* dk, void* dv, void* workspace,
                                  int64_t batch, int64_t heads, int64_t kv_heads, int64_t seq,
                                  int64_t head_dim, float scale, int dtype, void* stream) {
  static const char* name = "eg_llama3_attn_bwd";
  clear_error();
  if (check_attn(name, batch, heads, kv_heads, seq, head_dim, dtype, true)) return 1;
  if (batch == 0 || heads == 0 || seq == 0) return 0;
  if (!dout || !q || !k || !v || !o || !lse || !cos || !sin || !dq || !dk || !dv || !workspace) {
    set_error("%s: null pointer", name);
    return 1;
  }
  if (!attn_aligned({dout, q, k, v, o, cos, sin, dq, dk, dv, workspace})) {
    set_error("%s: tensors, tables and workspace must be 16-byte aligned", name);
    return 1;
  }
  hipStream_t st = as_stream(stream);
  char* ws = (char*)workspace;
  void* q_r = ws;
  void* k_r = ws + llama3_ws_qr(batch, heads, seq, head_dim);
  float* delta = (float*)((char*)k_r + llama3_ws_kr(batch, kv_heads, seq, head_dim));
  if (int rc = rope_apply(q, k, q_r, k_r, cos, sin, batch, heads, kv_heads, seq, head_dim, dtype,
                          EG_F32, false, st))
    return rc;
  const int64_t BH = batch * heads;
  const int group = (int)(heads / kv_heads);
  return llama3_dispatch(dtype, head_dim, [&](auto tc, auto dc) {
    using T = decltype(tc);
    return attn_bwd_launch<T, decltype(dc)::value, true>(dout, q_r, k_r, v, o, lse, dq, dk, dv,
                                                         delta, BH, seq, group, scale, st, cos,
                                                         sin);
  });
}
