// Causal grouped-query attention over packed sequences for the shapes the 16-bit MFMA
// kernels do not take: fp32 tensors, head sizes other than 64 and 128, and rows that 16-byte
// loads cannot read. The arithmetic is attn_generic_kernel.hpp's (fp32 MFMA, masked pairs
// left out of the sums even beside infinite or NaN values); here are the kernels that place
// its workgroups over sequences of any lengths (packed_seqs.hpp).
//
// A 16-row block is a workgroup of four waves. The dK/dV walk of a key block is cut where it
// is long against the work of the whole batch: into as many of at most `parts` pieces as
// keep each near 1 / 512 of it (two workgroups per CU) and two steps per wave, whose fp32
// slabs a last kernel adds in order. No atomics: every sum has a fixed order.
#include "attn_generic_kernel.hpp"
#include "packed_attention.hpp"

#include <algorithm>

namespace eg {
namespace {

constexpr int kRows = 16;
constexpr int64_t kMaxParts = 8;

// Pieces of a walk of `steps` steps, `total` of them in the batch.
__device__ __forceinline__ int walk_parts(float steps, float total, int most) {
  const float each = fmaxf(total * (1.f / 512.f), 2.f * kGenWaves);
  return min(most, max(1, (int)(steps / each + 0.999f)));
}

template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, 2) void packed_gen_fwd_kernel(PackedAttn a, int tiles,
                                                                        float scale_log2) {
  const int h = blockIdx.x % a.heads, rank = blockIdx.x / a.heads;
  T* os = (T*)a.o + h * a.head_dim;
  const int64_t ldo = (int64_t)a.heads * a.head_dim;
  SeqTile t;
  int spare;
  float walk;
  if (!find_tile<kRows, false>(a.seqs, rank, t, spare, walk)) {
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, os, ldo, a.head_dim);
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, a.lse + (int64_t)h * a.seqs.tokens, 1, 1);
    return;
  }
  const int kvh = h / (a.heads / a.kv_heads);
  attn_gen_fwd_rows<T, DM, VEC>((const T*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token,
                                (const T*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
                                (const T*)a.v + t.begin * a.v_token + kvh * a.v_head, a.v_token,
                                os + t.begin * ldo, ldo,
                                a.lse + (int64_t)h * a.seqs.tokens + t.begin, t.len, a.head_dim,
                                t.tile * kRows, scale_log2);
}

template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, DM > 64 ? 1 : 2) void packed_gen_dq_kernel(PackedAttn a,
                                                                                     int tiles) {
  const int h = blockIdx.x % a.heads, rank = blockIdx.x / a.heads;
  const int64_t ldo = (int64_t)a.heads * a.head_dim;
  T* dqs = (T*)a.dq + h * a.head_dim;
  SeqTile t;
  int spare;
  float walk;
  if (!find_tile<kRows, false>(a.seqs, rank, t, spare, walk)) {
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, dqs, ldo, a.head_dim);
    return;
  }
  const int kvh = h / (a.heads / a.kv_heads);
  const int64_t own = t.begin * ldo + h * a.head_dim;
  const int64_t row = (int64_t)h * a.seqs.tokens + t.begin;
  attn_gen_dq_rows<T, DM, VEC>((const T*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token,
                               (const T*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
                               (const T*)a.v + t.begin * a.v_token + kvh * a.v_head, a.v_token,
                               (const T*)a.dout + own, ldo, (const T*)a.o + own, ldo, a.lse + row,
                               a.delta + row, dqs + t.begin * ldo, ldo, t.len, a.head_dim,
                               t.tile * kRows, a.scale);
}

// Workgroup = 16 keys of one kv head, one piece of their walk; key blocks are counted from
// the end of their sequence, so the longest walks come first. Slabs: [most][tokens][kv_heads]
// [D] of dK, then of dV.
template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, DM > 64 ? 1 : 2) void packed_gen_dkdv_kernel(
    PackedAttn a, int tiles, int most) {
  __shared__ float buf[kGenWaves][16][DM + 4];
  const int u = blockIdx.x % (a.kv_heads * most), rank = blockIdx.x / (a.kv_heads * most);
  const int kvh = u % a.kv_heads, pi = u / a.kv_heads;
  const int group = a.heads / a.kv_heads, D = a.head_dim;
  const int64_t ldkv = (int64_t)a.kv_heads * D, ldo = (int64_t)a.heads * D;
  T *dks = (T*)a.dk + kvh * D, *dvs = (T*)a.dv + kvh * D;
  SeqTile t;
  int spare;
  float walk;
  if (!find_tile<kRows, true>(a.seqs, rank, t, spare, walk)) {
    if (pi != 0) return;
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, dks, ldkv, D);
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, dvs, ldkv, D);
    return;
  }
  const int parts = walk_parts((float)group * (t.tile + 1), walk * a.heads, most);
  if (pi >= parts) return;
  const int k0 = (t.tiles - 1 - t.tile) * kRows, h0 = kvh * group;
  const int64_t row = (int64_t)h0 * a.seqs.tokens + t.begin;
  f32x4 adk[DM / 16], adv[DM / 16];
  attn_gen_dkdv_keys<T, DM, VEC>(
      (const T*)a.q + t.begin * a.q_token + h0 * a.q_head, a.q_token, a.q_head,
      (const T*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
      (const T*)a.v + t.begin * a.v_token + kvh * a.v_head, a.v_token,
      (const T*)a.dout + t.begin * ldo + h0 * D, ldo, D, a.lse + row, a.delta + row,
      a.seqs.tokens, t.len, D, group, k0, parts, pi, a.scale, adk, adv);
  if (parts > 1) {
    const int64_t slab = a.seqs.tokens * ldkv, own = t.begin * ldkv + kvh * D;
    store_sum<float, DM>(buf, adk, a.part + pi * slab + own, ldkv, k0, t.len, D, a.scale);
    store_sum<float, DM>(buf, adv, a.part + (most + pi) * slab + own, ldkv, k0, t.len, D, 1.f);
  } else {
    store_sum<T, DM>(buf, adk, dks + t.begin * ldkv, ldkv, k0, t.len, D, a.scale);
    store_sum<T, DM>(buf, adv, dvs + t.begin * ldkv, ldkv, k0, t.len, D, 1.f);
  }
}

// dK and dV of the walks that were cut: their slabs in order, rounded once. Workgroup = the
// 16 keys of a dK/dV workgroup.
template <typename T>
__global__ __launch_bounds__(kGenThreads) void packed_gen_reduce_kernel(PackedAttn a, int most) {
  const int kvh = blockIdx.x % a.kv_heads, rank = blockIdx.x / a.kv_heads;
  SeqTile t;
  int spare;
  float walk;
  if (!find_tile<kRows, true>(a.seqs, rank, t, spare, walk)) return;
  const int parts = walk_parts((float)(a.heads / a.kv_heads) * (t.tile + 1), walk * a.heads, most);
  if (parts == 1) return;
  const int k0 = (t.tiles - 1 - t.tile) * kRows, n = min(kRows, t.len - k0), D = a.head_dim;
  const int64_t ldkv = (int64_t)a.kv_heads * D, slab = a.seqs.tokens * ldkv;
  for (int e = threadIdx.x; e < n * D; e += kGenThreads) {
    const int64_t at = (t.begin + k0 + e / D) * ldkv + kvh * D + e % D;
    float x = a.part[at], y = a.part[most * slab + at];
    for (int p = 1; p < parts; ++p) {
      x += a.part[p * slab + at];
      y += a.part[(most + p) * slab + at];
    }
    ((T*)a.dk)[at] = from_f32<T>(x);
    ((T*)a.dv)[at] = from_f32<T>(y);
  }
}

// The most pieces that a walk is cut into: what the workspace holds slabs for. None where
// the key blocks alone are two workgroups per CU and more.
int64_t most_parts(int64_t tokens, int64_t kv_heads) {
  const int64_t blocks = kv_heads * ((tokens + kRows - 1) / kRows);
  return std::max<int64_t>(1, std::min(kMaxParts, 2 * kGenTarget / blocks));
}

// Rows that can be read four columns at a time.
bool strides_vec(const PackedAttn& a) {
  for (int64_t s : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head})
    if (s % 4) return false;
  return true;
}

// gen_dispatch with the strides looked at too: an odd address takes the element loads.
template <typename F>
int dispatch(const PackedAttn& a, int dtype, bool backward, const char* name, F&& f) {
  const void* odd = strides_vec(a) ? nullptr : (const void*)1;
  const void *o = backward ? a.o : nullptr, *d = backward ? a.dout : nullptr;
  return gen_dispatch(dtype, a.head_dim, {a.q, a.k, a.v, o, d, odd}, name, std::forward<F>(f));
}

}  // namespace

size_t packed_generic_part_bytes(int64_t tokens, int64_t kv_heads, int64_t head_dim) {
  const int64_t most = most_parts(tokens, kv_heads);
  return most > 1 ? (size_t)2 * most * tokens * kv_heads * head_dim * sizeof(float) : 0;
}

int packed_generic_fwd(const PackedAttn& a, int dtype, hipStream_t st) {
  const int64_t tiles = packed_tiles(a.seqs.tokens, a.seqs.n, kRows);
  return dispatch(a, dtype, false, "eg_packed_attn_fwd", [&](auto tag, auto dm, auto vec) {
    EG_LAUNCH((packed_gen_fwd_kernel<decltype(tag), decltype(dm)::value, decltype(vec)::value>),
              dim3((unsigned)(tiles * a.heads)), dim3(kGenThreads), 0, st, a, (int)tiles,
              a.scale * kGenLog2e);
    return check_launch("eg_packed_attn_fwd(generic)");
  });
}

int packed_generic_bwd(const PackedAttn& a, int dtype, hipStream_t st) {
  const int64_t tiles = packed_tiles(a.seqs.tokens, a.seqs.n, kRows);
  const int most = (int)most_parts(a.seqs.tokens, a.kv_heads);
  return dispatch(a, dtype, true, "eg_packed_attn_bwd", [&](auto tag, auto dm, auto vec) {
    using T = decltype(tag);
    constexpr int DM = decltype(dm)::value;
    constexpr bool VEC = decltype(vec)::value;
    EG_LAUNCH((packed_gen_dq_kernel<T, DM, VEC>), dim3((unsigned)(tiles * a.heads)),
              dim3(kGenThreads), 0, st, a, (int)tiles);
    if (int e = check_launch("eg_packed_attn_bwd(generic dq)")) return e;
    EG_LAUNCH((packed_gen_dkdv_kernel<T, DM, VEC>), dim3((unsigned)(tiles * a.kv_heads * most)),
              dim3(kGenThreads), 0, st, a, (int)tiles, most);
    if (int e = check_launch("eg_packed_attn_bwd(generic dkdv)")) return e;
    if (most == 1) return 0;
    EG_LAUNCH((packed_gen_reduce_kernel<T>), dim3((unsigned)(tiles * a.kv_heads)),
              dim3(kGenThreads), 0, st, a, most);
    return check_launch("eg_packed_attn_bwd(generic dkdv reduce)");
  });
}

}  // namespace eg
