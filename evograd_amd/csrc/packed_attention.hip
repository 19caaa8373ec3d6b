// Causal grouped-query attention over packed sequences: the entry points.
//
//   o_i = sum over j <= i of i's sequence of p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i)
//   delta_i = do_i o_i,  dS_ij = p_ij (do_i v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i p_ij do_i
// with query head h reading kv head h / (heads / kv_heads), dk and dv summed over the group.
//
// 16-bit tensors of head size 64 or 128 run attention_kernel.hpp's MFMA workgroups (the
// arithmetic is described in attention.hip), everything else packed_attn_generic.hip. Where
// the workgroups of [B, H, S, D] tensors know their rows from their index, those here find
// their sequence and tile themselves (packed_seqs.hpp), longest walks first, and where a
// masked pair meets an infinite or NaN value the sums are done again without it.
#include "attention_kernel.hpp"
#include "packed_attention.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

// Workgroup -> (head slot, rank): with a multiple of 8 slots every workgroup of a slot runs
// on one XCD, whose L2 its keys and values stay in; other counts are dealt out evenly.
__device__ __forceinline__ void packed_coords(int slots, int& slot, int& rank) {
  const int i = blockIdx.x;
  if (slots % 8 == 0) {
    const int rest = i / 8, per = slots / 8;
    slot = i % 8 + 8 * (rest % per);
    rank = rest / per;
  } else {
    slot = i % slots;
    rank = i / slots;
  }
}

// Slot v -> query head: the heads of a group have the same v % 8 when kv_heads is a
// multiple of 8, so they share an XCD's L2.
__device__ __forceinline__ int slot_head(const PackedAttn& a, int v) {
  return (v % a.kv_heads) * (a.heads / a.kv_heads) + v / a.kv_heads;
}

template <typename T, int D, int NW, int KG>
__global__ __launch_bounds__(NW * KG * 64, 2) void packed_fwd_kernel(PackedAttn a, int tiles,
                                                                     float scale_log2) {
  int slot, rank, spare;
  packed_coords(a.heads, slot, rank);
  const int h = slot_head(a, slot), kvh = h / (a.heads / a.kv_heads);
  const int64_t ldo = (int64_t)a.heads * D;
  uint16_t* o = (uint16_t*)a.o + h * D;
  float* lse = a.lse + (int64_t)h * a.seqs.tokens;
  SeqTile t;
  float walk;
  if (!find_tile<32 * NW, false>(a.seqs, rank, t, spare, walk)) {
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, (T*)o, ldo, D);
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, lse, 1, 1);
    return;
  }
  attn_fwd_rows<T, D, NW, KG, false, true>(
      (const uint16_t*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token,
      (const uint16_t*)a.k + t.begin * a.k_token + kvh * a.k_head, (int)a.k_token,
      (const uint16_t*)a.v + t.begin * a.v_token + kvh * a.v_head, (int)a.v_token,
      o + t.begin * ldo, ldo, lse + t.begin, t.len, scale_log2, t.tile * 32 * NW, nullptr, nullptr);
}

template <typename T, int D, int NW, int KG>
__global__ __launch_bounds__(NW * KG * 64, 2) void packed_dq_kernel(PackedAttn a, int tiles,
                                                                    float scale_log2) {
  int slot, rank, spare;
  packed_coords(a.heads, slot, rank);
  const int h = slot_head(a, slot), kvh = h / (a.heads / a.kv_heads);
  const int64_t ldo = (int64_t)a.heads * D;
  uint16_t* dq = (uint16_t*)a.dq + h * D;
  SeqTile t;
  float walk;
  if (!find_tile<32 * NW, false>(a.seqs, rank, t, spare, walk)) {
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, (T*)dq, ldo, D);
    return;
  }
  const int64_t own = t.begin * ldo + h * D, row = (int64_t)h * a.seqs.tokens + t.begin;
  attn_dq_rows<T, D, NW, KG, false, true>(
      (const uint16_t*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token,
      (const uint16_t*)a.k + t.begin * a.k_token + kvh * a.k_head, (int)a.k_token,
      (const uint16_t*)a.v + t.begin * a.v_token + kvh * a.v_head, (int)a.v_token,
      (const uint16_t*)a.dout + own, ldo, (const uint16_t*)a.o + own, ldo, a.lse + row,
      a.delta + row, dq + t.begin * ldo, ldo, t.len, a.scale, scale_log2, t.tile * 32 * NW,
      nullptr, nullptr);
}

// The dK/dV walk of a block of 128 keys, cut where it is long against the work of the whole
// batch: into as many of at most `most` pieces as keep each near 1 / 512 of it (two
// workgroups per CU), but no shorter than kMinSteps steps of 32 rows, about what a piece's
// fp32 slabs cost to write and read.
constexpr int kKeyWaves = 4, kKeys = 32 * kKeyWaves, kWalkRows = 32;
constexpr float kMinSteps = 16.f;
__device__ __forceinline__ int mfma_parts(const PackedAttn& a, const SeqTile& t, float walk,
                                          int most) {
  const float per_tile = (float)(a.heads / a.kv_heads) * (kKeys / kWalkRows);
  const float each = fmaxf(walk * per_tile * a.kv_heads * (1.f / 512.f), kMinSteps);
  return min(most, max(1, (int)(per_tile * (t.tile + 1) / each + 0.999f)));
}

// Key blocks are counted from the end of their sequence, so the longest walks come first.
// Slabs: [most][tokens][kv_heads][D] fp32 of dK, then of dV.
template <typename T, int D>
__global__ __launch_bounds__(kKeyWaves * 64, 2) void packed_dkdv_kernel(PackedAttn a, int tiles,
                                                                        int most,
                                                                        float scale_log2) {
  int slot, rank, spare;
  packed_coords(a.kv_heads * most, slot, rank);
  const int kvh = slot % a.kv_heads, pi = slot / a.kv_heads;
  const int group = a.heads / a.kv_heads, h0 = kvh * group;
  const int64_t ldkv = (int64_t)a.kv_heads * D, ldo = (int64_t)a.heads * D;
  uint16_t *dk = (uint16_t*)a.dk + kvh * D, *dv = (uint16_t*)a.dv + kvh * D;
  SeqTile t;
  float walk;
  if (!find_tile<kKeys, true>(a.seqs, rank, t, spare, walk)) {
    if (pi != 0) return;
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, (T*)dk, ldkv, D);
    zero_unused_rows(a.seqs, spare, tiles - rank + spare, (T*)dv, ldkv, D);
    return;
  }
  const int parts = mfma_parts(a, t, walk, most);
  if (pi >= parts) return;
  const int64_t own = t.begin * ldkv, slab = a.seqs.tokens * ldkv;
  const int64_t row = (int64_t)h0 * a.seqs.tokens + t.begin;
  float* part = parts > 1 ? a.part + pi * slab + own + kvh * D : nullptr;
  attn_dkdv_keys<T, D, kKeyWaves, kWalkRows, false, true>(
      (const uint16_t*)a.q + t.begin * a.q_token + h0 * a.q_head, (int)a.q_token, a.q_head,
      (const uint16_t*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
      (const uint16_t*)a.v + t.begin * a.v_token + kvh * a.v_head, (int)a.v_token,
      (const uint16_t*)a.dout + t.begin * ldo + h0 * D, (int)ldo, D, a.lse + row, a.delta + row,
      a.seqs.tokens, dk + own, dv + own, ldkv, t.len, a.scale, scale_log2,
      (t.tiles - 1 - t.tile) * kKeys, group, nullptr, nullptr, parts, pi, part,
      part ? part + most * slab : nullptr);
}

// dK and dV of the walks that were cut: their slabs in order, rounded once. Workgroup = the
// 128 keys of a dK/dV workgroup.
template <typename T, int D>
__global__ __launch_bounds__(256) void packed_reduce_kernel(PackedAttn a, int most) {
  int kvh, rank, spare;
  packed_coords(a.kv_heads, kvh, rank);
  SeqTile t;
  float walk;
  if (!find_tile<kKeys, true>(a.seqs, rank, t, spare, walk)) return;
  const int parts = mfma_parts(a, t, walk, most);
  if (parts == 1) return;
  const int k0 = (t.tiles - 1 - t.tile) * kKeys, rows = min(kKeys, t.len - k0);
  const int64_t ldkv = (int64_t)a.kv_heads * D, slab = a.seqs.tokens * ldkv;
  for (int e = threadIdx.x; e < rows * (D / 4); e += 256) {
    const int64_t at = (t.begin + k0 + e / (D / 4)) * ldkv + kvh * D + e % (D / 4) * 4;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float* p = a.part + which * most * slab + at;
      float4 x = *reinterpret_cast<const float4*>(p);
      for (int i = 1; i < parts; ++i) {
        const float4 y = *reinterpret_cast<const float4*>(p + i * slab);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
      uint2 u;
      u.x = MM<T>::pack2(x.x, x.y);
      u.y = MM<T>::pack2(x.z, x.w);
      *reinterpret_cast<uint2*>((uint16_t*)(which ? a.dv : a.dk) + at) = u;
    }
  }
}

// The most pieces a walk is cut into, what the workspace holds slabs for: none where the
// key blocks alone fill the chip several times over.
int64_t most_parts(int64_t tokens, int64_t kv_heads) {
  const int64_t blocks = kv_heads * ((tokens + kKeys - 1) / kKeys);
  return std::max<int64_t>(1, std::min<int64_t>(8, (2048 + blocks - 1) / blocks));
}

size_t mfma_part_bytes(int64_t tokens, int64_t kv_heads, int64_t D) {
  const int64_t most = most_parts(tokens, kv_heads);
  return most > 1 ? (size_t)2 * most * tokens * kv_heads * D * 4 : 0;
}

bool mfma_sizes(int64_t D, int dtype) {
  return (D == 64 || D == 128) && (dtype == EG_BF16 || dtype == EG_F16);
}

// Rows that 16-byte loads can read and that do not overlap (a tile's loads are bounded by its
// last row's end); others take the generic kernels.
bool mfma_rows(const PackedAttn& a) {
  for (int64_t s : {a.q_token, a.k_token, a.v_token})
    if (s < a.head_dim) return false;
  for (int64_t s : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head})
    if (s % 8) return false;
  for (const void* p : {a.q, a.k, a.v, (const void*)a.o, a.dout, (const void*)a.dq,
                        (const void*)a.dk, (const void*)a.dv})
    if (!aligned16(p)) return false;
  return true;
}

template <int N> using Int = std::integral_constant<int, N>;

template <typename F>
int by_type(const PackedAttn& a, int dtype, F&& f) {
  if (dtype == EG_BF16)
    return a.head_dim == 128 ? f(bf16_t{}, Int<128>{}) : f(bf16_t{}, Int<64>{});
  return a.head_dim == 128 ? f(f16_t{}, Int<128>{}) : f(f16_t{}, Int<64>{});
}

int mfma_fwd(const PackedAttn& a, int dtype, hipStream_t st) {
  return by_type(a, dtype, [&](auto tc, auto dc) {
    using T = decltype(tc);
    constexpr int D = decltype(dc)::value;
    auto go = [&](auto nwc, auto kgc) {
      constexpr int NW = decltype(nwc)::value, KG = decltype(kgc)::value;
      const int64_t tiles = packed_tiles(a.seqs.tokens, a.seqs.n, 32 * NW);
      EG_LAUNCH((packed_fwd_kernel<T, D, NW, KG>), dim3((unsigned)(tiles * a.heads)),
                dim3(NW * KG * 64), 0, st, a, (int)tiles, a.scale * kLog2e);
      return check_launch("eg_packed_attn_fwd");
    };
    return go(Int<4>{}, Int<1>{});
  });
}

int mfma_bwd(const PackedAttn& a, int dtype, hipStream_t st) {
  const int64_t tiles = packed_tiles(a.seqs.tokens, a.seqs.n, kKeys);
  const int most = (int)most_parts(a.seqs.tokens, a.kv_heads);
  return by_type(a, dtype, [&](auto tc, auto dc) {
    using T = decltype(tc);
    constexpr int D = decltype(dc)::value;
    EG_LAUNCH((packed_dq_kernel<T, D, 4, 1>), dim3((unsigned)(tiles * a.heads)), dim3(256), 0, st,
              a, (int)tiles, a.scale * kLog2e);
    if (int e = check_launch("eg_packed_attn_bwd(dq)")) return e;
    EG_LAUNCH((packed_dkdv_kernel<T, D>), dim3((unsigned)(tiles * a.kv_heads * most)),
              dim3(kKeyWaves * 64), 0, st, a, (int)tiles, most, a.scale * kLog2e);
    if (int e = check_launch("eg_packed_attn_bwd(dkdv)")) return e;
    if (most == 1) return 0;
    EG_LAUNCH((packed_reduce_kernel<T, D>), dim3((unsigned)(tiles * a.kv_heads)), dim3(256), 0, st,
              a, most);
    return check_launch("eg_packed_attn_bwd(dkdv reduce)");
  });
}

}  // namespace
}  // namespace eg

using namespace eg;

namespace {

constexpr int64_t kMaxTokens = (int64_t)1 << 28, kMaxSeqs = (int64_t)1 << 24;

size_t delta_bytes(int64_t tokens, int64_t heads) {
  return ((size_t)(tokens * heads) * 4 + 255) / 256 * 256;
}

int check_packed(const char* name, const PackedAttn& a, int64_t tokens, int64_t seqs,
                 int64_t heads, int64_t kv_heads, int64_t D, int dtype) {
  if (tokens < 0 || seqs < 0 || heads < 0) { set_error("%s: negative size", name); return 1; }
  if (heads > 0 && (kv_heads <= 0 || heads % kv_heads != 0)) {
    set_error("%s: heads (%lld) must be a positive multiple of kv_heads (%lld)", name,
              (long long)heads, (long long)kv_heads);
    return 1;
  }
  if (D < 2 || D > 128 || D % 2) {
    set_error("%s: head_dim must be even and at most 128, got %lld", name, (long long)D);
    return 1;
  }
  if (dtype != EG_BF16 && dtype != EG_F16 && dtype != EG_F32) {
    set_error("%s: dtype must be fp32, bf16 or fp16", name);
    return 1;
  }
  // a tile's rows are addressed with 32-bit offsets, its head and first row with 64
  auto in = [](int64_t s, int64_t most) { return s >= 0 && s <= most; };
  for (int64_t s : {a.q_token, a.k_token, a.v_token})
    if (!in(s, (int64_t)1 << 22)) {
      set_error("%s: token strides must be at least 0 and at most 4194304 elements", name);
      return 1;
    }
  for (int64_t s : {a.q_head, a.k_head, a.v_head})
    if (!in(s, (int64_t)1 << 40)) {
      set_error("%s: head strides must be at least 0 and at most 2^40 elements", name);
      return 1;
    }
  // tiles of 16 rows times heads and walk pieces index one grid
  if (tokens > kMaxTokens || seqs > kMaxSeqs || heads > 4096 ||
      packed_tiles(tokens, seqs, 16) * heads * 8 > 0x7fffffffLL) {
    set_error("%s: size out of range (tokens <= 268435456, sequences <= 16777216, heads <= 4096, "
              "(tokens / 16 + sequences) * heads < 2^28)", name);
    return 1;
  }
  return 0;
}

PackedAttn describe(const void* q, const void* k, const void* v, const int* cu, int64_t tokens,
                    int64_t seqs, int64_t heads, int64_t kv_heads, int64_t D,
                    const int64_t* strides, float scale) {
  PackedAttn a = {};
  a.seqs = {cu, (int)seqs, (int)tokens};
  a.q = q, a.k = k, a.v = v;
  a.q_token = strides[0], a.q_head = strides[1];
  a.k_token = strides[2], a.k_head = strides[3];
  a.v_token = strides[4], a.v_head = strides[5];
  a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.head_dim = (int)D;
  a.scale = scale;
  return a;
}

}  // namespace

extern "C" size_t eg_packed_attn_workspace_bytes(int64_t tokens, int64_t seqs, int64_t heads,
                                                 int64_t kv_heads, int64_t head_dim, int dtype) {
  if (tokens <= 0 || seqs < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
  const size_t generic = packed_generic_part_bytes(tokens, kv_heads, head_dim);
  // rows of any alignment may come: the larger of the two where both kernels may run
  return delta_bytes(tokens, heads) +
         (mfma_sizes(head_dim, dtype) ? std::max(generic, mfma_part_bytes(tokens, kv_heads, head_dim))
                                      : generic);
}

extern "C" int eg_packed_attn_fwd(const void* q, const void* k, const void* v, const int* cu_seqlens,
                                  void* o, float* lse, int64_t tokens, int64_t seqs, int64_t heads,
                                  int64_t kv_heads, int64_t head_dim, const int64_t* strides,
                                  float scale, int dtype, void* stream) {
  static const char* name = "eg_packed_attn_fwd";
  clear_error();
  if (!strides) { set_error("%s: null strides", name); return 1; }
  PackedAttn a = describe(q, k, v, cu_seqlens, tokens, seqs, heads, kv_heads, head_dim, strides,
                          scale);
  if (check_packed(name, a, tokens, seqs, heads, kv_heads, head_dim, dtype)) return 1;
  if (tokens == 0 || heads == 0) return 0;
  if (!q || !k || !v || !cu_seqlens || !o || !lse) { set_error("%s: null pointer", name); return 1; }
  a.o = o, a.lse = lse;
  if (mfma_sizes(head_dim, dtype) && mfma_rows(a)) return mfma_fwd(a, dtype, as_stream(stream));
  return packed_generic_fwd(a, dtype, as_stream(stream));
}

extern "C" int eg_packed_attn_bwd(const void* dout, const void* q, const void* k, const void* v,
                                  const int* cu_seqlens, const void* o, const float* lse, void* dq,
                                  void* dk, void* dv, void* workspace, int64_t tokens, int64_t seqs,
                                  int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  const int64_t* strides, float scale, int dtype, void* stream) {
  static const char* name = "eg_packed_attn_bwd";
  clear_error();
  if (!strides) { set_error("%s: null strides", name); return 1; }
  PackedAttn a = describe(q, k, v, cu_seqlens, tokens, seqs, heads, kv_heads, head_dim, strides,
                          scale);
  if (check_packed(name, a, tokens, seqs, heads, kv_heads, head_dim, dtype)) return 1;
  if (tokens == 0 || heads == 0) return 0;
  if (!dout || !q || !k || !v || !cu_seqlens || !o || !lse || !dq || !dk || !dv || !workspace) {
    set_error("%s: null pointer", name);
    return 1;
  }
  a.o = const_cast<void*>(o), a.lse = const_cast<float*>(lse);
  a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + delta_bytes(tokens, heads));
  if (mfma_sizes(head_dim, dtype) && mfma_rows(a)) return mfma_bwd(a, dtype, as_stream(stream));
  return packed_generic_bwd(a, dtype, as_stream(stream));
}
