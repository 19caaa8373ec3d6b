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
//
// Rounding: scores, softmax statistics, dP and every sum are fp32. P and dS are rounded to the
// tensors' 16 bits before their products, which take both operands in one type (splitting
// dS into two parts would add two products to the backward's seven). delta is formed in fp32
// from a tile's own P and dP for a sequence's first 64 rows, whose keys are that tile, and from
// the stored o for the others. Of the norm of dq and dk that leaves, with standard normal
// inputs and 4 to 1000 tokens a sequence, 0.23 to 0.24% in bf16 where a single rounding of the
// result leaves 0.17% (0.030% and 0.021% in fp16), with o and dv between. Where scores are
// peaked (of a spread of 4), o's rounding in delta shows past the first 64 rows: 0.23% at 4 to 64
// tokens, 0.31% at 120, 0.37% at 1000 (0.030, 0.039 and 0.046% in fp16). Leaving it out there
// would take a fourth product in dQ (sum p k).
//
// What bounds it, kernel times at 32 query and 8 kv heads of 128, bf16 (forward + dQ + dK/dV):
// 32768 tokens in 7 sequences 2.46 + 3.47 + 5.39 ms, 1107, 1175 and 1011 TFLOP/s of the 4, 6
// and 8 D H pairs they execute, where a large matrix product reaches 1270: LDS operand
// traffic, as in attention.hip. 8192 tokens in 11 sequences (the longest of 3001) 0.14 + 0.19 +
// 0.28 ms, 2/3 of that rate: the longest sequence's last tiles take as long as an even share
// of the work. 4096 tokens in 160 prompts 40 + 54 + 57 us, 2.5 times the bytes' time: a
// workgroup's chain of loads, one or two tiles and the stores, of which two fit a CU.
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

// HW heads of a group share a workgroup, its keys and its values (attn_fwd_rows). Slot v ->
// first of them: the slots of a group have the same v % 8 when kv_heads is a multiple of
// 8, so they share an XCD's L2.
template <int HW>
__device__ __forceinline__ int slot_head(const PackedAttn& a, int v) {
  return (v % a.kv_heads) * (a.heads / a.kv_heads) + v / a.kv_heads * HW;
}

template <typename T, int D, int NW, int KG, int HW>
__global__ __launch_bounds__(NW * KG * 64, 2) void packed_fwd_kernel(PackedAttn a, int ranks,
                                                                     float scale_log2) {
  constexpr int ROWS = 32 * NW / HW;
  int slot, rank;
  packed_coords(a.heads / HW, slot, rank);
  const int h = slot_head<HW>(a, slot), kvh = h / (a.heads / a.kv_heads);
  const int64_t ldo = (int64_t)a.heads * D;
  uint16_t* o = (uint16_t*)a.o + h * D;
  float* lse = a.lse + (int64_t)h * a.seqs.tokens;
  SeqTile t;
  if (!find_tile<ROWS, false>(a.seqs, rank, t)) {
    zero_unused_rows(a.seqs, t, rank, ranks, (T*)o, ldo, HW * D);
#pragma unroll
    for (int i = 0; i < HW; ++i)
      zero_unused_rows(a.seqs, t, rank, ranks, lse + i * (int64_t)a.seqs.tokens, 1, 1);
    return;
  }
  attn_fwd_rows<T, D, NW, KG, HW, false, true>(
      (const uint16_t*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token, a.q_head,
      (const uint16_t*)a.k + t.begin * a.k_token + kvh * a.k_head, (int)a.k_token,
      (const uint16_t*)a.v + t.begin * a.v_token + kvh * a.v_head, (int)a.v_token,
      o + t.begin * ldo, ldo, D, lse + t.begin, a.seqs.tokens, t.len, scale_log2, t.tile * ROWS,
      nullptr, nullptr);
}

template <typename T, int D, int NW, int KG, int HW>
__global__ __launch_bounds__(NW * KG * 64, 2) void packed_dq_kernel(PackedAttn a, int ranks,
                                                                    float scale_log2) {
  constexpr int ROWS = 32 * NW / HW;
  int slot, rank;
  packed_coords(a.heads / HW, slot, rank);
  const int h = slot_head<HW>(a, slot), kvh = h / (a.heads / a.kv_heads);
  const int64_t ldo = (int64_t)a.heads * D;
  SeqTile t;
  if (!find_tile<ROWS, false>(a.seqs, rank, t)) {
    zero_unused_rows(a.seqs, t, rank, ranks, (T*)a.dq + h * D, ldo, HW * D);
    return;
  }
  const int64_t own = t.begin * ldo + h * D, row = (int64_t)h * a.seqs.tokens + t.begin;
  attn_dq_rows<T, D, NW, KG, HW, false, true>(
      (const uint16_t*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token, a.q_head,
      (const uint16_t*)a.k + t.begin * a.k_token + kvh * a.k_head, (int)a.k_token,
      (const uint16_t*)a.v + t.begin * a.v_token + kvh * a.v_head, (int)a.v_token,
      (const uint16_t*)a.dout + own, (const uint16_t*)a.o + own, (uint16_t*)a.dq + own, ldo, D,
      a.lse + row, a.delta + row, a.seqs.tokens, t.len, a.scale, scale_log2, t.tile * ROWS, nullptr,
      nullptr);
}

// A workgroup's rows or keys lie in one sequence, so where sequences are shorter than a block
// on the mean a narrower one leaves fewer waves without rows: key blocks of two waves instead of
// four, and at D = 64 row blocks of two for one or two heads a workgroup. Backward, four waves
// (with dQ's key groups, below 128 tokens) against two, bf16: 12 heads of 64, 160 prompts of 24
// tokens 90 / 40 us, 50 of 96 48 / 42, 40 of 128 46 / 41; 32 / 8 heads of 64, 100 of 48 73 / 61, 40
// of 128 the same; 32 / 8 heads of 128, 160 of 24 97 / 92, but 100 of 48 104 / 109 and 40 of 128
// 104 / 115. One limit lies between them.
constexpr int64_t kShort = 112;
inline bool short_seqs(int64_t tokens, int64_t seqs) { return tokens < kShort * seqs; }

// The dK/dV walk of a block of keys (32 a wave), cut where it is long against the work of the
// whole batch: each piece is at most 1 / kTarget of it (two workgroups per CU), but no
// shorter than kMinSteps steps of 32 rows, about what a piece's fp32 slab costs to write and
// read (4, 8 and 16 steps, backward: 12 heads of 64, 4 prompts of 256 tokens 31.7, 32.4 and 32.7
// us, 2 of 512 41.1, 39.9 and 43.1; 32 / 8 heads of 128 within 0.3%).
constexpr int kWalkRows = 32;
constexpr int64_t kTarget = 512, kMinSteps = 8;

struct WalkCut {
  int least;        // find_tile's arguments
  float share;
  int ranks, slabs;  // pieces of a kv head at most; those of them that belong to cut walks
  int waves;         // of 32 keys each
};
WalkCut walk_cut(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads) {
  WalkCut c;
  c.waves = short_seqs(tokens, seqs) ? 2 : 4;
  // Walks are not cut: a document among many prompts then has its first keys' walk as a tail (32
  // / 8 heads of 128, 301 sequences, one of 4096 of 7096 tokens, backward 1101 us, against 829
  // with 251; with one of 8192 of 12288 tokens 2754 and 2767).
  if (seqs > kSearchSeqs) {
    c.least = 1, c.share = 1.f, c.slabs = 0;
    c.ranks = (int)packed_tiles(tokens, seqs, 32 * c.waves);
    return c;
  }
  const int64_t per_tile = heads / kv_heads * (32 * c.waves / kWalkRows);
  c.least = (int)((kMinSteps + per_tile - 1) / per_tile);
  c.share = (float)kv_heads / kTarget;
  // a tile of index j makes at most 1 + j / m pieces, a cut one (j >= m) at most 2 j / m, and
  // the sum of j / m over a kv head's tiles is at most kTarget / kv_heads
  const int64_t more = (kTarget + kv_heads - 1) / kv_heads;
  c.ranks = (int)(packed_tiles(tokens, seqs, 32 * c.waves) + more);
  c.slabs = (int)std::min<int64_t>(c.ranks, 2 * more + 1);
  // no sequence has a tile of index `least`: nothing is cut
  if ((tokens + 32 * c.waves - 1) / (32 * c.waves) <= c.least) c.slabs = 0;
  return c;
}

// Key blocks are counted from the end of their sequence, so the longest walks come first, and
// the pieces of cut walks before the others: slab [kv head][rank][2][keys][D], dK then dV.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void packed_dkdv_kernel(PackedAttn a, WalkCut c,
                                                                 float scale_log2) {
  constexpr int kKeys = 32 * NW;
  int kvh, rank;
  packed_coords(a.kv_heads, kvh, rank);
  const int h0 = kvh * (a.heads / a.kv_heads);
  const int64_t ldkv = (int64_t)a.kv_heads * D, ldo = (int64_t)a.heads * D;
  uint16_t *dk = (uint16_t*)a.dk + kvh * D, *dv = (uint16_t*)a.dv + kvh * D;
  SeqTile t;
  if (!find_tile<kKeys, true>(a.seqs, rank, t, c.least, c.share)) {
    zero_unused_rows(a.seqs, t, rank, c.ranks, (T*)dk, ldkv, D);
    zero_unused_rows(a.seqs, t, rank, c.ranks, (T*)dv, ldkv, D);
    return;
  }
  const int k0 = (t.tiles - 1 - t.tile) * kKeys;
  float* part = nullptr;
  if (t.pieces > 1) {
    if (rank >= c.slabs) return;  // no batch's: the bound is walk_cut's
    part = a.part + ((int64_t)kvh * c.slabs + rank) * (2 * kKeys * D) - (int64_t)k0 * D;
  }
  const int64_t own = t.begin * ldkv, row = (int64_t)h0 * a.seqs.tokens + t.begin;
  attn_dkdv_keys<T, D, NW, kWalkRows, false, true>(
      (const uint16_t*)a.q + t.begin * a.q_token + h0 * a.q_head, (int)a.q_token, a.q_head,
      (const uint16_t*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
      (const uint16_t*)a.v + t.begin * a.v_token + kvh * a.v_head, (int)a.v_token,
      (const uint16_t*)a.dout + t.begin * ldo + h0 * D, (int)ldo, D, a.lse + row, a.delta + row,
      a.seqs.tokens, dk + own, dv + own, ldkv, t.len, a.scale, scale_log2, k0,
      a.heads / a.kv_heads, nullptr, nullptr, t.pieces, t.piece, part,
      part ? part + kKeys * D : nullptr, D);
}

// dK and dV of the walks that were cut: their slabs in order, rounded once. The workgroups of
// a walk's pieces share its keys.
template <typename T, int D, int NW>
__global__ __launch_bounds__(256) void packed_reduce_kernel(PackedAttn a, WalkCut c) {
  constexpr int kKeys = 32 * NW;
  int kvh, rank;
  packed_coords(a.kv_heads, kvh, rank);
  SeqTile t;
  if (!find_tile<kKeys, true>(a.seqs, rank, t, c.least, c.share)) return;
  const int head = rank - t.piece;  // the walk's first piece
  if (t.pieces == 1 || head < 0 || head + t.pieces > c.slabs) return;
  const int k0 = (t.tiles - 1 - t.tile) * kKeys, rows = min(kKeys, t.len - k0);
  const float* part = a.part + ((int64_t)kvh * c.slabs + head) * (2 * kKeys * D);
  const int64_t ldkv = (int64_t)a.kv_heads * D, first = (t.begin + k0) * ldkv + kvh * D;
  for (int e = t.piece * 256 + threadIdx.x; e < 2 * rows * (D / 4); e += 256 * t.pieces) {
    const int which = e >= rows * (D / 4), f = e - which * rows * (D / 4);
    const float* p = part + which * (kKeys * D) + f * 4;
    float4 x = *reinterpret_cast<const float4*>(p);
    for (int i = 1; i < t.pieces; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(p + i * (2 * kKeys * D));
      x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    uint2 u;
    u.x = MM<T>::pack2(x.x, x.y);
    u.y = MM<T>::pack2(x.z, x.w);
    *reinterpret_cast<uint2*>((uint16_t*)(which ? a.dv : a.dk) + first + f / (D / 4) * ldkv +
                              f % (D / 4) * 4) = u;
  }
}

size_t mfma_part_bytes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t D) {
  const WalkCut c = walk_cut(tokens, seqs, heads, kv_heads);
  return (size_t)kv_heads * c.slabs * 2 * (32 * c.waves) * D * 4;
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

// Two key groups per workgroup (KG = 2), which halve a row block's chain of key tiles: for few
// long walks. Forward, one group against two, bf16, 8 and 32 heads of 128, by the grid (blocks of
// 128 rows times heads): 128, one sequence of 2048 39 / 32 us; 256, one of 1024 25.6 / 23.2, 4 of
// 1024 30.0 / 25.5; 384, 2 of 768 28.5 / 28.0; 512, one of 2048 50 / 52. Below 512 tokens a sequence it
// costs more than it gives, most where the grid fills the CUs: 128, 4 of 128 10.8 / 12.3; 512, 4
// of 512 25 / 36, 16 of 128 22 / 30. The host knows the mean length alone, which does not tell such
// a batch from one long sequence among short ones (12 heads of 64, one of 1111 and 7 of 250 19.6 /
// 16.7, one of 1024 and 7 of 120 16.8 / 14.8), so both take it. dQ at D = 64, backward: 128, one of
// 2048 79 / 76; 256, 4 of 1024 67.6 / 65.0; 384, 2 of 768 65.5 / 67.5; 128, 4 of 128 38.3 / 39.8. dQ
// at D = 128 loses throughout (3 to 8 us).
template <int D, bool DQ>
inline bool split_keys(const PackedAttn& a) {
  if (DQ && D != 64) return false;
  const int64_t grid = ((int64_t)a.seqs.tokens + 127) / 128 * a.heads;
  return !short_seqs(a.seqs.tokens, a.seqs.n) && grid <= (DQ ? 384 : 512);
}

// Workgroups of the forward and dQ: f(HW, NW, KG).
// HW heads of a group share their keys and values: their waves walk the same keys, where the
// waves of one head's rows end one after the other, and short sequences fill a tile of 32
// rows where 128 of one head would be mostly empty.
template <int D, bool DQ, typename F>
int by_rows(const PackedAttn& a, F&& f) {
  const int group = a.heads / a.kv_heads;
  const bool split = split_keys<D, DQ>(a);
  auto go = [&](auto hw) -> int {
    constexpr int HW = decltype(hw)::value;
    if constexpr (!DQ || D == 64) {
      if (split) return f(hw, Int<4>{}, Int<2>{});
    }
    if constexpr (D == 64 && HW < 4) {
      if (short_seqs(a.seqs.tokens, a.seqs.n)) return f(hw, Int<2>{}, Int<1>{});
    }
    return f(hw, Int<4>{}, Int<1>{});
  };
  if (group % 4 == 0) return go(Int<4>{});
  if (group % 2 == 0) return go(Int<2>{});
  return go(Int<1>{});
}

int mfma_fwd(const PackedAttn& a, int dtype, hipStream_t st) {
  return by_type(a, dtype, [&](auto tc, auto dc) {
    using T = decltype(tc);
    constexpr int D = decltype(dc)::value;
    return by_rows<D, false>(a, [&](auto hw, auto nw, auto kg) {
      constexpr int HW = decltype(hw)::value, NW = decltype(nw)::value, KG = decltype(kg)::value;
      const int64_t ranks = packed_tiles(a.seqs.tokens, a.seqs.n, 32 * NW / HW);
      const int rows = 32 * NW / HW;
      PackedAttn b = a;
      if (check_grid("eg_packed_attn_fwd", ranks * (a.heads / HW), NW * KG * 64)) return 1;
      if (int e = packed_plan(a.seqs, 1, &rows, a.plan, &b.seqs, st)) return e;
      EG_LAUNCH((packed_fwd_kernel<T, D, NW, KG, HW>), dim3((unsigned)(ranks * (a.heads / HW))),
                dim3(NW * KG * 64), 0, st, b, (int)ranks, a.scale * kLog2e);
      return check_launch("eg_packed_attn_fwd");
    });
  });
}

int mfma_bwd(const PackedAttn& a, int dtype, hipStream_t st) {
  const WalkCut cut = walk_cut(a.seqs.tokens, a.seqs.n, a.heads, a.kv_heads);
  return by_type(a, dtype, [&](auto tc, auto dc) {
    using T = decltype(tc);
    constexpr int D = decltype(dc)::value;
    PackedAttn keys_of = a;
    const int rc = by_rows<D, true>(a, [&](auto hw, auto nw, auto kg) {
      constexpr int HW = decltype(hw)::value, NW = decltype(nw)::value, KG = decltype(kg)::value;
      const int64_t ranks = packed_tiles(a.seqs.tokens, a.seqs.n, 32 * NW / HW);
      const int rows[2] = {32 * NW / HW, 32 * cut.waves};
      PackedSeqs seqs[2];
      if (check_grid("eg_packed_attn_bwd", ranks * (a.heads / HW), NW * KG * 64) ||
          check_grid("eg_packed_attn_bwd", (int64_t)cut.ranks * a.kv_heads, cut.waves * 64))
        return 1;
      if (int e = packed_plan(a.seqs, 2, rows, a.plan, seqs, st)) return e;
      PackedAttn b = a;
      b.seqs = seqs[0];
      keys_of.seqs = seqs[1];
      EG_LAUNCH((packed_dq_kernel<T, D, NW, KG, HW>), dim3((unsigned)(ranks * (a.heads / HW))),
                dim3(NW * KG * 64), 0, st, b, (int)ranks, a.scale * kLog2e);
      return check_launch("eg_packed_attn_bwd(dq)");
    });
    if (rc) return rc;
    auto keys = [&](auto nwc) {
      constexpr int NW = decltype(nwc)::value;
      EG_LAUNCH((packed_dkdv_kernel<T, D, NW>), dim3((unsigned)(cut.ranks * a.kv_heads)),
                dim3(NW * 64), 0, st, keys_of, cut, a.scale * kLog2e);
      if (int e = check_launch("eg_packed_attn_bwd(dkdv)")) return e;
      if (cut.slabs == 0) return 0;
      EG_LAUNCH((packed_reduce_kernel<T, D, NW>), dim3((unsigned)(cut.slabs * a.kv_heads)),
                dim3(256), 0, st, keys_of, cut);
      return check_launch("eg_packed_attn_bwd(dkdv reduce)");
    };
    return cut.waves == 2 ? keys(Int<2>{}) : keys(Int<4>{});
  });
}

// One workgroup per table. Sequences go into classes by the bits of their tile count, the
// largest class first; where a sequence stands inside its class is left to the order in which
// the atomics come and moves no result, only which workgroup finds it.
constexpr int kPlanThreads = 1024, kClasses = 32;
struct PlanJob {
  int rows[2];
  int* table[2];
};
__global__ __launch_bounds__(kPlanThreads) void packed_plan_kernel(PackedSeqs p, PlanJob job) {
  __shared__ int at[kClasses], sums[kPlanThreads / 64];
  const int rows = job.rows[blockIdx.x], tid = threadIdx.x, lane = tid & 63;
  int *order = job.table[blockIdx.x], *start = order + p.n;
  auto tiles = [&](int s) {
    int b, len;
    seq_bounds(p, s, b, len);
    return (int)(((unsigned)len + rows - 1) / rows);
  };
  auto size_class = [](int nt) { return nt ? 32 - __builtin_clz(nt) : 0; };
  if (tid < kClasses) at[tid] = 0;
  __syncthreads();
  for (int s = tid; s < p.n; s += kPlanThreads) atomicAdd(&at[size_class(tiles(s))], 1);
  __syncthreads();
  if (tid == 0) {
    int before = 0;
    for (int c = kClasses - 1; c >= 0; --c) {
      const int n = at[c];
      at[c] = before;
      before += n;
    }
  }
  __syncthreads();
  for (int s = tid; s < p.n; s += kPlanThreads) order[atomicAdd(&at[size_class(tiles(s))], 1)] = s;
  __syncthreads();
  // running count of tiles: a run of slots per thread
  const int run = (p.n + kPlanThreads - 1) / kPlanThreads;
  const int first = min(p.n, tid * run), last = min(p.n, first + run);
  int mine = 0;
  for (int i = first; i < last; ++i) mine += tiles(order[i]);
  int upto = mine;  // inclusive over the wave
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const int x = __shfl_up(upto, off, 64);
    if (lane >= off) upto += x;
  }
  if (lane == 63) sums[tid >> 6] = upto;
  __syncthreads();
  int count = upto - mine;
  for (int w = 0; w < (tid >> 6); ++w) count += sums[w];
  for (int i = first; i < last; ++i) {
    start[i] = count;
    count += tiles(order[i]);
  }
  if (tid == kPlanThreads - 1) start[p.n] = count;
}

}  // namespace

int packed_plan(const PackedSeqs& seqs, int tables, const int* rows, void* const* table,
                PackedSeqs* out, hipStream_t st) {
  PlanJob job = {};
  for (int i = 0; i < tables; ++i) {
    out[i] = seqs;
    if (seqs.n <= kSearchSeqs) continue;
    job.rows[i] = rows[i];
    job.table[i] = (int*)table[i];
    out[i].order = job.table[i];
    out[i].start = job.table[i] + seqs.n;
  }
  if (seqs.n <= kSearchSeqs) return 0;
  EG_LAUNCH(packed_plan_kernel, dim3((unsigned)tables), dim3(kPlanThreads), 0, st, seqs, job);
  return check_launch("eg_packed_attn(plan)");
}

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
  if (heads == 0 || kv_heads <= 0 || heads % kv_heads != 0) {
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
  // tiles of 16 rows (and pieces of walks) times heads index one grid
  if (tokens > kMaxTokens || seqs > kMaxSeqs || heads > 4096 ||
      packed_tiles(tokens, seqs, 16) * heads > ((int64_t)1 << 30)) {
    set_error("%s: size out of range (tokens <= 268435456, sequences <= 16777216, heads <= 4096, "
              "(tokens / 16 + sequences) * heads < 2^30)", name);
    return 1;
  }
  return 0;
}

PackedAttn describe(const void* q, const void* k, const void* v, const int* cu, int64_t tokens,
                    int64_t seqs, int64_t heads, int64_t kv_heads, int64_t D,
                    const int64_t* strides, float scale) {
  PackedAttn a = {};
  a.seqs = {cu, (int)seqs, (int)tokens, nullptr, nullptr};
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
  if (tokens <= 0 || seqs < 0 || heads <= 0 || kv_heads <= 0 || heads < kv_heads || head_dim <= 0)
    return 0;
  const size_t generic = packed_generic_part_bytes(tokens, seqs, heads, kv_heads, head_dim);
  // rows of any alignment may come: the larger of the two where both kernels may run
  return delta_bytes(tokens, heads) + 2 * plan_bytes(seqs) +
         (mfma_sizes(head_dim, dtype) ? std::max(generic,
                                               mfma_part_bytes(tokens, seqs, heads, kv_heads, head_dim))
                                      : generic);
}

extern "C" size_t eg_packed_attn_fwd_workspace_bytes(int64_t seqs) {
  return seqs > 0 ? plan_bytes(seqs) : 0;
}

extern "C" int eg_packed_attn_fwd(const void* q, const void* k, const void* v, const int* cu_seqlens,
                                  void* o, float* lse, void* workspace, int64_t tokens,
                                  int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  const int64_t* strides, float scale, int dtype, void* stream) {
  static const char* name = "eg_packed_attn_fwd";
  clear_error();
  if (!strides) { set_error("%s: null strides", name); return 1; }
  PackedAttn a = describe(q, k, v, cu_seqlens, tokens, seqs, heads, kv_heads, head_dim, strides,
                          scale);
  if (check_packed(name, a, tokens, seqs, heads, kv_heads, head_dim, dtype)) return 1;
  if (tokens == 0) return 0;
  if (!q || !k || !v || !cu_seqlens || !o || !lse || (plan_bytes(seqs) && !workspace)) {
    set_error("%s: null pointer", name);
    return 1;
  }
  a.o = o, a.lse = lse;
  a.plan[0] = workspace;
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
  if (tokens == 0) return 0;
  if (!dout || !q || !k || !v || !cu_seqlens || !o || !lse || !dq || !dk || !dv || !workspace) {
    set_error("%s: null pointer", name);
    return 1;
  }
  if (!aligned16(workspace)) { set_error("%s: workspace must be 16-byte aligned", name); return 1; }
  a.o = const_cast<void*>(o), a.lse = const_cast<float*>(lse);
  a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  char* ws = (char*)workspace;
  a.delta = (float*)ws;
  a.plan[0] = ws += delta_bytes(tokens, heads);
  a.plan[1] = ws += plan_bytes(seqs);
  a.part = (float*)(ws + plan_bytes(seqs));
  if (mfma_sizes(head_dim, dtype) && mfma_rows(a)) return mfma_bwd(a, dtype, as_stream(stream));
  return packed_generic_bwd(a, dtype, as_stream(stream));
}
