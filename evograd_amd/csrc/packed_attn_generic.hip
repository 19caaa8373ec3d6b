// Causal grouped-query attention over packed sequences for the shapes the 16-bit MFMA
// kernels do not take: fp32 tensors, head sizes other than 64 and 128, and rows that 16-byte
// loads cannot read. The arithmetic is attn_generic_kernel.hpp's (fp32 MFMA, masked pairs
// left out of the sums even beside infinite or NaN values); here are the kernels that place
// its workgroups over sequences of any lengths (packed_seqs.hpp).
//
// A 16-row block is a workgroup of four waves. The dK/dV walk of a key block is cut where it
// is long against the work of the whole batch: each piece is at most 1 / kGenTarget of it (two
// workgroups per CU), but no shorter than eight steps per wave; a last kernel adds the pieces'
// fp32 slabs in order. No atomics: every sum has a fixed order.
#include "attn_generic_kernel.hpp"
#include "packed_attention.hpp"

#include <algorithm>

namespace eg {
namespace {

constexpr int kRows = 16;

struct WalkCut {
  int least;         // find_tile's arguments
  float share;
  int ranks, slabs;  // pieces of a kv head at most; those of them that belong to cut walks
};
WalkCut walk_cut(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads) {
  const int64_t group = heads / kv_heads, steps = 8 * kGenWaves;
  WalkCut c;
  // walks are not cut (8 / 2 heads of 64, fp32, one sequence of 2048 of 3548 tokens, backward: 301
  // sequences 379 us, 251 305)
  if (seqs > kSearchSeqs) {
    c.least = 1, c.share = 1.f, c.slabs = 0;
    c.ranks = (int)packed_tiles(tokens, seqs, kRows);
    return c;
  }
  c.least = (int)((steps + group - 1) / group);
  c.share = (float)kv_heads / kGenTarget;
  // a tile of index j makes at most 1 + j / m pieces, a cut one (j >= m) at most 2 j / m, and
  // the sum of j / m over a kv head's tiles is at most kGenTarget / kv_heads
  const int64_t more = (kGenTarget + kv_heads - 1) / kv_heads;
  c.ranks = (int)(packed_tiles(tokens, seqs, kRows) + more);
  c.slabs = (int)std::min<int64_t>(c.ranks, 2 * more + 1);
  // no sequence has a tile of index `least`: nothing is cut
  if ((tokens + kRows - 1) / kRows <= c.least) c.slabs = 0;
  return c;
}

template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, 2) void packed_gen_fwd_kernel(PackedAttn a, int ranks,
                                                                        float scale_log2) {
  const int h = blockIdx.x % a.heads, rank = blockIdx.x / a.heads;
  T* os = (T*)a.o + h * a.head_dim;
  float* lse = a.lse + (int64_t)h * a.seqs.tokens;
  const int64_t ldo = (int64_t)a.heads * a.head_dim;
  SeqTile t;
  if (!find_tile<kRows, false>(a.seqs, rank, t)) {
    zero_unused_rows(a.seqs, t, rank, ranks, os, ldo, a.head_dim);
    zero_unused_rows(a.seqs, t, rank, ranks, lse, 1, 1);
    return;
  }
  const int kvh = h / (a.heads / a.kv_heads);
  attn_gen_fwd_rows<T, DM, VEC>((const T*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token,
                                (const T*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
                                (const T*)a.v + t.begin * a.v_token + kvh * a.v_head, a.v_token,
                                os + t.begin * ldo, ldo, lse + t.begin, t.len, a.head_dim,
                                t.tile * kRows, scale_log2);
}

template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, DM > 64 ? 1 : 2) void packed_gen_dq_kernel(PackedAttn a,
                                                                                     int ranks) {
  const int h = blockIdx.x % a.heads, rank = blockIdx.x / a.heads;
  const int64_t ldo = (int64_t)a.heads * a.head_dim;
  T* dqs = (T*)a.dq + h * a.head_dim;
  SeqTile t;
  if (!find_tile<kRows, false>(a.seqs, rank, t)) {
    zero_unused_rows(a.seqs, t, rank, ranks, dqs, ldo, a.head_dim);
    return;
  }
  const int kvh = h / (a.heads / a.kv_heads);
  const int64_t own = t.begin * ldo + h * a.head_dim;
  const int64_t row = (int64_t)h * a.seqs.tokens + t.begin;
  attn_gen_dq_rows<T, DM, VEC, true>(
      (const T*)a.q + t.begin * a.q_token + h * a.q_head, a.q_token,
      (const T*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
      (const T*)a.v + t.begin * a.v_token + kvh * a.v_head, a.v_token, (const T*)a.dout + own, ldo,
      (const T*)a.o + own, ldo, a.lse + row, a.delta + row, dqs + t.begin * ldo, ldo, t.len,
      a.head_dim, t.tile * kRows, a.scale);
}

// Workgroup = 16 keys of one kv head, one piece of their walk; key blocks are counted from
// the end of their sequence, so the longest walks come first, and the pieces of cut walks
// before the others: slab [kv head][rank][2][16][D], dK then dV.
template <typename T, int DM, bool VEC>
__global__ __launch_bounds__(kGenThreads, DM > 64 ? 1 : 2) void packed_gen_dkdv_kernel(
    PackedAttn a, WalkCut c) {
  __shared__ float buf[kGenWaves][16][DM + 4];
  const int kvh = blockIdx.x % a.kv_heads, rank = blockIdx.x / a.kv_heads;
  const int group = a.heads / a.kv_heads, D = a.head_dim;
  const int64_t ldkv = (int64_t)a.kv_heads * D, ldo = (int64_t)a.heads * D;
  T *dks = (T*)a.dk + kvh * D, *dvs = (T*)a.dv + kvh * D;
  SeqTile t;
  if (!find_tile<kRows, true>(a.seqs, rank, t, c.least, c.share)) {
    zero_unused_rows(a.seqs, t, rank, c.ranks, dks, ldkv, D);
    zero_unused_rows(a.seqs, t, rank, c.ranks, dvs, ldkv, D);
    return;
  }
  if (t.pieces > 1 && rank >= c.slabs) return;  // no batch's: the bound is walk_cut's
  const int k0 = (t.tiles - 1 - t.tile) * kRows, h0 = kvh * group;
  const int64_t row = (int64_t)h0 * a.seqs.tokens + t.begin;
  f32x4 adk[DM / 16], adv[DM / 16];
  attn_gen_dkdv_keys<T, DM, VEC>(
      (const T*)a.q + t.begin * a.q_token + h0 * a.q_head, a.q_token, a.q_head,
      (const T*)a.k + t.begin * a.k_token + kvh * a.k_head, a.k_token,
      (const T*)a.v + t.begin * a.v_token + kvh * a.v_head, a.v_token,
      (const T*)a.dout + t.begin * ldo + h0 * D, ldo, D, a.lse + row, a.delta + row,
      a.seqs.tokens, t.len, D, group, k0, t.pieces, t.piece, a.scale, adk, adv);
  if (t.pieces > 1) {
    float* part = a.part + ((int64_t)kvh * c.slabs + rank) * (2 * kRows * D) - (int64_t)k0 * D;
    store_sum<float, DM>(buf, adk, part, D, k0, t.len, D, a.scale);
    store_sum<float, DM>(buf, adv, part + kRows * D, D, k0, t.len, D, 1.f);
  } else {
    store_sum<T, DM>(buf, adk, dks + t.begin * ldkv, ldkv, k0, t.len, D, a.scale);
    store_sum<T, DM>(buf, adv, dvs + t.begin * ldkv, ldkv, k0, t.len, D, 1.f);
  }
}

// dK and dV of the walks that were cut: their slabs in order, rounded once. The workgroups of
// a walk's pieces share its 16 keys.
template <typename T>
__global__ __launch_bounds__(kGenThreads) void packed_gen_reduce_kernel(PackedAttn a, WalkCut c) {
  const int kvh = blockIdx.x % a.kv_heads, rank = blockIdx.x / a.kv_heads;
  SeqTile t;
  if (!find_tile<kRows, true>(a.seqs, rank, t, c.least, c.share)) return;
  const int head = rank - t.piece;  // the walk's first piece
  if (t.pieces == 1 || head < 0 || head + t.pieces > c.slabs) return;
  const int k0 = (t.tiles - 1 - t.tile) * kRows, n = min(kRows, t.len - k0), D = a.head_dim;
  const float* part = a.part + ((int64_t)kvh * c.slabs + head) * (2 * kRows * D);
  const int64_t ldkv = (int64_t)a.kv_heads * D, first = (t.begin + k0) * ldkv + kvh * D;
  for (int e = t.piece * kGenThreads + threadIdx.x; e < 2 * n * D; e += kGenThreads * t.pieces) {
    const int which = e >= n * D, f = e - which * n * D;
    const float* p = part + which * kRows * D + f;
    float x = *p;
    for (int i = 1; i < t.pieces; ++i) x += p[i * 2 * kRows * D];
    ((T*)(which ? a.dv : a.dk))[first + f / D * ldkv + f % D] = from_f32<T>(x);
  }
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

size_t packed_generic_part_bytes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads,
                                 int64_t head_dim) {
  return (size_t)kv_heads * walk_cut(tokens, seqs, heads, kv_heads).slabs * 2 * kRows * head_dim *
         sizeof(float);
}

int packed_generic_fwd(const PackedAttn& given, int dtype, hipStream_t st) {
  PackedAttn a = given;
  const int64_t ranks = packed_tiles(a.seqs.tokens, a.seqs.n, kRows);
  if (check_grid("eg_packed_attn_fwd", ranks * a.heads, kGenThreads)) return 1;
  if (int e = packed_plan(given.seqs, 1, &kRows, given.plan, &a.seqs, st)) return e;
  return dispatch(a, dtype, false, "eg_packed_attn_fwd", [&](auto tag, auto dm, auto vec) {
    EG_LAUNCH((packed_gen_fwd_kernel<decltype(tag), decltype(dm)::value, decltype(vec)::value>),
              dim3((unsigned)(ranks * a.heads)), dim3(kGenThreads), 0, st, a, (int)ranks,
              a.scale * kGenLog2e);
    return check_launch("eg_packed_attn_fwd(generic)");
  });
}

int packed_generic_bwd(const PackedAttn& given, int dtype, hipStream_t st) {
  PackedAttn a = given;  // query and key tiles are of one size: one plan
  const int64_t ranks = packed_tiles(a.seqs.tokens, a.seqs.n, kRows);
  const WalkCut cut = walk_cut(a.seqs.tokens, a.seqs.n, a.heads, a.kv_heads);
  if (check_grid("eg_packed_attn_bwd", std::max(ranks * a.heads, (int64_t)cut.ranks * a.kv_heads),
                 kGenThreads))
    return 1;
  if (int e = packed_plan(given.seqs, 1, &kRows, given.plan, &a.seqs, st)) return e;
  return dispatch(a, dtype, true, "eg_packed_attn_bwd", [&](auto tag, auto dm, auto vec) {
    using T = decltype(tag);
    constexpr int DM = decltype(dm)::value;
    constexpr bool VEC = decltype(vec)::value;
    EG_LAUNCH((packed_gen_dq_kernel<T, DM, VEC>), dim3((unsigned)(ranks * a.heads)),
              dim3(kGenThreads), 0, st, a, (int)ranks);
    if (int e = check_launch("eg_packed_attn_bwd(generic dq)")) return e;
    EG_LAUNCH((packed_gen_dkdv_kernel<T, DM, VEC>), dim3((unsigned)(cut.ranks * a.kv_heads)),
              dim3(kGenThreads), 0, st, a, cut);
    if (int e = check_launch("eg_packed_attn_bwd(generic dkdv)")) return e;
    if (cut.slabs == 0) return 0;
    EG_LAUNCH((packed_gen_reduce_kernel<T>), dim3((unsigned)(cut.slabs * a.kv_heads)),
              dim3(kGenThreads), 0, st, a, cut);
    return check_launch("eg_packed_attn_bwd(generic dkdv reduce)");
  });
}

}  // namespace eg
