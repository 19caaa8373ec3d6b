// Device code of the generic attention (attn_generic.hip): causal attention of one head's
// sequence in fp32 MFMA arithmetic, any 16- or 32-bit type and even head size up to 128,
// as workgroup-wide functions over rows of any stride. The kernels that place them on a
// grid are in attn_generic.hip ([B, H, S, D] tensors) and packed_attn_generic.hip (packed
// sequences); the operand layouts are described in the former.
#pragma once

#include "eg_common.hpp"

#include <initializer_list>
#include <type_traits>

namespace eg {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kGenWaves = 4;
constexpr int kGenThreads = kGenWaves * 64;
constexpr int64_t kGenTarget = 512;  // workgroups: two per CU
constexpr float kGenLog2e = 1.4426950408889634f;
constexpr float kGenLn2 = 0.6931471805599453f;

__device__ __forceinline__ f32x4 gmma(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Columns per lane and load of the column layout, and the column of lane index m
// (0..15), tile t: runs of kRun<DM> consecutive columns.
template <int DM> constexpr int kRun = DM >= 64 ? 4 : DM / 16;
template <int DM> __device__ __forceinline__ int dcol(int m, int t) {
  return (t / kRun<DM>) * (16 * kRun<DM>) + m * kRun<DM> + t % kRun<DM>;
}

// W consecutive columns c .. c + W - 1 of a row of D, zero past D. VEC: W | D and
// aligned rows, so one load; the address of a column past D is replaced by column 0.
template <typename T, int W, bool VEC>
__device__ __forceinline__ void load_run(const T* __restrict__ row, int c, int D, float (&x)[W]) {
  if constexpr (VEC) {
    const bool in = c < D;
    load_f32<T, W>(row + (in ? c : 0), x);
#pragma unroll
    for (int i = 0; i < W; ++i) x[i] = in ? x[i] : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const bool in = c + i < D;
      const float y = to_f32(row[in ? c + i : 0]);
      x[i] = in ? y : 0.f;
    }
  }
}

// Row layout: this lane's columns of `row` (the row l%16 of the tile).
template <typename T, int DM, bool VEC>
__device__ __forceinline__ void load_rows(const T* __restrict__ row, int D, int g,
                                          float (&f)[DM / 4]) {
#pragma unroll
  for (int j = 0; j < DM / 16; ++j) {
    float x[4];
    load_run<T, 4, VEC>(row, 16 * j + 4 * g, D, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[4 * j + e] = x[e];
  }
}

// Column layout: rows r0 + 4g + r (clamped to the slice's last row) of an [S, D] slice
// whose rows lie ld elements apart.
template <typename T, int DM, bool VEC>
__device__ __forceinline__ void load_cols(const T* __restrict__ slice, int64_t ld, int r0, int S, int D,
                                          int g, int m, float (&f)[4][DM / 16]) {
  constexpr int W = kRun<DM>;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const T* row = slice + min(r0 + 4 * g + r, S - 1) * ld;
#pragma unroll
    for (int t0 = 0; t0 < DM / 16; t0 += W) {
      float x[W];
      load_run<T, W, VEC>(row, dcol<DM>(m, t0), D, x);
#pragma unroll
      for (int i = 0; i < W; ++i) f[r][t0 + i] = x[i];
    }
  }
}

template <int DT>
__device__ __forceinline__ bool all_finite(const float (&f)[4][DT]) {
  bool ok = true;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < DT; ++t) ok &= __builtin_fabsf(f[r][t]) < INFINITY;
  return __builtin_amdgcn_ballot_w64(!ok) == 0;
}

// acc += (column-layout tile f)^T w over the tile's 16 rows.
template <int DT>
__device__ __forceinline__ void add_tile(f32x4 (&acc)[DT], const float (&f)[4][DT], f32x4 w) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = gmma(f[r][t], w[r], acc[t]);
}

// The same sum pair by pair, leaving masked pairs out: bit 4G + r of `on` says whether
// row 4G + r of the tile counts for this lane's column.
template <int DT>
__device__ __forceinline__ void add_pairs(f32x4 (&acc)[DT], const float (&f)[4][DT], f32x4 w,
                                          unsigned on, int lane) {
  const int m = lane & 15, g = lane >> 4;
  for (int G = 0; G < 4; ++G)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float wr = __shfl(w[r], 16 * G + m, 64);
      const bool in = (on >> (4 * G + r)) & 1;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __shfl(f[r][t], 16 * G + 4 * g + e, 64);
          acc[t][e] = in ? __builtin_fmaf(wr, x, acc[t][e]) : acc[t][e];
        }
    }
}

// Sum over the workgroup's waves of a 16-row result (acc tiles: this lane's row l%16,
// columns dcol(4g + e, t)), through LDS in wave order: rows row0 .. row0 + 15 below
// `rows` of dst, row stride ld, times f. Every wave calls it; `buf` holds one [16][DM + 4]
// tile per wave.
template <typename TO, int DM>
__device__ __forceinline__ void store_sum(float (*buf)[16][DM + 4], const f32x4 (&acc)[DM / 16],
                                          TO* __restrict__ dst, int64_t ld, int row0, int rows,
                                          int D, float f) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  __syncthreads();  // the buffer's last use is over
#pragma unroll
  for (int t = 0; t < DM / 16; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) buf[w][m][dcol<DM>(4 * g + e, t)] = acc[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * DM; i += kGenThreads) {
    const int r = i / DM, d = i % DM;
    float s = buf[0][r][d];
#pragma unroll
    for (int k = 1; k < kGenWaves; ++k) s += buf[k][r][d];
    if (row0 + r < rows && d < D) dst[(row0 + r) * ld + d] = from_f32<TO>(s * f);
  }
}

__device__ __forceinline__ float over_groups(float v, bool is_max) {
#pragma unroll
  for (int off = 16; off <= 32; off <<= 1) {
    const float o = __shfl_xor(v, off, 64);
    v = is_max ? fmaxf(v, o) : v + o;
  }
  return v;
}

// Forward: workgroup = the 16 query rows from q0 on of one head's sequence of S rows, its
// waves cutting the keys in tiles of 16 KT. Rows of the slices lie ldq, ldk, ldv and ldo
// elements apart.
template <typename T, int DM, bool VEC>
__device__ __forceinline__ void attn_gen_fwd_rows(
    const T* __restrict__ qs, int64_t ldq, const T* __restrict__ ks, int64_t ldk,
    const T* __restrict__ vs, int64_t ldv, T* __restrict__ os, int64_t ldo,
    float* __restrict__ lse, int S, int D, int q0, float scale_log2) {
  constexpr int NS = DM / 4, DT = DM / 16, KT = DM > 64 ? 1 : 2;
  __shared__ float buf[kGenWaves][16][DM + 4];
  __shared__ float wm[kGenWaves][16], wl[kGenWaves][16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m16 = lane & 15, g = lane >> 4;
  const int query = q0 + m16;
  float qf[NS];
  load_rows<T, DM, VEC>(qs + min(query, S - 1) * ldq, D, g, qf);
#pragma unroll
  for (int i = 0; i < NS; ++i) qf[i] *= scale_log2;
  f32x4 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x4{};
  float m = -INFINITY, l = 0.f;
  const int nt = (min(S, q0 + 16) + 16 * KT - 1) / (16 * KT);
  float kf[KT][NS];
  auto load_k = [&](int tile) {
#pragma unroll
    for (int i = 0; i < KT; ++i)
      load_rows<T, DM, VEC>(ks + min(16 * (KT * tile + i) + m16, S - 1) * ldk, D, g, kf[i]);
  };
  if (w < nt) load_k(w);
  for (int tile = w; tile < nt; tile += kGenWaves) {
    const int key0 = 16 * KT * tile;
    float vf[KT][4][DT];
#pragma unroll
    for (int i = 0; i < KT; ++i) load_cols<T, DM, VEC>(vs, ldv, key0 + 16 * i, S, D, g, m16, vf[i]);
    f32x4 s[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) s[i] = f32x4{};
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < KT; ++i) s[i] = gmma(kf[i][st], qf[st], s[i]);
    if (tile + kGenWaves < nt) load_k(tile + kGenWaves);
    const bool masked = key0 + 16 * KT - 1 > q0;
    if (masked) {
#pragma unroll
      for (int i = 0; i < KT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key0 + 16 * i + 4 * g + r > query) s[i][r] = -INFINITY;
    }
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < KT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) mt = fmaxf(mt, s[i][r]);
    const float mn = fmaxf(m, over_groups(mt, true));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    l *= alpha;
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] *= alpha;
    m = mn;
#pragma unroll
    for (int i = 0; i < KT; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - ref);
        l += s[i][r];
      }
      if (masked && !all_finite<DT>(vf[i])) {
        const int n = query - (key0 + 16 * i) + 1;  // keys of the tile this query sees
        add_pairs<DT>(acc, vf[i], s[i], n >= 16 ? 0xffffu : n <= 0 ? 0u : (1u << n) - 1, lane);
      } else {
        add_tile<DT>(acc, vf[i], s[i]);
      }
    }
  }
  // The waves' maxima and sums, then their outputs, each scaled to the common maximum.
  l = over_groups(l, false);
  if (g == 0) { wm[w][m16] = m; wl[w][m16] = l; }
  __syncthreads();
  float M = wm[0][m16];
#pragma unroll
  for (int i = 1; i < kGenWaves; ++i) M = fmaxf(M, wm[i][m16]);
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
#pragma unroll
  for (int i = 0; i < kGenWaves; ++i) L += wl[i][m16] * __builtin_amdgcn_exp2f(wm[i][m16] - ref);
  const float f = __builtin_amdgcn_exp2f(m - ref) / L;
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] *= f;
  store_sum<T, DM>(buf, acc, os, ldo, q0, S, D, 1.f);
  if (w == 0 && g == 0 && query < S) lse[query] = (M + __log2f(L)) * kGenLn2;
}

// dQ (and delta = rowsum(do * o) for the dK/dV kernel): workgroup and waves as above, key
// tiles of 16 KT. PACKED: where the rows' keys fit one tile, delta is sum p dp / sum p, which
// has no rounding of o in it (bf16 rows of 4 keys, dq's error 0.28 -> 0.17% of its norm).
template <typename T, int DM, bool VEC, bool PACKED>
__device__ __forceinline__ void attn_gen_dq_rows(
    const T* __restrict__ qs, int64_t ldq, const T* __restrict__ ks, int64_t ldk,
    const T* __restrict__ vs, int64_t ldv, const T* __restrict__ dos, int64_t lddo,
    const T* __restrict__ os, int64_t ldo, const float* __restrict__ lse,
    float* __restrict__ delta, T* __restrict__ dqs, int64_t lddq, int S, int D, int q0,
    float scale) {
  constexpr int NS = DM / 4, DT = DM / 16, KT = DM > 64 ? 1 : 2;
  __shared__ float buf[kGenWaves][16][DM + 4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m16 = lane & 15, g = lane >> 4;
  const int query = q0 + m16, qc = min(query, S - 1);
  const float sl2 = scale * kGenLog2e;
  float qf[NS], df[NS], dl = 0.f;
  load_rows<T, DM, VEC>(qs + qc * ldq, D, g, qf);
  load_rows<T, DM, VEC>(dos + qc * lddo, D, g, df);
  {
    float of[NS];
    load_rows<T, DM, VEC>(os + qc * ldo, D, g, of);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      dl = __builtin_fmaf(df[i], of[i], dl);
      qf[i] *= sl2;
    }
  }
  dl = over_groups(dl, false);
  const float l2 = lse[qc] * kGenLog2e;
  if constexpr (!PACKED)
    if (w == 0 && g == 0 && query < S) delta[query] = dl;
  f32x4 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x4{};
  const int nt = (min(S, q0 + 16) + 16 * KT - 1) / (16 * KT);
  float kf[KT][NS], vf[KT][NS];
  auto load_kv = [&](int tile) {
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const int row = min(16 * (KT * tile + i) + m16, S - 1);
      load_rows<T, DM, VEC>(ks + row * ldk, D, g, kf[i]);
      load_rows<T, DM, VEC>(vs + row * ldv, D, g, vf[i]);
    }
  };
  if (w < nt) load_kv(w);
  for (int tile = w; tile < nt; tile += kGenWaves) {
    const int key0 = 16 * KT * tile;
    float kc[KT][4][DT];
#pragma unroll
    for (int i = 0; i < KT; ++i) load_cols<T, DM, VEC>(ks, ldk, key0 + 16 * i, S, D, g, m16, kc[i]);
    f32x4 s[KT], dp[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) { s[i] = f32x4{}; dp[i] = f32x4{}; }
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        s[i] = gmma(kf[i][st], qf[st], s[i]);
        dp[i] = gmma(vf[i][st], df[st], dp[i]);
      }
    if (tile + kGenWaves < nt) load_kv(tile + kGenWaves);
    const bool masked = key0 + 16 * KT - 1 > q0;
    if constexpr (PACKED) {
      if (nt == 1) {
        float pd = 0.f, ps = 0.f;
#pragma unroll
        for (int i = 0; i < KT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool in = 16 * i + 4 * g + r <= query;
            const float p = in ? __builtin_amdgcn_exp2f(s[i][r] - l2) : 0.f;
            pd += in ? p * dp[i][r] : 0.f;
            ps += p;
          }
        dl = over_groups(pd, false) / over_groups(ps, false);
      }
    }
#pragma unroll
    for (int i = 0; i < KT; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float ds = __builtin_amdgcn_exp2f(s[i][r] - l2) * (dp[i][r] - dl);
        s[i][r] = key0 + 16 * i + 4 * g + r > query ? 0.f : ds;
      }
      if (masked && !all_finite<DT>(kc[i])) {
        const int n = query - (key0 + 16 * i) + 1;
        add_pairs<DT>(acc, kc[i], s[i], n >= 16 ? 0xffffu : n <= 0 ? 0u : (1u << n) - 1, lane);
      } else {
        add_tile<DT>(acc, kc[i], s[i]);
      }
    }
  }
  if constexpr (PACKED)
    if (w == 0 && g == 0 && query < S) delta[query] = dl;
  store_sum<T, DM>(buf, acc, dqs, lddq, q0, S, D, scale);
}

// dK, dV: workgroup = the 16 keys from k0 on of one kv head, part pi of `parts`; the walk
// over the group's query heads and their 16-row tiles from the diagonal on is dealt out step
// by step over the parts' waves. qs, dos, lse and delta are those of the group's first
// head; the next head's lie hq, hdo and hl elements on. Leaves each wave's sums, dK's unscaled.
template <typename T, int DM, bool VEC>
__device__ __forceinline__ void attn_gen_dkdv_keys(
    const T* __restrict__ qs, int64_t ldq, int64_t hq, const T* __restrict__ ks, int64_t ldk,
    const T* __restrict__ vs, int64_t ldv, const T* __restrict__ dos, int64_t lddo, int64_t hdo,
    const float* __restrict__ lse, const float* __restrict__ delta, int64_t hl,
    int S, int D, int group, int k0, int parts, int pi, float scale, f32x4 (&adk)[DM / 16],
    f32x4 (&adv)[DM / 16]) {
  constexpr int NS = DM / 4, DT = DM / 16;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, m16 = lane & 15, g = lane >> 4;
  const int key = k0 + m16;
  const float sl2 = scale * kGenLog2e;
  float kf[NS], vf[NS];
  load_rows<T, DM, VEC>(ks + min(key, S - 1) * ldk, D, g, kf);
  load_rows<T, DM, VEC>(vs + min(key, S - 1) * ldv, D, g, vf);
#pragma unroll
  for (int i = 0; i < NS; ++i) kf[i] *= sl2;
#pragma unroll
  for (int t = 0; t < DT; ++t) { adk[t] = f32x4{}; adv[t] = f32x4{}; }
  const int ntq = (S - k0 + 15) / 16, nsteps = group * ntq, stride = parts * kGenWaves;
  float qf[NS], df[NS];
  auto load_qd = [&](int step) {
    const int h = step / ntq, row = min(k0 + 16 * (step % ntq) + m16, S - 1);
    load_rows<T, DM, VEC>(qs + h * hq + row * ldq, D, g, qf);
    load_rows<T, DM, VEC>(dos + h * hdo + row * lddo, D, g, df);
  };
  const int first = pi * kGenWaves + w;
  if (first < nsteps) load_qd(first);
  for (int step = first; step < nsteps; step += stride) {
    const int h = step / ntq;
    const int q0 = k0 + 16 * (step % ntq);
    float qc[4][DT], dc[4][DT];
    load_cols<T, DM, VEC>(dos + h * hdo, lddo, q0, S, D, g, m16, dc);
    load_cols<T, DM, VEC>(qs + h * hq, ldq, q0, S, D, g, m16, qc);
    float lr[4], er[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t at = h * hl + min(q0 + 4 * g + r, S - 1);
      lr[r] = lse[at] * kGenLog2e;
      er[r] = delta[at];
    }
    f32x4 s = f32x4{}, dp = f32x4{};
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      s = gmma(qf[st], kf[st], s);
      dp = gmma(df[st], vf[st], dp);
    }
    if (step + stride < nsteps) load_qd(step + stride);
    unsigned on = 0;  // this lane's rows
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = q0 + 4 * g + r;
      const bool in = row >= key && row < S;
      on |= (unsigned)in << (4 * g + r);
      const float p = __builtin_amdgcn_exp2f(s[r] - lr[r]);
      dp[r] = in ? p * (dp[r] - er[r]) : 0.f;
      s[r] = in ? p : 0.f;
    }
    if ((q0 < k0 + 16 || q0 + 16 > S) && !(all_finite<DT>(qc) && all_finite<DT>(dc))) {
      on |= __shfl_xor(on, 16, 64);
      on |= __shfl_xor(on, 32, 64);
      add_pairs<DT>(adv, dc, s, on, lane);
      add_pairs<DT>(adk, qc, dp, on, lane);
    } else {
      add_tile<DT>(adv, dc, s);
      add_tile<DT>(adk, qc, dp);
    }
  }
}

// f(type, DM, VEC): DM the smallest of 16, 32, 64, 128 that holds D; VEC when rows can
// be read four columns at a time (D % 4 == 0 and every tensor aligned to four elements).
template <typename F>
int gen_dispatch(int dtype, int64_t D, std::initializer_list<const void*> ptrs, const char* name,
                 F&& f) {
  auto by_vec = [&](auto tag, auto dm) -> int {
    bool vec = D % 4 == 0;
    for (const void* p : ptrs) vec = vec && (uintptr_t)p % (4 * sizeof(tag)) == 0;
    return vec ? f(tag, dm, std::true_type{}) : f(tag, dm, std::false_type{});
  };
  auto by_dim = [&](auto tag) -> int {
    if (D <= 16) return by_vec(tag, std::integral_constant<int, 16>{});
    if (D <= 32) return by_vec(tag, std::integral_constant<int, 32>{});
    if (D <= 64) return by_vec(tag, std::integral_constant<int, 64>{});
    return by_vec(tag, std::integral_constant<int, 128>{});
  };
  switch (dtype) {
    case EG_F32: return by_dim(float{});
    case EG_F16: return by_dim(f16_t{});
    case EG_BF16: return by_dim(bf16_t{});
    default: set_error("%s: unsupported dtype %d", name, dtype); return 1;
  }
}

}  // namespace
}  // namespace eg
