// Distillation from a teacher's top logits over vocabulary-wide rows, for gfx950.
//
// Per row r with target != ignore_index (n of them), student logits z [cols], teacher values
// t_k at columns i_k (k < K; a negative i_k is no entry, entries of one column all count):
//   p = softmax over the entries of t / tau,  q = softmax(z / tau) over all columns
//   soft = tau^2 sum_k p_k (log p_k - log q_{i_k}), 0 for a row without entries
//   hard = logsumexp(z) - z_target
//   loss = sum_r (soft_weight soft + hard_weight hard) / n
//   dz_c = dloss / n (hard_weight (softmax(z)_c - [c = target])
//                     + soft_weight tau (P q_c - sum over k with i_k = c of p_k)),
// P = 1 with entries, else 0; zero in ignored rows. Everything in fp32, dz rounded once.
//
// Memory-bound: the forward reads the logits once, for both normalisers (they share the row's
// maximum, tau being positive), the backward reads them and writes dz. Ignored rows are read by
// neither. Saved per row: (max, 1 / sum exp(z - max), P / sum exp((z - max) / tau)), so that
// the backward's exponents are small differences, and p with the entries of one column added
// up in the first of them: every column of the backward has one term at most, which it finds in
// LDS.
#include "rowwise.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

using rowwise::kLog2e;
using rowwise::kUnroll;
using rowwise::lse_ref;

constexpr int kMaxEntries = 1024;
constexpr int kFinishBlock = 256, kMeanBlock = 1024;
constexpr int kFlatBlock = rowwise::kFlatBlock, kFlatUnroll = rowwise::kFlatUnroll,
              kFlatPer = rowwise::kFlatPer;

struct DistillArgs {
  const void *logits, *teacher, *ids;
  const int64_t* target;
  const float* dloss;
  float *loss, *stats, *probs, *n_valid;
  void* dlogits;
  float *rowloss, *part;  // part: [rows][splits][3] (max, sum, sum at tau)
  int64_t rows, ignore_index;
  int cols, k, slots, splits, ids_64, teacher_type;
  float tau, soft, hard;
};

__device__ __forceinline__ int64_t entry_id(const DistillArgs& a, int64_t i) {
  return a.ids_64 ? ((const int64_t*)a.ids)[i] : (int64_t)((const int*)a.ids)[i];
}
__device__ __forceinline__ float entry_value(const DistillArgs& a, int64_t i) {
  return a.teacher_type == EG_F32    ? ((const float*)a.teacher)[i]
         : a.teacher_type == EG_F16 ? to_f32(((const f16_t*)a.teacher)[i])
                                    : to_f32(((const bf16_t*)a.teacher)[i]);
}

// A running (max, sum of exp(z - max), sum of exp((z - max) / tau)) of a row's part.
struct RowSums {
  float m, s1, st;
};
// Brings `s`, a sum relative to `from`, to the reference `to` (both as lse_ref gives them).
__device__ __forceinline__ float rescale(float s, float from, float to, float c) {
  return s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f((from - to) * c);
}

// One workgroup's columns [c0, c1) of a row, the same result in every thread.
template <typename T, int VEC, int BLOCK, bool RAG>
__device__ __forceinline__ RowSums row_sums(const T* __restrict__ xr, int c0, int c1, int cols,
                                            float ct, float* red) {
  constexpr int STEP = BLOCK * VEC;
  RowSums r = {-INFINITY, 0.f, 0.f};
  for (int64_t base = c0 + (int64_t)threadIdx.x * VEC; base < c1; base += STEP * kUnroll) {
    float v[kUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t c = base + u * STEP;
      if (c < c1) {
        rowwise::load_pack<T, VEC, VEC * sizeof(T) == 16, RAG>(xr, (int)c, cols, -INFINITY, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[u][i] = -INFINITY;
      }
    }
    float bm = r.m;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) bm = fmaxf(bm, v[u][i]);
    const float ref = lse_ref(bm);
    float a1 = 0.f, at = 0.f;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = v[u][i] - ref;
        a1 += __builtin_amdgcn_exp2f(d * kLog2e);
        at += __builtin_amdgcn_exp2f(d * ct);
      }
    r.s1 = rescale(r.s1, lse_ref(r.m), ref, kLog2e) + a1;
    r.st = rescale(r.st, lse_ref(r.m), ref, ct) + at;
    r.m = bm;
  }
  const float gm = block_reduce<BLOCK>(r.m, MaxOp(), red), ref = lse_ref(gm);
  r.s1 = block_reduce<BLOCK>(rescale(r.s1, lse_ref(r.m), ref, kLog2e), SumOp(), red);
  r.st = block_reduce<BLOCK>(rescale(r.st, lse_ref(r.m), ref, ct), SumOp(), red);
  r.m = gm;
  return r;
}

// The rest of a counted row by one workgroup: its loss, saved statistics and probabilities.
// `lds` holds slots x 2 ints and K floats.
template <typename T, int BLOCK>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, RowSums r, int* lds,
                                           float* red) {
  int *table = lds, *holder = lds + a.slots;
  float* p = (float*)(lds + 2 * a.slots);
  const T* xr = (const T*)a.logits + row * a.cols;
  const int64_t e0 = row * a.k;
  const float ref = lse_ref(r.m), rtau = 1.f / a.tau;
  for (int i = threadIdx.x; i < a.slots; i += BLOCK) table[i] = -1, holder[i] = kMaxEntries;
  float tm = -INFINITY, bad = 0.f;
  for (int k = threadIdx.x; k < a.k; k += BLOCK) {
    const int64_t id = entry_id(a, e0 + k);
    if (id >= a.cols) bad = 1.f;
    if (id >= 0 && id < a.cols) tm = fmaxf(tm, entry_value(a, e0 + k));
  }
  __syncthreads();
  tm = lse_ref(block_reduce<BLOCK>(tm, MaxOp(), red));
  bad = block_reduce<BLOCK>(bad, SumOp(), red);
  float total = 0.f;
  for (int k = threadIdx.x; k < a.k; k += BLOCK) {
    const int64_t id = entry_id(a, e0 + k);
    const bool in = id >= 0 && id < a.cols;
    total += p[k] = in ? expf((entry_value(a, e0 + k) - tm) * rtau) : 0.f;
  }
  total = block_reduce<BLOCK>(total, SumOp(), red);
  const bool some = total != 0.f;  // a NaN is one
  const float lt = logf(total), lq = logf(r.st);
  float kl = 0.f;
  for (int k = threadIdx.x; k < a.k; k += BLOCK) {
    const int64_t id = entry_id(a, e0 + k);
    const float pk = some && id >= 0 && id < a.cols ? p[k] / total : 0.f;
    p[k] = pk;
    if (pk == 0.f) continue;
    const float logq = (to_f32(xr[id]) - ref) * rtau - lq;
    kl += pk * ((entry_value(a, e0 + k) - tm) * rtau - lt - logq);
    // the first entry of each column, in a hash table of at least twice the entries
    unsigned s = (unsigned)id * 2654435761u >> 16;
    for (;; ++s) {
      s &= a.slots - 1;
      const int was = atomicCAS(&table[s], -1, (int)id);
      if (was == -1 || was == (int)id) break;
    }
    atomicMin(&holder[s], k);
  }
  kl = block_reduce<BLOCK>(kl, SumOp(), red);
  __syncthreads();
  for (int k = threadIdx.x; k < a.k; k += BLOCK) {
    const int64_t id = entry_id(a, e0 + k);
    float sum = p[k];
    if (sum != 0.f) {
      unsigned s = (unsigned)id * 2654435761u >> 16;
      for (;; ++s) {
        s &= a.slots - 1;
        if (table[s] == (int)id) break;
      }
      if (holder[s] != k) {
        sum = 0.f;
      } else {
        for (int j = k + 1; j < a.k; ++j)
          if (entry_id(a, e0 + j) == id) sum += p[j];
      }
    }
    a.probs[e0 + k] = sum;
  }
  if (threadIdx.x == 0) {
    float loss = 0.f;
    const int64_t t = a.target[row];
    if (a.soft != 0.f && some) loss += a.soft * a.tau * a.tau * kl;
    if (a.hard != 0.f) {
      if (t < 0 || t >= a.cols) bad = 1.f;
      else loss += a.hard * (logf(r.s1) - (to_f32(xr[t]) - ref));
    }
    const float fail = bad != 0.f ? NAN : 0.f;
    a.rowloss[row] = loss + fail;
    float* s = a.stats + row * 4;
    s[0] = ref;
    s[1] = 1.f / r.s1 + fail;
    s[2] = some ? 1.f / r.st + fail : fail;
    s[3] = 0.f;
  }
}

template <int BLOCK>
__device__ __forceinline__ void skip_row(const DistillArgs& a, int64_t row) {
  for (int k = threadIdx.x; k < a.k; k += BLOCK) a.probs[row * a.k + k] = 0.f;
  if (threadIdx.x < 4) a.stats[row * 4 + threadIdx.x] = 0.f;
  if (threadIdx.x == 0) a.rowloss[row] = 0.f;
}

// A workgroup a row, or (splits > 1) a part of one.
template <typename T, int VEC, int BLOCK, bool RAG>
__global__ __launch_bounds__(BLOCK) void distill_row_kernel(DistillArgs a) {
  extern __shared__ int lds[];
  __shared__ float red[BLOCK / kWave];
  const int64_t row = blockIdx.x;
  if (a.target[row] == a.ignore_index) {
    if (a.splits == 1) skip_row<BLOCK>(a, row);
    return;
  }
  const T* xr = (const T*)a.logits + row * a.cols;
  const int64_t packs = (a.cols + VEC - 1) / VEC;
  const int64_t each = (packs + a.splits - 1) / a.splits * VEC;
  const int c0 = (int)min((int64_t)blockIdx.y * each, (int64_t)a.cols);
  const int c1 = (int)min(c0 + each, (int64_t)a.cols);
  const RowSums r = row_sums<T, VEC, BLOCK, RAG>(xr, c0, c1, a.cols, kLog2e / a.tau, red);
  if (a.splits == 1) {
    finish_row<T, BLOCK>(a, row, r, lds, red);
  } else if (threadIdx.x == 0) {
    float* p = a.part + (row * a.splits + blockIdx.y) * 3;
    p[0] = r.m, p[1] = r.s1, p[2] = r.st;
  }
}

template <typename T>
__global__ __launch_bounds__(kFinishBlock) void distill_finish_kernel(DistillArgs a) {
  extern __shared__ int lds[];
  __shared__ float red[kFinishBlock / kWave];
  const int64_t row = blockIdx.x;
  if (a.target[row] == a.ignore_index) {
    skip_row<kFinishBlock>(a, row);
    return;
  }
  const float ct = kLog2e / a.tau;
  RowSums r = {-INFINITY, 0.f, 0.f};
  for (int i = 0; i < a.splits; ++i) r.m = fmaxf(r.m, a.part[(row * a.splits + i) * 3]);
  const float ref = lse_ref(r.m);
  for (int i = 0; i < a.splits; ++i) {
    const float* p = a.part + (row * a.splits + i) * 3;
    r.s1 += rescale(p[1], lse_ref(p[0]), ref, kLog2e);
    r.st += rescale(p[2], lse_ref(p[0]), ref, ct);
  }
  finish_row<T, kFinishBlock>(a, row, r, lds, red);
}

__global__ __launch_bounds__(kMeanBlock) void distill_mean_kernel(DistillArgs a) {
  __shared__ float red[kMeanBlock / kWave];
  float sum = 0.f, count = 0.f;
  for (int64_t r = threadIdx.x; r < a.rows; r += kMeanBlock) {
    sum += a.rowloss[r];
    count += a.target[r] != a.ignore_index ? 1.f : 0.f;
  }
  sum = block_reduce<kMeanBlock>(sum, SumOp(), red);
  count = block_reduce<kMeanBlock>(count, SumOp(), red);
  if (threadIdx.x == 0) {
    a.loss[0] = sum / count;
    a.n_valid[0] = count;
  }
}

// What a row's gradient takes: dz = g1 exp(z - m) + gt exp((z - m) / tau) - gp p - [target] gh.
struct RowGrad {
  float m, g1, gt;
  int target;
  bool live;
};

// The matrix as one run of packs, kFlatPer a workgroup (rowwise.hpp). The entries' terms of its
// packs are laid out in LDS first. TWO: both exponentials, else the one of factor c.
template <typename T, int VEC, bool RAG, bool TWO>
__global__ __launch_bounds__(kFlatBlock) void distill_bwd_kernel(DistillArgs a) {
  __shared__ __attribute__((aligned(16))) float terms[kFlatPer * VEC];
  constexpr bool NT = VEC * sizeof(T) == 16;
  const unsigned ppr = (a.cols + VEC - 1) / VEC;  // packs per row
  const int64_t npack = a.rows * ppr, first = (int64_t)blockIdx.x * kFlatPer;
  const int64_t row0 = first / ppr;
  const unsigned in0 = (unsigned)(first - row0 * ppr);  // the workgroup's first pack in its row
  const float scale = a.dloss[0] / a.n_valid[0];
  const float gh = scale * a.hard, gp = scale * a.soft * a.tau;
  const float ct = kLog2e / a.tau;
  float v[kFlatUnroll][VEC];
  RowGrad g[kFlatUnroll];
  unsigned rows[kFlatUnroll], packs[kFlatUnroll];
#pragma unroll
  for (int u = 0; u < kFlatUnroll; ++u) {
    const unsigned q = in0 + u * kFlatBlock + threadIdx.x;
    rows[u] = q / ppr, packs[u] = q - rows[u] * ppr;
    g[u].live = false;
    if (first + u * kFlatBlock + threadIdx.x >= npack) continue;
    const int64_t row = row0 + rows[u];
    const int64_t t = a.target[row];
    g[u].live = t != a.ignore_index;
    if (!g[u].live) continue;
    rowwise::load_pack<T, VEC, NT, RAG>((const T*)a.logits + row * a.cols, packs[u] * VEC, a.cols, 0.f,
                                        v[u]);
    const float* s = a.stats + row * 4;
    g[u].m = s[0], g[u].g1 = gh * s[1], g[u].gt = gp * s[2];
    g[u].target = a.hard != 0.f && t >= 0 && t < a.cols ? (int)t : -1;
  }
  const bool entries = a.k > 0 && a.soft != 0.f;
  if (entries) {
#pragma unroll
    for (int u = 0; u < kFlatUnroll; ++u)
#pragma unroll
      for (int i = 0; i < VEC; ++i) terms[(u * kFlatBlock + threadIdx.x) * VEC + i] = 0.f;
    __syncthreads();
    const int64_t last = min(first + kFlatPer, npack) - 1;
    const int64_t e0 = row0 * a.k, n = (last / ppr + 1) * a.k - e0;
    for (int64_t i = threadIdx.x; i < n; i += kFlatBlock) {
      const float p = a.probs[e0 + i];
      if (p == 0.f) continue;
      const int64_t id64 = entry_id(a, e0 + i);
      if (id64 < 0 || id64 >= a.cols) continue;  // written over since the forward
      const int id = (int)id64;
      const int64_t at = i / a.k * ppr - in0;  // the row's first pack, from the workgroup's first
      const int64_t k = at + id / VEC;
      const int lo = RAG ? a.cols - VEC : 0;
      if (RAG && id >= lo) {  // the last pack, which overlaps the one before it
        const int64_t l = at + ppr - 1;
        if (l >= 0 && l < kFlatPer) terms[l * VEC + id - lo] = p;
        if (id / VEC == (int)ppr - 1) continue;
      }
      if (k >= 0 && k < kFlatPer) terms[k * VEC + id % VEC] = p;
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < kFlatUnroll; ++u) {
    if (first + u * kFlatBlock + threadIdx.x >= npack) continue;
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = 0.f;
    if (g[u].live) {
      const int c = packs[u] * VEC, c0 = RAG ? min(c, a.cols - VEC) : c;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = v[u][i] - g[u].m;
        if constexpr (TWO)
          o[i] = g[u].g1 * __builtin_amdgcn_exp2f(d * kLog2e) +
                 g[u].gt * __builtin_amdgcn_exp2f(d * ct);
        else
          o[i] = a.soft != 0.f ? (g[u].g1 + g[u].gt) * __builtin_amdgcn_exp2f(d * ct)
                               : g[u].g1 * __builtin_amdgcn_exp2f(d * kLog2e);
        if (entries) o[i] -= gp * terms[(u * kFlatBlock + threadIdx.x) * VEC + i];
        if (c0 + i == g[u].target) o[i] -= gh;
      }
    }
    rowwise::store_pack<T, VEC, NT, RAG>((T*)a.dlogits + (row0 + rows[u]) * a.cols, packs[u] * VEC,
                                         a.cols, o);
  }
}

int slots_for(int k) {
  int s = 64;
  while (s < 2 * k) s *= 2;
  return s;
}
size_t finish_lds(const DistillArgs& a) { return (2 * a.slots + a.k) * sizeof(int); }

// Parts of a row, where rows are few.
constexpr int kMostSplits = 64;
int splits_for(int64_t rows, int64_t cols) {
  const int64_t want = 512 / std::max<int64_t>(rows, 1), most = cols / 8192;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMostSplits}));
}

template <typename T, int VEC, bool RAG>
struct RowLaunch {
  const DistillArgs& a;
  hipStream_t st;
  template <int BLOCK>
  void go() {
    EG_LAUNCH((distill_row_kernel<T, VEC, BLOCK, RAG>), dim3((unsigned)a.rows, a.splits), dim3(BLOCK),
              a.splits == 1 ? finish_lds(a) : 0, st, a);
  }
};

// go(VEC, RAG) for the rows' alignment and width
template <typename T, typename F>
int by_width(int64_t cols, std::initializer_list<const void*> tensors, F&& go) {
  using std::integral_constant;
  constexpr int V = 16 / (int)sizeof(T);
  if (cols < V) return go(integral_constant<int, 1>{}, std::false_type{});
  bool aligned = cols % V == 0;
  for (const void* p : tensors) aligned = aligned && aligned16(p);
  const integral_constant<int, V> vec;
  return aligned ? go(vec, std::false_type{}) : go(vec, std::true_type{});
}

int check(const char* name, int64_t rows, int64_t cols, int64_t k, float temperature) {
  if (rows < 0 || cols < 0 || k < 0) { set_error("%s: negative size", name); return 1; }
  if (rows > 0 && cols == 0) { set_error("%s: distillation over zero classes", name); return 1; }
  if (rows > ((int64_t)1 << 22) || cols > ((int64_t)1 << 30) || k > kMaxEntries) {
    set_error("%s: size out of range (rows <= 2^22, cols <= 2^30, entries <= %d)", name, kMaxEntries);
    return 1;
  }
  if (!(temperature > 0.f) || __builtin_isinf(temperature)) {
    set_error("%s: temperature must be positive and finite", name);
    return 1;
  }
  return 0;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" size_t eg_topk_distill_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  const int splits = splits_for(rows, cols);
  return (size_t)rows * (1 + (splits > 1 ? 3 * splits : 0)) * sizeof(float);
}

extern "C" int eg_topk_distill_fwd(const void* logits, const int64_t* target, const void* teacher,
                                   int teacher_dtype, const void* teacher_ids, int ids_64,
                                   float* loss, float* stats, float* probs, float* n_valid,
                                   void* workspace, int64_t rows, int64_t cols, int64_t entries,
                                   float temperature, float soft_weight, float hard_weight,
                                   int64_t ignore_index, int dtype, void* stream) {
  static const char* name = "eg_topk_distill_fwd";
  clear_error();
  if (check(name, rows, cols, entries, temperature)) return 1;
  if (!loss || !n_valid || (rows && (!logits || !target || !stats || !workspace)) ||
      (rows && entries && (!teacher || !teacher_ids || !probs))) {
    set_error("%s: null pointer", name);
    return 1;
  }
  if (teacher_dtype != EG_F32 && teacher_dtype != EG_F16 && teacher_dtype != EG_BF16) {
    set_error("%s: unsupported dtype %d of the teacher's logits", name, teacher_dtype);
    return 1;
  }
  DistillArgs a = {};
  a.logits = logits, a.teacher = teacher, a.ids = teacher_ids, a.target = target;
  a.loss = loss, a.stats = stats, a.probs = probs, a.n_valid = n_valid;
  a.rowloss = (float*)workspace, a.part = a.rowloss + rows;
  a.rows = rows, a.cols = (int)cols, a.k = (int)entries, a.ignore_index = ignore_index;
  a.slots = slots_for(a.k), a.splits = splits_for(rows, cols), a.ids_64 = ids_64;
  a.teacher_type = teacher_dtype;
  a.tau = temperature, a.soft = soft_weight, a.hard = hard_weight;
  hipStream_t st = as_stream(stream);
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    using T = scalar_t;
    if (rows) {
      if (check_grid(name, rows, 1024)) return 1;
      by_width<T>(cols, {logits}, [&](auto vec, auto rag) {
        constexpr int V = decltype(vec)::value;
        const int64_t packs = ((cols + V - 1) / V + a.splits - 1) / a.splits;
        rowwise::pick_row_block(packs, RowLaunch<T, V, decltype(rag)::value>{a, st});
        return 0;
      });
      if (a.splits > 1)
        EG_LAUNCH((distill_finish_kernel<T>), dim3((unsigned)rows), dim3(kFinishBlock), finish_lds(a),
                  st, a);
    }
    EG_LAUNCH(distill_mean_kernel, dim3(1), dim3(kMeanBlock), 0, st, a);
    return check_launch(name);
  });
}

extern "C" int eg_topk_distill_bwd(const float* dloss, const void* logits, const int64_t* target,
                                   const void* teacher_ids, int ids_64, const float* stats,
                                   const float* probs, const float* n_valid, void* dlogits,
                                   int64_t rows, int64_t cols, int64_t entries, float temperature,
                                   float soft_weight, float hard_weight, int64_t ignore_index,
                                   int dtype, void* stream) {
  static const char* name = "eg_topk_distill_bwd";
  clear_error();
  if (check(name, rows, cols, entries, temperature)) return 1;
  if (rows == 0) return 0;
  if (!dloss || !logits || !target || !stats || !n_valid || !dlogits ||
      (entries && (!teacher_ids || !probs))) {
    set_error("%s: null pointer", name);
    return 1;
  }
  DistillArgs a = {};
  a.logits = logits, a.ids = teacher_ids, a.target = target, a.dloss = dloss;
  a.stats = const_cast<float*>(stats), a.probs = const_cast<float*>(probs);
  a.n_valid = const_cast<float*>(n_valid), a.dlogits = dlogits;
  a.rows = rows, a.cols = (int)cols, a.k = (int)entries, a.ignore_index = ignore_index;
  a.ids_64 = ids_64, a.tau = temperature, a.soft = soft_weight, a.hard = hard_weight;
  const bool two = soft_weight != 0.f && hard_weight != 0.f && temperature != 1.f;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    using T = scalar_t;
    return by_width<T>(cols, {logits, (const void*)dlogits}, [&](auto vec, auto rag) -> int {
      constexpr int V = decltype(vec)::value;
      constexpr bool R = decltype(rag)::value;
      const int64_t blocks = (rows * ((cols + V - 1) / V) + kFlatPer - 1) / kFlatPer;
      if (check_grid(name, blocks, kFlatBlock)) return 1;
      const dim3 grid((unsigned)blocks), block(kFlatBlock);
      if (two)
        EG_LAUNCH((distill_bwd_kernel<T, V, R, true>), grid, block, 0, as_stream(stream), a);
      else
        EG_LAUNCH((distill_bwd_kernel<T, V, R, false>), grid, block, 0, as_stream(stream), a);
      return check_launch(name);
    });
  });
}
