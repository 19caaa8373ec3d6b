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
//
// Kernels: distill_row_kernel streams the rows (a workgroup a row, or a part of one where rows
// are few), leaves their sums and reads the entries' logits while the row is near;
// distill_finish_kernel does the rest of a row, whose work is a chain of short steps, in one wave;
// distill_mean_kernel adds the rows; distill_bwd_kernel. bf16 [8192, 128256] with 64 entries at a
// temperature of 2 with hard labels, a tenth of the rows ignored: 306 + 12 + 5 us forward (6.2
// TB/s) and 684 backward (5.8 TB/s), medians over whole steps; the figures below that compare variants
// are least means of 20 launches of one kernel in a row, where this backward takes 655. With the
// finish at the end of the row's own workgroup the forward took 597, as the streams of a CU's other
// workgroup do not fill it, and with the entries loaded after the first barrier the backward 939. Rows
// that are no multiple of a pack: fp16 [2047, 50257] 36 + 6 + 5 and 58; with the non-temporal hint on
// their loads 52 and 68, for unaligned packs share cache lines.
#include "rowwise.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

using rowwise::kLog2e;
using rowwise::lse_ref;

constexpr int kMaxEntries = 1024;
constexpr int kMeanBlock = 1024;
// Rows that one workgroup finishes, a wave each, with their mean. Forward of 128256 columns, us, so
// and with a launch for each: 1 row 10.0 / 10.9, 4 rows 10.6 / 11.5, 16 rows 11.3 / 11.5, 32 rows (two
// a wave) 17.3 / 12.6.
constexpr int64_t kFewRows = 16;
// Threads of a row's workgroup at most and packs in flight per thread. Forward, us, at 1024 / 512
// / 256 threads: bf16 [8192, 128256] with one exponential 308 / 309 / 308, a squared one 330 / 309 /
// 314, two 366 / 338 / 336, 16 rows 11.4 / 11.8 / 11.6; with 512 threads at 8 / 4 / 2 packs: 316 / 313
// / 305, 328 / 315 / 308, 362 / 344 / 338.
// A narrower row takes the smallest workgroup that walks it in kRowSteps (forward, us, in 1 / 2 / 4
// steps: bf16 [8192, 4096] 33.6 / 30.0 / 29.6, [8192, 8192] 47.4 / 38.2 / 36.3, [4096, 1000] 15.2 / 15.1 /
// 15.3, fp16 [3000, 2001] 15.0 / 14.6 / 14.5, fp32 [4096, 5000] 29.5 / 29.3 / 24.9).
constexpr int kMostRow = 512, kUnroll = 2, kRowSteps = 2;
// The backward's workgroup (bf16 [8192, 128256], a tenth of the rows ignored, us: 512 threads 671, 256
// 655, 128 652 but 814 with 256 entries a row for 690, 256 of four packs 788).
constexpr int kFlatBlock = 256, kFlatUnroll = 2, kFlatPer = kFlatBlock * kFlatUnroll;

// The exponentials of a column: one of them (no hard label, no soft part or a temperature of 1),
// both, or, at a temperature of 2, the hard label's as the soft one's square (bf16 [8192, 128256],
// forward and backward, us: one 308 and 635, both 350 and 675, the square 306 and 655).
enum Exps { kOne, kTwo, kSquare };

struct DistillArgs {
  const void *logits, *teacher, *ids;
  const int64_t* target;
  const float* dloss;
  float *loss, *stats, *probs, *n_valid;
  void* dlogits;
  float *rowloss, *part, *zs;  // part: [rows][splits][3] (max, sum, sum at tau); zs: [rows][k]
  int64_t rows, ignore_index;
  int cols, k, slots, splits, ids_64, teacher_type;
  float tau, soft, hard;
  float c1, ct;  // log2(e), log2(e) / tau
};

__device__ __forceinline__ int64_t entry_id(const DistillArgs& a, int64_t i) {
  return a.ids_64 ? ((const int64_t*)a.ids)[i] : (int64_t)((const int*)a.ids)[i];
}
__device__ __forceinline__ float entry_value(const DistillArgs& a, int64_t i) {
  return a.teacher_type == EG_F32    ? ((const float*)a.teacher)[i]
         : a.teacher_type == EG_F16 ? to_f32(((const f16_t*)a.teacher)[i])
                                    : to_f32(((const bf16_t*)a.teacher)[i]);
}

// exp(d) and exp(d / tau) of a difference to the row's maximum; kOne: both the one that is used.
template <int E>
__device__ __forceinline__ void exps(const DistillArgs& a, float d, float& e1, float& et) {
  et = __builtin_amdgcn_exp2f(d * a.ct);
  e1 = E == kTwo ? __builtin_amdgcn_exp2f(d * a.c1) : E == kSquare ? et * et : et;
}

// Brings `s`, a sum relative to `from`, to the reference `to` (both as lse_ref gives them).
__device__ __forceinline__ float rescale(float s, float from, float to, float c) {
  return s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f((from - to) * c);
}

// (max, sum of exp(z - max), sum of exp((z - max) / tau)) of a row's part, by a workgroup.
template <typename T, int VEC, int BLOCK, bool RAG, int E>
__global__ __launch_bounds__(BLOCK) void distill_row_kernel(DistillArgs a) {
  __shared__ float red[BLOCK / kWave], red2[BLOCK / kWave];
  constexpr int STEP = BLOCK * VEC;
  const int64_t row = blockIdx.x;
  if (a.target[row] == a.ignore_index) return;
  const T* __restrict__ xr = (const T*)a.logits + row * a.cols;
  const int64_t packs = (a.cols + VEC - 1) / VEC;
  const int64_t each = (packs + a.splits - 1) / a.splits * VEC;
  const int c0 = (int)min((int64_t)blockIdx.y * each, (int64_t)a.cols);
  const int c1 = (int)min(c0 + each, (int64_t)a.cols);
  // the entries' logits: read while the row is still near, for the finish
  int64_t id = -1;
  if (blockIdx.y == 0 && (int)threadIdx.x < a.k) id = entry_id(a, row * a.k + threadIdx.x);
  float m = -INFINITY, s1 = 0.f, st = 0.f;
  for (int64_t base = c0 + (int64_t)threadIdx.x * VEC; base < c1; base += STEP * kUnroll) {
    float v[kUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t c = base + u * STEP;
      if (c < c1) {
        rowwise::load_pack<T, VEC, VEC * sizeof(T) == 16 && !RAG, RAG>(xr, (int)c, a.cols, -INFINITY, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[u][i] = -INFINITY;
      }
    }
    float bm = m;
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
        float e1, et;
        exps<E>(a, v[u][i] - ref, e1, et);
        a1 += e1;
        if (E != kOne) at += et;
      }
    s1 = rescale(s1, lse_ref(m), ref, E == kOne ? a.ct : a.c1) + a1;
    if (E != kOne) st = rescale(st, lse_ref(m), ref, a.ct) + at;
    m = bm;
  }
  float z = 0.f;
  if (id >= 0 && id < a.cols) z = to_f32(xr[id]);
  const float gm = block_reduce<BLOCK>(m, MaxOp(), red), ref = lse_ref(gm);
  s1 = block_reduce<BLOCK>(rescale(s1, lse_ref(m), ref, E == kOne ? a.ct : a.c1), SumOp(), red2);
  if (E == kOne) st = s1;
  else st = block_reduce<BLOCK>(rescale(st, lse_ref(m), ref, a.ct), SumOp(), red);
  if (threadIdx.x == 0) {
    float* p = a.part + (row * a.splits + blockIdx.y) * 3;
    p[0] = gm, p[1] = s1, p[2] = st;
  }
  if (blockIdx.y) return;
  float* zr = a.zs + row * a.k;
  if ((int)threadIdx.x < a.k) zr[threadIdx.x] = z;
  for (int k = threadIdx.x + BLOCK; k < a.k; k += BLOCK) {
    id = entry_id(a, row * a.k + k);
    zr[k] = id >= 0 && id < a.cols ? to_f32(xr[id]) : 0.f;
  }
}

// A wave's stores to LDS before its later loads of them by other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The rest of a row by one wave: its parts joined, the teacher's distribution, the loss, what the
// backward needs. `lds` holds 2 slots + 3 K words. Returns the row's loss.
template <typename T>
__device__ __forceinline__ float finish_row(const DistillArgs& a, int64_t row, int* lds) {
  const int lane = threadIdx.x & 63;
  const int64_t e0 = row * a.k, t = a.target[row];
  float* s = a.stats + row * 4;
  if (t == a.ignore_index) {
    for (int k = lane; k < a.k; k += kWave) a.probs[e0 + k] = 0.f;
    if (lane < 4) s[lane] = 0.f;
    return 0.f;
  }
  wave_sync();  // an earlier row's words have been read
  int *table = lds, *holder = lds + a.slots, *ids = lds + 2 * a.slots;
  float *p = (float*)(ids + a.k), *zs = p + a.k;
  const T* xr = (const T*)a.logits + row * a.cols;
  // every load first: parts, the target's logit, entries
  const bool part = lane < a.splits;
  const float* q = a.part + (row * a.splits + (part ? lane : 0)) * 3;
  const float pm = part ? q[0] : -INFINITY, p1 = part ? q[1] : 0.f, pt = part ? q[2] : 0.f;
  const bool label = t >= 0 && t < a.cols;
  const float zt = label ? to_f32(xr[t]) : NAN;
  float tm = -INFINITY, bad = a.hard != 0.f && !label ? 1.f : 0.f;
  for (int i = lane; i < a.slots; i += kWave) table[i] = -1, holder[i] = kMaxEntries;
  for (int k = lane; k < a.k; k += kWave) {
    const int64_t id = entry_id(a, e0 + k);
    const float v = entry_value(a, e0 + k);
    if (id >= a.cols) bad = 1.f;
    const bool in = id >= 0 && id < a.cols;
    ids[k] = in ? (int)id : -1;
    p[k] = v;
    zs[k] = a.zs[e0 + k];
    if (in) tm = fmaxf(tm, v);
  }
  const float m = wave_reduce(pm, MaxOp()), ref = lse_ref(m);
  const bool one = a.soft == 0.f || a.hard == 0.f || a.tau == 1.f;
  const float s1 = wave_reduce(rescale(p1, lse_ref(pm), ref, one ? a.ct : a.c1), SumOp());
  const float st = wave_reduce(rescale(pt, lse_ref(pm), ref, a.ct), SumOp());
  tm = lse_ref(wave_reduce(tm, MaxOp()));
  bad = wave_reduce(bad, SumOp());
  const float rtau = 1.f / a.tau;
  float total = 0.f;
  for (int k = lane; k < a.k; k += kWave)
    if (ids[k] >= 0) total += expf((p[k] - tm) * rtau);
  total = wave_reduce(total, SumOp());
  const bool some = total != 0.f;  // a NaN is one
  const float lt = logf(total), lq = logf(st);
  float kl = 0.f;
  bool again = false;  // an entry of another one's column
  wave_sync();
  for (int k = lane; k < a.k; k += kWave) {
    const int id = ids[k];
    const float logit = (p[k] - tm) * rtau, pk = some && id >= 0 ? expf(logit) / total : 0.f;
    p[k] = pk;
    if (pk == 0.f) continue;
    kl += pk * (logit - lt - ((zs[k] - ref) * rtau - lq));
    // the first entry of each column, in a hash table of at least twice the entries
    unsigned at = (unsigned)id * 2654435761u >> 16;
    for (;; ++at) {
      at &= a.slots - 1;
      const int was = atomicCAS(&table[at], -1, id);
      again = again || was == id;
      if (was == -1 || was == id) break;
    }
    atomicMin(&holder[at], k);
  }
  kl = wave_reduce(kl, SumOp());
  again = __any(again);
  wave_sync();
  for (int k = lane; k < a.k; k += kWave) {
    float sum = p[k];
    if (again && sum != 0.f) {
      const int id = ids[k];
      unsigned at = (unsigned)id * 2654435761u >> 16;
      for (;; ++at) {
        at &= a.slots - 1;
        if (table[at] == id) break;
      }
      if (holder[at] != k) {
        sum = 0.f;
      } else {
        for (int j = k + 1; j < a.k; ++j)
          if (ids[j] == id) sum += p[j];
      }
    }
    a.probs[e0 + k] = sum;
  }
  float loss = 0.f;
  if (a.soft != 0.f && some) loss += a.soft * a.tau * a.tau * kl;
  if (a.hard != 0.f && label) loss += a.hard * (logf(s1) - (zt - ref));
  // a NaN or +inf among the entries is one in p's sum, which every column's gradient has
  const float fail = bad != 0.f || !(total < INFINITY) ? NAN : 0.f;
  if (lane == 0) {
    s[0] = ref;
    s[1] = 1.f / s1 + fail;
    s[2] = some ? 1.f / st + fail : fail;
    s[3] = 0.f;
  }
  return loss + fail;
}

// A wave a row.
template <typename T>
__global__ __launch_bounds__(kWave) void distill_finish_kernel(DistillArgs a) {
  extern __shared__ int lds[];
  const float loss = finish_row<T>(a, blockIdx.x, lds);
  if (threadIdx.x == 0) a.rowloss[blockIdx.x] = loss;
}

__device__ __forceinline__ void write_mean(const DistillArgs& a, float sum, float count, float* red) {
  sum = block_reduce<kMeanBlock>(sum, SumOp(), red);
  count = block_reduce<kMeanBlock>(count, SumOp(), red);
  if (threadIdx.x == 0) {
    a.loss[0] = sum / count;
    a.n_valid[0] = count;
  }
}

constexpr int kMeanRows = 8;  // in flight per thread
__global__ __launch_bounds__(kMeanBlock) void distill_mean_kernel(DistillArgs a) {
  __shared__ float red[kMeanBlock / kWave];
  float sum = 0.f, count = 0.f;
  for (int64_t r0 = threadIdx.x; r0 < a.rows; r0 += kMeanBlock * kMeanRows) {
    float l[kMeanRows], ok[kMeanRows];
#pragma unroll
    for (int j = 0; j < kMeanRows; ++j) {
      const int64_t r = r0 + (int64_t)j * kMeanBlock;
      const bool in = r < a.rows;
      ok[j] = in && a.target[r] != a.ignore_index ? 1.f : 0.f;
      l[j] = in ? a.rowloss[r] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kMeanRows; ++j) sum += l[j], count += ok[j];
  }
  write_mean(a, sum, count, red);
}

// Both, by one workgroup, where rows are few: a launch less.
template <typename T>
__global__ __launch_bounds__(kMeanBlock) void distill_finish_all_kernel(DistillArgs a) {
  extern __shared__ int lds[];
  __shared__ float red[kMeanBlock / kWave];
  const int wave = threadIdx.x >> 6;
  float sum = 0.f, count = 0.f;
  for (int64_t row = wave; row < a.rows; row += kMeanBlock / kWave) {
    const float loss = finish_row<T>(a, row, lds + wave * (2 * a.slots + 3 * a.k));
    if ((threadIdx.x & 63) == 0) {
      sum += loss;
      count += a.target[row] != a.ignore_index ? 1.f : 0.f;
    }
  }
  write_mean(a, sum, count, red);
}

// What a row's gradient takes: dz = g1 exp(z - m) + gt exp((z - m) / tau), less what its entries
// and target have.
struct RowGrad {
  float m, g1, gt;
  bool live;
};
__device__ __forceinline__ RowGrad row_grad(const DistillArgs& a, int64_t row, float gh, float gp) {
  RowGrad g;
  g.live = a.target[row] != a.ignore_index;
  const float* s = a.stats + row * 4;
  g.m = s[0], g.g1 = gh * s[1], g.gt = gp * s[2];
  return g;
}

// The matrix as one run of packs, kFlatPer a workgroup (rowwise.hpp). What entries and targets
// take from its columns is laid out in LDS, while the packs are on their way: entries of a column
// are one (finish_row), so that a place has two addends at most and their order does not matter.
// MANY: rows of fewer than kFlatPer packs.
template <typename T, int VEC, bool RAG, int E, bool MANY>
__global__ __launch_bounds__(kFlatBlock) void distill_bwd_kernel(DistillArgs a) {
  __shared__ __attribute__((aligned(16))) float terms[kFlatPer * VEC];
  constexpr bool NT = VEC * sizeof(T) == 16;
  const unsigned ppr = (a.cols + VEC - 1) / VEC;  // packs per row
  const int64_t npack = a.rows * ppr, first = (int64_t)blockIdx.x * kFlatPer;
  const int64_t row0 = npack >> 32 ? first / ppr : (unsigned)first / ppr;
  const unsigned in0 = (unsigned)(first - row0 * ppr);  // the workgroup's first pack in its row
  const int64_t last = min(first + kFlatPer, npack) - 1;
  const int rows = 1 + (MANY ? (int)((in0 + (unsigned)(last - first)) / ppr)
                             : in0 + (unsigned)(last - first) >= ppr ? 1 : 0);
  const float scale = a.dloss[0] / a.n_valid[0];
  const float gh = scale * a.hard, gp = scale * a.soft * a.tau;
  // this thread's first entry
  const int64_t e0 = row0 * a.k;
  const int n = rows * a.k;
  float p0 = 0.f;
  int64_t id0 = -1;
  if ((int)threadIdx.x < n) p0 = a.probs[e0 + threadIdx.x], id0 = entry_id(a, e0 + threadIdx.x);
  RowGrad g[MANY ? kFlatUnroll : 2];
  if constexpr (!MANY) {
    g[0] = row_grad(a, row0, gh, gp);
    g[1] = rows > 1 ? row_grad(a, row0 + 1, gh, gp) : g[0];
  }
  float v[kFlatUnroll][VEC];
  unsigned at[kFlatUnroll], pack[kFlatUnroll];  // row, counted from row0, and pack in it
#pragma unroll
  for (int u = 0; u < kFlatUnroll; ++u) {
    const unsigned q = in0 + u * kFlatBlock + threadIdx.x;
    at[u] = MANY ? q / ppr : q >= ppr ? 1 : 0;
    pack[u] = q - at[u] * ppr;
    if (first + u * kFlatBlock + threadIdx.x > last) continue;
    if constexpr (MANY) g[u] = row_grad(a, row0 + at[u], gh, gp);
    if (MANY ? g[u].live : at[u] ? g[1].live : g[0].live)
      rowwise::load_pack<T, VEC, NT && !RAG, RAG>((const T*)a.logits + (row0 + at[u]) * a.cols, pack[u] * VEC,
                                          a.cols, 0.f, v[u]);
  }
  float* own[kFlatUnroll];
#pragma unroll
  for (int u = 0; u < kFlatUnroll; ++u) {
    own[u] = terms + (u * kFlatBlock + threadIdx.x) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) own[u][i] = 0.f;
  }
  __syncthreads();
  // takes `value` from a column of row r (from row0)
  auto take = [&](int r, int64_t id64, float value) {
    if (id64 < 0 || id64 >= a.cols) return;
    const int id = (int)id64;
    const int64_t row = (int64_t)r * ppr - in0;  // its first pack, from the workgroup's first
    const int64_t k = row + id / VEC;
    if (RAG && id >= a.cols - VEC) {  // the last pack, which overlaps the one before it
      const int64_t l = row + ppr - 1;
      if (l >= 0 && l < kFlatPer) atomicAdd(&terms[l * VEC + id - (a.cols - VEC)], value);
      if (id / VEC == (int)ppr - 1) return;
    }
    if (k >= 0 && k < kFlatPer) atomicAdd(&terms[k * VEC + id % VEC], value);
  };
  if (p0 != 0.f) take((int)threadIdx.x / a.k, id0, gp * p0);
  for (int i = threadIdx.x + kFlatBlock; i < n; i += kFlatBlock) {
    const float p = a.probs[e0 + i];
    if (p != 0.f) take(i / a.k, entry_id(a, e0 + i), gp * p);
  }
  if (a.hard != 0.f)
    for (int r = threadIdx.x; r < rows; r += kFlatBlock) take(r, a.target[row0 + r], gh);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kFlatUnroll; ++u) {
    if (first + u * kFlatBlock + threadIdx.x > last) continue;
    const RowGrad& r = g[MANY ? u : at[u] ? 1 : 0];
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = 0.f;
    if (r.live) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float e1, et;
        exps<E>(a, v[u][i] - r.m, e1, et);
        if constexpr (E == kOne) o[i] = __builtin_fmaf(r.g1 + r.gt, et, -own[u][i]);
        else if constexpr (E == kTwo) o[i] = __builtin_fmaf(r.g1, e1, __builtin_fmaf(r.gt, et, -own[u][i]));
        else o[i] = __builtin_fmaf(__builtin_fmaf(r.g1, et, r.gt), et, -own[u][i]);
      }
    }
    rowwise::store_pack<T, VEC, NT, RAG>((T*)a.dlogits + (row0 + at[u]) * a.cols, pack[u] * VEC, a.cols,
                                         o);
  }
}

// How the exponentials are formed; for kOne the factor of the one that is used becomes ct.
int exps_of(DistillArgs& a) {
  a.c1 = kLog2e, a.ct = kLog2e / a.tau;
  if (a.soft == 0.f) a.ct = kLog2e;
  if (a.soft == 0.f || a.hard == 0.f || a.tau == 1.f) return kOne;
  return a.tau == 2.f ? kSquare : kTwo;
}
template <typename F>
int by_exps(int e, F&& f) {
  switch (e) {
    case kOne: return f(std::integral_constant<int, kOne>{});
    case kTwo: return f(std::integral_constant<int, kTwo>{});
    default: return f(std::integral_constant<int, kSquare>{});
  }
}

int slots_for(int k) {
  int s = 64;
  while (s < 2 * k) s *= 2;
  return s;
}
size_t finish_lds(const DistillArgs& a) { return (2 * a.slots + 3 * a.k) * sizeof(int); }

// Parts of a row, where rows are few: up to the card's 1024 workgroups, of 4096 columns or more; a
// lane each in the finish. Forward of bf16 rows of 128256, us, whole / so: 1 row 17.5 / 9.7, 16 rows
// 21.2 / 11.6, 64 rows 24.5 / 14.3, 300 rows 31.2 / 24.6 (with up to 512 workgroups 32.8); 100 rows of
// 32000 14.4 / 12.6 (in parts of 8192 13.5), 500 of them 17.2 / 17.4.
constexpr int kMostSplits = 64;
int splits_for(int64_t rows, int64_t cols) {
  const int64_t want = 1024 / std::max<int64_t>(rows, 1), most = cols / 4096;
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kMostSplits}));
}

template <typename T, int VEC, bool RAG, int E>
struct RowLaunch {
  const DistillArgs& a;
  hipStream_t st;
  template <int BLOCK>
  void go() {
    EG_LAUNCH((distill_row_kernel<T, VEC, BLOCK, RAG, E>), dim3((unsigned)a.rows, a.splits),
              dim3(BLOCK), 0, st, a);
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
  // farther out its square or the logits' quotients leave fp32, and the loss would be NaN
  if (!(temperature >= 0x1p-100f && temperature <= 0x1p60f)) {
    set_error("%s: temperature must be positive, from 2^-100 to 2^60", name);
    return 1;
  }
  return 0;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" size_t eg_topk_distill_workspace_bytes(int64_t rows, int64_t cols, int64_t entries) {
  if (rows <= 0 || cols <= 0 || entries < 0) return 0;
  return (size_t)rows * (1 + 3 * splits_for(rows, cols) + entries) * sizeof(float);
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
  a.zs = a.part + rows * 3 * splits_for(rows, cols);
  a.rows = rows, a.cols = (int)cols, a.ignore_index = ignore_index;
  a.k = soft_weight != 0.f ? (int)entries : 0;  // else they have no part
  a.slots = slots_for(a.k), a.splits = splits_for(rows, cols), a.ids_64 = ids_64;
  a.teacher_type = teacher_dtype;
  a.tau = temperature, a.soft = soft_weight, a.hard = hard_weight;
  hipStream_t st = as_stream(stream);
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    using T = scalar_t;
    if (rows) {
      if (check_grid(name, rows, 1024)) return 1;
      by_exps(exps_of(a), [&](auto e) {
        return by_width<T>(cols, {logits}, [&](auto vec, auto rag) {
          constexpr int V = decltype(vec)::value;
          const int64_t packs = ((cols + V - 1) / V + a.splits - 1) / a.splits;
          RowLaunch<T, V, decltype(rag)::value, decltype(e)::value> row{a, st};
          const int64_t threads = (packs + kUnroll * kRowSteps - 1) / (kUnroll * kRowSteps);
          if (threads <= 64) row.template go<64>();
          else if (threads <= 128) row.template go<128>();
          else if (threads <= 256) row.template go<256>();
          else row.template go<kMostRow>();
          return 0;
        });
      });
      const size_t lds = finish_lds(a);
      if (rows <= kFewRows && kMeanBlock / kWave * lds <= 65536) {
        EG_LAUNCH((distill_finish_all_kernel<T>), dim3(1), dim3(kMeanBlock), kMeanBlock / kWave * lds, st,
                  a);
        return check_launch(name);
      }
      EG_LAUNCH((distill_finish_kernel<T>), dim3((unsigned)rows), dim3(kWave), lds, st, a);
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
  a.rows = rows, a.cols = (int)cols, a.ignore_index = ignore_index;
  a.k = soft_weight != 0.f ? (int)entries : 0;  // else they have no part
  a.ids_64 = ids_64, a.tau = temperature, a.soft = soft_weight, a.hard = hard_weight;
  const int exponentials = exps_of(a);
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    using T = scalar_t;
    return by_width<T>(cols, {logits, (const void*)dlogits}, [&](auto vec, auto rag) -> int {
      constexpr int V = decltype(vec)::value;
      constexpr bool R = decltype(rag)::value;
      const int64_t ppr = (cols + V - 1) / V, blocks = (rows * ppr + kFlatPer - 1) / kFlatPer;
      if (check_grid(name, blocks, kFlatBlock)) return 1;
      return by_exps(exponentials, [&](auto e) -> int {
        const dim3 grid((unsigned)blocks), block(kFlatBlock);
        if (ppr >= kFlatPer)
          EG_LAUNCH((distill_bwd_kernel<T, V, R, decltype(e)::value, false>), grid, block, 0,
                    as_stream(stream), a);
        else
          EG_LAUNCH((distill_bwd_kernel<T, V, R, decltype(e)::value, true>), grid, block, 0,
                    as_stream(stream), a);
        return check_launch(name);
      });
    });
  });
}
