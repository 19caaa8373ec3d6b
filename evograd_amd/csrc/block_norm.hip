// The norms around a block for gfx950, fused with its gate, residual scale and residual:
//
//   n = h rstd_h w1            (RMSNorm of the block's output, gain w1)
//   s = x + alpha g n          (residual stream; gate g per channel, row or element, or 1)
//   y = s rstd_s w2            (RMSNorm before the next block, gain w2)
// rstd = rsqrt(mean(.^2) + eps), everything in fp32 and each output rounded once; y is
// formed from the unrounded s. Backward, with hhat = h rstd_h, shat = s rstd_s:
//   e  = ds + rstd_s (dy w2 - shat mean(dy w2 shat))         dx = e
//   dn = alpha g e
//   dh = rstd_h (dn w1 - hhat mean(dn w1 hhat))
//   dw1 = sum over rows of dn hhat,  dw2 = sum over rows of dy shat
//   dg = alpha e n, summed over the rows (channel), the columns (row) or not at all
// s is formed again from x and h: the same bytes as reading a saved s, and unrounded. A
// gate per channel shares its column sum with w1: with C = sum alpha e hhat, dw1 = g C and
// dg = w1 C.
//
// Memory-bound: the forward reads x and h and writes s and y, the backward reads x, h, ds
// and dy and writes dx and dh. A row stays in its workgroup's registers between the two
// reductions, so each element is moved once. The backward's workgroups walk the rows in
// steps of the grid and keep the column sums of their rows in registers; they leave one
// partial row each, which a second kernel adds in order (no atomics).
//
// Kernel times, forward + backward + column sums: bf16 [16384, 4096] with a gate per channel
// 100 + 148 + 8 us, the backward at 5.4 TB/s, behind two dependent row sums; bf16 [4099, 1538]
// with a gate per element 14.4 + 26.5 + 5.9 us, the backward at 3.8 TB/s on unaligned packs; fp32
// [64, 768] 3.8 + 4.3 + 3.3 us, launches. Without the backward's loads of the next row under
// the present one the first took 393 us a step instead of 273, before the non-temporal
// accesses (240 to 244 with them).
#include "eg_common.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

enum Gate { kNone, kChannel, kRow, kElement };

struct NormArgs {
  const void *x, *h, *w1, *gate, *w2;
  void *s, *y;
  float* rstd;  // [2][rows]: of h, of s
  const void *ds, *dy;
  void *dx, *dh, *dw1, *dgate, *dw2;
  float* part;  // [workgroups][2][cols]
  int64_t rows;
  int cols;
  float alpha, eps;
};

// A pack of a row: whole 16-byte packs, or (RAG) packs at any element, the last of a row
// overlapping its neighbour (eg_common.hpp); VEC = 1 takes elements.
template <typename T, int VEC, bool RAG>
struct RowPack {
  int c, lo;
  bool in;
  __device__ __forceinline__ void set(int pack, int cols) {
    const int at = pack * VEC;
    in = at < cols;
    c = at, lo = 0;
    if constexpr (RAG) {
      const RaggedPack p = ragged_pack<VEC>(in ? at : 0, cols);
      c = p.c, lo = p.lo;
    }
    if (!in) c = 0;
  }
  // zeros where the pack's elements are not its own, so sums skip them
  __device__ __forceinline__ void load(const void* row, float (&v)[VEC]) const {
    if (!in) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = 0.f;
      return;
    }
    if constexpr (RAG) {
      load_ragged<T, VEC, false>((const T*)row + c, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = i < lo ? 0.f : v[i];
    } else {
      load_f32<T, VEC>((const T*)row + c, v);
    }
  }
  __device__ __forceinline__ void store(void* row, const float (&v)[VEC]) const {
    if (!in) return;
    if constexpr (RAG) store_ragged<T, VEC, true>((T*)row + c, lo, v);
    else store_vec<T, VEC, true>((T*)row + c, v);
  }
};

// Sum over the workgroup, in wave order. One barrier: a kernel gives each of its sums a buffer
// of its own, and another sum's barrier lies between two uses of one.
__device__ __forceinline__ float row_sum(float v, float* lds) {
  v = wave_reduce(v, SumOp());
  const int waves = blockDim.x / 64;
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = lds[0];
  for (int w = 1; w < waves; ++w) r += lds[w];
  return r;
}

template <typename T>
__device__ __forceinline__ const void* row_of(const void* p, int64_t row, int cols) {
  return (const T*)p + row * cols;
}
template <typename T>
__device__ __forceinline__ void* row_of(void* p, int64_t row, int cols) {
  return (T*)p + row * cols;
}

// A workgroup per row, PPT packs per thread: pack p of thread t is p * threads + t.
constexpr int kFwdThreads = 256, kBwdThreads = 512;

template <typename T, int VEC, int PPT, bool RAG, int GATE>
__global__ __launch_bounds__(kFwdThreads) void block_norm_fwd_kernel(NormArgs a) {
  __shared__ float red[2][kFwdThreads / 64];
  const int64_t row = blockIdx.x;
  const int cols = a.cols;
  RowPack<T, VEC, RAG> at[PPT];
  float h[PPT][VEC], x[PPT][VEC];
#pragma unroll
  for (int p = 0; p < PPT; ++p) {
    at[p].set(threadIdx.x + p * blockDim.x, cols);
    at[p].load(row_of<T>(a.h, row, cols), h[p]);
  }
#pragma unroll
  for (int p = 0; p < PPT; ++p) at[p].load(row_of<T>(a.x, row, cols), x[p]);
  float scale = a.alpha;
  if (GATE == kRow) scale *= to_f32(((const T*)a.gate)[row]);
  float sum = 0.f;
#pragma unroll
  for (int p = 0; p < PPT; ++p)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += h[p][i] * h[p][i];
  const float rh = rsqrtf(row_sum(sum, red[0]) / cols + a.eps);
  sum = 0.f;
#pragma unroll
  for (int p = 0; p < PPT; ++p) {
    float w[VEC], g[VEC];
    at[p].load(a.w1, w);
    if (GATE == kChannel) at[p].load(a.gate, g);
    if (GATE == kElement) at[p].load(row_of<T>(a.gate, row, cols), g);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float n = h[p][i] * rh * w[i];
      x[p][i] += GATE == kChannel || GATE == kElement ? scale * g[i] * n : scale * n;
      sum += x[p][i] * x[p][i];
    }
    at[p].store(row_of<T>(a.s, row, cols), x[p]);
  }
  const float rs = rsqrtf(row_sum(sum, red[1]) / cols + a.eps);
#pragma unroll
  for (int p = 0; p < PPT; ++p) {
    float w[VEC];
    at[p].load(a.w2, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[p][i] = x[p][i] * rs * w[i];
    at[p].store(row_of<T>(a.y, row, cols), x[p]);
  }
  if (threadIdx.x == 0) {
    a.rstd[row] = rh;
    a.rstd[a.rows + row] = rs;
  }
}

// A row's packs as they lie in memory: the backward loads the next row's while it works on
// this one's, in half the registers (16-bit types) that fp32 values take.
template <typename T, int VEC, int PPT, bool RAG, bool NT>
struct RawRow {
  Pack<T, VEC> v[PPT];
  __device__ __forceinline__ void load(const RowPack<T, VEC, RAG> (&at)[PPT], const void* row) {
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      if (!at[p].in) continue;
      if constexpr (RAG || NT) v[p] = load_ragged_raw<T, VEC, NT>((const T*)row + at[p].c);
      else v[p] = *reinterpret_cast<const Pack<T, VEC>*>((const T*)row + at[p].c);
    }
  }
  __device__ __forceinline__ void get(const RowPack<T, VEC, RAG> (&at)[PPT], int p,
                                      float (&f)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = at[p].in && i >= at[p].lo ? to_f32(v[p].v[i]) : 0.f;
  }
};

// One pack per thread up to 256 packs, then two, on up to 512 threads: a CU's registers hold
// the values of three or four rows, and of the rows after them, either way. Whole 16-bit packs,
// one a thread, are held to four waves per SIMD's registers, which spills 7 of them with a channel
// gate, 1 to 3 with a row's and 16 with an element's. At three waves (bf16, backward): [8192, 2048]
// 53 -> 48 us, 50 -> 49 and 63 -> 51, but [4099, 1536] 32 -> 34, 30 -> 37 and 36 -> 35.
template <typename T, int VEC, int PPT, bool RAG, bool NT, int GATE>
__global__ __launch_bounds__(PPT == 1 ? kBwdThreads / 2 : kBwdThreads,
                             PPT == 2 ? 2 : RAG ? 3 : 4) void block_norm_bwd_kernel(NormArgs a) {
  __shared__ float red[3][kBwdThreads / 64];
  const int cols = a.cols;
  RowPack<T, VEC, RAG> at[PPT];
#pragma unroll
  for (int p = 0; p < PPT; ++p) at[p].set(threadIdx.x + p * blockDim.x, cols);
  RawRow<T, VEC, PPT, RAG, false> w1, w2, gate;
  RawRow<T, VEC, PPT, RAG, NT> rawg, rawh, rawx, rawdy, rawds;
  w1.load(at, a.w1);
  w2.load(at, a.w2);
  if (GATE == kChannel) gate.load(at, a.gate);
  auto fetch = [&](int64_t row) {
    rawh.load(at, row_of<T>(a.h, row, cols));
    rawx.load(at, row_of<T>(a.x, row, cols));
    rawdy.load(at, row_of<T>(a.dy, row, cols));
    rawds.load(at, row_of<T>(a.ds, row, cols));
    if (GATE == kElement) rawg.load(at, row_of<T>(a.gate, row, cols));
  };
  // the gate of a pack's columns in the present row
  auto gates = [&](int p, float grow, float (&g)[VEC]) {
    if constexpr (GATE == kChannel || GATE == kElement) {
      gate.get(at, p, g);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[i] = grow;
    }
  };
  float acc1[PPT][VEC], acc2[PPT][VEC];
#pragma unroll
  for (int p = 0; p < PPT; ++p)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc1[p][i] = acc2[p][i] = 0.f;
  fetch(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float rh = a.rstd[row], rs = a.rstd[a.rows + row];
    const float grow = GATE == kRow ? to_f32(((const T*)a.gate)[row]) : 1.f;
    float hhat[PPT][VEC], shat[PPT][VEC], e[PPT][VEC], dyw[PPT][VEC];
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      rawh.get(at, p, hhat[p]);
      rawx.get(at, p, shat[p]);
      rawdy.get(at, p, dyw[p]);
      rawds.get(at, p, e[p]);
    }
    if constexpr (GATE == kElement) {
#pragma unroll
      for (int p = 0; p < PPT; ++p) gate.v[p] = rawg.v[p];
    }
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      float w[VEC], v[VEC], g[VEC];
      w1.get(at, p, w);
      w2.get(at, p, v);
      gates(p, grow, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        hhat[p][i] *= rh;
        shat[p][i] = (shat[p][i] + a.alpha * g[i] * (hhat[p][i] * w[i])) * rs;
        acc2[p][i] += dyw[p][i] * shat[p][i];
        dyw[p][i] *= v[i];
        sum += dyw[p][i] * shat[p][i];
      }
    }
    const float m1 = row_sum(sum, red[0]) / cols;
    float dot = 0.f, dgrow = 0.f;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
      float w[VEC], g[VEC], dg[VEC];
      w1.get(at, p, w);
      gates(p, grow, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        e[p][i] += rs * (dyw[p][i] - shat[p][i] * m1);
        const float ae = a.alpha * e[p][i];
        dyw[p][i] = g[i] * ae * w[i];  // dn w1 from here on
        dot += dyw[p][i] * hhat[p][i];
        acc1[p][i] += (GATE == kChannel ? ae : g[i] * ae) * hhat[p][i];
        dg[i] = ae * (hhat[p][i] * w[i]);
        dgrow += dg[i];
      }
      at[p].store(row_of<T>(a.dx, row, cols), e[p]);
      if (GATE == kElement) at[p].store(row_of<T>(a.dgate, row, cols), dg);
    }
    if (GATE == kRow) {
      dgrow = row_sum(dgrow, red[2]);
      if (threadIdx.x == 0) ((T*)a.dgate)[row] = from_f32<T>(dgrow);
    }
    const float m2 = row_sum(dot, red[1]) / cols;
#pragma unroll
    for (int p = 0; p < PPT; ++p) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) dyw[p][i] = rh * (dyw[p][i] - hhat[p][i] * m2);
      at[p].store(row_of<T>(a.dh, row, cols), dyw[p]);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int p = 0; p < PPT; ++p) {
    if (!at[p].in) continue;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= at[p].lo) {
        part[at[p].c + i] = acc1[p][i];
        part[cols + at[p].c + i] = acc2[p][i];
      }
  }
}

// Rows too wide for a workgroup's registers: the row is read again for every reduction (from
// L2: a workgroup's row is at most a few hundred KB), and the backward's column sums are kept
// in the workgroup's partial row, where each column belongs to one thread. With a gate per channel
// fp32 [8192, 8192] takes 240 us forward and 753 backward, bf16 [8192, 16384] 292 and 1519, where the
// bytes take 174 and 261.
constexpr int kWideBlock = 1024;

template <typename T, int VEC, int GATE>
struct WideRow {
  const NormArgs& a;
  int64_t row;
  float rh, scale;  // scale: alpha, times a row's gate
  __device__ __forceinline__ void gate(const RowPack<T, VEC, true>& at, float (&g)[VEC]) const {
    if constexpr (GATE == kChannel) at.load(a.gate, g);
    else if constexpr (GATE == kElement) at.load(row_of<T>(a.gate, row, a.cols), g);
    else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[i] = 1.f;
    }
  }
  // hhat, w1, the gate and the residual stream of one pack
  __device__ __forceinline__ void stream(const RowPack<T, VEC, true>& at, float (&hhat)[VEC],
                                         float (&w)[VEC], float (&g)[VEC], float (&s)[VEC]) const {
    at.load(row_of<T>(a.h, row, a.cols), hhat);
    at.load(row_of<T>(a.x, row, a.cols), s);
    at.load(a.w1, w);
    gate(at, g);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      hhat[i] *= rh;
      s[i] += scale * g[i] * (hhat[i] * w[i]);
    }
  }
};

template <typename T, int VEC, int GATE>
__global__ __launch_bounds__(kWideBlock) void block_norm_fwd_wide_kernel(NormArgs a) {
  __shared__ float red[kWideBlock / 64];
  const int64_t row = blockIdx.x;
  const int cols = a.cols, packs = (cols + VEC - 1) / VEC;
  RowPack<T, VEC, true> at;
  float sum = 0.f;
  for (int p = threadIdx.x; p < packs; p += kWideBlock) {
    float v[VEC];
    at.set(p, cols);
    at.load(row_of<T>(a.h, row, cols), v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += v[i] * v[i];
  }
  WideRow<T, VEC, GATE> r{a, row, 0.f, a.alpha};
  if (GATE == kRow) r.scale *= to_f32(((const T*)a.gate)[row]);
  r.rh = rsqrtf(block_reduce<kWideBlock>(sum, SumOp(), red) / cols + a.eps);
  sum = 0.f;
  float hhat[VEC], w[VEC], g[VEC], s[VEC];
  for (int p = threadIdx.x; p < packs; p += kWideBlock) {
    at.set(p, cols);
    r.stream(at, hhat, w, g, s);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += s[i] * s[i];
  }
  const float rs = rsqrtf(block_reduce<kWideBlock>(sum, SumOp(), red) / cols + a.eps);
  for (int p = threadIdx.x; p < packs; p += kWideBlock) {
    at.set(p, cols);
    r.stream(at, hhat, w, g, s);
    at.store(row_of<T>(a.s, row, cols), s);
    at.load(a.w2, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[i] = s[i] * rs * w[i];
    at.store(row_of<T>(a.y, row, cols), s);
  }
  if (threadIdx.x == 0) {
    a.rstd[row] = r.rh;
    a.rstd[a.rows + row] = rs;
  }
}

template <typename T, int VEC, int GATE>
__global__ __launch_bounds__(kWideBlock) void block_norm_bwd_wide_kernel(NormArgs a) {
  __shared__ float red[kWideBlock / 64];
  const int cols = a.cols, packs = (cols + VEC - 1) / VEC;
  float* part = a.part + (int64_t)blockIdx.x * 2 * cols;
  RowPack<T, VEC, true> at;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const bool first = row == blockIdx.x;
    WideRow<T, VEC, GATE> r{a, row, a.rstd[row], a.alpha};
    const float rs = a.rstd[a.rows + row];
    const float grow = GATE == kRow ? to_f32(((const T*)a.gate)[row]) : 1.f;
    r.scale *= grow;
    float hhat[VEC], w[VEC], g[VEC], s[VEC], dy[VEC], v[VEC], e[VEC];
    float sum = 0.f;
    for (int p = threadIdx.x; p < packs; p += kWideBlock) {
      at.set(p, cols);
      r.stream(at, hhat, w, g, s);
      at.load(row_of<T>(a.dy, row, cols), dy);
      at.load(a.w2, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum += dy[i] * v[i] * (s[i] * rs);
    }
    const float m1 = block_reduce<kWideBlock>(sum, SumOp(), red) / cols;
    // e of a pack, and shat and dy beside it
    auto upstream = [&] {
      r.stream(at, hhat, w, g, s);
      at.load(row_of<T>(a.dy, row, cols), dy);
      at.load(row_of<T>(a.ds, row, cols), e);
      at.load(a.w2, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        s[i] *= rs;
        e[i] += rs * (dy[i] * v[i] - s[i] * m1);
      }
    };
    float dot = 0.f, dgrow = 0.f;
    for (int p = threadIdx.x; p < packs; p += kWideBlock) {
      at.set(p, cols);
      upstream();
      at.store(row_of<T>(a.dx, row, cols), e);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float ae = a.alpha * e[i], dn = grow * g[i] * ae;
        dot += dn * w[i] * hhat[i];
        dgrow += ae * (hhat[i] * w[i]);
        if (i >= at.lo) {
          float* c = part + at.c + i;
          const float p1 = (GATE == kChannel ? ae : dn) * hhat[i], p2 = dy[i] * s[i];
          c[0] = first ? p1 : c[0] + p1;
          c[cols] = first ? p2 : c[cols] + p2;
        }
        e[i] = ae * (hhat[i] * w[i]);
      }
      if (GATE == kElement) at.store(row_of<T>(a.dgate, row, cols), e);
    }
    if (GATE == kRow) {
      dgrow = block_reduce<kWideBlock>(dgrow, SumOp(), red);
      if (threadIdx.x == 0) ((T*)a.dgate)[row] = from_f32<T>(dgrow);
    }
    const float m2 = block_reduce<kWideBlock>(dot, SumOp(), red) / cols;
    for (int p = threadIdx.x; p < packs; p += kWideBlock) {
      at.set(p, cols);
      upstream();
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        e[i] = r.rh * (grow * g[i] * (a.alpha * e[i]) * w[i] - hhat[i] * m2);
      at.store(row_of<T>(a.dh, row, cols), e);
    }
  }
}

// dw1, dw2 and a channel gate's gradient from the workgroups' partial rows: 16 columns (a
// 64-byte run of each row) per workgroup, its rows dealt to 64 adders whose sums are added
// in order.
constexpr int kSumCols = 16, kSumRows = 64;
template <typename T, int GATE>
__global__ __launch_bounds__(kSumCols * kSumRows) void block_norm_sum_kernel(NormArgs a, int parts) {
  __shared__ float sums[2][kSumRows][kSumCols];
  const int lane = threadIdx.x % kSumCols, adder = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + lane;
  float s1 = 0.f, s2 = 0.f;
  if (c < a.cols) {
    const float* p = a.part + c;
#pragma unroll 4
    for (int r = adder; r < parts; r += kSumRows) {
      s1 += p[(int64_t)r * 2 * a.cols];
      s2 += p[((int64_t)r * 2 + 1) * a.cols];
    }
  }
  sums[0][adder][lane] = s1;
  sums[1][adder][lane] = s2;
  __syncthreads();
#pragma unroll
  for (int n = kSumRows / 2; n >= 1; n /= 2) {
    if (adder < n) {
      sums[0][adder][lane] = s1 += sums[0][adder + n][lane];
      sums[1][adder][lane] = s2 += sums[1][adder + n][lane];
    }
    __syncthreads();
  }
  if (adder != 0 || c >= a.cols) return;
  if (GATE == kChannel) {
    ((T*)a.dgate)[c] = from_f32<T>(s1 * to_f32(((const T*)a.w1)[c]));
    s1 *= to_f32(((const T*)a.gate)[c]);
  }
  ((T*)a.dw1)[c] = from_f32<T>(s1);
  ((T*)a.dw2)[c] = from_f32<T>(s2);
}

constexpr int64_t kMaxCols = (int64_t)1 << 24;

// Packs per thread and threads of a row's workgroup, whole waves. Rows of more than 1024 packs
// (8192 16-bit columns, 4096 fp32) take the wide kernels.
constexpr int64_t kRowPacks = 1024;
struct RowShape {
  int ppt, threads;
};
RowShape row_shape(int64_t cols, int vec, bool backward) {
  const int64_t packs = (cols + vec - 1) / vec;
  RowShape r = {packs <= 256 ? 1 : backward || packs <= 512 ? 2 : 4, 0};
  r.threads = (int)((packs + 64 * r.ppt - 1) / (64 * r.ppt)) * 64;
  return r;
}
// Past this size of one tensor its six do not fit the 256 MB last-level cache twice over, and
// the backward reads them with the non-temporal hint: bf16 [16384, 4096] step 261 -> 248 us,
// [8192, 8192] 307 -> 294; fp16 [8192, 5000] would go 222 -> 240.
constexpr int64_t kStreamBytes = 96 << 20;
// Workgroups of the backward, a partial row each: as many whole ones as are resident at once, for
// they walk the rows in steps of the grid and a second round of a few would leave the others'
// CUs idle. The 16-bit kernels' registers allow three waves per SIMD with one pack a thread
// (four without RAG and an element's gate, which gain nothing) and two with two packs: 12 and 8
// per CU. Against 16 and 8 without counting whole workgroups (step times, bf16): [4099, 1538] 51
// -> 44 us, [2048, 2050] 57 -> 45, [6000, 6001] 336 -> 273, [8192, 1024] fp16 70 -> 62,
// [16384, 4096] the same; fp32 [5000, 1027] 50 -> 52. At most 2048, whose partial rows the sum
// kernel reads in a few us.
int64_t parts_for(int64_t rows, int64_t cols, int vec) {
  if (cols > kRowPacks * vec) return std::min<int64_t>(rows, 512);
  const RowShape r = row_shape(cols, vec, true);
  const int64_t resident = (r.ppt == 1 ? 12 : 8) / (r.threads / 64);
  return std::min<int64_t>({rows, 2048, 256 * std::max<int64_t>(resident, 1)});
}

// go(VEC, RAG) for a row that a workgroup's registers hold, else wide(VEC).
template <typename T, typename F, typename W>
int by_shape(const NormArgs& a, F&& go, W&& wide) {
  using std::integral_constant;
  constexpr int V = 16 / (int)sizeof(T);
  if (a.cols < V) return go(integral_constant<int, 1>{}, std::false_type{});
  bool aligned = a.cols % V == 0;
  for (const void* p : {a.x, a.h, a.w1, a.gate, a.w2, (const void*)a.s, (const void*)a.y, a.ds, a.dy,
                        (const void*)a.dx, (const void*)a.dh, (const void*)a.dgate})
    aligned = aligned && aligned16(p);
  const integral_constant<int, V> vec;
  if (a.cols > kRowPacks * V) return wide(vec);
  return aligned ? go(vec, std::false_type{}) : go(vec, std::true_type{});
}

template <typename F>
int by_gate(int gate, F&& f) {
  switch (gate) {
    case kChannel: return f(std::integral_constant<int, kChannel>{});
    case kRow: return f(std::integral_constant<int, kRow>{});
    case kElement: return f(std::integral_constant<int, kElement>{});
    default: return f(std::integral_constant<int, kNone>{});
  }
}

int check(const char* name, int64_t rows, int64_t cols, int gate) {
  if (rows < 0 || cols < 0) { set_error("%s: negative size", name); return 1; }
  if (rows > ((int64_t)1 << 30) || cols > kMaxCols) {
    set_error("%s: size out of range (rows <= 1073741824, cols <= %lld)", name,
              (long long)kMaxCols);
    return 1;
  }
  if (gate < kNone || gate > kElement) { set_error("%s: unknown gate kind %d", name, gate); return 1; }
  return 0;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" size_t eg_block_norm_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  // the narrower packs (fp32) of the dtype not known here have the wider workgroups
  return (size_t)std::max(parts_for(rows, cols, 4), parts_for(rows, cols, 8)) * 2 * cols *
         sizeof(float);
}

extern "C" int eg_block_norm_fwd(const void* x, const void* h, const void* post_weight,
                                 const void* gate, const void* pre_weight, void* s, void* y,
                                 float* rstd, int64_t rows, int64_t cols, int gate_kind,
                                 float alpha, float eps, int dtype, void* stream) {
  static const char* name = "eg_block_norm_fwd";
  clear_error();
  if (check(name, rows, cols, gate_kind)) return 1;
  if (rows == 0 || cols == 0) return 0;
  if (!x || !h || !post_weight || !pre_weight || !s || !y || !rstd || (gate_kind && !gate)) {
    set_error("%s: null pointer", name);
    return 1;
  }
  NormArgs a = {};
  a.x = x, a.h = h, a.w1 = post_weight, a.gate = gate, a.w2 = pre_weight;
  a.s = s, a.y = y, a.rstd = rstd;
  a.rows = rows, a.cols = (int)cols, a.alpha = alpha, a.eps = eps;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    return by_gate(gate_kind, [&](auto g) {
      return by_shape<scalar_t>(a, [&](auto vec, auto rag) {
        constexpr int V = decltype(vec)::value, G = decltype(g)::value;
        const RowShape r = row_shape(cols, V, false);
        if (check_grid(name, rows, r.threads)) return 1;
        auto go = [&](auto ppt) {
          EG_LAUNCH((block_norm_fwd_kernel<scalar_t, V, decltype(ppt)::value, decltype(rag)::value, G>),
                    dim3((unsigned)rows), dim3(r.threads), 0, as_stream(stream), a);
          return check_launch(name);
        };
        if constexpr (V > 1) {
          if (r.ppt == 4) return go(std::integral_constant<int, 4>{});
          if (r.ppt == 2) return go(std::integral_constant<int, 2>{});
        }
        return go(std::integral_constant<int, 1>{});
      }, [&](auto vec) {
        constexpr int V = decltype(vec)::value, G = decltype(g)::value;
        if (check_grid(name, rows, kWideBlock)) return 1;
        EG_LAUNCH((block_norm_fwd_wide_kernel<scalar_t, V, G>), dim3((unsigned)rows),
                  dim3(kWideBlock), 0, as_stream(stream), a);
        return check_launch(name);
      });
    });
  });
}

extern "C" int eg_block_norm_bwd(const void* ds, const void* dy, const void* x, const void* h,
                                 const void* post_weight, const void* gate, const void* pre_weight,
                                 const float* rstd, void* dx, void* dh, void* dpost_weight,
                                 void* dgate, void* dpre_weight, void* workspace, int64_t rows,
                                 int64_t cols, int gate_kind, float alpha, int dtype,
                                 void* stream) {
  static const char* name = "eg_block_norm_bwd";
  clear_error();
  if (check(name, rows, cols, gate_kind)) return 1;
  if (cols == 0) {  // nothing but a row gate's gradient, a sum over no columns
    if (gate_kind != kRow) return 0;
    if (dtype != EG_F32 && dtype != EG_F16 && dtype != EG_BF16) {
      set_error("%s: unsupported dtype %d", name, dtype);
      return 1;
    }
    return zero_fill(dgate, (size_t)rows * (dtype == EG_F32 ? 4 : 2), as_stream(stream), name);
  }
  // without rows the weights' gradients (and a channel gate's) are zero, and nothing is read
  const bool gated = gate_kind == kChannel || (gate_kind && rows > 0);
  if (!dpost_weight || !dpre_weight || !post_weight || !pre_weight || (gated && (!gate || !dgate))) {
    set_error("%s: null pointer", name);
    return 1;
  }
  if (rows > 0 && (!ds || !dy || !x || !h || !rstd || !dx || !dh || !workspace)) {
    set_error("%s: null pointer", name);
    return 1;
  }
  NormArgs a = {};
  a.x = x, a.h = h, a.w1 = post_weight, a.gate = gate, a.w2 = pre_weight;
  a.ds = ds, a.dy = dy, a.rstd = const_cast<float*>(rstd);
  a.dx = dx, a.dh = dh, a.dw1 = dpost_weight, a.dgate = dgate, a.dw2 = dpre_weight;
  a.part = (float*)workspace;
  a.rows = rows, a.cols = (int)cols, a.alpha = alpha;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    const int parts = (int)parts_for(rows, cols, 16 / (int)sizeof(scalar_t));
    return by_gate(gate_kind, [&](auto g) -> int {
      constexpr int G = decltype(g)::value;
      if (rows > 0) {
        const int rc = by_shape<scalar_t>(a, [&](auto vec, auto rag) {
          constexpr int V = decltype(vec)::value;
          const RowShape r = row_shape(cols, V, true);
          auto go = [&](auto ppt, auto nt) {
            EG_LAUNCH((block_norm_bwd_kernel<scalar_t, V, decltype(ppt)::value,
                                             decltype(rag)::value, decltype(nt)::value, G>),
                      dim3((unsigned)parts), dim3(r.threads), 0, as_stream(stream), a);
            return check_launch(name);
          };
          if constexpr (V > 1) {
            if (r.ppt == 2 && rows * cols * (int64_t)sizeof(scalar_t) > kStreamBytes)
              return go(std::integral_constant<int, 2>{}, std::true_type{});
            if (r.ppt == 2) return go(std::integral_constant<int, 2>{}, std::false_type{});
          }
          return go(std::integral_constant<int, 1>{}, std::false_type{});
        }, [&](auto vec) {
          EG_LAUNCH((block_norm_bwd_wide_kernel<scalar_t, decltype(vec)::value, G>),
                    dim3((unsigned)parts), dim3(kWideBlock), 0, as_stream(stream), a);
          return check_launch(name);
        });
        if (rc) return rc;
      }
      EG_LAUNCH((block_norm_sum_kernel<scalar_t, G>), dim3((unsigned)((cols + kSumCols - 1) / kSumCols)),
                dim3(kSumCols * kSumRows), 0, as_stream(stream), a, parts);
      return check_launch(name);
    });
  });
}
