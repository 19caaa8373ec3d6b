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
    if constexpr (RAG) store_ragged<T, VEC, false>((T*)row + c, lo, v);
    else store_f32<T, VEC>((T*)row + c, v);
  }
};

// Sum over the workgroup, in wave order. One barrier: a kernel gives each of its sums a buffer
// of its own, and another sum's barrier lies between two uses of one.
template <int BLOCK>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  v = wave_reduce(v, SumOp());
  if constexpr (BLOCK == 64) return v;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = lds[0];
#pragma unroll
  for (int w = 1; w < BLOCK / 64; ++w) r += lds[w];
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

// Workgroup of BLOCK threads per row, a pack per thread.
template <typename T, int VEC, int BLOCK, bool RAG, int GATE>
__global__ __launch_bounds__(BLOCK) void block_norm_fwd_kernel(NormArgs a) {
  __shared__ float red[2][BLOCK / 64];
  const int64_t row = blockIdx.x;
  const int cols = a.cols;
  RowPack<T, VEC, RAG> at;
  at.set(threadIdx.x, cols);
  float h[VEC], x[VEC], w[VEC], g[VEC], w2[VEC];
  at.load(row_of<T>(a.h, row, cols), h);
  at.load(row_of<T>(a.x, row, cols), x);
  at.load(a.w1, w);
  if (GATE == kChannel) at.load(a.gate, g);
  if (GATE == kElement) at.load(row_of<T>(a.gate, row, cols), g);
  at.load(a.w2, w2);
  float scale = a.alpha;
  if (GATE == kRow) scale *= to_f32(((const T*)a.gate)[row]);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum += h[i] * h[i];
  const float rh = rsqrtf(row_sum<BLOCK>(sum, red[0]) / cols + a.eps);
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float n = h[i] * rh * w[i];
    x[i] += GATE == kChannel || GATE == kElement ? scale * g[i] * n : scale * n;
    sum += x[i] * x[i];
  }
  at.store(row_of<T>(a.s, row, cols), x);
  const float rs = rsqrtf(row_sum<BLOCK>(sum, red[1]) / cols + a.eps);
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = x[i] * rs * w2[i];
  at.store(row_of<T>(a.y, row, cols), x);
  if (threadIdx.x == 0) {
    a.rstd[row] = rh;
    a.rstd[a.rows + row] = rs;
  }
}

// A row's packs as they lie in memory: the backward loads the next row's while it works on
// this one's, in a quarter (16-bit types: half) of the registers that fp32 values take.
template <typename T, int VEC, bool RAG>
struct RawPack {
  Pack<T, VEC> v;
  __device__ __forceinline__ void load(const RowPack<T, VEC, RAG>& at, const void* row) {
    if (!at.in) return;
    if constexpr (RAG) v = load_ragged_raw<T, VEC, false>((const T*)row + at.c);
    else v = *reinterpret_cast<const Pack<T, VEC>*>((const T*)row + at.c);
  }
  __device__ __forceinline__ void get(const RowPack<T, VEC, RAG>& at, float (&f)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = at.in && i >= at.lo ? to_f32(v.v[i]) : 0.f;
  }
};

template <typename T, int VEC, int BLOCK, bool RAG, int GATE>
__global__ __launch_bounds__(BLOCK) void block_norm_bwd_kernel(NormArgs a) {
  __shared__ float red[3][BLOCK / 64];
  const int cols = a.cols;
  RowPack<T, VEC, RAG> at;
  at.set(threadIdx.x, cols);
  RawPack<T, VEC, RAG> w1, w2, gate, rh_, rx, rdy, rds;
  w1.load(at, a.w1);
  w2.load(at, a.w2);
  if (GATE == kChannel) gate.load(at, a.gate);
  auto fetch = [&](int64_t row) {
    rh_.load(at, row_of<T>(a.h, row, cols));
    rx.load(at, row_of<T>(a.x, row, cols));
    rdy.load(at, row_of<T>(a.dy, row, cols));
    rds.load(at, row_of<T>(a.ds, row, cols));
    if (GATE == kElement) gate.load(at, row_of<T>(a.gate, row, cols));
  };
  float acc1[VEC], acc2[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc1[i] = acc2[i] = 0.f;
  fetch(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float rh = a.rstd[row], rs = a.rstd[a.rows + row];
    const float grow = GATE == kRow ? to_f32(((const T*)a.gate)[row]) : 1.f;
    float hhat[VEC], shat[VEC], e[VEC], dyw[VEC], g[VEC];
    rh_.get(at, hhat);
    rx.get(at, shat);
    rdy.get(at, dyw);
    rds.get(at, e);
    if (GATE == kElement) gate.get(at, g);
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
    if (GATE == kChannel) gate.get(at, g);
    float w[VEC], v[VEC], sum = 0.f;
    w1.get(at, w);
    w2.get(at, v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      hhat[i] *= rh;
      if (GATE != kChannel && GATE != kElement) g[i] = grow;
      shat[i] = (shat[i] + a.alpha * g[i] * (hhat[i] * w[i])) * rs;
      acc2[i] += dyw[i] * shat[i];
      dyw[i] *= v[i];
      sum += dyw[i] * shat[i];
    }
    const float m1 = row_sum<BLOCK>(sum, red[0]) / cols;
    float dot = 0.f, dgrow = 0.f, dg[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      e[i] += rs * (dyw[i] - shat[i] * m1);
      const float ae = a.alpha * e[i];
      dyw[i] = g[i] * ae * w[i];  // dn w1 from here on
      dot += dyw[i] * hhat[i];
      acc1[i] += (GATE == kChannel ? ae : g[i] * ae) * hhat[i];
      dg[i] = ae * (hhat[i] * w[i]);
      dgrow += dg[i];
    }
    at.store(row_of<T>(a.dx, row, cols), e);
    if (GATE == kElement) at.store(row_of<T>(a.dgate, row, cols), dg);
    if (GATE == kRow) {
      dgrow = row_sum<BLOCK>(dgrow, red[2]);
      if (threadIdx.x == 0) ((T*)a.dgate)[row] = from_f32<T>(dgrow);
    }
    const float m2 = row_sum<BLOCK>(dot, red[1]) / cols;
#pragma unroll
    for (int i = 0; i < VEC; ++i) dyw[i] = rh * (dyw[i] - hhat[i] * m2);
    at.store(row_of<T>(a.dh, row, cols), dyw);
  }
  float* part = a.part + (int64_t)blockIdx.x * 2 * cols;
  if (at.in) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i >= at.lo) {
        part[at.c + i] = acc1[i];
        part[cols + at.c + i] = acc2[i];
      }
  }
}

// Rows too wide for a workgroup's registers: the row is read again for every reduction (from
// L2: a workgroup's row is at most a few hundred KB), and the backward's column sums are kept
// in the workgroup's partial row, where each column belongs to one thread.
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

// Threads of a row's workgroup: as many as packs (up to 1024 packs: 8192 16-bit columns, 4096
// fp32), 0 where the row is too wide.
int block_of(int64_t cols, int vec) {
  const int64_t packs = (cols + vec - 1) / vec;
  for (int b = 64; b <= 1024; b *= 2)
    if (packs <= b) return b;
  return 0;
}
// Workgroups of the backward, a partial row each: about 16 waves per CU, 2048 at most, whose
// partial rows the sum kernel reads in a few us.
int64_t parts_for(int64_t rows, int64_t cols, int vec) {
  const int block = block_of(cols, vec);
  const int64_t most = block ? std::min<int64_t>(2048, 256 * 1024 / block) : 512;
  return std::min(rows, most);
}

// go(VEC, BLOCK, RAG) for a row that a workgroup's registers hold, else wide(VEC).
template <typename T, typename F, typename W>
int by_shape(const NormArgs& a, F&& go, W&& wide) {
  using std::integral_constant;
  constexpr int V = 16 / (int)sizeof(T);
  if (a.cols < V)
    return go(integral_constant<int, 1>{}, integral_constant<int, 64>{}, std::false_type{});
  bool aligned = a.cols % V == 0;
  for (const void* p : {a.x, a.h, a.w1, a.gate, a.w2, (const void*)a.s, (const void*)a.y, a.ds, a.dy,
                        (const void*)a.dx, (const void*)a.dh, (const void*)a.dgate})
    aligned = aligned && aligned16(p);
  const integral_constant<int, V> vec;
  auto by_row = [&](auto rag) -> int {
    switch (block_of(a.cols, V)) {
      case 64: return go(vec, integral_constant<int, 64>{}, rag);
      case 128: return go(vec, integral_constant<int, 128>{}, rag);
      case 256: return go(vec, integral_constant<int, 256>{}, rag);
      case 512: return go(vec, integral_constant<int, 512>{}, rag);
      case 1024: return go(vec, integral_constant<int, 1024>{}, rag);
      default: return wide(vec);
    }
  };
  return aligned ? by_row(std::false_type{}) : by_row(std::true_type{});
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
      return by_shape<scalar_t>(a, [&](auto vec, auto block, auto rag) {
        constexpr int V = decltype(vec)::value, B = decltype(block)::value, G = decltype(g)::value;
        EG_LAUNCH((block_norm_fwd_kernel<scalar_t, V, B, decltype(rag)::value, G>),
                  dim3((unsigned)rows), dim3(B), 0, as_stream(stream), a);
        return check_launch(name);
      }, [&](auto vec) {
        constexpr int V = decltype(vec)::value, G = decltype(g)::value;
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
  if (cols == 0) return 0;
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
        const int rc = by_shape<scalar_t>(a, [&](auto vec, auto block, auto rag) {
          constexpr int V = decltype(vec)::value, B = decltype(block)::value;
          EG_LAUNCH((block_norm_bwd_kernel<scalar_t, V, B, decltype(rag)::value, G>),
                    dim3((unsigned)parts), dim3(B), 0, as_stream(stream), a);
          return check_launch(name);
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
