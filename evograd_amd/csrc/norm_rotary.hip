// Norms of queries and keys for each head with the position rotation behind them, for gfx950.
//
//   n = x rstd w,  rstd = rsqrt(mean(x^2) + eps) over a head's columns
//   y = rotation of n by position * freq (amp (n1 c - n2 s, n2 c + n1 s)); columns past
//       2 * pairs are n itself
// in fp32, rounded once. Backward, with dn the transposed rotation of dy and xhat = x rstd:
//   dx = rstd (dn w - xhat mean(dn w xhat)),  dw = sum over tokens and heads of dn xhat
// rstd is formed again from x, which the backward reads anyway: its two sums over a head,
// x^2 and dn w x, do not wait for one another.
//
// Layout: q [tokens, heads_q, head_dim] and k [tokens, heads_k, head_dim], head_dim contiguous,
// other strides free, each with its own weight [head_dim]; outputs contiguous. A head lies in
// `group` neighbouring lanes (a power of two), each with two packs of VEC columns: the two
// halves of VEC pairs, or neighbours where pairs are interleaved or columns are not turned.
// Neighbouring groups take neighbouring heads of a token, q's and then k's. Sines are formed
// once for a workgroup's tokens, into LDS.
//
// Memory-bound: the forward reads x and writes y, the backward reads x and dy and writes dx.
// Workgroups walk the tokens, a head a thread group, and load the next token's packs under the
// present one's work; the backward's keep the sums for dw in registers over the walk and leave one
// partial row each of q's and k's, which a second kernel adds in order.
//
// Kernel times, bf16 32768 tokens, 32 + 8 heads of 128: forward 125 us (5.4 TB/s), backward 171 to
// 184 us (5.5 to 5.9 TB/s) and 5; fp16 5003 tokens, 16 + 16 heads of 96, 64 columns interleaved: 13
// and 21 + 4; 32 tokens 4 us, a launch. With a workgroup per token and heads summed by LDS
// permutes the first took 163 and 362 us; with branches around the walk's loads and stores,
// where each step waited for the last one's stores, 127 and 236.
#include "rotary_angles.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

constexpr int kMostThreads = 512;
// The backward's workgroups, which leave a partial row each, at most; or as many as one token's
// heads take.
constexpr int64_t kMostParts = 2048;
// Waves per SIMD that the registers leave room for, and of them those that the backward's walk
// starts (32768 tokens, 32 + 8 heads of 128, us: one or two 185, three 189, four 194, and 254 where
// four have to fit the registers; the forward 122 to 124 with four to six, 239 with eight).
constexpr int kFrontWaves = 6, kBackWaves = 3, kBackGrid = 2;
// Past this size of q and k together a call streams: stores, and the backward's loads, with the
// non-temporal hint. Plain and streamed, us, forward and backward: 32768 tokens, 32 + 8 heads of
// 128 bf16 (336 MB) 132 / 126 and 191 / 172; 8192 of them (84 MB) 28 / 28 and 49 / 48; 5003 tokens,
// 32 heads of 96 fp16 (31 MB) 12 / 13 and 23 / 26. The forward's loads gain nothing (126 / 124) and
// lose in small calls.
constexpr int64_t kStreamBytes = 64 << 20;

struct HeadArgs {
  const void *q, *k, *dqo, *dko, *qw, *kw;
  void *qo, *ko;  // y, or dx
  void *dqw, *dkw;
  float* part;  // [workgroups][2][head_dim]
  const void* pos;
  const double* freq;
  int64_t tokens, q_token, q_head, k_token, k_head, dq_token, dq_head, dk_token, dk_head;
  int heads_q, heads_k, head_dim, pairs, pos64;
  int group, lanes, per_block;  // lanes of a head; heads along a token's threads; tokens
  int ahead;                    // steps whose sines are formed at a time
  float amp, eps, share;        // share: 1 / head_dim
};

// Sum over the `group` lanes of a head, the same bits in each: neighbours, pairs of a quad, and
// mirrored halves and rows of 16 lanes are register accesses of the addition itself (DPP).
template <int CTRL>
__device__ __forceinline__ float plus_lane(float v) {
  const int other = __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false);
  return v + __int_as_float(other);
}
__device__ __forceinline__ float group_sum(float v, int group) {
  if (group > 1) v = plus_lane<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  if (group > 2) v = plus_lane<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  if (group > 4) v = plus_lane<0x141>(v);  // row_half_mirror
  if (group > 8) v = plus_lane<0x140>(v);  // row_mirror
  if (group > 16) v += __shfl_xor(v, 16);
  if (group > 32) v += __shfl_xor(v, 32);
  return v;
}

// A thread's place: token of the workgroup, head, columns. Every thread has valid ones: a lane
// past its head's packs does the first lane's work again, a group past the workgroup's heads the
// first group's, and a second pack past the head is the first one again. They store the same bits
// to the same places and are left out of the sums, so that the walk's loads and stores need no
// branches, which would keep a step's stores from staying in flight over the next one's loads.
template <int VEC, bool INTER>
struct Place {
  int tl, hl, c1, c2;
  bool in, one, two;  // of the workgroup's tokens; the lane and its second pack are a head's own
  bool turn;          // turned columns
  int pair;           // first pair
  __device__ __forceinline__ Place(const HeadArgs& a) {
    const unsigned per = a.lanes * a.group;  // threads of a token
    const unsigned e = blockIdx.y * blockDim.x + threadIdx.x;
    tl = e / per;
    const unsigned r = e - tl * per;
    hl = r / a.group;
    int ch = r - hl * a.group;
    in = tl < a.per_block;
    if (!in) tl = hl = 0;
    const int turned = a.pairs / VEC;
    one = ch < turned || 2 * a.pairs + (ch - turned) * 2 * VEC < a.head_dim;
    if (!one) ch = 0;
    turn = ch < turned;
    pair = ch * VEC;
    c1 = !turn ? 2 * a.pairs + (ch - turned) * 2 * VEC : INTER ? 2 * ch * VEC : ch * VEC;
    c2 = turn && !INTER ? c1 + a.pairs : c1 + VEC;
    two = one && c2 < a.head_dim;
    if (c2 >= a.head_dim) c2 = c1;
  }
};

// The rows of head h (q's heads, then k's).
struct Head {
  bool isq;
  int at;
  __device__ __forceinline__ Head(const HeadArgs& a, int h) {
    isq = h < a.heads_q;
    at = isq ? h : h - a.heads_q;
  }
  template <typename T>
  __device__ __forceinline__ const T* x(const HeadArgs& a, int64_t t) const {
    return isq ? (const T*)a.q + t * a.q_token + at * a.q_head
               : (const T*)a.k + t * a.k_token + at * a.k_head;
  }
  template <typename T>
  __device__ __forceinline__ const T* dy(const HeadArgs& a, int64_t t) const {
    return isq ? (const T*)a.dqo + t * a.dq_token + at * a.dq_head
               : (const T*)a.dko + t * a.dk_token + at * a.dk_head;
  }
  template <typename T>
  __device__ __forceinline__ T* out(const HeadArgs& a, int64_t t) const {
    return isq ? (T*)a.qo + (t * a.heads_q + at) * a.head_dim
               : (T*)a.ko + (t * a.heads_k + at) * a.head_dim;
  }
  template <typename T>
  __device__ __forceinline__ const T* weight(const HeadArgs& a) const {
    return (const T*)(isq ? a.qw : a.kw);
  }
};

// (cos, sin) of `steps` runs of per_block tokens, the first from t0 on, `stride` apart.
__device__ __forceinline__ void form_table(const HeadArgs& a, int64_t t0, int steps, int64_t stride,
                                           float sign, float2* table) {
  const int each = a.per_block * a.pairs;
  for (int i = threadIdx.x; i < steps * each; i += blockDim.x) {
    const int step = i / each, tl = (i - step * each) / a.pairs;
    const int64_t t = min(t0 + step * stride + tl, a.tokens - 1);
    table[i] = rotary_turn(rotary_position(a.pos, a.pos64, t), a.freq[i % a.pairs], a.amp, sign);
  }
}

// Elements of pair i of a thread's two packs.
template <int VEC, bool INTER>
struct PairAt {
  int u, v;  // of the 2 * VEC elements
  __device__ __forceinline__ PairAt(int i) : u(INTER ? 2 * i : i), v(INTER ? 2 * i + 1 : VEC + i) {}
};

// Turns the packs in place.
template <int VEC, bool INTER>
__device__ __forceinline__ void turn_packs(const float2* table, float (&n)[2 * VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const PairAt<VEC, INTER> p(i);
    const float2 cs = table[i];
    const float a = n[p.u], b = n[p.v];
    n[p.u] = __builtin_fmaf(a, cs.x, -(b * cs.y));
    n[p.v] = __builtin_fmaf(b, cs.x, a * cs.y);
  }
}

// A thread's two packs of a row as they lie in memory.
template <typename T, int VEC, bool NT>
struct RawPacks {
  Pack<T, VEC> v[2];
  static __device__ __forceinline__ Pack<T, VEC> read(const T* p) {
    if constexpr (NT && sizeof(T) * VEC == 16) return load_ragged_raw<T, VEC, true>(p);
    else return *reinterpret_cast<const Pack<T, VEC>*>(p);
  }
  template <bool INTER>
  __device__ __forceinline__ void load(const T* row, const Place<VEC, INTER>& at) {
    v[0] = read(row + at.c1);
    v[1] = read(row + at.c2);
  }
  __device__ __forceinline__ void get(float (&f)[2 * VEC]) const {
#pragma unroll
    for (int i = 0; i < 2 * VEC; ++i) f[i] = to_f32(v[i / VEC].v[i % VEC]);
  }
};

template <bool NT, typename T, int VEC, bool INTER>
__device__ __forceinline__ void put(T* row, const Place<VEC, INTER>& at, const float (&f)[2 * VEC]) {
  float u[VEC], v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) u[i] = f[i], v[i] = f[VEC + i];
  store_vec<T, VEC, NT>(row + at.c1, u);
  store_vec<T, VEC, NT>(row + at.c2, v);
}

// Sum of a head's products u v, over the packs that are its own.
template <int GROUP, int VEC, bool INTER>
__device__ __forceinline__ float head_dot(const Place<VEC, INTER>& at, const float (&u)[2 * VEC],
                                          const float (&v)[2 * VEC], int group) {
  float s = 0.f, s2 = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) s += u[i] * v[i], s2 += u[VEC + i] * v[VEC + i];
  s += at.two ? s2 : 0.f;
  return group_sum(at.one ? s : 0.f, GROUP ? GROUP : group);
}

// A workgroup walks the tokens in steps of the grid, one head a thread group, and loads the next
// step's packs under the present one's work. The sines of a.ahead steps are formed at a time.
template <typename T, int VEC, bool INTER, bool NT>
__global__ __launch_bounds__(kMostThreads, kFrontWaves) void norm_rotary_fwd_kernel(HeadArgs a) {
  extern __shared__ float2 table[];  // [ahead][per_block][pairs]
  const Place<VEC, INTER> at(a);
  const Head h(a, at.hl);
  const int64_t stride = (int64_t)gridDim.x * a.per_block;
  int64_t t0 = (int64_t)blockIdx.x * a.per_block, t = min(t0 + at.tl, a.tokens - 1);
  const T* x = h.x<T>(a, t);
  RawPacks<T, VEC, false> raw, w;
  raw.load(x, at);
  w.load(h.weight<T>(a), at);
  for (int ahead = 0; t0 < a.tokens; t0 += stride) {
    if (ahead == 0) {
      __syncthreads();
      form_table(a, t0, a.ahead, stride, 1.f, table);
      __syncthreads();
    }
    const float2* turns = table + (ahead * a.per_block + at.tl) * a.pairs + at.pair;
    if (++ahead == a.ahead) ahead = 0;
    float n[2 * VEC], g[2 * VEC];
    raw.get(n);
    T* out = h.out<T>(a, t);
    t = min(t0 + stride + at.tl, a.tokens - 1);
    raw.load(h.x<T>(a, t), at);
    w.get(g);
    const float rstd = rsqrtf(head_dot<0>(at, n, n, a.group) * a.share + a.eps);
#pragma unroll
    for (int i = 0; i < 2 * VEC; ++i) n[i] = n[i] * rstd * g[i];
    if (at.turn) turn_packs<VEC, INTER>(turns, n);
    put<NT>(out, at, n);
  }
}

// The backward's walk is the forward's.
template <typename T, int VEC, bool INTER, int GROUP, bool NT>
__global__ __launch_bounds__(kMostThreads, kBackWaves) void norm_rotary_bwd_kernel(HeadArgs a) {
  extern __shared__ float2 table[];  // [ahead][per_block][pairs]; sums at the end
  const Place<VEC, INTER> at(a);
  const Head h(a, at.hl);
  const int64_t stride = (int64_t)gridDim.x * a.per_block;
  float acc[2 * VEC];
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) acc[i] = 0.f;
  int64_t t0 = (int64_t)blockIdx.x * a.per_block, t = min(t0 + at.tl, a.tokens - 1);
  RawPacks<T, VEC, NT> rawx, rawd;
  RawPacks<T, VEC, false> w;
  rawx.load(h.x<T>(a, t), at);
  rawd.load(h.dy<T>(a, t), at);
  w.load(h.weight<T>(a), at);
  for (int ahead = 0; t0 < a.tokens; t0 += stride) {
    if (ahead == 0) {
      __syncthreads();
      form_table(a, t0, a.ahead, stride, -1.f, table);
      __syncthreads();
    }
    const float2* turns = table + (ahead * a.per_block + at.tl) * a.pairs + at.pair;
    if (++ahead == a.ahead) ahead = 0;
    float x[2 * VEC], d[2 * VEC], g[2 * VEC];
    rawx.get(x);
    rawd.get(d);
    T* out = h.out<T>(a, t);
    t = min(t0 + stride + at.tl, a.tokens - 1);
    rawx.load(h.x<T>(a, t), at);
    rawd.load(h.dy<T>(a, t), at);
    w.get(g);
    if (at.turn) turn_packs<VEC, INTER>(turns, d);  // dn
#pragma unroll
    for (int i = 0; i < 2 * VEC; ++i) g[i] *= d[i];
    const float squares = head_dot<GROUP>(at, x, x, a.group), dot = head_dot<GROUP>(at, g, x, a.group);
    const float rstd = rsqrtf(squares * a.share + a.eps), mean = dot * rstd * a.share;
#pragma unroll
    for (int i = 0; i < 2 * VEC; ++i) {
      x[i] *= rstd;
      g[i] = rstd * (g[i] - x[i] * mean);
    }
    put<NT>(out, at, g);
    if (t0 + at.tl < a.tokens)
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) acc[i] += d[i] * x[i];
  }
  // this workgroup's sums, column by column over its heads' rows
  float* rows = (float*)table;
  const int heads = blockDim.x / a.group, me = threadIdx.x / a.group;
  float* part = a.part + ((int64_t)blockIdx.x * gridDim.y + blockIdx.y) * 2 * a.head_dim;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if (at.one) rows[me * a.head_dim + at.c1 + i] = acc[i];
    if (at.two) rows[me * a.head_dim + at.c2 + i] = acc[VEC + i];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.head_dim; c += blockDim.x) {
    float sum[2] = {0.f, 0.f};
    const int first = blockIdx.y * heads, left = a.per_block * a.lanes - first;
    int head = first % a.lanes;
#pragma unroll 8
    for (int m = 0; m < min(heads, left); ++m) {
      const float v = rows[m * a.head_dim + c];
      sum[0] += head < a.heads_q ? v : 0.f;
      sum[1] += head < a.heads_q ? 0.f : v;
      if (++head == a.lanes) head = 0;
    }
    part[c] = sum[0];
    part[a.head_dim + c] = sum[1];
  }
}

// Heads of more than 64 lanes' packs (single columns of wide heads): a wave per head, which reads
// its columns again for every step and forms its own sines. Column sums lie in LDS, each
// column with the lane that works on it. Bound by the loads, a column a lane and two waves a SIMD, and
// not by the sines (8192 tokens, 8 heads of 513 bf16, forward: 65 pairs 179 us, 256 pairs 160): 2048
// tokens, 8 heads of 514 42 + 90 us, of 130 with 65 pairs 19 + 38.

template <typename T, bool INTER, bool BACK>
__global__ __launch_bounds__(kWave) void norm_rotary_wide_kernel(HeadArgs a) {
  extern __shared__ float2 table[];
  float* sums = (float*)table;  // [2][head_dim]
  const int lane = threadIdx.x;
  const int64_t heads = a.heads_q + a.heads_k, items = a.tokens * heads;
  if (BACK)
    for (int c = lane; c < 2 * a.head_dim; c += kWave) sums[c] = 0.f;
  __syncthreads();
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t t = item / heads;
    const Head h(a, (int)(item - t * heads));
    const T *x = h.x<T>(a, t), *w = h.weight<T>(a), *d = BACK ? h.dy<T>(a, t) : nullptr;
    T* out = h.out<T>(a, t);
    const double pos = rotary_position(a.pos, a.pos64, t);
    // f(first column, second or -1, the columns' dn) for every pair and single column
    auto columns = [&](auto f) {
      for (int p = lane; p < a.pairs; p += kWave) {
        const int u = INTER ? 2 * p : p, v = INTER ? 2 * p + 1 : p + a.pairs;
        const float2 cs = rotary_turn(pos, a.freq[p], a.amp, BACK ? -1.f : 1.f);
        f(u, v, cs);
      }
      for (int c = 2 * a.pairs + lane; c < a.head_dim; c += kWave) f(c, -1, make_float2(1.f, 0.f));
    };
    // the two columns' dn
    auto upstream = [&](int u, int v, float2 cs, float& du, float& dv) {
      const float p = to_f32(d[u]), r = v < 0 ? 0.f : to_f32(d[v]);
      du = __builtin_fmaf(p, cs.x, -(r * cs.y));
      dv = __builtin_fmaf(r, cs.x, p * cs.y);
    };
    float squares = 0.f, dot = 0.f;
    columns([&](int u, int v, float2 cs) {
      const float xu = to_f32(x[u]), xv = v < 0 ? 0.f : to_f32(x[v]);
      squares += xu * xu + xv * xv;
      if constexpr (BACK) {
        float du, dv;
        upstream(u, v, cs, du, dv);
        dot += du * to_f32(w[u]) * xu;
        if (v >= 0) dot += dv * to_f32(w[v]) * xv;
      }
    });
    const float rstd = rsqrtf(wave_reduce(squares, SumOp()) / a.head_dim + a.eps);
    const float mean = BACK ? wave_reduce(dot, SumOp()) * rstd / a.head_dim : 0.f;
    float* sum = sums + (h.isq ? 0 : a.head_dim);
    columns([&](int u, int v, float2 cs) {
      const float xu = to_f32(x[u]) * rstd, xv = v < 0 ? 0.f : to_f32(x[v]) * rstd;
      const float wu = to_f32(w[u]), wv = v < 0 ? 0.f : to_f32(w[v]);
      if constexpr (BACK) {
        float du, dv;
        upstream(u, v, cs, du, dv);
        sum[u] += du * xu;
        out[u] = from_f32<T>(rstd * (du * wu - xu * mean));
        if (v >= 0) {
          sum[v] += dv * xv;
          out[v] = from_f32<T>(rstd * (dv * wv - xv * mean));
        }
      } else {
        const float p = xu * wu, r = xv * wv;
        out[u] = from_f32<T>(__builtin_fmaf(p, cs.x, -(r * cs.y)));
        if (v >= 0) out[v] = from_f32<T>(__builtin_fmaf(r, cs.x, p * cs.y));
      }
    });
  }
  if (BACK) {
    __syncthreads();
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.head_dim;
    for (int c = lane; c < 2 * a.head_dim; c += kWave) part[c] = sums[c];
  }
}

// The weights' gradients from the partial rows: 16 columns a workgroup, its rows dealt to 64
// adders whose sums are added in order.
constexpr int kSumCols = 16, kSumRows = 64;
template <typename T>
__global__ __launch_bounds__(kSumCols* kSumRows) void norm_rotary_sum_kernel(HeadArgs a, int parts) {
  __shared__ float sums[kSumRows][kSumCols];
  const int lane = threadIdx.x % kSumCols, adder = threadIdx.x / kSumCols;
  const int c = blockIdx.x * kSumCols + lane, cols = 2 * a.head_dim;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int r = adder; r < parts; r += kSumRows) s += a.part[(int64_t)r * cols + c];
  }
  sums[adder][lane] = s;
  __syncthreads();
#pragma unroll
  for (int n = kSumRows / 2; n >= 1; n /= 2) {
    if (adder < n) sums[adder][lane] = s += sums[adder + n][lane];
    __syncthreads();
  }
  if (adder != 0 || c >= cols) return;
  if (c < a.head_dim) ((T*)a.dqw)[c] = from_f32<T>(s);
  else if (a.dkw) ((T*)a.dkw)[c - a.head_dim] = from_f32<T>(s);
}

// How a call's heads lie on threads: 0 lanes if a head does not fit a wave.
struct Shape {
  int group, lanes, per_block, threads;
  int64_t gx, gy;
};
Shape shape_of(const HeadArgs& a, int vec) {
  Shape s = {};
  const int64_t heads = a.heads_q + a.heads_k;
  const int chunks = a.pairs / vec + (a.head_dim - 2 * a.pairs + 2 * vec - 1) / (2 * vec);
  s.group = 1;
  while (s.group < chunks) s.group *= 2;
  if (s.group > kWave) return s;
  s.lanes = (int)heads;
  // As many whole tokens as fill the waves of a workgroup best, from 256 threads on; a token of
  // more than 512 threads lies over several workgroups.
  const int64_t per = (int64_t)s.group * s.lanes;
  int64_t best = std::max<int64_t>(1, 256 / per), unused = 64;
  for (int64_t n = best; n * per <= kMostThreads; ++n) {
    const int64_t idle = (64 - n * per % 64) % 64;
    if (idle < unused) best = n, unused = idle;
  }
  s.per_block = (int)best;
  const int64_t used = best * per;
  s.gy = (used + kMostThreads - 1) / kMostThreads;
  s.threads = (int)((used + 64 * s.gy - 1) / (64 * s.gy)) * 64;
  s.gx = (a.tokens + s.per_block - 1) / s.per_block;
  return s;
}

// A walk of `waves` waves per SIMD: a grid of the workgroups that are resident, and sines of as
// many steps at a time as give each thread two, within 16 KB.
void place(HeadArgs& a, Shape& s, int waves) {
  a.group = s.group, a.lanes = s.lanes, a.per_block = s.per_block;
  const int64_t resident = 256 * std::max(1, 4 * waves / (s.threads / 64));
  s.gx = std::min(s.gx, std::max<int64_t>(1, std::min(resident, kMostParts) / s.gy));
  const int64_t steps = (a.tokens + s.gx * s.per_block - 1) / (s.gx * s.per_block);
  const int each = std::max(1, a.per_block * a.pairs);
  a.ahead = (int)std::max<int64_t>(1, std::min<int64_t>(steps, std::min(2 * s.threads, 2048) / each));
}

// go(VEC) with the widest pack (at most 16 bytes) that divides the halves, the head and every
// stride, and to which the tensors are aligned. bf16, 8192 tokens, forward + backward, us: 32 heads of
// 80 with 40 / 20 / 10 pairs (16, 8, 4 bytes) 16 + 31 / 19 + 38 / 27 + 59; of 128 at 16 bytes 22 + 39,
// an element off it (2 bytes) 50 + 116.
template <typename T, int VEC, typename F>
int by_width(const HeadArgs& a, F&& go) {
  if constexpr (VEC > 1) {
    bool fits = a.pairs % VEC == 0 && a.head_dim % VEC == 0;
    for (int64_t s : {a.q_token, a.q_head, a.k_token, a.k_head, a.dq_token, a.dq_head, a.dk_token,
                      a.dk_head})
      fits = fits && s % VEC == 0;
    for (const void* p : {a.q, a.k, a.dqo, a.dko, a.qw, a.kw, (const void*)a.qo, (const void*)a.ko})
      fits = fits && (uintptr_t)p % (VEC * sizeof(T)) == 0;
    if (!fits) return by_width<T, VEC / 2>(a, go);
  }
  return go(std::integral_constant<int, VEC>{});
}

// f(NT): whether the call streams.
template <int VEC, typename T, typename F>
int by_size(const HeadArgs& a, F&& f) {
  if constexpr (VEC * sizeof(T) == 16) {
    const int64_t heads = a.heads_q + a.heads_k;
    if (a.tokens * heads * a.head_dim * (int64_t)sizeof(T) > kStreamBytes) return f(std::true_type{});
  }
  return f(std::false_type{});
}

// f(GROUP): the backward's lanes of a head where 16-byte packs make it a usual count, else 0, the
// count at run time. 32768 tokens, 32 + 8 heads of 128 bf16 173 us / 181 at run time, 16384 tokens,
// 18 heads of 256 93 / 103; the forward is the same either way.
template <int VEC, typename T, typename F>
int by_group(const HeadArgs& a, F&& f) {
  if constexpr (VEC * sizeof(T) == 16) {
    if (a.group == 4) return f(std::integral_constant<int, 4>{});
    if (a.group == 8) return f(std::integral_constant<int, 8>{});
    if (a.group == 16) return f(std::integral_constant<int, 16>{});
  }
  return f(std::integral_constant<int, 0>{});
}

template <typename F>
int by_layout(bool interleaved, F&& f) {
  return interleaved ? f(std::true_type{}) : f(std::false_type{});
}

int check(const char* name, int64_t tokens, int64_t heads_q, int64_t heads_k, int64_t head_dim,
          int64_t pairs, const int64_t* strides, int n) {
  if (tokens < 0 || heads_q < 0 || heads_k < 0 || head_dim < 0) {
    set_error("%s: negative size", name);
    return 1;
  }
  if (pairs < 0 || 2 * pairs > head_dim) {
    set_error("%s: %lld pairs do not fit head_dim %lld", name, (long long)pairs,
              (long long)head_dim);
    return 1;
  }
  if (heads_q > (1 << 16) || heads_k > (1 << 16) || head_dim > (1 << 13) ||
      tokens > ((int64_t)1 << 32)) {
    set_error("%s: size out of range (heads <= 65536, head_dim <= 8192, tokens <= 2^32)", name);
    return 1;
  }
  if (!strides) { set_error("%s: null strides", name); return 1; }
  for (int i = 0; i < n; ++i) {  // token steps and head steps
    const int bits = i % 2 ? 40 : 32;
    if (strides[i] < 0 || strides[i] > ((int64_t)1 << bits)) {
      set_error("%s: strides must be at least 0 and at most 2^32 (tokens) or 2^40 (heads) elements",
                name);
      return 1;
    }
  }
  return 0;
}

int64_t part_rows(int64_t tokens, int64_t heads) {
  // a token of more than 512 threads (64 lanes a head at most) takes several workgroups
  return tokens ? std::max(kMostParts, (heads * kWave + kMostThreads - 1) / kMostThreads) : 0;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" int eg_norm_rotary_fwd(const void* q, const void* k, const void* q_weight,
                                  const void* k_weight, void* q_out, void* k_out,
                                  const void* positions, int positions_64, const double* freqs,
                                  int64_t tokens, int64_t heads_q, int64_t heads_k,
                                  int64_t head_dim, int64_t pairs, const int64_t* strides,
                                  float eps, float amplitude, int interleaved, int dtype,
                                  void* stream) {
  static const char* name = "eg_norm_rotary_fwd";
  clear_error();
  if (check(name, tokens, heads_q, heads_k, head_dim, pairs, strides, 4)) return 1;
  if (tokens == 0 || head_dim == 0 || heads_q + heads_k == 0) return 0;
  if ((heads_q && (!q || !q_weight || !q_out)) || (heads_k && (!k || !k_weight || !k_out)) ||
      !positions || (pairs && !freqs)) {
    set_error("%s: null pointer", name);
    return 1;
  }
  HeadArgs a = {};
  a.q = q, a.k = heads_k ? k : nullptr, a.qw = q_weight, a.kw = heads_k ? k_weight : nullptr;
  a.qo = q_out, a.ko = heads_k ? k_out : nullptr, a.pos = positions, a.freq = freqs;
  a.tokens = tokens;
  a.q_token = strides[0], a.q_head = strides[1], a.k_token = strides[2], a.k_head = strides[3];
  a.heads_q = (int)heads_q, a.heads_k = (int)heads_k, a.head_dim = (int)head_dim;
  a.pairs = (int)pairs, a.pos64 = positions_64, a.amp = amplitude, a.eps = eps, a.share = 1.f / head_dim;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    using T = scalar_t;
    return by_layout(interleaved, [&](auto inter) -> int {
      constexpr bool I = decltype(inter)::value;
      return by_width<T, 16 / (int)sizeof(T)>(a, [&](auto vec) -> int {
        constexpr int V = decltype(vec)::value;
        Shape s = shape_of(a, V);
        if (s.lanes == 0) {
          const int64_t waves = std::min<int64_t>(tokens * (heads_q + heads_k), kMostParts);
          EG_LAUNCH((norm_rotary_wide_kernel<T, I, false>), dim3((unsigned)waves), dim3(kWave), 0,
                    as_stream(stream), a);
          return check_launch(name);
        }
        place(a, s, kFrontWaves);
        if (s.gy > 65535) { set_error("%s: grid too large", name); return 1; }
        return by_size<V, T>(a, [&](auto nt) -> int {
          EG_LAUNCH((norm_rotary_fwd_kernel<T, V, I, decltype(nt)::value>),
                    dim3((unsigned)s.gx, (unsigned)s.gy), dim3(s.threads),
                    (size_t)a.ahead * a.per_block * a.pairs * sizeof(float2), as_stream(stream), a);
          return check_launch(name);
        });
      });
    });
  });
}

extern "C" size_t eg_norm_rotary_workspace_bytes(int64_t tokens, int64_t heads_q, int64_t heads_k,
                                                 int64_t head_dim) {
  if (tokens <= 0 || heads_q < 0 || heads_k < 0 || head_dim <= 0) return 0;
  return (size_t)part_rows(tokens, heads_q + heads_k) * 2 * head_dim * sizeof(float);
}

extern "C" int eg_norm_rotary_bwd(const void* dq_out, const void* dk_out, const void* q,
                                  const void* k, const void* q_weight, const void* k_weight,
                                  const void* positions, int positions_64, const double* freqs,
                                  void* dq, void* dk, void* dq_weight, void* dk_weight,
                                  void* workspace, int64_t tokens, int64_t heads_q,
                                  int64_t heads_k, int64_t head_dim, int64_t pairs,
                                  const int64_t* strides, float eps, float amplitude,
                                  int interleaved, int dtype, void* stream) {
  static const char* name = "eg_norm_rotary_bwd";
  clear_error();
  if (check(name, tokens, heads_q, heads_k, head_dim, pairs, strides, 8)) return 1;
  if (head_dim == 0) return 0;
  const bool some = tokens > 0 && heads_q + heads_k > 0;
  if (!dq_weight || (heads_k && !dk_weight) ||
      (some && (!positions || (pairs && !freqs) || !workspace)) ||
      (some && heads_q && (!dq_out || !q || !q_weight || !dq)) ||
      (some && heads_k && (!dk_out || !k || !k_weight || !dk))) {
    set_error("%s: null pointer", name);
    return 1;
  }
  HeadArgs a = {};
  a.dqo = dq_out, a.q = q, a.qw = q_weight, a.qo = dq, a.dqw = dq_weight;
  a.dkw = dk_weight;  // of no heads: zeros
  if (heads_k) a.dko = dk_out, a.k = k, a.kw = k_weight, a.ko = dk;
  a.part = (float*)workspace, a.pos = positions, a.freq = freqs, a.tokens = tokens;
  a.q_token = strides[0], a.q_head = strides[1], a.k_token = strides[2], a.k_head = strides[3];
  a.dq_token = strides[4], a.dq_head = strides[5], a.dk_token = strides[6], a.dk_head = strides[7];
  a.heads_q = (int)heads_q, a.heads_k = (int)heads_k, a.head_dim = (int)head_dim;
  a.pairs = (int)pairs, a.pos64 = positions_64, a.amp = amplitude, a.eps = eps, a.share = 1.f / head_dim;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    using T = scalar_t;
    int parts = 0;
    if (some) {
      const int rc = by_layout(interleaved, [&](auto inter) -> int {
        constexpr bool I = decltype(inter)::value;
        return by_width<T, 16 / (int)sizeof(T)>(a, [&](auto vec) -> int {
          constexpr int V = decltype(vec)::value;
          Shape s = shape_of(a, V);
          if (s.lanes == 0) {
            parts = (int)std::min<int64_t>(tokens * (heads_q + heads_k), kMostParts);
            EG_LAUNCH((norm_rotary_wide_kernel<T, I, true>), dim3((unsigned)parts), dim3(kWave),
                      2 * head_dim * sizeof(float), as_stream(stream), a);
            return check_launch(name);
          }
          place(a, s, kBackGrid);
          if (s.gy > 65535) { set_error("%s: grid too large", name); return 1; }
          parts = (int)(s.gx * s.gy);
          const size_t lds = std::max<size_t>((size_t)a.ahead * a.per_block * a.pairs * sizeof(float2),
                                              (size_t)s.threads / s.group * head_dim * sizeof(float));
          return by_group<V, T>(a, [&](auto group) -> int {
            return by_size<V, T>(a, [&](auto nt) -> int {
              EG_LAUNCH((norm_rotary_bwd_kernel<T, V, I, decltype(group)::value, decltype(nt)::value>),
                        dim3((unsigned)s.gx, (unsigned)s.gy), dim3(s.threads), lds, as_stream(stream),
                        a);
              return check_launch(name);
            });
          });
        });
      });
      if (rc) return rc;
    }
    EG_LAUNCH((norm_rotary_sum_kernel<T>), dim3((unsigned)((2 * head_dim + kSumCols - 1) / kSumCols)),
              dim3(kSumCols * kSumRows), 0, as_stream(stream), a, parts);
    return check_launch(name);
  });
}
