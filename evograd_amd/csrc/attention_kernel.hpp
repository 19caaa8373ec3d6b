// Device code of the 16-bit MFMA attention (head size 64 or 128), as workgroup-wide functions
// over one head's sequence, with rows of any step. The kernels that place them on a grid are
// in attention.hip ([B, H, S, D] tensors; the arithmetic, operand layouts and LDS tiles are
// described there) and packed_attention.hip (packed sequences).
#pragma once

#include "eg_common.hpp"

#include <type_traits>

namespace eg {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
#define EG_LDS __attribute__((address_space(3)))

template <typename T> struct MM;
template <> struct MM<bf16_t> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack2_bf16(lo, hi); }
};
template <> struct MM<f16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack2_f16(lo, hi); }
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescaleBound = 256.0f;  // largest P term kept without a max refresh
constexpr int kFwdPrefetch = 4;            // forward S operand reads in flight
constexpr int kDqPrefetch = 2;             // dQ S / dP operand reads in flight

// Eight fp32 values (registers off..off+7 of a result tile) rounded and packed
// as one MFMA operand.
template <typename T>
__device__ __forceinline__ typename MM<T>::v8 pack8(const f32x16& c, int off) {
  uint4 u;
  u.x = MM<T>::pack2(c[off + 0], c[off + 1]);
  u.y = MM<T>::pack2(c[off + 2], c[off + 3]);
  u.z = MM<T>::pack2(c[off + 4], c[off + 5]);
  u.w = MM<T>::pack2(c[off + 6], c[off + 7]);
  typename MM<T>::v8 r;
  __builtin_memcpy(&r, &u, 16);
  return r;
}

// The two 16-bit values of a packed word, widened to fp32 (element 0 is bits 0..15).
template <typename T> __device__ __forceinline__ float half_lo(uint32_t u);
template <typename T> __device__ __forceinline__ float half_hi(uint32_t u);
template <> __device__ __forceinline__ float half_lo<bf16_t>(uint32_t u) { return __uint_as_float(u << 16); }
template <> __device__ __forceinline__ float half_hi<bf16_t>(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
template <> __device__ __forceinline__ float half_lo<f16_t>(uint32_t u) {
  const uint16_t b = (uint16_t)(u & 0xffffu);
  f16_t h;
  __builtin_memcpy(&h, &b, 2);
  return (float)h;
}
template <> __device__ __forceinline__ float half_hi<f16_t>(uint32_t u) {
  const uint16_t b = (uint16_t)(u >> 16);
  f16_t h;
  __builtin_memcpy(&h, &b, 2);
  return (float)h;
}

// Writes the rows of a transposed 32 x 32 result (lane = row of the output, its
// registers = 32 consecutive columns in C's order), scaled, as 8-byte stores.
template <typename T>
__device__ __forceinline__ void store_rows(uint16_t* __restrict__ row, const f32x16& c, int t,
                                           int hh, float f) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint2 u;
    u.x = MM<T>::pack2(c[4 * g + 0] * f, c[4 * g + 1] * f);
    u.y = MM<T>::pack2(c[4 * g + 2] * f, c[4 * g + 3] * f);
    *reinterpret_cast<uint2*>(row + 32 * t + 8 * g + 4 * hh) = u;
  }
}

// The same rows as fp32 (16-byte stores), for a split walk's partial sums.
__device__ __forceinline__ void store_rows_f32(float* __restrict__ row, const f32x16& c, int t,
                                               int hh, float f) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    *reinterpret_cast<float4*>(row + 32 * t + 8 * g + 4 * hh) =
        make_float4(c[4 * g + 0] * f, c[4 * g + 1] * f, c[4 * g + 2] * f, c[4 * g + 3] * f);
}

// RoPE on a query row held as MFMA operands (the decoder layer's q rotation,
// src/evograd/ops/level3/llama3_decoder_layer/forward_ref.py:42-51, fused into the
// forward's Q load): f[kk] holds columns 16kk + 8hh .. +7, so f[kk] and
// f[kk + KSTEPS/2] are the two halves of the same 8 rotation pairs.
//   y1 = x1 cos1 - x2 sin1,  y2 = x2 cos2 + x1 sin2   (fp32, rounded once)
template <typename T, int D>
__device__ __forceinline__ void rotate_row(typename MM<T>::v8* f, const float* __restrict__ cr,
                                           const float* __restrict__ sr, int hh) {
  constexpr int H2 = D / 32;  // KSTEPS / 2
#pragma unroll
  for (int kk = 0; kk < H2; ++kk) {
    const int col = 16 * kk + 8 * hh;
    uint4 u1, u2;
    __builtin_memcpy(&u1, &f[kk], 16);
    __builtin_memcpy(&u2, &f[kk + H2], 16);
    const uint32_t w1[4] = {u1.x, u1.y, u1.z, u1.w}, w2[4] = {u2.x, u2.y, u2.z, u2.w};
    float c1[8], s1[8], c2[8], s2[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 a = *reinterpret_cast<const float4*>(cr + col + 4 * h);
      const float4 b = *reinterpret_cast<const float4*>(sr + col + 4 * h);
      const float4 c = *reinterpret_cast<const float4*>(cr + col + D / 2 + 4 * h);
      const float4 d = *reinterpret_cast<const float4*>(sr + col + D / 2 + 4 * h);
      c1[4 * h] = a.x; c1[4 * h + 1] = a.y; c1[4 * h + 2] = a.z; c1[4 * h + 3] = a.w;
      s1[4 * h] = b.x; s1[4 * h + 1] = b.y; s1[4 * h + 2] = b.z; s1[4 * h + 3] = b.w;
      c2[4 * h] = c.x; c2[4 * h + 1] = c.y; c2[4 * h + 2] = c.z; c2[4 * h + 3] = c.w;
      s2[4 * h] = d.x; s2[4 * h + 1] = d.y; s2[4 * h + 2] = d.z; s2[4 * h + 3] = d.w;
    }
    uint32_t o1[4], o2[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x1l = half_lo<T>(w1[e]), x1h = half_hi<T>(w1[e]);
      const float x2l = half_lo<T>(w2[e]), x2h = half_hi<T>(w2[e]);
      const int i = 2 * e;
      o1[e] = MM<T>::pack2(x1l * c1[i] - x2l * s1[i], x1h * c1[i + 1] - x2h * s1[i + 1]);
      o2[e] = MM<T>::pack2(x2l * c2[i] + x1l * s2[i], x2h * c2[i + 1] + x1h * s2[i + 1]);
    }
    u1 = make_uint4(o1[0], o1[1], o1[2], o1[3]);
    u2 = make_uint4(o2[0], o2[1], o2[2], o2[3]);
    __builtin_memcpy(&f[kk], &u1, 16);
    __builtin_memcpy(&f[kk + H2], &u2, 16);
  }
}

// The transpose of RoPE applied to a gradient held as transposed result tiles
// (lane = one row of the output, register r of tile t = column 32t + 8(r/4) +
// 4hh + r%4; tiles t and t + DT/2 hold the two halves): with a the first-half and
// b the second-half entries,
//   a' = a cos1 + b sin2,  b' = b cos2 - a sin1
// the gradient of the rotation above (cr, sr: this row of the tables).
template <int D>
__device__ __forceinline__ void unrotate_rows(f32x16* acc, const float* __restrict__ cr,
                                              const float* __restrict__ sr, int hh) {
  constexpr int H2 = D / 64;  // DT / 2
#pragma unroll
  for (int t = 0; t < H2; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * t + 8 * g + 4 * hh;
      const float4 c1 = *reinterpret_cast<const float4*>(cr + d);
      const float4 s1 = *reinterpret_cast<const float4*>(sr + d);
      const float4 c2 = *reinterpret_cast<const float4*>(cr + d + D / 2);
      const float4 s2 = *reinterpret_cast<const float4*>(sr + d + D / 2);
      const float cv1[4] = {c1.x, c1.y, c1.z, c1.w}, sv1[4] = {s1.x, s1.y, s1.z, s1.w};
      const float cv2[4] = {c2.x, c2.y, c2.z, c2.w}, sv2[4] = {s2.x, s2.y, s2.z, s2.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = acc[t][4 * g + i], b = acc[t + H2][4 * g + i];
        acc[t][4 * g + i] = a * cv1[i] + b * sv2[i];
        acc[t + H2][4 * g + i] = b * cv2[i] - a * sv1[i];
      }
    }
}

template <int D>
__device__ __forceinline__ int swz(int row) {
  return (((row & 3) << 2) | ((row >> 2) & 3)) & (D / 8 - 1);
}
template <int D>
__device__ __forceinline__ int toff(int row, int chunk) {
  return row * D + ((chunk ^ swz<D>(row)) << 3);
}

__device__ __forceinline__ int wave_id() {
  return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
}

// A operand from the rows of a tile (row `row`, k = D columns 16kk + 8hh ..+7).
template <typename V, int D>
__device__ __forceinline__ V rd_rows(const uint16_t* lds, int row, int kk, int hh) {
  return *reinterpret_cast<const V*>(lds + toff<D>(row, 2 * kk + hh));
}

// A operand of a transposed tile: rows = D index dd0 + l%32, k = 16 tile rows
// from r16 in the permuted order r16 + 4hh + {0..3}, r16 + 8 + 4hh + {0..3}.
// ds_read_b64_tr_b16: within each 16-lane group, lane j receives element j%4 of
// the 8 bytes addressed by lanes 4i + j/4 (i = 0..3), so lane j points at row
// 4hh + j/4, columns 4*(j%4) .. +3 and receives column j of rows +0..3.
template <typename V, int D>
__device__ __forceinline__ V rd_tr(const uint16_t* lds, int r16, int dd0, int lane) {
  const int m = lane & 15, gs = (lane >> 4) & 1, hh = lane >> 5;
  const int col = dd0 + 16 * gs + 4 * (m & 3);
  const int chunk = col >> 3, sub = col & 7;
  const int r0 = r16 + 4 * hh + (m >> 2);
  const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EG_LDS i16x4*)(lds + toff<D>(r0, chunk) + sub));
  const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EG_LDS i16x4*)(lds + toff<D>(r0 + 8, chunk) + sub));
  V r;
  __builtin_memcpy(&r, &a, 8);
  __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &b, 8);
  return r;
}

// Copies rows [row0, row0 + ROWS) of an [nrows, D] slice, whose rows lie ld elements apart,
// into a swizzled LDS tile with 16-byte buffer->LDS loads. Each lane's offset inside the tile is fixed;
// the buffer resource starts at row0 and ends at the slice's last row, so rows
// past the slice are not fetched: their LDS rows are written with zeros (the
// bounded-access rules in eg_common.hpp).
template <int ROWS, int D, int NW, bool PACKED>
struct TileLoader {
  static constexpr int CPR = D / 8;
  static constexpr int ITER = ROWS * CPR / (64 * NW);
  static_assert(ITER >= 1 && ITER * 64 * NW == ROWS * CPR, "tile must split evenly over the waves");
  int voff[ITER], w, ld;  // w: this wave among the NW that load the tile
  __device__ __forceinline__ void init(int wave, int row_step) {
    const int lane = threadIdx.x & 63;
    w = wave;
    ld = row_step;
#pragma unroll
    for (int it = 0; it < ITER; ++it) {
      const int p = (it * NW + w) * 64 + lane;
      const int r = p / CPR;
      const int c = (p % CPR) ^ swz<D>(r);
      voff[it] = (r * ld + c * 8) * 2;
    }
  }
  __device__ __forceinline__ void load(const uint16_t* slice, int row0, int nrows,
                                       uint16_t* lds) const {
    // The range ends with the slice's last row and, of packed sequences, with the tile's: it
    // stays below 2^31 bytes for a tile of any row step taken, but not for any sequence.
    const int rows = PACKED ? min(nrows - row0, ROWS) : nrows - row0;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(slice + (int64_t)row0 * ld), (short)0, rows * ld * 2, 0x00020000);
    // Where the rows of a lane's loads are 16 apart or a multiple, their swizzles agree and the
    // later offsets follow from the first. Packed tiles at D = 128 form them so: with two row
    // steps in a loop registers are short there (packed dK/dV held in scratch what the loop
    // needs; bf16 32768 tokens, 32 / 8 heads, forward and backward 11.8 -> 11.4 ms. The 22 registers
    // a lane that it still spills belong to the second walk; of the two-wave form's 35, three are
    // read again in every step).
    constexpr int STEP = 64 * NW / CPR;
    constexpr bool FORM = PACKED && D == 128 && STEP % 16 == 0;
    int base = voff[0];
    if constexpr (FORM) asm volatile("" : "+v"(base));
#pragma unroll
    for (int it = 0; it < ITER; ++it)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (EG_LDS void*)(lds + (it * NW + w) * 64 * 8), 16,
          FORM ? base + it * STEP * ld * 2 : voff[it], 0, 0, 0);
  }
};

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <int NT>
__device__ __forceinline__ void zero_lds(void* p, int bytes) {
  uint4* z = reinterpret_cast<uint4*>(p);
  for (int e = threadIdx.x; e < bytes / 16; e += NT) z[e] = make_uint4(0, 0, 0, 0);
}

// A masked score's weight is an exact 0, but 0 times an infinite or NaN value is NaN. The
// PACKED variants look at the finished sums (a few instructions per workgroup, nothing in the
// loops): where one is not finite, the walk is done again with the masked pairs left out
// of the products (add_seen), so that such values reach the rows that see them and no
// others. The second walk also takes what fp16 cannot hold: a dS past 65504 (the gradients of a
// scaled loss) is infinite as an operand though dq and dk may be well in range, so there a
// row's or key's dS of a tile is rounded as a multiple of a power of two (half_range). It is
// slow, a product per row: with one NaN in q, bf16 8192 tokens in 11 sequences 150 + 461 -> 203 +
// 2063 us.
template <int DT>
__device__ __forceinline__ bool all_finite(const f32x16 (&acc)[DT]) {
  float z = 0.f;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = __builtin_fmaf(acc[t][r], 0.f, z);
  return z == 0.f;
}

// fp16: scales the values of this lane's column (its own and those of the lane 32 on) by the power
// of two that brings the largest finite one below 2^15, if it is not, and returns that power's
// inverse. The product's column is this lane's too, so no other row's (dQ) or key's (dK) share it.
template <typename T>
__device__ __forceinline__ float half_range(f32x16& w) {
  if constexpr (!std::is_same_v<T, f16_t>) return 1.f;
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float x = __builtin_fabsf(w[r]);
    most = x < INFINITY ? fmaxf(most, x) : most;
  }
  most = fmaxf(most, __shfl_xor(most, 32, 64));
  const int over = max(0, __builtin_amdgcn_frexp_expf(most) - 15);  // most < 2^(over + 15)
  const float back = ldexpf(1.f, over), to = ldexpf(1.f, -over);
#pragma unroll
  for (int r = 0; r < 16; ++r) w[r] *= to;
  return back;
}

// acc += back * (16 tile rows, transposed)^T w for the rows that this lane's column sees: a product
// per row, of the row's operand elements alone, whose result a lane takes or leaves. The
// row's element: rows 4hh + 0..3 are elements 0..3 of half hh's lanes, rows 8 + 4hh + 0..3
// elements 4..7.
template <typename T, int D, typename Seen>
__device__ __forceinline__ void add_seen(f32x16 (&acc)[D / 32], const uint16_t* rows,
                                         typename MM<T>::v8 w, int lane, Seen seen,
                                         float back = 1.f) {
  using v8 = typename MM<T>::v8;
  const int hh = lane >> 5;
  uint32_t ww[4];
  __builtin_memcpy(ww, &w, 16);
#pragma unroll 1
  for (int r = 0; r < 16; ++r) {
    const int e = (r & 3) | ((r >> 3) << 2);
    const uint32_t half = hh == ((r >> 2) & 1) ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
    auto alone = [&](const uint32_t (&x)[4]) {
      uint32_t y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = i == (e >> 1) ? x[i] & half : 0u;
      v8 z;
      __builtin_memcpy(&z, y, 16);
      return z;
    };
    const v8 wr = alone(ww);
    const bool in = seen(r);
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      uint32_t x[4];
      const v8 a = rd_tr<v8, D>(rows, 0, 32 * t, lane);
      __builtin_memcpy(x, &a, 16);
      const f32x16 one = MM<T>::mma(alone(x), wr, f32x16{});
#pragma unroll
      for (int i = 0; i < 16; ++i)
        acc[t][i] = in ? __builtin_fmaf(back, one[i], acc[t][i]) : acc[t][i];
    }
  }
}

// ------------------------------------------------------------------ forward
// KG = 2: two groups of NW waves share the workgroup's rows and take the key tiles by
// turns, each with tile buffers, a reference max, sums and an output of its own; group 1
// hands these to group 0 through LDS at the end. Halves the chain of tiles of a row block,
// which is what bounds a grid that leaves the chip's SIMDs with one wave or less.
// The workgroup's rows are those from q0 on of HW heads' sequences of S rows; the heads share
// their keys and values, the waves are dealt out over them, and the next head's q, o and lse
// lie hq, ho and hl elements on. Rows of q, k, v and o lie ldq, ldk, ldv and ldo elements
// apart. PACKED: see all_finite and TileLoader.
template <typename T, int D, int NW, int KG, int HW, bool ROPE, bool PACKED>
__device__ __forceinline__ void attn_fwd_rows(
    const uint16_t* __restrict__ q, int64_t ldq, int64_t hq, const uint16_t* __restrict__ kp,
    int ldk, const uint16_t* __restrict__ vp, int ldv, uint16_t* __restrict__ o, int64_t ldo,
    int64_t ho, float* __restrict__ lse, int64_t hl, int S, float scale_log2, int q0,
    const float* __restrict__ rope_cos, const float* __restrict__ rope_sin) {
  using v8 = typename MM<T>::v8;
  constexpr int HR = NW / HW, BM = 32 * HR, BN = 64;  // HR: waves of a head
  constexpr int KSTEPS = D / 16, DT = D / 32;
  // One __shared__ object per buffer (see the file comment): LDS reads of one
  // buffer never wait for the loads in flight into the other.
  __shared__ __align__(16) uint16_t Ks0[KG * BN * D], Ks1[KG * BN * D];
  __shared__ __align__(16) uint16_t Vs0[KG * BN * D], Vs1[KG * BN * D];

  const int lane = threadIdx.x & 63;
  const int w = KG == 1 ? wave_id() : wave_id() % NW, kg = KG == 1 ? 0 : wave_id() / NW;
  const int kvo = kg * BN * D;  // this group's tile buffers
  const int l32 = lane & 31, hh = lane >> 5;
  const int wr = HW == 1 ? w : w % HR;  // among the waves of its head
  if constexpr (HW > 1) {
    q += w / HR * hq;
    o += w / HR * ho;
    lse += w / HR * hl;
  }

  const int qrow = q0 + 32 * wr + l32;
  const int qrc = qrow < S ? qrow : S - 1;
  v8 qf[KSTEPS];
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk)
    qf[kk] = *reinterpret_cast<const v8*>(q + qrc * ldq + kk * 16 + 8 * hh);

  // Element offsets of this lane's operand reads inside a tile, computed once: the
  // S reads (row l32, chunk 2kk + hh; the second 32-row half adds 32 * D) and the
  // transposed V reads (rows 4hh + m/4 and +8 of each 16-row step, column block t;
  // step ms adds 16 * D). With the tile loop unrolled over the two buffers, each
  // read is one of these registers plus an immediate.
  int offS[KSTEPS], offV[DT][2];
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk) offS[kk] = toff<D>(l32, 2 * kk + hh);
  {
    const int mq = lane & 15, gs = (lane >> 4) & 1, r0 = 4 * hh + (mq >> 2);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int col = 32 * t + 16 * gs + 4 * (mq & 3);
      offV[t][0] = toff<D>(r0, col >> 3) + (col & 7);
      offV[t][1] = toff<D>(r0 + 8, col >> 3) + (col & 7);
    }
  }

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
  float m = -INFINITY, lsum = 0.f;
  const int kv_end = min(S, q0 + BM);
  const int ntiles = (kv_end + BN - 1) / BN;
  const int nturns = (ntiles + KG - 1) / KG;  // tile KG * j + kg in turn j
  const int wave_first_row = q0 + 32 * wr;

  zero_lds<NW * KG * 64>(Ks0, sizeof(Ks0));
  zero_lds<NW * KG * 64>(Ks1, sizeof(Ks1));
  zero_lds<NW * KG * 64>(Vs0, sizeof(Vs0));
  zero_lds<NW * KG * 64>(Vs1, sizeof(Vs1));
  __syncthreads();
  TileLoader<BN, D, NW, PACKED> lk, lv;
  lk.init(w, ldk);
  lv.init(w, ldv);
  if (kg < ntiles) {
    lk.load(kp, kg * BN, S, Ks0 + kvo);
    lv.load(vp, kg * BN, S, Vs0 + kvo);
  }
  // The rotation waits for q and the tables, so it comes after the first tile's
  // loads are issued: those are in flight meanwhile.
  if constexpr (ROPE)
    rotate_row<T, D>(qf, rope_cos + (int64_t)qrc * D, rope_sin + (int64_t)qrc * D, hh);
  auto tile = [&](auto bufc, int j) {
    constexpr int buf = decltype(bufc)::value;
    wait_loads();
    __syncthreads();
    const int next = KG * (j + 1) + kg;
    if (next < ntiles) {
      lk.load(kp, next * BN, S, (buf ? Ks0 : Ks1) + kvo);
      lv.load(vp, next * BN, S, (buf ? Vs0 : Vs1) + kvo);
    }
    const int k0 = (KG * j + kg) * BN;
    // every key of the tile is above this wave's rows (a tile past the last one too)
    if (k0 > wave_first_row + 31) return;
    if (KG > 1 && k0 >= kv_end) return;
    const uint16_t* Kb = (buf ? Ks1 : Ks0) + kvo;
    const uint16_t* Vb = (buf ? Vs1 : Vs0) + kvo;
    f32x16 s[2];
    // S^T = K Q^T with the K operand reads kFwdPrefetch MFMAs ahead of their use
    // (MFMA i takes (kk, T2) = (i / 2, i % 2)); the scheduling groups keep that
    // order, which the default schedule would collapse to one read ahead. Keys past
    // the diagonal (and past S) are set to -inf (diagonal tiles only).
    auto scores = [&]() {
      s[0] = f32x16{};
      s[1] = f32x16{};
      constexpr int NM = 2 * KSTEPS, PF = kFwdPrefetch;
      v8 ring[PF];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < PF; ++i)
        ring[i] = *reinterpret_cast<const v8*>(Kb + offS[i >> 1] + 32 * D * (i & 1));
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        s[i & 1] = MM<T>::mma(ring[i % PF], qf[i >> 1], s[i & 1]);
        if (i + PF < NM)
          ring[i % PF] =
              *reinterpret_cast<const v8*>(Kb + offS[(i + PF) >> 1] + 32 * D * ((i + PF) & 1));
      }
      __builtin_amdgcn_sched_group_barrier(0x100, PF, 0);  // the first PF LDS reads
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one MFMA
        if (i + PF < NM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one read
      }
      __builtin_amdgcn_sched_barrier(0);
      if (k0 + BN - 1 > wave_first_row) {
#pragma unroll
        for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = k0 + 32 * T2 + (r >> 2) * 8 + 4 * hh + (r & 3);
            if (key > qrow) s[T2][r] = -INFINITY;
          }
      }
    };
    auto exps = [&](float nm) {
      float sum = 0.f;
#pragma unroll
      for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[T2][r], scale_log2, nm));
          s[T2][r] = p;
          sum += p;
        }
      return sum;
    };
    scores();
    // P against the running reference max m (log2 units), in place. A lane's sum of
    // its 32 terms bounds each of them, so a sum <= 2^8 shows that no score of its
    // row grew past m + 8. Otherwise (and on the first tile, where m is -inf, or
    // on overflow) the tile's scores are formed again, the row max is taken, the
    // running sums are rescaled to it and P is recomputed.
    float ps = 0.f;
    bool refresh = j == 0;
    if (!refresh) {
      ps = exps(-m);
      refresh = __builtin_amdgcn_ballot_w64(!(ps <= kRescaleBound)) != 0;
      if (refresh) scores();
    }
    if (refresh) {
      float mt = -INFINITY;
#pragma unroll
      for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[T2][r]);
      mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * scale_log2;
      const float m_new = fmaxf(m, mt);
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      lsum *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= alpha;
      m = m_new;
      ps = exps(m == -INFINITY ? 0.f : -m);
    }
    lsum += ps;
#pragma unroll
    for (int ms = 0; ms < BN / 16; ++ms) {
      const v8 pb = pack8<T>(s[ms >> 1], 8 * (ms & 1));
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (EG_LDS i16x4*)(Vb + offV[t][0] + 16 * D * ms));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (EG_LDS i16x4*)(Vb + offV[t][1] + 16 * D * ms));
        v8 va;
        __builtin_memcpy(&va, &lo, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&va) + 8, &hi, 8);
        acc[t] = MM<T>::mma(va, pb, acc[t]);
      }
    }
  };
  for (int j = 0; j < nturns; j += 2) {
    tile(std::integral_constant<int, 0>{}, j);
    if (j + 1 < nturns) tile(std::integral_constant<int, 1>{}, j + 1);
  }
  if constexpr (PACKED) {
    if (__syncthreads_or(qrow < S && !all_finite<DT>(acc))) {
      m = -INFINITY;
      lsum = 0.f;
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
      for (int j = 0; j < nturns; ++j) {
        const int k0 = (KG * j + kg) * BN;
        __syncthreads();
        if (k0 < kv_end) {
          lk.load(kp, k0, S, Ks0 + kvo);
          lv.load(vp, k0, S, Vs0 + kvo);
        }
        wait_loads();
        __syncthreads();
        if (k0 > wave_first_row + 31 || k0 >= kv_end) continue;
        f32x16 s[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
          for (int T2 = 0; T2 < 2; ++T2)
            s[T2] = MM<T>::mma(
                *reinterpret_cast<const v8*>(Ks0 + kvo + offS[kk] + 32 * D * T2), qf[kk], s[T2]);
        float mt = -INFINITY;
#pragma unroll
        for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (k0 + 32 * T2 + (r >> 2) * 8 + 4 * hh + (r & 3) > qrow) s[T2][r] = -INFINITY;
            mt = fmaxf(mt, s[T2][r]);
          }
        const float m_new = fmaxf(m, fmaxf(mt, __shfl_xor(mt, 32, 64)) * scale_log2);
        const float alpha = m == m_new ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
        lsum *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t) acc[t] *= alpha;
        m = m_new;
        // every score so far may be -inf: weights of zero, not -inf + inf
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[T2][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[T2][r], scale_log2, -ref));
            lsum += s[T2][r];
          }
#pragma unroll
        for (int ms = 0; ms < BN / 16; ++ms)
          add_seen<T, D>(acc, Vs0 + kvo + 16 * D * ms, pack8<T>(s[ms >> 1], 8 * (ms & 1)), lane,
                         [&](int r) { return k0 + 16 * ms + r <= qrow; });
      }
    }
  }
  if constexpr (KG > 1) {
    // Group 1's values in the lane that holds the same rows in group 0, half of the output
    // tiles in each K buffer.
    constexpr int HT = DT / 2, STRIDE = NW * 64;
    static_assert(HT * 16 * STRIDE * 4 <= (int)sizeof(Ks0), "half the output fits a buffer");
    float* half0 = reinterpret_cast<float*>(Ks0);
    float* half1 = reinterpret_cast<float*>(Ks1);
    float* ml = reinterpret_cast<float*>(Vs0);
    const int at = w * 64 + lane;
    __syncthreads();  // the last tiles are consumed
    if (kg == 1) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          (t < HT ? half0 : half1)[((t % HT) * 16 + r) * STRIDE + at] = acc[t][r];
      ml[at] = m;
      ml[STRIDE + at] = lsum;
    }
    __syncthreads();
    if (kg == 1) return;
    const float m1 = ml[at], mx = fmaxf(m, m1), ref = mx == -INFINITY ? 0.f : mx;
    const float a0 = __builtin_amdgcn_exp2f(m - ref), a1 = __builtin_amdgcn_exp2f(m1 - ref);
    lsum = lsum * a0 + ml[STRIDE + at] * a1;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[t][r] = acc[t][r] * a0 +
                    (t < HT ? half0 : half1)[((t % HT) * 16 + r) * STRIDE + at] * a1;
    m = mx;
  }

  const float ltot = lsum + __shfl_xor(lsum, 32, 64);
  if (qrow < S) {
    const float inv = 1.0f / ltot;
    uint16_t* op = o + qrow * ldo;
#pragma unroll
    for (int t = 0; t < DT; ++t) store_rows<T>(op, acc[t], t, hh, inv);
    if (hh == 0) lse[qrow] = (m + log2f(ltot)) * kLn2;
  }
}

// ------------------------------------------------------------ dK, dV
// The workgroup's keys are those from k0 on of one kv head's sequence of S rows; q, dout, lse
// and delta are those of its group's first query head, the next head's lie hq, hdo and hl
// elements on, rows ldq, ldk, ldv and lddo apart. With parts > 1 the walk below is cut into
// ranges of steps, and part pi's sums go to the fp32 rows pk, pv, ldp apart; else to dk and dv,
// ldd apart. PACKED: see all_finite and TileLoader.
template <typename T, int D, int NW, int BQ, bool ROPE, bool PACKED>
__device__ __forceinline__ void attn_dkdv_keys(
    const uint16_t* __restrict__ q, int ldq, int64_t hq, const uint16_t* __restrict__ k,
    int64_t ldk, const uint16_t* __restrict__ v, int ldv, const uint16_t* __restrict__ dout,
    int lddo, int64_t hdo, const float* __restrict__ lse, const float* __restrict__ delta,
    int64_t hl, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv, int64_t ldd, int S,
    float scale, float scale_log2, int k0, int group, const float* __restrict__ rope_cos,
    const float* __restrict__ rope_sin, int parts, int pi, float* __restrict__ pk,
    float* __restrict__ pv, int64_t ldp) {
  using v8 = typename MM<T>::v8;
  constexpr int BK = 32 * NW;
  constexpr int KSTEPS = D / 16, DT = D / 32;
  static_assert(BQ == 32, "one 32-row Q / dO tile per step");
  __shared__ __align__(16) uint16_t Qs0[BQ * D], Qs1[BQ * D];  // one object per buffer
  __shared__ __align__(16) uint16_t Ds0[BQ * D], Ds1[BQ * D];
  // V of the workgroup's keys: the B operand of dP = dO V^T, read from LDS so
  // that its 64 registers per wave stay free for operand staging.
  __shared__ __align__(16) uint16_t Vk[BK * D];
  __shared__ __align__(16) float Ls[2][BQ];
  __shared__ __align__(16) float Es[2][BQ];

  const int lane = threadIdx.x & 63, w = wave_id();
  const int l32 = lane & 31, hh = lane >> 5;

  const int key = k0 + 32 * w + l32;
  const int krc = key < S ? key : S - 1;
  v8 kf[KSTEPS];
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk)
    kf[kk] = *reinterpret_cast<const v8*>(k + krc * ldk + kk * 16 + 8 * hh);
  f32x16 dka[DT], dva[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) { dka[t] = f32x16{}; dva[t] = f32x16{}; }

  // Operand read offsets as one register per read family. The fields of toff() are
  // disjoint bit ranges (row * D, chunk ^ swizzle in bits 3-6, the 4-column
  // sub-offset in bit 2), and the swizzle depends on the row's low 4 bits only, so
  //   rows as A operand, row l32 (+32 for this wave's V rows), chunk 2kk + hh:  R0 ^ 16kk
  //   transposed reads, column block t, rows r0 / r0 + 8 (+16 per ms step):    T0[j] ^ 32t
  const int R0 = toff<D>(l32, hh);
  int T0[2];
  {
    const int mq = lane & 15, gs = (lane >> 4) & 1, r0 = 4 * hh + (mq >> 2);
    const int col = 16 * gs + 4 * (mq & 3);
    T0[0] = toff<D>(r0, col >> 3) + (col & 7);
    T0[1] = toff<D>(r0 + 8, col >> 3) + (col & 7);
  }
  const uint16_t* Vw = Vk + 32 * w * D;  // this wave's 32 keys

  zero_lds<NW * 64>(Qs0, sizeof(Qs0));
  zero_lds<NW * 64>(Qs1, sizeof(Qs1));
  zero_lds<NW * 64>(Ds0, sizeof(Ds0));
  zero_lds<NW * 64>(Ds1, sizeof(Ds1));
  zero_lds<NW * 64>(Vk, sizeof(Vk));
  // The walk: for each query head of the group (in order), the q tiles from the
  // diagonal block to S. dK and dV accumulate over all of them in registers, so
  // the kv-head gradient is the group sum without atomics or a second pass.
  const int i_first = k0 / BQ;
  const int ntq = (S + BQ - 1) / BQ - i_first;
  const int nsteps = group * ntq;
  const int per = (nsteps + parts - 1) / parts;
  const int s_begin = min(nsteps, pi * per), s_end = min(nsteps, s_begin + per);
  const int wave_first_key = k0 + 32 * w;
  TileLoader<BQ, D, NW, PACKED> lq, ldo;
  lq.init(w, ldq);
  ldo.init(w, lddo);
  auto qhead = [&](int step) { return step / ntq; };  // in the group
  auto qtile = [&](int step) { return i_first + step % ntq; };
  // lse and delta of a tile's rows: wave 0 loads them when the tile is requested
  // and converts and stores them to LDS only after the current step's compute, so
  // that waiting for them does not hold that compute behind the tile loads.
  float lraw = 0.f, eraw = 0.f;
  bool lrow = false;
  auto load_stats = [&](int step) {
    if (w == 0 && lane < BQ) {
      const int64_t hb = qhead(step) * hl;
      const int row = qtile(step) * BQ + lane;
      const int rc = row < S ? row : S - 1;
      lraw = lse[hb + rc];
      eraw = delta[hb + rc];
      lrow = row < S;
    }
  };
  auto store_stats = [&](float* ls, float* es) {
    if (w == 0 && lane < BQ) {
      ls[lane] = lrow ? lraw * kLog2e : INFINITY;  // rows past S: p = 0
      es[lane] = lrow ? eraw : 0.f;
    }
  };
  __syncthreads();
  {
    TileLoader<BK, D, NW, PACKED> lv;  // keys past S stay zero
    lv.init(w, ldv);
    lv.load(v, k0, S, Vk);
  }
  if (s_begin < s_end) {
    lq.load(q + qhead(s_begin) * hq, qtile(s_begin) * BQ, S, Qs0);
    ldo.load(dout + qhead(s_begin) * hdo, qtile(s_begin) * BQ, S, Ds0);
    load_stats(s_begin);
    store_stats(Ls[0], Es[0]);
  }
  auto step_fn = [&](auto bufc, int step) {
    constexpr int buf = decltype(bufc)::value;
    wait_loads();
    __syncthreads();
    const bool more = step + 1 < s_end;
    if (more) {
      lq.load(q + qhead(step + 1) * hq, qtile(step + 1) * BQ, S, buf ? Qs0 : Qs1);
      ldo.load(dout + qhead(step + 1) * hdo, qtile(step + 1) * BQ, S, buf ? Ds0 : Ds1);
      load_stats(step + 1);
    }
    const int qi0 = qtile(step) * BQ;
    if (qi0 + BQ - 1 >= wave_first_key) {  // some row of the tile sees some key of this wave
      const uint16_t* Qb = buf ? Qs1 : Qs0;
      const uint16_t* Db = buf ? Ds1 : Ds0;
      // Opaque copies of the offset registers: the XORs are redone in each step
      // instead of being hoisted out of the loop into 24 live registers.
      int r0 = R0, t0 = T0[0], t1 = T0[1];
      asm volatile("" : "+v"(r0), "+v"(t0), "+v"(t1));
      auto offR = [&](int kk) { return r0 ^ (16 * kk); };
      auto offT = [&](int t, int j) { return (j ? t1 : t0) ^ (32 * t); };
      // S = Q K^T and dP = dO V^T, the three operand reads of step kk + 1 issued
      // before the two MFMAs of step kk (scheduling groups keep that order).
      f32x16 s = f32x16{}, dp = f32x16{};
      {
        v8 qa[2], da[2], vb[2];
        __builtin_amdgcn_sched_barrier(0);
        qa[0] = *reinterpret_cast<const v8*>(Qb + offR(0));
        da[0] = *reinterpret_cast<const v8*>(Db + offR(0));
        vb[0] = *reinterpret_cast<const v8*>(Vw + offR(0));
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          if (kk + 1 < KSTEPS) {
            qa[(kk + 1) & 1] = *reinterpret_cast<const v8*>(Qb + offR(kk + 1));
            da[(kk + 1) & 1] = *reinterpret_cast<const v8*>(Db + offR(kk + 1));
            vb[(kk + 1) & 1] = *reinterpret_cast<const v8*>(Vw + offR(kk + 1));
          }
          s = MM<T>::mma(qa[kk & 1], kf[kk], s);
          dp = MM<T>::mma(da[kk & 1], vb[kk & 1], dp);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          if (kk + 1 < KSTEPS) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // P = exp(S * scale - lse); register r holds row 8(r/4) + 4hh + r%4.
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 l4 = *reinterpret_cast<const float4*>(&Ls[buf][8 * g + 4 * hh]);
        const float lv[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          s[4 * g + i4] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + i4], scale_log2, -lv[i4]));
      }
      // Causal mask, in the diagonal steps only (a wave-uniform branch): row
      // qi0 + 8g + 4hh + i4 sees this lane's key iff 8g + i4 >= key - qi0 - 4hh.
      if (qi0 < wave_first_key + 31) {
        const int mask_below = key - qi0 - 4 * hh;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + (r & 3) < mask_below) s[r] = 0.f;
      }
      // dS = P (dP - delta)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 e4 = *reinterpret_cast<const float4*>(&Es[buf][8 * g + 4 * hh]);
        const float ev[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          dp[4 * g + i4] = s[4 * g + i4] * (dp[4 * g + i4] - ev[i4]);
      }
      // dV^T += dO^T P and dK^T += Q^T dS in the order (ms, t, dV then dK), each
      // MFMA's transposed operand read one MFMA ahead (two ds_read_b64_tr_b16); the
      // scheduling groups keep that order, which the default schedule collapses to
      // a wait before every MFMA.
      constexpr int NM = 2 * DT * (BQ / 16);
      auto rd = [&](int i) {
        const int ms = i / (2 * DT), t = (i / 2) % DT;
        const uint16_t* tb = (i & 1) ? Qb : Db;
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (EG_LDS i16x4*)(tb + offT(t, 0) + 16 * D * ms));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (EG_LDS i16x4*)(tb + offT(t, 1) + 16 * D * ms));
        v8 r;
        __builtin_memcpy(&r, &lo, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&r) + 8, &hi, 8);
        return r;
      };
      v8 op[2], pb, sb;
      __builtin_amdgcn_sched_barrier(0);
      op[0] = rd(0);
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        if (i + 1 < NM) op[(i + 1) & 1] = rd(i + 1);
        const int ms = i / (2 * DT), t = (i / 2) % DT;
        if (i % (2 * DT) == 0) {
          pb = pack8<T>(s, 8 * ms);
          sb = pack8<T>(dp, 8 * ms);
        }
        if (i & 1) dka[t] = MM<T>::mma(op[i & 1], sb, dka[t]);
        else dva[t] = MM<T>::mma(op[i & 1], pb, dva[t]);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        if (i + 1 < NM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (more) store_stats(Ls[buf ^ 1], Es[buf ^ 1]);
  };
  // Unrolled over the two buffers, so every LDS address is a register plus an
  // immediate and the buffers are distinct objects at compile time.
  for (int step = s_begin; step < s_end; step += 2) {
    step_fn(std::integral_constant<int, 0>{}, step);
    if (step + 1 < s_end) step_fn(std::integral_constant<int, 1>{}, step + 1);
  }

  if constexpr (PACKED) {
    if (__syncthreads_or(key < S && !(all_finite<DT>(dka) && all_finite<DT>(dva)))) {
#pragma unroll
      for (int t = 0; t < DT; ++t) { dka[t] = f32x16{}; dva[t] = f32x16{}; }
      for (int step = s_begin; step < s_end; ++step) {
        __syncthreads();
        lq.load(q + qhead(step) * hq, qtile(step) * BQ, S, Qs0);
        ldo.load(dout + qhead(step) * hdo, qtile(step) * BQ, S, Ds0);
        load_stats(step);
        store_stats(Ls[0], Es[0]);
        wait_loads();
        __syncthreads();
        const int qi0 = qtile(step) * BQ;
        if (qi0 + BQ - 1 < wave_first_key) continue;
        f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          const int at = R0 ^ (16 * kk);
          s = MM<T>::mma(*reinterpret_cast<const v8*>(Qs0 + at), kf[kk], s);
          dp = MM<T>::mma(*reinterpret_cast<const v8*>(Ds0 + at),
                          *reinterpret_cast<const v8*>(Vw + at), dp);
        }
        // (rows past S are zeros, which an infinite key turns into a NaN score)
        auto seen = [&](int r) { return qi0 + r >= key && qi0 + r < S; };
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = (r >> 2) * 8 + 4 * hh + (r & 3);
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale_log2, -Ls[0][row]));
          s[r] = seen(row) ? p : 0.f;
          dp[r] = seen(row) ? p * (dp[r] - Es[0][row]) : 0.f;
        }
        const float back = half_range<T>(dp);
#pragma unroll
        for (int ms = 0; ms < BQ / 16; ++ms) {
          auto seen16 = [&](int r) { return seen(16 * ms + r); };
          add_seen<T, D>(dva, Ds0 + 16 * D * ms, pack8<T>(s, 8 * ms), lane, seen16);
          add_seen<T, D>(dka, Qs0 + 16 * D * ms, pack8<T>(dp, 8 * ms), lane, seen16, back);
        }
      }
    }
  }
  if (key < S) {
    uint16_t* dkp = dk + key * ldd;
    uint16_t* dvp = dv + key * ldd;
    float fk = scale;
    if constexpr (ROPE) {  // dk of the pre-rotation keys: the rotation's transpose
#pragma unroll
      for (int t = 0; t < DT; ++t) dka[t] *= scale;
      unrotate_rows<D>(dka, rope_cos + (int64_t)key * D, rope_sin + (int64_t)key * D, hh);
      fk = 1.0f;
    }
    if (pk) {  // this part's sums, scaled (and unrotated) like the direct store
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        store_rows_f32(pk + key * ldp, dka[t], t, hh, fk);
        store_rows_f32(pv + key * ldp, dva[t], t, hh, 1.0f);
      }
    } else {
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        store_rows<T>(dkp, dka[t], t, hh, fk);
        store_rows<T>(dvp, dva[t], t, hh, 1.0f);
      }
    }
  }
}

// ------------------------------------------------------------------- dQ
// KG as in the forward.
// Rows and heads as in attn_fwd_rows; dout, o and dq share their steps, as lse and delta do.
template <typename T, int D, int NW, int KG, int HW, bool ROPE, bool PACKED>
__device__ __forceinline__ void attn_dq_rows(
    const uint16_t* __restrict__ q, int64_t ldq, int64_t hq, const uint16_t* __restrict__ kp,
    int ldk, const uint16_t* __restrict__ vp, int ldv, const uint16_t* __restrict__ dout,
    const uint16_t* __restrict__ o, uint16_t* __restrict__ dq, int64_t ldo, int64_t ho,
    const float* __restrict__ lse, float* __restrict__ delta, int64_t hl, int S, float scale,
    float scale_log2, int q0, const float* __restrict__ rope_cos,
    const float* __restrict__ rope_sin) {
  using v8 = typename MM<T>::v8;
  constexpr int HR = NW / HW, BM = 32 * HR, BN = 64;  // HR: waves of a head
  constexpr int KSTEPS = D / 16, DT = D / 32;
  // one object per buffer
  __shared__ __align__(16) uint16_t Ks0[KG * BN * D], Ks1[KG * BN * D];
  __shared__ __align__(16) uint16_t Vs0[KG * BN * D], Vs1[KG * BN * D];

  const int lane = threadIdx.x & 63;
  const int w = KG == 1 ? wave_id() : wave_id() % NW, kg = KG == 1 ? 0 : wave_id() / NW;
  const int kvo = kg * BN * D;  // this group's tile buffers
  const int l32 = lane & 31, hh = lane >> 5;
  const int wr = HW == 1 ? w : w % HR;  // among the waves of its head
  if constexpr (HW > 1) {
    q += w / HR * hq;
    dout += w / HR * ho;
    o += w / HR * ho;
    dq += w / HR * ho;
    lse += w / HR * hl;
    delta += w / HR * hl;
  }

  const int qrow = q0 + 32 * wr + l32;
  const int qrc = qrow < S ? qrow : S - 1;
  v8 qf[KSTEPS], df[KSTEPS];
  // delta = rowsum(do * o) for this row: the lane pair (l, l + 32) holds the
  // row's D columns between them; summed in a fixed order and written for the
  // dK/dV kernel, which runs after this one.
  float dsum = 0.f;
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk) {
    const int col = kk * 16 + 8 * hh;
    qf[kk] = *reinterpret_cast<const v8*>(q + qrc * ldq + col);
    df[kk] = *reinterpret_cast<const v8*>(dout + qrc * ldo + col);
    const uint4 ou = *reinterpret_cast<const uint4*>(o + qrc * ldo + col);
    uint4 du;
    __builtin_memcpy(&du, &df[kk], 16);
    const uint32_t ow[4] = {ou.x, ou.y, ou.z, ou.w}, dw[4] = {du.x, du.y, du.z, du.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      dsum += half_lo<T>(dw[e]) * half_lo<T>(ow[e]);
      dsum += half_hi<T>(dw[e]) * half_hi<T>(ow[e]);
    }
  }
  dsum += __shfl_xor(dsum, 32, 64);
  const float lraw = lse[qrc];
  const float l2 = qrow < S ? lraw * kLog2e : INFINITY;
  float dl = qrow < S ? dsum : 0.f;
  if constexpr (!PACKED)
    if (qrow < S && hh == 0 && kg == 0) delta[qrow] = dsum;

  f32x16 acc[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
  const int kv_end = min(S, q0 + BM);
  const int ntiles = (kv_end + BN - 1) / BN;
  const int nturns = (ntiles + KG - 1) / KG;
  const int wave_first_row = q0 + 32 * wr;

  // Element offsets of this lane's operand reads inside a tile, computed once (as in
  // the forward): rows for S and dP (the K and V tiles share the layout), transposed
  // rows of K for dQ; the tile loop is unrolled over the two buffers.
  int offS[KSTEPS], offV[DT][2];
#pragma unroll
  for (int kk = 0; kk < KSTEPS; ++kk) offS[kk] = toff<D>(l32, 2 * kk + hh);
  {
    const int mq = lane & 15, gs = (lane >> 4) & 1, r0 = 4 * hh + (mq >> 2);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const int col = 32 * t + 16 * gs + 4 * (mq & 3);
      offV[t][0] = toff<D>(r0, col >> 3) + (col & 7);
      offV[t][1] = toff<D>(r0 + 8, col >> 3) + (col & 7);
    }
  }
  zero_lds<NW * KG * 64>(Ks0, sizeof(Ks0));
  zero_lds<NW * KG * 64>(Ks1, sizeof(Ks1));
  zero_lds<NW * KG * 64>(Vs0, sizeof(Vs0));
  zero_lds<NW * KG * 64>(Vs1, sizeof(Vs1));
  __syncthreads();
  TileLoader<BN, D, NW, PACKED> lk, lv;
  lk.init(w, ldk);
  lv.init(w, ldv);
  if (kg < ntiles) {
    lk.load(kp, kg * BN, S, Ks0 + kvo);
    lv.load(vp, kg * BN, S, Vs0 + kvo);
  }
  auto tile = [&](auto bufc, int j) {
    constexpr int buf = decltype(bufc)::value;
    wait_loads();
    __syncthreads();
    const int next = KG * (j + 1) + kg;
    if (next < ntiles) {
      lk.load(kp, next * BN, S, (buf ? Ks0 : Ks1) + kvo);
      lv.load(vp, next * BN, S, (buf ? Vs0 : Vs1) + kvo);
    }
    const int k0 = (KG * j + kg) * BN;
    if (k0 > wave_first_row + 31) return;
    if (KG > 1 && k0 >= kv_end) return;
    const uint16_t* Kb = (buf ? Ks1 : Ks0) + kvo;
    const uint16_t* Vb = (buf ? Vs1 : Vs0) + kvo;
    f32x16 s[2] = {f32x16{}, f32x16{}}, dp[2] = {f32x16{}, f32x16{}};
    // S^T = K Q^T and dP^T = V dO^T interleaved, each operand read kDqPrefetch MFMAs
    // ahead (read i: kk = i / 4, T2 = (i / 2) % 2, K for even i and V for odd i);
    // the scheduling groups keep that order.
    {
      constexpr int NR = 4 * KSTEPS, PF = kDqPrefetch;
      auto rd = [&](int i) {
        const uint16_t* tb = (i & 1) ? Vb : Kb;
        return *reinterpret_cast<const v8*>(tb + offS[i >> 2] + 32 * D * ((i >> 1) & 1));
      };
      v8 ring[PF];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < PF; ++i) ring[i] = rd(i);
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const int kk = i >> 2, T2 = (i >> 1) & 1;
        if (i & 1) dp[T2] = MM<T>::mma(ring[i % PF], df[kk], dp[T2]);
        else s[T2] = MM<T>::mma(ring[i % PF], qf[kk], s[T2]);
        if (i + PF < NR) ring[i % PF] = rd(i + PF);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, PF, 0);  // the first PF LDS reads
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one MFMA
        if (i + PF < NR) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one read
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[T2][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[T2][r], scale_log2, -l2));
    // Keys past the diagonal only in the diagonal tiles: a wave-uniform branch
    // around the per-element selects, so the other tiles skip them.
    if (k0 + BN - 1 > wave_first_row) {
#pragma unroll
      for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kkey = k0 + 32 * T2 + (r >> 2) * 8 + 4 * hh + (r & 3);
          if (kkey > qrow) s[T2][r] = 0.f;
        }
    }
    if constexpr (PACKED) {
      // Rows whose keys are this tile's: delta = sum p dp / sum p, from fp32 registers. The
      // stored o's rounding enters dS by p times its part of delta, which for rows of few keys,
      // and peaked ones, is most of what dq and dk are off by (at 4 keys bf16 0.34 -> 0.24% of
      // their norm). Rows of one key get dS = 0 exactly.
      if (k0 == 0 && wave_first_row < BN) {
        float pd = 0.f, ps = 0.f;
#pragma unroll
        for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int kkey = 32 * T2 + (r >> 2) * 8 + 4 * hh + (r & 3);
            pd += kkey > qrow ? 0.f : s[T2][r] * dp[T2][r];
            ps += s[T2][r];
          }
        pd += __shfl_xor(pd, 32, 64);
        ps += __shfl_xor(ps, 32, 64);
        dl = qrow < S ? pd / ps : 0.f;
      }
    }
#pragma unroll
    for (int T2 = 0; T2 < 2; ++T2)
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[T2][r] = s[T2][r] * (dp[T2][r] - dl);
#pragma unroll
    for (int ms = 0; ms < BN / 16; ++ms) {
      const v8 sb = pack8<T>(dp[ms >> 1], 8 * (ms & 1));
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (EG_LDS i16x4*)(Kb + offV[t][0] + 16 * D * ms));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (EG_LDS i16x4*)(Kb + offV[t][1] + 16 * D * ms));
        v8 ka;
        __builtin_memcpy(&ka, &lo, 8);
        __builtin_memcpy(reinterpret_cast<char*>(&ka) + 8, &hi, 8);
        acc[t] = MM<T>::mma(ka, sb, acc[t]);
      }
    }
  };
  for (int j = 0; j < nturns; j += 2) {
    tile(std::integral_constant<int, 0>{}, j);
    if (j + 1 < nturns) tile(std::integral_constant<int, 1>{}, j + 1);
  }
  if constexpr (PACKED) {
    if (qrow < S && hh == 0 && kg == 0) delta[qrow] = dl;
    if (__syncthreads_or(qrow < S && !all_finite<DT>(acc))) {
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] = f32x16{};
      for (int j = 0; j < nturns; ++j) {
        const int k0 = (KG * j + kg) * BN;
        __syncthreads();
        if (k0 < kv_end) {
          lk.load(kp, k0, S, Ks0 + kvo);
          lv.load(vp, k0, S, Vs0 + kvo);
        }
        wait_loads();
        __syncthreads();
        if (k0 > wave_first_row + 31 || k0 >= kv_end) continue;
#pragma unroll
        for (int T2 = 0; T2 < 2; ++T2) {
          f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
          for (int kk = 0; kk < KSTEPS; ++kk) {
            const int at = kvo + offS[kk] + 32 * D * T2;
            s = MM<T>::mma(*reinterpret_cast<const v8*>(Ks0 + at), qf[kk], s);
            dp = MM<T>::mma(*reinterpret_cast<const v8*>(Vs0 + at), df[kk], dp);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale_log2, -l2));
            const bool in = k0 + 32 * T2 + (r >> 2) * 8 + 4 * hh + (r & 3) <= qrow;
            dp[r] = in ? p * (dp[r] - dl) : 0.f;
          }
          const float back = half_range<T>(dp);
#pragma unroll
          for (int ms = 0; ms < 2; ++ms)
            add_seen<T, D>(acc, Ks0 + kvo + 16 * D * (2 * T2 + ms), pack8<T>(dp, 8 * ms), lane,
                           [&](int r) { return k0 + 32 * T2 + 16 * ms + r <= qrow; }, back);
        }
      }
    }
  }
  if constexpr (KG > 1) {
    constexpr int HT = DT / 2, STRIDE = NW * 64;
    static_assert(HT * 16 * STRIDE * 4 <= (int)sizeof(Ks0), "half of dQ fits a buffer");
    float* half0 = reinterpret_cast<float*>(Ks0);
    float* half1 = reinterpret_cast<float*>(Ks1);
    const int at = w * 64 + lane;
    __syncthreads();  // the last tiles are consumed
    if (kg == 1) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          (t < HT ? half0 : half1)[((t % HT) * 16 + r) * STRIDE + at] = acc[t][r];
    }
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[t][r] += (t < HT ? half0 : half1)[((t % HT) * 16 + r) * STRIDE + at];
  }

  if (qrow < S) {
    uint16_t* op = dq + qrow * ldo;
    float fq = scale;
    if constexpr (ROPE) {  // dq of the pre-rotation queries: the rotation's transpose
#pragma unroll
      for (int t = 0; t < DT; ++t) acc[t] *= scale;
      unrotate_rows<D>(acc, rope_cos + (int64_t)qrow * D, rope_sin + (int64_t)qrow * D, hh);
      fq = 1.0f;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t) store_rows<T>(op, acc[t], t, hh, fq);
  }
}

}  // namespace
}  // namespace eg
