// Rotary positions by a position per token for gfx950: q and k of packed tokens in one
// launch, forward and (with the angle negated) backward.
//
//   angle[t, i] = pos[t] * freq[i], i < pairs;  (x1, x2) -> amp (x1 c - x2 s, x2 c + x1 s)
// over the pairs (x[i], x[i + pairs]) of the half layout or (x[2i], x[2i + 1]) of the
// interleaved one; columns past 2 * pairs are copied. The backward is the transpose,
// amp (dy1 c + dy2 s, dy2 c - dy1 s).
//
// Angles: a position of a long context times a frequency leaves few bits of an fp32 product
// behind its whole turns (at position 131072 an fp32 angle is off by 0.004), so the turns
// pos * freq / 2 pi are formed in fp64 and reduced there to an eighth of a turn; only that
// remainder is rounded to fp32 for the sine and cosine. A workgroup forms them once for its
// tokens, into LDS, while its loads are on their way, and uses them for every head.
//
// Layout: q [tokens, heads_q, head_dim] and k [tokens, heads_k, head_dim], head_dim
// contiguous, other strides free; outputs contiguous. A thread owns a chunk of VEC pairs of one
// token in HPT heads, `lanes` apart in the list of q's heads and then k's, so neighbouring
// threads read neighbouring heads of a token. (With neighbouring threads on neighbouring
// tokens instead, a wave's load is eight runs of 128 bytes a token's 8 KB apart: q and k of
// 32768 tokens, 32 + 8 heads of 128, forward and backward 304 us against 254, both with sines
// formed per thread; 226 with the sines in LDS.)
//
// Memory-bound: each element is read and written once. bf16 32768 tokens, 32 + 8 heads of 128:
// 115 us each way, 5.9 TB/s; fp16 5003 tokens, 16 + 16 heads of 96, 64 columns interleaved:
// 13 us each way; 32 tokens 4 us, a launch.
#include "eg_common.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

constexpr int kMostThreads = 512;

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  const void* pos;
  const double* freq;
  int64_t tokens, q_token, q_head, k_token, k_head;
  int heads_q, heads_k, head_dim, pairs, pos64;
  int lanes, per_block;  // threads along the heads; tokens of a workgroup
  float amp, sign;
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> read(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
// Results are written past the caches (whole 16-byte packs): each is touched once.
template <typename T, int VEC>
__device__ __forceinline__ void write(T* p, const Pack<T, VEC>& v) {
  if constexpr (sizeof(T) * VEC == 16) {
    typedef unsigned int words __attribute__((ext_vector_type(4)));
    words raw;
    __builtin_memcpy(&raw, &v, 16);
    __builtin_nontemporal_store(raw, reinterpret_cast<words*>(p));
  } else {
    *reinterpret_cast<Pack<T, VEC>*>(p) = v;
  }
}

// Chunks of a head: pairs / VEC of them rotate two packs of VEC columns, the rest copy one
// 16-byte pack or two narrower ones.
template <typename T, int VEC> constexpr int kCopies = VEC * sizeof(T) == 16 ? 1 : 2;
template <typename T, int VEC>
__host__ __device__ inline int chunks_of(int head_dim, int pairs) {
  constexpr int COPY = kCopies<T, VEC> * VEC;
  return pairs / VEC + (head_dim - 2 * pairs + COPY - 1) / COPY;
}
template <typename T, int VEC, int HPT, bool INTER>
__global__ __launch_bounds__(kMostThreads) void rotary_kernel(RotaryArgs a) {
  const unsigned turned = a.pairs / VEC, chunks = chunks_of<T, VEC>(a.head_dim, a.pairs);
  const unsigned per = chunks * a.lanes;  // threads of a token
  const unsigned e = blockIdx.y * blockDim.x + threadIdx.x, tl = e / per, in = e - tl * per;
  const int64_t t = (int64_t)blockIdx.x * a.per_block + tl;
  const bool live = (int)tl < a.per_block && t < a.tokens;
  const int hl = in / chunks, ch = in - hl * chunks;
  const bool turn = ch < (int)turned;
  // columns of the chunk's packs
  const int c1 = !turn   ? 2 * a.pairs + (ch - (int)turned) * (kCopies<T, VEC> * VEC)
                 : INTER ? 2 * ch * VEC
                         : ch * VEC;
  const int c2 = turn && !INTER ? c1 + a.pairs : c1 + VEC;
  const bool two = turn || (kCopies<T, VEC> == 2 && c2 < a.head_dim);
  Pack<T, VEC> x1[HPT], x2[HPT];
  T* dst[HPT];
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    const int h = hl + j * a.lanes, hk = h - a.heads_q;
    const bool isq = hk < 0;
    dst[j] = nullptr;
    if (!live || hk >= a.heads_k) continue;
    const T* src = isq ? (const T*)a.q + t * a.q_token + h * a.q_head
                       : (const T*)a.k + t * a.k_token + hk * a.k_head;
    dst[j] = isq ? (T*)a.qo + (t * a.heads_q + h) * a.head_dim
                 : (T*)a.ko + (t * a.heads_k + hk) * a.head_dim;
    x1[j] = read<T, VEC>(src + c1);
    if (two) x2[j] = read<T, VEC>(src + c2);
  }
  // (cos, sin) of the workgroup's tokens, while the packs are on their way
  extern __shared__ float2 table[];
  const int64_t t0 = (int64_t)blockIdx.x * a.per_block;
  for (int i = threadIdx.x; i < a.per_block * a.pairs; i += blockDim.x) {
    const int64_t tok = min(t0 + i / a.pairs, a.tokens - 1);
    const double pos =
        a.pos64 ? (double)((const int64_t*)a.pos)[tok] : (double)((const int*)a.pos)[tok];
    // explicit fma, here and below: every width of packs gives the same bits
    const double f = a.freq[i % a.pairs] * 0.15915494309189533577;
    const double rest = __builtin_fma(pos, f, -rint(pos * f)), quarter = rint(4.0 * rest);
    float s0, c0;
    sincospif(2.f * (float)__builtin_fma(-0.25, quarter, rest), &s0, &c0);
    const int n = (int)quarter & 3;  // s0, c0 turned by n quarters
    const float s1 = n & 1 ? c0 : s0, c1 = n & 1 ? s0 : c0;
    table[i] = make_float2(a.amp * ((n + 1) & 2 ? -c1 : c1), a.amp * a.sign * (n & 2 ? -s1 : s1));
  }
  __syncthreads();
  if (!live) return;
  if (!turn) {
#pragma unroll
    for (int j = 0; j < HPT; ++j) {
      if (!dst[j]) continue;
      write(dst[j] + c1, x1[j]);
      if (two) write(dst[j] + c2, x2[j]);
    }
    return;
  }
  float cs[VEC], sn[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const float2 e = table[tl * a.pairs + ch * VEC + i];
    cs[i] = e.x;
    sn[i] = e.y;
  }
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    if (!dst[j]) continue;
    Pack<T, VEC> y1, y2;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      // pair i: elements i of the two packs, or 2i and 2i + 1 of the two as one run
      const int p = INTER ? 2 * i : i, r = INTER ? 2 * i + 1 : i;
      const float u = to_f32(INTER && p >= VEC ? x2[j].v[p % VEC] : x1[j].v[p % VEC]);
      const float v = to_f32(!INTER || r >= VEC ? x2[j].v[r % VEC] : x1[j].v[r % VEC]);
      float fu = __builtin_fmaf(u, cs[i], -(v * sn[i])), fv = __builtin_fmaf(v, cs[i], u * sn[i]);
      // fp32 values: not to be merged with the conversion into v_fma_mix, which rounds once
      asm("" : "+v"(fu), "+v"(fv));
      const T yu = from_f32<T>(fu), yv = from_f32<T>(fv);
      if (INTER && p >= VEC) y2.v[p % VEC] = yu; else y1.v[p % VEC] = yu;
      if (!INTER || r >= VEC) y2.v[r % VEC] = yv; else y1.v[r % VEC] = yv;
    }
    write(dst[j] + c1, y1);
    write(dst[j] + c2, y2);
  }
}

template <typename T, int VEC, bool INTER>
int launch(RotaryArgs a, hipStream_t st) {
  const int64_t chunks = chunks_of<T, VEC>(a.head_dim, a.pairs);
  const int64_t heads = a.heads_q + a.heads_k;
  auto go = [&](auto hpt) {
    constexpr int HPT = decltype(hpt)::value;
    a.lanes = (int)((heads + HPT - 1) / HPT);
    // As many whole tokens as fill the waves of a workgroup best, from 256 threads on; a token
    // of more than 512 threads lies over several workgroups.
    const int64_t per = chunks * a.lanes;
    int64_t best = std::max<int64_t>(1, 256 / per), unused = 64;
    for (int64_t n = best; n * per <= kMostThreads; ++n) {
      const int64_t idle = (64 - n * per % 64) % 64;
      if (idle < unused) best = n, unused = idle;
    }
    a.per_block = (int)best;
    const int64_t used = best * per, gy = (used + kMostThreads - 1) / kMostThreads;
    const int threads = (int)((used + 64 * gy - 1) / (64 * gy)) * 64;
    const int64_t gx = (a.tokens + a.per_block - 1) / a.per_block;
    if (gx > 0x7fffffffLL || gy > 65535) {
      set_error("eg_rotary: grid too large");
      return 1;
    }
    if (check_grid("eg_rotary", gx, threads)) return 1;
    EG_LAUNCH((rotary_kernel<T, VEC, HPT, INTER>), dim3((unsigned)gx, (unsigned)gy), dim3(threads),
              a.per_block * a.pairs * sizeof(float2), st, a);
    return check_launch("eg_rotary");
  };
  // Two heads a thread (q and k of 32768 tokens, 32 + 8 heads of 128, forward and backward: one
  // 270 us, two 230, four 233, eight 254), one where tokens are few. Kernel times of one and two at
  // 32 + 8 heads, bf16, tokens 32: 3.1 / 3.6 us, 256: 3.3 / 3.9, 512: 3.8 / 4.1, 2048: 6.2 / 6.3,
  // 4096: 16.3 / 15.8; fp32, 128: 3.1 / 3.3, 512: 4.0 / 4.0, 2048: 14.9 / 14.0.
  if (a.tokens * chunks * ((heads + 1) / 2) < 65536) return go(std::integral_constant<int, 1>{});
  return go(std::integral_constant<int, 2>{});
}

// The widest pack (at most 16 bytes) that divides the halves, the copied columns and every
// stride, and to which the tensors are aligned.
template <typename T, int VEC>
int by_width(const RotaryArgs& a, bool inter, hipStream_t st) {
  if constexpr (VEC > 1) {
    bool fits = a.pairs % VEC == 0 && a.head_dim % VEC == 0;
    for (int64_t s : {a.q_token, a.q_head, a.k_token, a.k_head}) fits = fits && s % VEC == 0;
    for (const void* p : {a.q, a.k, (const void*)a.qo, (const void*)a.ko})
      fits = fits && (uintptr_t)p % (VEC * sizeof(T)) == 0;
    if (!fits) return by_width<T, VEC / 2>(a, inter, st);
  }
  return inter ? launch<T, VEC, true>(a, st) : launch<T, VEC, false>(a, st);
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" int eg_rotary(const void* q, const void* k, void* q_out, void* k_out,
                         const void* positions, int positions_64, const double* freqs,
                         int64_t tokens, int64_t heads_q, int64_t heads_k, int64_t head_dim,
                         int64_t pairs, const int64_t* strides, float amplitude, int interleaved,
                         int inverse, int dtype, void* stream) {
  static const char* name = "eg_rotary";
  clear_error();
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
  for (int i = 0; i < 4; ++i) {  // token steps and head steps
    const int bits = i % 2 ? 40 : 32;
    if (strides[i] < 0 || strides[i] > ((int64_t)1 << bits)) {
      set_error("%s: strides must be at least 0 and at most 2^32 (tokens) or 2^40 (heads) elements",
                name);
      return 1;
    }
  }
  if (tokens == 0 || head_dim == 0 || heads_q + heads_k == 0) return 0;
  if ((heads_q && (!q || !q_out)) || (heads_k && (!k || !k_out)) || !positions ||
      (pairs && !freqs)) {
    set_error("%s: null pointer", name);
    return 1;
  }
  RotaryArgs a = {};
  a.q = q, a.k = heads_k ? k : nullptr, a.qo = q_out, a.ko = heads_k ? k_out : nullptr;
  a.pos = positions, a.freq = freqs;
  a.tokens = tokens;
  a.q_token = strides[0], a.q_head = strides[1], a.k_token = strides[2], a.k_head = strides[3];
  a.heads_q = (int)heads_q, a.heads_k = (int)heads_k, a.head_dim = (int)head_dim;
  a.pairs = (int)pairs, a.pos64 = positions_64;
  a.amp = amplitude, a.sign = inverse ? -1.f : 1.f;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    return by_width<scalar_t, 16 / (int)sizeof(scalar_t)>(a, interleaved != 0, as_stream(stream));
  });
}
