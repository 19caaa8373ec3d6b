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
// remainder is rounded to fp32 for the sine and cosine. A thread does that once for its pairs of a token and uses
// it for all of its heads, so no table is stored, gathered or read.
//
// Layout: q [tokens, heads_q, head_dim] and k [tokens, heads_k, head_dim], head_dim
// contiguous, other strides free; outputs contiguous. A thread owns a (token, chunk of VEC
// pairs) and serves groups of four heads, the group's loads issued together; the heads'
// groups are dealt out along grid y as far as that fills the chip.
#include "eg_common.hpp"

namespace eg {
namespace {

constexpr int kBlock = 256;
constexpr int kHeads = 4;  // heads whose loads are in flight together

struct RotaryArgs {
  const void *q, *k;
  void *qo, *ko;
  const void* pos;
  const double* freq;
  int64_t tokens, q_token, q_head, k_token, k_head;
  int heads_q, heads_k, head_dim, pairs, pos64;
  float amp, sign;
};

// Chunks of a head: pairs / VEC of them rotate 2 VEC columns, the rest copy VEC each.
template <typename T, int VEC, bool INTER>
__global__ __launch_bounds__(kBlock) void rotary_kernel(RotaryArgs a) {
  const int turned = a.pairs / VEC, chunks = turned + (a.head_dim - 2 * a.pairs) / VEC;
  const int64_t idx = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  const int64_t t = idx / chunks;
  if (t >= a.tokens) return;
  const int ch = (int)(idx - t * chunks);
  const bool turn = ch < turned;
  // columns of the chunk's two packs (a copying chunk has the first alone)
  const int c1 = !turn ? 2 * a.pairs + (ch - turned) * VEC : INTER ? 2 * ch * VEC : ch * VEC;
  const int c2 = !turn ? c1 : INTER ? c1 + VEC : c1 + a.pairs;
  float cs[VEC], sn[VEC];
  if (turn) {
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[t] : (double)((const int*)a.pos)[t];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const double turns = pos * (a.freq[ch * VEC + i] * 0.15915494309189533577);
      const double rest = turns - rint(turns), quarter = rint(4.0 * rest);
      float s0, c0;
      sincospif(2.f * (float)(rest - 0.25 * quarter), &s0, &c0);
      const int n = (int)quarter & 3;  // s0, c0 turned by n quarters
      const float s1 = n & 1 ? c0 : s0, c1 = n & 1 ? s0 : c0;
      cs[i] = a.amp * ((n + 1) & 2 ? -c1 : c1);
      sn[i] = a.amp * a.sign * (n & 2 ? -s1 : s1);
    }
  }
  const int groups_q = (a.heads_q + kHeads - 1) / kHeads;
  const int groups = groups_q + (a.heads_k + kHeads - 1) / kHeads;
  for (int g = blockIdx.y; g < groups; g += gridDim.y) {
    const bool isq = g < groups_q;
    const int heads = isq ? a.heads_q : a.heads_k, h0 = (isq ? g : g - groups_q) * kHeads;
    const int64_t step = isq ? a.q_head : a.k_head;
    const T* src = (const T*)(isq ? a.q : a.k) + t * (isq ? a.q_token : a.k_token) + h0 * step;
    T* dst = (T*)(isq ? a.qo : a.ko) + (t * heads + h0) * a.head_dim;
    Pack<T, VEC> x1[kHeads], x2[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j)
      if (h0 + j < heads) {
        x1[j] = *reinterpret_cast<const Pack<T, VEC>*>(src + j * step + c1);
        if (turn) x2[j] = *reinterpret_cast<const Pack<T, VEC>*>(src + j * step + c2);
      }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      if (h0 + j >= heads) continue;
      T* row = dst + (int64_t)j * a.head_dim;
      if (turn) {
        Pack<T, VEC> y1, y2;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          // pair i: elements i of the two packs, or 2i and 2i + 1 of the two as one run
          const int e = INTER ? 2 * i : i, f = INTER ? 2 * i + 1 : i;
          const float u = to_f32(INTER && e >= VEC ? x2[j].v[e % VEC] : x1[j].v[e % VEC]);
          const float v = to_f32(!INTER || f >= VEC ? x2[j].v[f % VEC] : x1[j].v[f % VEC]);
          const T yu = from_f32<T>(u * cs[i] - v * sn[i]), yv = from_f32<T>(v * cs[i] + u * sn[i]);
          if (INTER && e >= VEC) y2.v[e % VEC] = yu; else y1.v[e % VEC] = yu;
          if (!INTER || f >= VEC) y2.v[f % VEC] = yv; else y1.v[f % VEC] = yv;
        }
        *reinterpret_cast<Pack<T, VEC>*>(row + c1) = y1;
        *reinterpret_cast<Pack<T, VEC>*>(row + c2) = y2;
      } else {
        *reinterpret_cast<Pack<T, VEC>*>(row + c1) = x1[j];
      }
    }
  }
}

template <typename T, int VEC, bool INTER>
int launch(const RotaryArgs& a, hipStream_t st) {
  const int64_t chunks = a.pairs / VEC + (a.head_dim - 2 * a.pairs) / VEC;
  const int64_t gx = (a.tokens * chunks + kBlock - 1) / kBlock;
  const int64_t groups = (a.heads_q + kHeads - 1) / kHeads + (a.heads_k + kHeads - 1) / kHeads;
  if (gx > 0x7fffffffLL) { set_error("eg_rotary: grid too large"); return 1; }
  EG_LAUNCH((rotary_kernel<T, VEC, INTER>), dim3((unsigned)gx, (unsigned)groups), dim3(kBlock), 0,
            st, a);
  return check_launch("eg_rotary");
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
  if (heads_q > (1 << 16) || heads_k > (1 << 16) || head_dim > (1 << 16) ||
      tokens > ((int64_t)1 << 32)) {
    set_error("%s: size out of range (heads and head_dim <= 65536, tokens <= 2^32)", name);
    return 1;
  }
  if (!strides) { set_error("%s: null strides", name); return 1; }
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || strides[i] > ((int64_t)1 << 32)) {
      set_error("%s: strides must be at least 0 and at most 2^32 elements", name);
      return 1;
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
