// Sequences packed along one token axis: sequence s holds the rows cu[s] .. cu[s + 1] - 1
// of [tokens, ...] tensors. Shared by the packed attention kernels.
//
// The lengths live on the GPU and are never read on the host, so a grid covers every tile
// that n sequences of `tokens` rows can have (packed_tiles) and each workgroup finds its
// own: the tiles are taken in the order of their index inside their sequence, highest
// first, which is the order of their work (a causal query tile walks the keys before it;
// key tiles are counted from the sequence's end), so the longest walks start first whatever
// the lengths are. The workgroup of rank r searches the index j of its tile by halving,
// with count(j) = sum over s of max(0, tiles(s) - j), the number of tiles with index >= j:
// one wave-wide sum per halving, and no list to build, sort or keep.
#pragma once

#include "eg_common.hpp"

namespace eg {

struct PackedSeqs {
  const int* cu;  // [n + 1]
  int n, tokens;
};

// Workgroups of one head: the tiles of `rows` rows, and one at least for the rows that no
// sequence holds.
inline int64_t packed_tiles(int64_t tokens, int64_t n, int rows) {
  return (tokens + n * (rows - 1)) / rows + 1;
}

// Sum over the wave of an int, in every lane.
__device__ __forceinline__ int wave_sum_int(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return __builtin_amdgcn_readlane(v, 63);
}

// First row and length of sequence s. Every bound is clamped to the tensors' rows, so
// whatever cu holds no access leaves them.
__device__ __forceinline__ int seq_begin(const PackedSeqs& p, int s, int& len) {
  const int b = min(max(p.cu[s], 0), p.tokens);
  len = min(max(p.cu[s + 1], b), p.tokens) - b;
  return b;
}

struct SeqTile {
  int begin, len;   // the sequence's first row and its length
  int tile, tiles;  // index among the tiles of the sequence
};

// The tile of rank `rank`, or false and, in `spare`, the index past the last tile (-1: none,
// bounds that are no sequence's). Called by whole waves; every lane gets the result. WALK:
// also the sum over all tiles of (index + 1), the work of a causal walk.
template <int ROWS, bool WALK>
__device__ __forceinline__ bool find_tile(const PackedSeqs& p, int rank, SeqTile& t, int& spare,
                                          float& walk) {
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](int s) {
    if (s >= p.n) return 0;
    int len;
    seq_begin(p, s, len);
    return (len + ROWS - 1) / ROWS;
  };
  const int first = tiles_of(lane);  // the whole table where n <= 64
  int most = first, all = wave_sum_int(first);
  float w = 0.5f * (float)first * (float)(first + 1);
  for (int s0 = 64; s0 < p.n; s0 += 64) {
    const int nt = tiles_of(s0 + lane);
    most = max(most, nt);
    all += wave_sum_int(nt);
    w += 0.5f * (float)nt * (float)(nt + 1);
  }
  if (WALK) walk = wave_reduce(w, SumOp());
  if (rank >= all) {
    spare = rank - all;
    return false;
  }
  auto count = [&](int j) {
    int c = wave_sum_int(max(0, first - j));
    for (int s0 = 64; s0 < p.n; s0 += 64) c += wave_sum_int(max(0, tiles_of(s0 + lane) - j));
    return c;
  };
  // count(lo) > rank >= count(hi)
  int lo = 0, hi = 1, above = 0;
  {
    int m = most;  // the longest sequence's tiles
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = max(m, __shfl_xor(m, off, 64));
    hi = __builtin_amdgcn_readfirstlane(m);
  }
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2, c = count(mid);
    if (c > rank) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  // `above` = count(lo + 1) tiles come before those of index lo; the sequences that have
  // such a tile follow in their order.
  int left = rank - above, seq = 0;
  for (int s0 = 0; s0 < p.n; s0 += 64) {
    uint64_t have = __builtin_amdgcn_ballot_w64((s0 == 0 ? first : tiles_of(s0 + lane)) > lo);
    const int c = __builtin_popcountll(have);
    if (left < c) {
      for (; left > 0; --left) have &= have - 1;
      seq = s0 + __builtin_ctzll(have);
      break;
    }
    left -= c;
  }
  t.begin = seq_begin(p, seq, t.len);
  t.tile = lo;
  t.tiles = (t.len + ROWS - 1) / ROWS;
  spare = -1;
  return lo < t.tiles;
}

// Zeroes the rows that no sequence holds (before cu[0], from cu[n] on) of one head's columns
// in a [tokens][ld] tensor; workgroup `spare` of `spares`, none where spare < 0.
template <typename T>
__device__ __forceinline__ void zero_unused_rows(const PackedSeqs& p, int spare, int spares, T* dst,
                                                 int64_t ld, int cols) {
  if (spare < 0) return;
  const int head = min(max(p.cu[0], 0), p.tokens);
  const int tail = min(max(p.cu[p.n], head), p.tokens);
  const int64_t unused = (int64_t)head + (p.tokens - tail);
  for (int64_t e = (int64_t)spare * blockDim.x + threadIdx.x; e < unused * cols;
       e += (int64_t)spares * blockDim.x) {
    const int64_t r = e / cols;
    dst[(r < head ? r : r - head + tail) * ld + e % cols] = from_f32<T>(0.f);
  }
}

}  // namespace eg
