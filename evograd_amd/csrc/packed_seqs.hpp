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
// one wave-wide sum per halving, and no list to build, sort, keep or launch for.
//
// A walk may also be cut into pieces (dK/dV): a tile of index j makes j / m + 1 of them, m
// being the same for all, so the pieces of the tiles below index j of a sequence have a
// closed form too (Cut::below) and the search is the same.
//
// What it costs: the bounds' load (from L2) and about 30 instructions a halving; up to
// kSearchSeqs sequences the bounds stay in registers, four per lane. Past that every halving
// would read them again (1024 sequences: 15 us a workgroup), so there one workgroup orders the
// sequences by size class first (packed_plan_kernel, packed_attention.hip) and a workgroup
// searches the running count of their tiles, 64 entries a step; walks are not cut then.
#pragma once

#include "eg_common.hpp"

namespace eg {

constexpr int kSearchSeqs = 256;

struct PackedSeqs {
  const int* cu;  // [n + 1]
  int n, tokens;
  // past kSearchSeqs sequences: their order [n], and the tiles before each in it [n + 1]
  const int *order, *start;
};

// First row and length of sequence s (none for s >= n). Every bound is clamped to the tensors'
// rows, so whatever cu holds no access leaves them.
__device__ __forceinline__ void seq_bounds(const PackedSeqs& p, int s, int& begin, int& len) {
  const int b = p.cu[min(s, p.n)], e = p.cu[min(s + 1, p.n)];
  begin = min(max(b, 0), p.tokens);
  len = min(max(e, begin), p.tokens) - begin;
}

// Tiles of `rows` rows that n sequences of `tokens` rows have at most, and one workgroup at
// least for the rows that no sequence holds.
inline int64_t packed_tiles(int64_t tokens, int64_t n, int rows) {
  return (tokens + n * (rows - 1)) / rows + 1;
}

// Wave-wide sums and maximum (of values >= 0), in every lane, in a fixed order.
template <typename T, typename Op>
__device__ __forceinline__ T wave_combine(T v, Op op) {
  auto step = [&](auto dpp) {
    int x;
    __builtin_memcpy(&x, &v, 4);
    x = dpp(x);
    T y;
    __builtin_memcpy(&y, &x, 4);
    v = op(v, y);
  };
  step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false); });  // row_shr:1
  step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false); });  // row_shr:2
  step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false); });  // row_shr:4
  step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false); });  // row_shr:8
  step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); });  // row_bcast:15
  step([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false); });  // row_bcast:31
  int x;
  __builtin_memcpy(&x, &v, 4);
  x = __builtin_amdgcn_readlane(x, 63);
  __builtin_memcpy(&v, &x, 4);
  return v;
}
__device__ __forceinline__ int wave_sum(int v) {
  return wave_combine(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_combine(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ int wave_max(int v) {
  return wave_combine(v, [](int a, int b) { return max(a, b); });
}

// How walks are cut: a tile of index j into j / m + 1 pieces; m = 0: not at all.
struct Cut {
  int m;
  float inv;
  __device__ __forceinline__ int over(int n) const {  // n / m
    int q = (int)((float)n * inv);
    const int r = n - q * m;
    if (r < 0) --q;
    else if (r >= m) ++q;
    return q;
  }
  __device__ __forceinline__ int pieces(int j) const { return m ? over(j) + 1 : 1; }
  // pieces of the tiles 0 .. n - 1
  __device__ __forceinline__ int below(int n) const {
    if (!m) return n;
    const int q = over(n), r = n - q * m;
    return n + m * (q * (q - 1) / 2) + q * r;
  }
};

struct SeqTile {
  int begin, len;     // the sequence's first row and its length
  int tile, tiles;    // index among the tiles of the sequence
  int piece, pieces;  // of the tile's walk
  int spare;          // no tile: index past the last piece, or -1 (bounds that are no sequence's)
};

// The tile of rank `rank` by the plan: the sequences in its order, each one's tiles from its
// last on. Wave-uniform; the search narrows [lo, hi) to a 64th a step.
template <int ROWS>
__device__ __forceinline__ bool find_planned(const PackedSeqs& p, int rank, SeqTile& t) {
  const int lane = threadIdx.x & 63;
  const int all = max(p.start[p.n], 0);  // a count past 2^31 is no sequences'
  t.piece = 0;
  t.pieces = 1;
  t.tile = t.tiles = 0;
  t.spare = rank - all;
  if (rank >= all) return false;
  int lo = 0, hi = p.n;  // start[lo] <= rank < start[hi]
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
    const bool before = at < hi && p.start[min(at, hi)] <= rank;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
    hi = min(hi, lo + (n + 1) * step);
    lo += n * step;
  }
  t.spare = -1;
  seq_bounds(p, p.order[lo], t.begin, t.len);
  t.tiles = (int)(((unsigned)t.len + ROWS - 1) / ROWS);
  t.tile = t.tiles - 1 - (rank - p.start[lo]);
  return t.tile >= 0 && t.tile < t.tiles;  // false: bounds that are no sequences'
}

// The piece of rank `rank`, or false. Called by whole waves; every lane gets the result.
// CUT: with the batch's work known, W = the sum over all tiles of (index + 1), walks are cut
// with m = max(least, ceil(W * share)); pass least and share > 0.
template <int ROWS, bool CUT>
__device__ __forceinline__ bool find_tile(const PackedSeqs& p, int rank, SeqTile& t, int least = 0,
                                          float share = 0.f) {
  constexpr int KEEP = kSearchSeqs / 64;
  const int lane = threadIdx.x & 63;
  if (p.n > kSearchSeqs) return find_planned<ROWS>(p, rank, t);
  auto bounds = [&](int s, int& begin, int& len) { seq_bounds(p, s, begin, len); };
  auto tiles_of = [](int len) { return (int)(((unsigned)len + ROWS - 1) / ROWS); };
  int begin[KEEP], len[KEEP];
  bounds(lane, begin[0], len[0]);
#pragma unroll
  for (int c = 1; c < KEEP; ++c) begin[c] = len[c] = 0;
  if (p.n > 64) {
#pragma unroll
    for (int c = 1; c < KEEP; ++c) bounds(64 * c + lane, begin[c], len[c]);
  }
  // f(tiles) of every sequence, each lane its own
  auto each = [&](auto f) {
    f(tiles_of(len[0]));
    if (p.n > 64) {
#pragma unroll
      for (int c = 1; c < KEEP; ++c) f(tiles_of(len[c]));
    }
  };
  Cut cut{0, 0.f};
  int most = 0;
  {
    float work = 0.f;
    each([&](int nt) {
      most = max(most, nt);
      if (CUT) work += 0.5f * (float)nt * (float)(nt + 1);
    });
    most = wave_max(most);
    if (CUT) {
      work = wave_sum(work);
      cut.m = max(least, (int)ceilf(work * share));
      cut.inv = 1.f / (float)cut.m;
    }
  }
  auto count = [&](int j) {  // pieces of the tiles of index >= j
    const int under = cut.below(j);
    int c = 0;
    each([&](int nt) { c += nt > j ? cut.below(nt) - under : 0; });
    return wave_sum(c);
  };
  const int all = max(count(0), 0);  // a count past 2^31 is no sequences'
  if (rank >= all) {
    t.spare = rank - all;
    return false;
  }
  int lo = 0, hi = most, above = 0;  // count(lo) > rank >= count(hi) = above
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2, c = count(mid);
    if (c > rank) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  // `above` pieces come before those of index lo; the sequences that have such a tile
  // follow in their order.
  t.spare = -1;
  t.tile = lo;
  t.pieces = cut.pieces(lo);
  int left = rank - above;
  const int nth = CUT ? left / t.pieces : left;
  t.piece = CUT ? left - nth * t.pieces : 0;
  left = nth;
  bool found = false;
  auto look = [&](int b, int l) {
    uint64_t have = __builtin_amdgcn_ballot_w64(tiles_of(l) > lo);
    const int c = __builtin_popcountll(have);
    if (left >= c) {
      left -= c;
      return;
    }
    for (; left > 0; --left) have &= have - 1;
    const int at = __builtin_ctzll(have);
    t.begin = __builtin_amdgcn_readlane(b, at);
    t.len = __builtin_amdgcn_readlane(l, at);
    found = true;
  };
  look(begin[0], len[0]);
#pragma unroll
  for (int c = 1; c < KEEP; ++c)
    if (!found && 64 * c < p.n) look(begin[c], len[c]);
  t.tiles = found ? tiles_of(t.len) : 0;
  return found;
}

// Zeroes the rows that no sequence holds (before cu[0], from cu[n] on) of `cols` columns of
// a [tokens][ld] tensor; the workgroups past the last of `ranks` pieces share them.
template <typename T>
__device__ __forceinline__ void zero_unused_rows(const PackedSeqs& p, const SeqTile& t, int rank,
                                                 int ranks, T* dst, int64_t ld, int cols) {
  if (t.spare < 0) return;
  const int spares = ranks - rank + t.spare;
  const int head = min(max(p.cu[0], 0), p.tokens);
  const int tail = min(max(p.cu[p.n], head), p.tokens);
  const int64_t unused = (int64_t)head + (p.tokens - tail);
  for (int64_t e = (int64_t)t.spare * blockDim.x + threadIdx.x; e < unused * cols;
       e += (int64_t)spares * blockDim.x) {
    const int64_t r = e / cols;
    dst[(r < head ? r : r - head + tail) * ld + e % cols] = from_f32<T>(0.f);
  }
}

}  // namespace eg
