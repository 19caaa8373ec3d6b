// Embedding lookup with scaling, and its gradient by sorted tokens, for gfx950.
//
//   out[t] = scale * weight[ids[t]]
//   dweight[v] = scale * sum of dout[t] over the tokens t with ids[t] == v
// in fp32, each output rounded once. An id's tokens are added in ascending pieces; the partial sums
// of a run over many pieces are dealt to kJoinAdders adders and joined in their order. A token equal to
// ignore_index gives a row of zeros, any other one outside [0, vocab) a row of NaN; neither is used
// as an index or has a gradient.
//
// The gradient of few tokens is one launch (embed_few_kernel), that of more runs in three, both
// without atomics on their sums:
//   embed_sort_kernel   orders the tokens by id, equal ones by position. The ids are dealt to
//                       buckets, id modulo their number (a power of two): frequent tokens tend
//                       to have low ids, which ranges of ids would put into one bucket. Each bucket's
//                       workgroup reads all tokens twice: first it counts its own ids per wave
//                       (a wave holds a range of positions) and those of the buckets before it,
//                       which is where its part of the order begins, then it places its tokens.
//                       Workgroups behind those zero the beginning of the table: most of it is
//                       rows without a token, and nothing else moves meanwhile.
//   embed_sum_kernel    cuts the order into pieces and adds the rows of each; a run of one id that
//                       lies within a piece is a finished row, the others leave an fp32 partial
//                       row per piece.
//   embed_join_kernel   adds the partial rows of the runs that cross pieces, in order; the same
//                       launch writes the rows of ids without a token behind the beginning.
//
// Memory-bound: the backward reads T rows and writes the table. bf16, 16384 tokens of [128256,
// 4096] whose frequencies fall as one over their rank: forward 32 us, backward 197 (6.0 TB/s);
// fp16 8191 tokens of [50257, 1538], a third of them the same: 9 and 40; 32 tokens forward 3 us, a
// launch. Steps of the first backward (259 us): ids loaded eight at a time and matched one by one
// where they are few, the zeros beside the join and not the sums, two packs of zeros a thread (4: 234,
// 8: 250, one: 242 where two took 213), zeros under the ordering.
#include "eg_common.hpp"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace eg {
namespace {

constexpr int kGatherThreads = 256;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kBucketIds = 1024;  // at most, an id per thread in the scan
constexpr int kMostPiece = 32;
constexpr int kSumThreads = 256, kFewestLanes = 16, kMostGroups = kSumThreads / kFewestLanes;
constexpr int kSingly = 4;      // ids of 64 positions that are placed one by one
constexpr int kEarlyPacks = 2;  // of 16 bytes, per thread
constexpr int kAhead = 8;       // loads of a thread on their way at once
constexpr int kFewTokens = 256, kFewThreads = 512, kFewLanes = 128;
constexpr int kJoinLanes = 64, kJoinAdders = 8, kJoinThreads = kJoinLanes * kJoinAdders;
constexpr int kJoinParts = 4;  // workgroups that share a piece's columns, at most
constexpr int kZeroPacks = 2;  // per thread

struct EmbedArgs {
  const void *weight, *dout;
  const void* ids;
  void *out, *dweight;
  int64_t tokens, vocab, ignore_index;
  int hidden, ids_64, accumulate;
  float scale;
  // the order: positions and their ids, and the first place of every id's run (by slot)
  int *order, *key;
  unsigned* first;
  float* part;  // [pieces][2][hidden]: of the run a piece begins in, of the one it ends in
  int64_t early;  // bytes from the table's beginning that are zeroed while the order is found
  int piece;      // tokens of a piece
  int shift;      // 2^shift buckets
  int per;        // ids of a bucket
};

// The token's id, or -1 for one that has no row of the table.
__device__ __forceinline__ int64_t token_id(const EmbedArgs& a, int64_t t) {
  const int64_t id = a.ids_64 ? ((const int64_t*)a.ids)[t] : (int64_t)((const int*)a.ids)[t];
  return id == a.ignore_index || id < 0 || id >= a.vocab ? -1 : id;
}
__device__ __forceinline__ bool ignored(const EmbedArgs& a, int64_t t) {
  return (a.ids_64 ? ((const int64_t*)a.ids)[t] : (int64_t)((const int*)a.ids)[t]) ==
         a.ignore_index;
}
// Where an id's run is noted: bucket by bucket.
__device__ __forceinline__ int64_t slot_of(const EmbedArgs& a, unsigned id) {
  return (int64_t)(id & ((1u << a.shift) - 1)) * a.per + (id >> a.shift);
}

// A pack of a row: c its first column, lo its first own element (RAG, eg_common.hpp).
template <typename T, int VEC, bool RAG>
struct RowAt {
  int c, lo;
  __device__ __forceinline__ RowAt(int pack, int cols) : c(pack * VEC), lo(0) {
    if constexpr (RAG) {
      const RaggedPack p = ragged_pack<VEC>(c, cols);
      c = p.c, lo = p.lo;
    }
  }
  __device__ __forceinline__ Pack<T, VEC> load(const T* row) const {
    if constexpr (RAG) return load_ragged_raw<T, VEC, false>(row + c);
    else return *reinterpret_cast<const Pack<T, VEC>*>(row + c);
  }
  __device__ __forceinline__ void store(T* row, const float (&v)[VEC]) const {
    if constexpr (RAG) store_ragged<T, VEC, true>(row + c, lo, v);
    else store_vec<T, VEC, true>(row + c, v);
  }
};

// `lanes` threads a token (a power of two), which walk its row in packs.
template <typename T, int VEC, bool RAG>
__global__ __launch_bounds__(kGatherThreads) void embed_gather_kernel(EmbedArgs a, int lanes) {
  const int64_t t = (int64_t)blockIdx.x * (kGatherThreads / lanes) + threadIdx.x / lanes;
  if (t >= a.tokens) return;
  const int64_t id = token_id(a, t);
  const float fill = ignored(a, t) ? 0.f : NAN;
  const T* src = (const T*)a.weight + (id < 0 ? 0 : id) * a.hidden;
  T* dst = (T*)a.out + t * a.hidden;
  const int packs = (a.hidden + VEC - 1) / VEC;
  for (int p = threadIdx.x & (lanes - 1); p < packs; p += lanes) {
    const RowAt<T, VEC, RAG> at(p, a.hidden);
    float v[VEC];
    if (id < 0) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = fill;
    } else {
      const Pack<T, VEC> x = at.load(src);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = a.scale * to_f32(x.v[i]);
    }
    at.store(dst, v);
  }
}

// Lanes of the wave whose `v` (below 2^bits) equals this lane's, among those of `in`.
__device__ __forceinline__ uint64_t same_value(unsigned v, uint64_t in, int bits) {
  for (int b = 0; b < bits; ++b) {
    const bool set = v >> b & 1;
    const uint64_t ones = __ballot(set);
    in &= set ? ones : ~ones;
  }
  return in;
}

template <typename ID>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedArgs a) {
  extern __shared__ unsigned counts[];  // [waves][per]
  __shared__ unsigned sums[kSortWaves], base;
  __shared__ unsigned staged[kSortWaves][kAhead * kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned bucket = blockIdx.x, mask = (1u << a.shift) - 1;
  if (bucket > mask) {  // the table's beginning
    typedef unsigned int words __attribute__((ext_vector_type(4)));
    words* p = (words*)a.dweight + (int64_t)(bucket - mask - 1) * (kSortThreads * kEarlyPacks);
#pragma unroll
    for (int u = 0; u < kEarlyPacks; ++u)
      __builtin_nontemporal_store((words){0, 0, 0, 0}, p + u * kSortThreads + threadIdx.x);
    return;
  }
  unsigned* mine = counts + wave * a.per;
  for (int i = threadIdx.x; i < kSortWaves * a.per; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  // this wave's positions
  const int tokens = (int)a.tokens, share = (tokens + kSortThreads - 1) / kSortThreads * kWave;
  const int from = (int)min((int64_t)wave * share, a.tokens), to = min(from + share, tokens);
  // The ids of kAhead runs of 64 positions, all on their way at once, as (bucket, place in it) in
  // one word; all bits set for a token of no row.
  unsigned code[kAhead];
  const unsigned first = bucket * kBucketIds;
  auto fetch = [&](int t0) {
    ID id[kAhead];
    const ID* at = (const ID*)a.ids + t0 + lane;
    if (t0 + kAhead * kWave <= to) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) id[u] = at[u * kWave];
    } else {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) id[u] = t0 + u * kWave + lane < to ? at[u * kWave] : (ID)-1;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const bool row = id[u] >= 0 && (int64_t)id[u] < a.vocab && id[u] != a.ignore_index;
      const unsigned v = (unsigned)id[u];
      code[u] = row ? (v & mask) * kBucketIds | v >> a.shift : ~0u;
    }
  };
  unsigned before = 0;  // the wave's tokens of earlier buckets
  for (int t0 = from; t0 < to; t0 += kAhead * kWave) {
    fetch(t0);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      before += __popcll(__ballot(code[u] < first));
      if (code[u] - first < kBucketIds) atomicAdd(&mine[code[u] - first], 1u);
    }
  }
  if (lane == 0) sums[wave] = before;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned s = 0;
    for (int w = 0; w < kSortWaves; ++w) s += sums[w];
    base = s;
  }
  // the ids' counts, and where each begins: a scan over the threads, one id each
  unsigned count = 0;
  if ((int)threadIdx.x < a.per)
    for (int w = 0; w < kSortWaves; ++w) count += counts[w * a.per + threadIdx.x];
  unsigned upto = count;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const unsigned other = __shfl_up(upto, off);
    if (lane >= off) upto += other;
  }
  __syncthreads();  // base is written, sums has been read
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  unsigned start = base + upto - count;
  for (int w = 0; w < wave; ++w) start += sums[w];
  if ((int)threadIdx.x < a.per) {
    a.first[(int64_t)bucket * a.per + threadIdx.x] = start;
    if (bucket == mask && (int)threadIdx.x == a.per - 1)
      a.first[((int64_t)bucket + 1) * a.per] = start + count;
    // each wave's tokens of an id stand behind those of the waves before it
    for (int w = 0; w < kSortWaves; ++w) {
      const unsigned n = counts[w * a.per + threadIdx.x];
      counts[w * a.per + threadIdx.x] = start;
      start += n;
    }
  }
  __syncthreads();
  const int bits = 32 - __clz(a.per);  // of a place in the bucket
  for (int t0 = from; t0 < to; t0 += kAhead * kWave) {
    if (share > kAhead * kWave) fetch(t0);  // else they are still there
    unsigned runs = 0;                      // that hold ids of the bucket
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (__ballot(code[u] - first < kBucketIds)) {
        staged[wave][u * kWave + lane] = code[u];
        runs |= 1u << u;
      }
    while (runs) {
      const int u = __ffs(runs) - 1;
      runs &= runs - 1;
      const unsigned local = staged[wave][u * kWave + lane] - first;  // the lane's own
      const bool in = local < kBucketIds;
      uint64_t left = __ballot(in);
      // `same`: the lanes of this lane's id, which stand behind the id's earlier ones in their order;
      // the last of them moves the id's place on, after all have read it and before any reads again
      auto put = [&](bool now, uint64_t same) {
        const uint64_t below = same & ((1ull << lane) - 1);
        const unsigned place = mine[now ? local : 0] + __popcll(below);
        if (now) {
          a.order[place] = t0 + u * kWave + lane;
          a.key[place] = (int)(local << a.shift | bucket);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (now && below == (same & ~(1ull << lane))) mine[local] = place + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      };
      // a few ids one by one, more of them by their bits
      for (int n = 0; n < kSingly && left; ++n) {
        const unsigned v = __builtin_amdgcn_readlane(local, __ffsll((unsigned long long)left) - 1);
        const uint64_t same = __ballot(local == v);
        put(local == v, same);
        left &= ~same;
      }
      if (left) put(left >> lane & 1, same_value(local, left, bits));
    }
  }
}

template <typename T, int VEC, bool RAG>
__device__ void write_row(const EmbedArgs& a, const RowAt<T, VEC, RAG>& at, int id,
                          const float (&sum)[VEC]) {
  T* row = (T*)a.dweight + (int64_t)id * a.hidden;
  float v[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = a.scale * sum[i];
  if (a.accumulate) {
    const Pack<T, VEC> old = at.load(row);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] += to_f32(old.v[i]);
  }
  at.store(row, v);
}

// Rows of ids without a token, over the table as one run of packs.
template <typename T, int VEC>
__device__ void zero_rows(const EmbedArgs& a, int64_t block) {
  constexpr int kChunk = kJoinThreads * kZeroPacks * VEC;
  __shared__ uint64_t bits[kChunk / kWave + 1];  // of the rows that the chunk touches
  const int64_t first = a.early / (int64_t)sizeof(T) + block * kChunk, total = a.vocab * a.hidden;
  const int64_t row0 = first / a.hidden;
  const unsigned rest = (unsigned)(first - row0 * a.hidden), hidden = a.hidden;
  const int rows = (int)min((int64_t)((rest + kChunk - 1) / hidden + 1), a.vocab - row0);
  for (int r = threadIdx.x; r < (rows + kWave - 1) / kWave * kWave; r += kJoinThreads) {
    const int64_t s = slot_of(a, (unsigned)(row0 + min(r, rows - 1)));
    const uint64_t b = __ballot(a.first[s] == a.first[s + 1]);
    if ((threadIdx.x & 63) == 0) bits[r / kWave] = b;
  }
  __syncthreads();
  auto empty = [&](unsigned r) { return (bool)(bits[r / kWave] >> (r % kWave) & 1); };
  T* p = (T*)a.dweight + first;
#pragma unroll
  for (int u = 0; u < kZeroPacks; ++u) {
    const unsigned e = (u * kJoinThreads + threadIdx.x) * VEC, in = rest + e;
    if (first + e >= total) break;
    // the pack's first row and the last one; between them lie others only in rows below a pack
    const unsigned r = in / hidden, end = min((unsigned)rows - 1, (in + VEC - 1) / hidden);
    const bool whole = first + e + VEC <= total && (hidden >= VEC || r == end);
    if (whole && empty(r) && empty(end)) {
      const float z[VEC] = {};
      store_vec<T, VEC, true>(p + e, z);
    } else if (!whole || empty(r) || empty(end)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (first + e + i < total && empty((in + i) / hidden)) p[e + i] = from_f32<T>(0.f);
    }
  }
}

// kSumThreads / lanes pieces a workgroup, `lanes` threads (a power of two) over the columns of one.
template <typename T, int VEC, bool RAG>
__global__ __launch_bounds__(kSumThreads) void embed_sum_kernel(EmbedArgs a, int lanes,
                                                                int column_blocks) {
  // a piece's tokens and ids, and the ids before and behind it
  __shared__ int where[kMostGroups][kMostPiece], ids[kMostGroups][kMostPiece + 2];
  const int64_t n = a.first[(int64_t)a.per << a.shift];
  const int groups = kSumThreads / lanes, group = threadIdx.x / lanes;
  const int64_t piece0 = (int64_t)(blockIdx.x / column_blocks) * groups;
  for (int i = threadIdx.x; i < groups * (a.piece + 2); i += kSumThreads) {
    const int g = i / (a.piece + 2), j = i - g * (a.piece + 2);
    const int64_t at = (piece0 + g) * a.piece + j - 1;
    const int64_t safe = max((int64_t)0, min(at, a.tokens - 1));  // read before n has come
    const int id = a.key[safe], pos = a.order[safe];
    ids[g][j] = at >= 0 && at < n ? id : -1;
    if (j >= 1 && j <= a.piece) where[g][j - 1] = pos;
  }
  __syncthreads();
  const int64_t piece = piece0 + group;
  const int pack = blockIdx.x % column_blocks * lanes + (threadIdx.x & (lanes - 1));
  if (piece * a.piece >= n || pack * VEC >= a.hidden) return;
  const int len = (int)min((int64_t)a.piece, n - piece * a.piece);
  const RowAt<T, VEC, RAG> at(pack, a.hidden);
  float acc[VEC] = {};
  bool crosses = ids[group][0] == ids[group][1];  // the run began before the piece
  auto finish = [&](int j) {  // the run that ends with the piece's j-th token
    const bool behind = j == len - 1 && ids[group][j + 2] == ids[group][j + 1];
    if (!crosses && !behind) {
      write_row(a, at, ids[group][j + 1], acc);
    } else {
      float* row = a.part + (piece * 2 + !crosses) * a.hidden + at.c;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (i >= at.lo) row[i] = acc[i];
    }
    crosses = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  };
  for (int j0 = 0; j0 < len; j0 += kAhead) {
    Pack<T, VEC> x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (j0 + u < len) x[u] = at.load((const T*)a.dout + (int64_t)where[group][j0 + u] * a.hidden);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = j0 + u;
      if (j >= len) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += to_f32(x[u].v[i]);
      if (j == len - 1 || ids[group][j + 2] != ids[group][j + 1]) finish(j);
    }
  }
}

// The run that begins in a piece and goes on behind it: the piece's second partial row and the
// first ones of the pieces behind, dealt to kJoinAdders adders whose sums are added in order.
// `parts` workgroups share the columns of a piece. Those past `joins` write the rows without tokens.
template <typename T, int VEC, int ZVEC>
__global__ __launch_bounds__(kJoinThreads) void embed_join_kernel(EmbedArgs a, int64_t joins, int parts) {
  if ((int64_t)blockIdx.x >= joins) {
    zero_rows<T, ZVEC>(a, (int64_t)blockIdx.x - joins);
    return;
  }
  __shared__ Pack<float, VEC> sums[kJoinAdders][kJoinLanes];
  const int64_t n = a.first[(int64_t)a.per << a.shift];
  const int64_t piece = blockIdx.x / parts, end = (piece + 1) * a.piece;
  if (end >= n) return;
  const int id = a.key[end];
  if (id != a.key[end - 1]) return;  // no run crosses the piece's end
  const int64_t slot = slot_of(a, (unsigned)id);
  if (a.first[slot] < piece * a.piece) return;  // it began in an earlier piece
  const int64_t last = (a.first[slot + 1] - 1) / a.piece;
  const int lane = threadIdx.x % kJoinLanes, adder = threadIdx.x / kJoinLanes;
  const int step = parts * kJoinLanes * VEC;
  for (int c0 = (int)(blockIdx.x % parts) * kJoinLanes * VEC; c0 < a.hidden; c0 += step) {
    const int c = c0 + lane * VEC;
    float s[VEC] = {}, v[VEC];
    if (c < a.hidden) {
      if (adder == 0) load_f32<float, VEC>(a.part + (piece * 2 + 1) * a.hidden + c, s);
#pragma unroll 8
      for (int64_t p = piece + 1 + adder; p <= last; p += kJoinAdders) {
        load_f32<float, VEC>(a.part + p * 2 * a.hidden + c, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[i] += v[i];
      }
    }
    __syncthreads();  // the last columns' sums have been read
    store_f32<float, VEC>(sums[adder][lane].v, s);
    __syncthreads();
    if (adder || c >= a.hidden) continue;
    for (int k = 1; k < kJoinAdders; ++k)
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] += sums[k][lane].v[i];
    RowAt<T, VEC, false> at(c / VEC, a.hidden);
    write_row(a, at, id, s);
  }
}

// All of it for few tokens: a workgroup of a bucket and a block of columns finds the bucket's tokens
// (one a thread), orders them by counting those before each, adds their rows and writes the rows
// without tokens. `lanes` threads (a power of two) hold the columns; each group of them adds a piece
// of the order, and the runs that cross pieces are joined through LDS.
template <typename T, int VEC, bool RAG, typename ID>
__global__ __launch_bounds__(kFewThreads) void embed_few_kernel(EmbedArgs a, int lanes, int column_blocks) {
  __shared__ int ids[kFewTokens], order[kFewTokens];
  __shared__ __align__(16) int found[kFewTokens + 4];  // (place in the bucket, which of its tokens)
  __shared__ unsigned used[kBucketIds / 32], waves[kFewThreads / kWave];
  __shared__ Pack<float, VEC> part[2][kFewThreads];  // as embed_sum_kernel's partial rows
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const unsigned bucket = blockIdx.x / column_blocks, mask = (1u << a.shift) - 1;
  const int64_t id = t < a.tokens ? (int64_t)((const ID*)a.ids)[t] : -1;
  const bool in = id >= 0 && id < a.vocab && id != a.ignore_index && ((unsigned)id & mask) == bucket;
  const int local = (int)((unsigned)id >> a.shift);  // its place in the bucket
  const uint64_t here = __ballot(in);
  if (lane == 0) waves[wave] = __popcll(here);
  if (t < kBucketIds / 32) used[t] = 0;
  __syncthreads();
  int n = 0, mine = 0;  // the bucket's tokens; those before this one
  for (int w = 0; w < kFewThreads / kWave; ++w) {
    if (w == wave) mine = n;
    n += waves[w];
  }
  mine += __popcll(here & ((1ull << lane) - 1));
  if (in) {
    found[mine] = local * kFewTokens + mine;
    atomicOr(&used[local / 32], 1u << local % 32);
  }
  if (t < 4) found[n + t] = INT_MAX;
  __syncthreads();
  const int groups = kFewThreads / lanes, group = t / lanes;
  const int pack = blockIdx.x % column_blocks * lanes + (t & (lanes - 1));
  const bool live = pack * VEC < a.hidden;
  const RowAt<T, VEC, RAG> at(live ? pack : 0, a.hidden);
  if (live && !a.accumulate) {
    const float zero[VEC] = {};
    const int rows = (int)((a.vocab - bucket + mask) >> a.shift);  // of the bucket
    for (int r = group; r < rows; r += groups)
      if (!(used[r / 32] >> r % 32 & 1))
        at.store((T*)a.dweight + ((int64_t)r << a.shift | bucket) * a.hidden, zero);
  }
  if (n == 0) return;
  if (in) {
    int before = 0;
    const int own = local * kFewTokens + mine;
    for (int j = 0; j < n; j += 4) {
      int other[4];
      *(Pack<int, 4>*)other = *(const Pack<int, 4>*)(found + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) before += other[i] < own;
    }
    order[before] = t, ids[before] = (int)id;
  }
  __syncthreads();
  const int piece = (n + groups - 1) / groups, from = min(group * piece, n), to = min(from + piece, n);
  if (live && from < to) {
    bool crosses = from > 0 && ids[from - 1] == ids[from];
    float acc[VEC] = {};
    for (int e0 = from; e0 < to; e0 += kAhead) {
      Pack<T, VEC> x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (e0 + u < to) x[u] = at.load((const T*)a.dout + (int64_t)order[e0 + u] * a.hidden);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int e = e0 + u;
        if (e >= to) break;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += to_f32(x[u].v[i]);
        const bool last = e + 1 == n || ids[e + 1] != ids[e];
        if (!last && e + 1 < to) continue;
        if (last && !crosses) write_row(a, at, ids[e], acc);
        else store_f32<float, VEC>(part[!crosses][t].v, acc);
        crosses = false;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
      }
    }
  }
  __syncthreads();
  // the run that begins in this piece and goes on behind it
  if (!live || from >= to || to == n || ids[to] != ids[to - 1]) return;
  const int id_out = ids[to - 1];
  if (from > 0 && ids[from - 1] == id_out) return;  // it began in an earlier piece
  float s[VEC];
  load_f32<float, VEC>(part[1][t].v, s);
  for (int g = group + 1; g * piece < n && ids[g * piece] == id_out; ++g) {
    const Pack<float, VEC>& other = part[0][g * lanes + (t & (lanes - 1))];
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[i] += other.v[i];
  }
  write_row(a, at, id_out, s);
}

// Tokens of a piece: a piece's rows are added one after the other, its partial rows are read again.
// Backward, us, with 8 / 16 / 32: 700 tokens of [5003, 768] fp32 15.2 / 16.8 / 19.9; 4096 of [32000,
// 1024] bf16 28.0 / 29.0 / 33.5; 8191 of [50257, 1538] fp16 59.7 / 55.9 / 57.7; 16384 of [128256,
// 4096] bf16 255 / 244 / 241; 65536 of [50257, 768] 137 / 122 / 111.
int piece_for(int64_t tokens) { return tokens < 4096 ? 8 : tokens < 16384 ? 16 : 32; }

// Bytes of the table that the ordering's launch zeroes under way, as many as its time has room
// for. Backward, us, none / 32 MB / this: 16384 tokens of [128256, 4096] bf16 211 / 206 / 197, 2048
// of [128256, 2048] 97 / 91 / 90, 65536 of [50257, 768] 83 / 79 / 75, 700 of [5003, 768] fp32 15 /
// 14 / 14.
int64_t early_bytes(int64_t tokens) { return ((int64_t)32 << 20) + tokens * 3500; }

// One launch for few tokens. It leaves HBM idle under its ordering, and its zeros of rows that are
// not whole packs are slower, which a large table outweighs. Backward, us, three launches / one: 1
// token of [5003, 768] fp32 10.8 / 5.2; 32 of [32000, 1024] bf16 18.4 / 11.8; 256 of [1000, 4096],
// a third of them one id, 16.0 / 11.9 and 512 of those 17.3 / 19.0; 256 equal ones of [1, 4096] 16.9
// / 21; 128 of [48000, 1024] bf16 23.4 / 17.8, of [30000, 4096] 43 / 46; rows in ragged packs, 128 of
// [20000, 1538] fp16 (62 MB) 19.8 / 18.6, of [50257, 770] (77 MB) 22.4 / 25.5; more than kBucketIds
// 2^8 ids, 4000000 of 8: 87 / 157. Added into a table, 128 of [30000, 4096] 12.1 / 4.9.
bool few_tokens(int64_t tokens, int64_t vocab, int64_t bytes, bool accumulate, bool ragged) {
  if (tokens > kFewTokens) return false;
  return accumulate || (vocab <= kBucketIds << 8 && bytes <= (int64_t)(ragged ? 64 : 96) << 20);
}

// A table [vocab, hidden] with `tokens` of it: how the ids are dealt and where the order lies.
struct Layout {
  int shift, per, piece;
  int64_t pieces;
  size_t order, key, first, part, bytes;  // offsets into the workspace
};
Layout layout(int64_t tokens, int64_t vocab, int64_t hidden) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Layout l = {};
  l.shift = 8;
  while (vocab > ((int64_t)kBucketIds << l.shift)) ++l.shift;
  l.per = (int)((vocab + ((int64_t)1 << l.shift) - 1) >> l.shift);
  l.piece = piece_for(tokens);
  l.pieces = (tokens + l.piece - 1) / l.piece;
  l.key = up(tokens * sizeof(int));
  l.first = l.key + up(tokens * sizeof(int));
  l.part = l.first + up((((size_t)l.per << l.shift) + 1) * sizeof(unsigned));
  l.bytes = l.part + (l.pieces > 1 ? (size_t)l.pieces * 2 * hidden * sizeof(float) : 0);
  return l;
}

int lanes_for(int64_t packs, int most) {
  int n = kFewestLanes;
  while (n < packs && n < most) n *= 2;
  return n;
}

template <typename T, typename F>
int by_width(int hidden, std::initializer_list<const void*> tensors, F&& go) {
  using std::integral_constant;
  constexpr int V = 16 / (int)sizeof(T);
  if (hidden < V) return go(integral_constant<int, 1>{}, std::false_type{});
  bool aligned = hidden % V == 0;
  for (const void* p : tensors) aligned = aligned && aligned16(p);
  const integral_constant<int, V> vec;
  return aligned ? go(vec, std::false_type{}) : go(vec, std::true_type{});
}

int check(const char* name, int64_t tokens, int64_t vocab, int64_t hidden) {
  if (tokens < 0 || vocab < 0 || hidden < 0) { set_error("%s: negative size", name); return 1; }
  if (tokens > ((int64_t)1 << 30) || vocab > ((int64_t)1 << 30) || hidden > ((int64_t)1 << 20)) {
    set_error("%s: size out of range (tokens, vocab <= 2^30, hidden <= 2^20)", name);
    return 1;
  }
  return 0;
}

}  // namespace
}  // namespace eg

using namespace eg;

extern "C" int eg_embedding_fwd(const void* weight, const void* ids, int ids_64, void* out,
                                int64_t tokens, int64_t vocab, int64_t hidden, float scale,
                                int64_t ignore_index, int dtype, void* stream) {
  static const char* name = "eg_embedding_fwd";
  clear_error();
  if (check(name, tokens, vocab, hidden)) return 1;
  if (tokens == 0 || hidden == 0) return 0;
  if ((vocab && !weight) || !ids || !out) { set_error("%s: null pointer", name); return 1; }
  EmbedArgs a = {};
  a.weight = weight, a.ids = ids, a.out = out, a.ids_64 = ids_64;
  a.tokens = tokens, a.vocab = vocab, a.hidden = (int)hidden, a.ignore_index = ignore_index;
  a.scale = scale;
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    return by_width<scalar_t>(a.hidden, {weight, (const void*)out}, [&](auto vec, auto rag) -> int {
      constexpr int V = decltype(vec)::value;
      const int lanes = lanes_for((hidden + V - 1) / V, kGatherThreads);
      const int64_t per = kGatherThreads / lanes, blocks = (tokens + per - 1) / per;
      if (check_grid(name, blocks, kGatherThreads)) return 1;
      EG_LAUNCH((embed_gather_kernel<scalar_t, V, decltype(rag)::value>), dim3((unsigned)blocks),
                dim3(kGatherThreads), 0, as_stream(stream), a, lanes);
      return check_launch(name);
    });
  });
}

extern "C" size_t eg_embedding_workspace_bytes(int64_t tokens, int64_t vocab, int64_t hidden) {
  if (tokens < 0 || vocab <= 0 || hidden <= 0) return 0;
  return layout(tokens, vocab, hidden).bytes;
}

extern "C" int eg_embedding_bwd(const void* dout, const void* ids, int ids_64, void* dweight,
                                void* workspace, int64_t tokens, int64_t vocab, int64_t hidden,
                                float scale, int64_t ignore_index, int accumulate, int dtype,
                                void* stream) {
  static const char* name = "eg_embedding_bwd";
  clear_error();
  if (check(name, tokens, vocab, hidden)) return 1;
  if (vocab == 0 || hidden == 0) return 0;
  if ((tokens && (!dout || !ids)) || !dweight || !workspace) {
    set_error("%s: null pointer", name);
    return 1;
  }
  if (!aligned16(workspace)) { set_error("%s: workspace must be 16-byte aligned", name); return 1; }
  const Layout l = layout(tokens, vocab, hidden);
  EmbedArgs a = {};
  a.dout = dout, a.ids = ids, a.dweight = dweight, a.ids_64 = ids_64;
  a.tokens = tokens, a.vocab = vocab, a.hidden = (int)hidden, a.ignore_index = ignore_index;
  a.scale = scale, a.accumulate = accumulate;
  char* ws = (char*)workspace;
  a.order = (int*)ws, a.key = (int*)(ws + l.key), a.first = (unsigned*)(ws + l.first);
  a.part = (float*)(ws + l.part);
  a.shift = l.shift, a.per = l.per, a.piece = l.piece;
  hipStream_t st = as_stream(stream);
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    return by_width<scalar_t>(a.hidden, {dout, (const void*)dweight}, [&](auto vec, auto rag) -> int {
      using T = scalar_t;
      constexpr int V = decltype(vec)::value, W = 16 / (int)sizeof(T);
      const int64_t packs = (hidden + V - 1) / V, bytes = vocab * hidden * (int64_t)sizeof(T);
      const int lanes = lanes_for(packs, kSumThreads), groups = kSumThreads / lanes;
      const int64_t columns = (packs + lanes - 1) / lanes;
      const int64_t sums = (l.pieces + groups - 1) / groups * columns;
      if (few_tokens(tokens, vocab, bytes, accumulate, decltype(rag)::value)) {
        const int wide = lanes_for(packs, kFewLanes);
        const int64_t blocks = (packs + wide - 1) / wide, grid = blocks << l.shift;
        if (check_grid(name, grid, kFewThreads)) return 1;
        auto few = [&](auto id) {
          EG_LAUNCH((embed_few_kernel<T, V, decltype(rag)::value, decltype(id)>), dim3((unsigned)grid),
                    dim3(kFewThreads), 0, st, a, wide, (int)blocks);
        };
        if (ids_64) few(int64_t{});
        else few(int{});
        return check_launch(name);
      }
      // the join in fours or twos of columns where a row's are aligned, zeros in whole packs (8191
      // tokens of [50257, 1538] fp16, a third of them one: 44 us in single columns, 40 in twos)
      const bool flat = aligned16(dweight);
      const bool fours = flat && hidden % 4 == 0, twos = flat && hidden % 2 == 0;
      const int64_t span = kJoinLanes * (fours ? 4 : twos ? 2 : 1);
      const int parts = (int)std::min<int64_t>((hidden + span - 1) / span, kJoinParts);
      const int64_t joins = l.pieces > 1 ? (l.pieces - 1) * parts : 0;
      const int64_t chunk = (int64_t)kJoinThreads * kZeroPacks * (flat ? W : 1);
      const int64_t at_once = kSortThreads * kEarlyPacks * 16;
      const int64_t early = accumulate || !flat ? 0 : std::min(early_bytes(tokens), bytes) / at_once;
      a.early = early * at_once;
      const int64_t zeros =
          accumulate ? 0 : ((bytes - a.early) / (int64_t)sizeof(T) + chunk - 1) / chunk;
      const int64_t sorts = ((int64_t)1 << l.shift) + early;
      if (check_grid(name, sorts, kSortThreads) ||
          check_grid(name, sums, kSumThreads) || check_grid(name, joins + zeros, kJoinThreads))
        return 1;
      const size_t lds = (size_t)kSortWaves * l.per * sizeof(unsigned);
      if (ids_64)
        EG_LAUNCH((embed_sort_kernel<int64_t>), dim3((unsigned)sorts), dim3(kSortThreads), lds, st, a);
      else
        EG_LAUNCH((embed_sort_kernel<int>), dim3((unsigned)sorts), dim3(kSortThreads), lds, st, a);
      if (sums)
        EG_LAUNCH((embed_sum_kernel<T, V, decltype(rag)::value>), dim3((unsigned)sums),
                  dim3(kSumThreads), 0, st, a, lanes, (int)columns);
      auto join = [&](auto c, auto z) {
        EG_LAUNCH((embed_join_kernel<T, decltype(c)::value, decltype(z)::value>),
                  dim3((unsigned)(joins + zeros)), dim3(kJoinThreads), 0, st, a, joins, parts);
      };
      if (joins + zeros) {
        using std::integral_constant;
        if (fours) join(integral_constant<int, 4>{}, integral_constant<int, W>{});
        else if (twos) join(integral_constant<int, 2>{}, integral_constant<int, W>{});
        else if (flat) join(integral_constant<int, 1>{}, integral_constant<int, W>{});
        else join(integral_constant<int, 1>{}, integral_constant<int, 1>{});
      }
      return check_launch(name);
    });
  });
}
