// Embedding lookup with scaling, and its gradient by sorted tokens, for gfx950.
//
//   out[t] = scale * weight[ids[t]]
//   dweight[v] = scale * sum of dout[t] over the tokens t with ids[t] == v, t ascending
// in fp32, each output rounded once. A token equal to ignore_index gives a row of zeros, any
// other one outside [0, vocab) a row of NaN; neither is used as an index or has a gradient.
//
// The gradient runs in three launches and without atomics on its sums:
//   embed_sort_kernel   orders the tokens by id, equal ones by position. The ids are dealt to
//                       buckets, id modulo their number (a power of two): frequent tokens tend
//                       to have low ids, which ranges of ids would put into one bucket. Each bucket's
//                       workgroup reads all tokens twice: first it counts its own ids per wave
//                       (a wave holds a range of positions) and those of the buckets before it,
//                       which is where its part of the order begins, then it places its tokens.
//   embed_sum_kernel    cuts the order into pieces of kPiece tokens and adds the rows of each; a
//                       run of one id that lies within a piece is a finished row, the others
//                       leave an fp32 partial row per piece. The same launch writes the rows of
//                       ids without a token.
//   embed_join_kernel   adds the partial rows of the runs that cross pieces, in order.
#include "eg_common.hpp"

#include <algorithm>
#include <type_traits>

namespace eg {
namespace {

constexpr int kGatherThreads = 256;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kBucketIds = 1024;  // at most, an id per thread in the scan
constexpr int kPiece = 32;
constexpr int kSumThreads = 256, kFewestLanes = 16, kMostGroups = kSumThreads / kFewestLanes;
constexpr int kZeroPacks = 8;  // per thread
constexpr int kJoinLanes = 64, kJoinAdders = 8;

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
  int shift;    // 2^shift buckets
  int per;      // ids of a bucket
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

__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedArgs a) {
  extern __shared__ unsigned counts[];  // [waves][per]
  __shared__ unsigned sums[kSortWaves], base;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned bucket = blockIdx.x, mask = (1u << a.shift) - 1;
  unsigned* mine = counts + wave * a.per;
  for (int i = threadIdx.x; i < kSortWaves * a.per; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  // this wave's positions
  const int64_t share = (a.tokens + kSortThreads - 1) / kSortThreads * kWave;
  const int64_t from = min((int64_t)wave * share, a.tokens), to = min(from + share, a.tokens);
  unsigned before = 0;
  for (int64_t t = from + lane; t < to; t += kWave) {
    const int64_t id = token_id(a, t);
    if (id < 0) continue;
    const unsigned b = (unsigned)id & mask;
    before += b < bucket;
    if (b == bucket) atomicAdd(&mine[id >> a.shift], 1u);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off);
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
  const int bits = 32 - __clz(a.per);  // of a bucket's id
  for (int64_t t0 = from; t0 < to; t0 += kWave) {
    const int64_t t = t0 + lane;
    const int64_t id = t < to ? token_id(a, t) : -1;
    const bool in = id >= 0 && ((unsigned)id & mask) == bucket;
    const uint64_t any = __ballot(in);
    if (!any) continue;
    const unsigned local = in ? (unsigned)(id >> a.shift) : 0;
    const uint64_t same = same_value(local, any, bits);
    const uint64_t below = same & ((1ull << lane) - 1);
    const unsigned place = mine[local] + __popcll(below);
    if (in) {
      a.order[place] = (int)t;
      a.key[place] = (int)id;
    }
    // the last of them moves the id's place on, after all have read it and before any reads again
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && below == (same & ~(1ull << lane))) mine[local] = place + 1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
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
  const int64_t first = block * (kSumThreads * kZeroPacks * VEC);
  const int64_t row0 = first / a.hidden, total = a.vocab * a.hidden;
  const int rest = (int)(first - row0 * a.hidden);
  auto empty = [&](int64_t row) {
    const int64_t s = slot_of(a, (unsigned)row);
    return a.first[s] == a.first[s + 1];
  };
  T* p = (T*)a.dweight + first;
  bool clear[kZeroPacks];
#pragma unroll
  for (int u = 0; u < kZeroPacks; ++u) {
    const unsigned e = (u * kSumThreads + threadIdx.x) * VEC, in = rest + e;
    clear[u] = first + e < total && empty(row0 + in / (unsigned)a.hidden);
  }
#pragma unroll
  for (int u = 0; u < kZeroPacks; ++u) {
    const unsigned e = (u * kSumThreads + threadIdx.x) * VEC, in = rest + e;
    if (first + e >= total) continue;
    const int64_t r = in / (unsigned)a.hidden, last = (in + VEC - 1) / (unsigned)a.hidden;
    if (r == last && first + e + VEC <= total) {
      float z[VEC] = {};
      if (clear[u]) store_vec<T, VEC, true>(p + e, z);
    } else {  // a pack of several rows, or the table's end
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (first + e + i < total && empty(row0 + (in + i) / (unsigned)a.hidden))
          p[e + i] = from_f32<T>(0.f);
    }
  }
}

// kSumThreads / lanes pieces a workgroup, `lanes` threads (a power of two) over the columns of one.
template <typename T, int VEC, bool RAG, int ZVEC>
__global__ __launch_bounds__(kSumThreads) void embed_sum_kernel(EmbedArgs a, int lanes, int column_blocks,
                                                                int64_t sum_blocks) {
  if ((int64_t)blockIdx.x >= sum_blocks) {
    zero_rows<T, ZVEC>(a, (int64_t)blockIdx.x - sum_blocks);
    return;
  }
  // a piece's tokens and ids, and the ids before and behind it
  __shared__ int where[kMostGroups][kPiece], ids[kMostGroups][kPiece + 2];
  const int64_t n = a.first[(int64_t)a.per << a.shift];
  const int groups = kSumThreads / lanes, group = threadIdx.x / lanes;
  const int64_t piece0 = (int64_t)(blockIdx.x / column_blocks) * groups;
  for (int i = threadIdx.x; i < groups * (kPiece + 2); i += kSumThreads) {
    const int g = i / (kPiece + 2), j = i - g * (kPiece + 2);
    const int64_t at = (piece0 + g) * kPiece + j - 1;
    const bool in = at >= 0 && at < n;
    ids[g][j] = in ? a.key[at] : -1;
    if (in && j >= 1 && j <= kPiece) where[g][j - 1] = a.order[at];
  }
  __syncthreads();
  const int64_t piece = piece0 + group;
  const int pack = blockIdx.x % column_blocks * lanes + (threadIdx.x & (lanes - 1));
  if (piece * kPiece >= n || pack * VEC >= a.hidden) return;
  const int len = (int)min((int64_t)kPiece, n - piece * kPiece);
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
  constexpr int kAhead = 8;
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
template <typename T>
__global__ __launch_bounds__(kJoinLanes* kJoinAdders) void embed_join_kernel(EmbedArgs a) {
  __shared__ float sums[kJoinAdders][kJoinLanes];
  const int64_t n = a.first[(int64_t)a.per << a.shift];
  const int64_t piece = blockIdx.x, end = (piece + 1) * kPiece;
  if (end >= n) return;
  const int id = a.key[end];
  if (id != a.key[end - 1]) return;  // no run crosses the piece's end
  const int64_t slot = slot_of(a, (unsigned)id);
  if (a.first[slot] < piece * kPiece) return;  // it began in an earlier piece
  const int64_t last = (a.first[slot + 1] - 1) / kPiece;
  const int lane = threadIdx.x % kJoinLanes, adder = threadIdx.x / kJoinLanes;
  const int c = blockIdx.y * kJoinLanes + lane;
  float s = 0.f;
  if (c < a.hidden) {
    if (adder == 0) s = a.part[(piece * 2 + 1) * a.hidden + c];
#pragma unroll 8
    for (int64_t p = piece + 1 + adder; p <= last; p += kJoinAdders) s += a.part[p * 2 * a.hidden + c];
  }
  sums[adder][lane] = s;
  __syncthreads();
  if (adder || c >= a.hidden) return;
  for (int i = 1; i < kJoinAdders; ++i) s += sums[i][lane];
  const float sum[1] = {s};
  RowAt<T, 1, false> at(c, a.hidden);
  write_row(a, at, id, sum);
}

// A table [vocab, hidden] with `tokens` of it: how the ids are dealt and where the order lies.
struct Layout {
  int shift, per;
  int64_t pieces;
  size_t order, key, first, part, bytes;  // offsets into the workspace
};
Layout layout(int64_t tokens, int64_t vocab, int64_t hidden) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Layout l = {};
  l.shift = 8;
  while (vocab > ((int64_t)kBucketIds << l.shift)) ++l.shift;
  l.per = (int)((vocab + ((int64_t)1 << l.shift) - 1) >> l.shift);
  l.pieces = (tokens + kPiece - 1) / kPiece;
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
  a.shift = l.shift, a.per = l.per;
  hipStream_t st = as_stream(stream);
  return EG_DISPATCH_FLOAT(dtype, name, [&]() -> int {
    return by_width<scalar_t>(a.hidden, {dout, (const void*)dweight}, [&](auto vec, auto rag) -> int {
      using T = scalar_t;
      constexpr int V = decltype(vec)::value, W = 16 / (int)sizeof(T);
      const int64_t packs = (hidden + V - 1) / V;
      const int lanes = lanes_for(packs, kSumThreads), groups = kSumThreads / lanes;
      const int64_t columns = (packs + lanes - 1) / lanes;
      const int64_t sums = (l.pieces + groups - 1) / groups * columns;
      const bool flat = aligned16(dweight);
      const int64_t zpacks = (vocab * hidden + (flat ? W : 1) - 1) / (flat ? W : 1);
      const int64_t zeros = accumulate ? 0 : (zpacks + kSumThreads * kZeroPacks - 1) /
                                                 (kSumThreads * kZeroPacks);
      if (check_grid(name, (int64_t)1 << l.shift, kSortThreads) ||
          check_grid(name, sums + zeros, kSumThreads) ||
          check_grid(name, l.pieces, kJoinLanes * kJoinAdders))
        return 1;
      const int64_t joins = (hidden + kJoinLanes - 1) / kJoinLanes;
      EG_LAUNCH((embed_sort_kernel), dim3(1u << l.shift), dim3(kSortThreads),
                (size_t)kSortWaves * l.per * sizeof(unsigned), st, a);
      if (sums + zeros) {
        if (flat)
          EG_LAUNCH((embed_sum_kernel<T, V, decltype(rag)::value, W>),
                    dim3((unsigned)(sums + zeros)), dim3(kSumThreads), 0, st, a, lanes,
                    (int)columns, sums);
        else
          EG_LAUNCH((embed_sum_kernel<T, V, decltype(rag)::value, 1>),
                    dim3((unsigned)(sums + zeros)), dim3(kSumThreads), 0, st, a, lanes,
                    (int)columns, sums);
      }
      if (l.pieces > 1)
        EG_LAUNCH((embed_join_kernel<T>), dim3((unsigned)(l.pieces - 1), (unsigned)joins),
                  dim3(kJoinLanes * kJoinAdders), 0, st, a);
      return check_launch(name);
    });
  });
}
