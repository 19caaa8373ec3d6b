// What the packed attention kernels are given: eg_packed_attn_fwd / eg_packed_attn_bwd's
// arguments, validated.
#pragma once

#include "packed_seqs.hpp"

namespace eg {

struct PackedAttn {
  PackedSeqs seqs;
  // q [tokens, heads, D], k, v [tokens, kv_heads, D] with D contiguous, the others' strides
  // in elements; o, dout, dq and dk, dv contiguous; lse, delta fp32 [heads, tokens].
  const void *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;
  void* o;
  float* lse;
  const void* dout;
  void *dq, *dk, *dv;
  float *delta, *part;  // workspace
  void* plan[2];        // plan_bytes each: for query tiles, for key tiles
  int heads, kv_heads, head_dim;
  float scale;
};

// Where there are so many sequences that the kernels search a plan (packed_attention.hip), orders
// them for tiles of rows[i] rows into table[i] (plan_bytes(n) bytes each), all in one launch; out[i]
// is seqs with that plan, or seqs as it is. Returns 0 or a launch error.
inline size_t plan_bytes(int64_t n) {
  return n > kSearchSeqs ? ((size_t)(2 * n + 1) * 4 + 255) / 256 * 256 : 0;
}
int packed_plan(const PackedSeqs& seqs, int tables, const int* rows, void* const* table,
                PackedSeqs* out, hipStream_t st);

// packed_attn_generic.hip: any type, even head size up to 128 and strides.
size_t packed_generic_part_bytes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads,
                                 int64_t head_dim);
int packed_generic_fwd(const PackedAttn& a, int dtype, hipStream_t st);
int packed_generic_bwd(const PackedAttn& a, int dtype, hipStream_t st);

}  // namespace eg
