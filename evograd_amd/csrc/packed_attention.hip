// Causal grouped-query attention over packed sequences: the entry points.
//
//   o_i = sum over j <= i of i's sequence of p_ij v_j,  p_ij = exp(scale q_i k_j - lse_i)
//   delta_i = do_i o_i,  dS_ij = p_ij (do_i v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i p_ij do_i
// with query head h reading kv head h / (heads / kv_heads), dk and dv summed over the group.
#include "packed_attention.hpp"

using namespace eg;

namespace {

constexpr int64_t kMaxTokens = (int64_t)1 << 28, kMaxSeqs = (int64_t)1 << 24;

size_t delta_bytes(int64_t tokens, int64_t heads) {
  return ((size_t)(tokens * heads) * 4 + 255) / 256 * 256;
}

int check_packed(const char* name, const PackedAttn& a, int64_t tokens, int64_t seqs,
                 int64_t heads, int64_t kv_heads, int64_t D, int dtype) {
  if (tokens < 0 || seqs < 0 || heads < 0) { set_error("%s: negative size", name); return 1; }
  if (heads > 0 && (kv_heads <= 0 || heads % kv_heads != 0)) {
    set_error("%s: heads (%lld) must be a positive multiple of kv_heads (%lld)", name,
              (long long)heads, (long long)kv_heads);
    return 1;
  }
  if (D < 2 || D > 128 || D % 2) {
    set_error("%s: head_dim must be even and at most 128, got %lld", name, (long long)D);
    return 1;
  }
  if (dtype != EG_BF16 && dtype != EG_F16 && dtype != EG_F32) {
    set_error("%s: dtype must be fp32, bf16 or fp16", name);
    return 1;
  }
  for (int64_t s : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head})
    if (s < 0 || s > ((int64_t)1 << 24)) {
      set_error("%s: strides must be at least 0 and at most 16777216 elements", name);
      return 1;
    }
  // tiles of 16 rows times heads and walk pieces index one grid
  if (tokens > kMaxTokens || seqs > kMaxSeqs || heads > 4096 ||
      packed_tiles(tokens, seqs, 16) * heads * 8 > 0x7fffffffLL) {
    set_error("%s: size out of range (tokens <= 268435456, sequences <= 16777216, heads <= 4096, "
              "(tokens / 16 + sequences) * heads < 2^28)", name);
    return 1;
  }
  return 0;
}

PackedAttn describe(const void* q, const void* k, const void* v, const int* cu, int64_t tokens,
                    int64_t seqs, int64_t heads, int64_t kv_heads, int64_t D,
                    const int64_t* strides, float scale) {
  PackedAttn a = {};
  a.seqs = {cu, (int)seqs, (int)tokens};
  a.q = q, a.k = k, a.v = v;
  a.q_token = strides[0], a.q_head = strides[1];
  a.k_token = strides[2], a.k_head = strides[3];
  a.v_token = strides[4], a.v_head = strides[5];
  a.heads = (int)heads, a.kv_heads = (int)kv_heads, a.head_dim = (int)D;
  a.scale = scale;
  return a;
}

}  // namespace

extern "C" size_t eg_packed_attn_workspace_bytes(int64_t tokens, int64_t seqs, int64_t heads,
                                                 int64_t kv_heads, int64_t head_dim, int dtype) {
  if (tokens <= 0 || seqs < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
  return delta_bytes(tokens, heads) + packed_generic_part_bytes(tokens, kv_heads, head_dim);
}

extern "C" int eg_packed_attn_fwd(const void* q, const void* k, const void* v, const int* cu_seqlens,
                                  void* o, float* lse, int64_t tokens, int64_t seqs, int64_t heads,
                                  int64_t kv_heads, int64_t head_dim, const int64_t* strides,
                                  float scale, int dtype, void* stream) {
  static const char* name = "eg_packed_attn_fwd";
  clear_error();
  if (!strides) { set_error("%s: null strides", name); return 1; }
  PackedAttn a = describe(q, k, v, cu_seqlens, tokens, seqs, heads, kv_heads, head_dim, strides,
                          scale);
  if (check_packed(name, a, tokens, seqs, heads, kv_heads, head_dim, dtype)) return 1;
  if (tokens == 0 || heads == 0) return 0;
  if (!q || !k || !v || !cu_seqlens || !o || !lse) { set_error("%s: null pointer", name); return 1; }
  a.o = o, a.lse = lse;
  return packed_generic_fwd(a, dtype, as_stream(stream));
}

extern "C" int eg_packed_attn_bwd(const void* dout, const void* q, const void* k, const void* v,
                                  const int* cu_seqlens, const void* o, const float* lse, void* dq,
                                  void* dk, void* dv, void* workspace, int64_t tokens, int64_t seqs,
                                  int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  const int64_t* strides, float scale, int dtype, void* stream) {
  static const char* name = "eg_packed_attn_bwd";
  clear_error();
  if (!strides) { set_error("%s: null strides", name); return 1; }
  PackedAttn a = describe(q, k, v, cu_seqlens, tokens, seqs, heads, kv_heads, head_dim, strides,
                          scale);
  if (check_packed(name, a, tokens, seqs, heads, kv_heads, head_dim, dtype)) return 1;
  if (tokens == 0 || heads == 0) return 0;
  if (!dout || !q || !k || !v || !cu_seqlens || !o || !lse || !dq || !dk || !dv || !workspace) {
    set_error("%s: null pointer", name);
    return 1;
  }
  a.o = const_cast<void*>(o), a.lse = const_cast<float*>(lse);
  a.dout = dout, a.dq = dq, a.dk = dk, a.dv = dv;
  a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + delta_bytes(tokens, heads));
  return packed_generic_bwd(a, dtype, as_stream(stream));
}
