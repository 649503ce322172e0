// Entry points of the attention over chains (attention.h).
#include "attention.h"

namespace {

bool attn_ok(const AttnArgs& a, int tile_rows, int splits, int dtype, bool backward) {
  for (int64_t row : {a.q_row, a.k_row, a.v_row})
    if (row < 0 || row >= (int64_t(1) << 22)) return false;
  return a.beads >= 0 && a.beads < (int64_t(1) << 31) - 256 && a.heads >= 1 && a.heads <= 1024 &&
         a.dim >= 1 && a.dim <= 128 && a.reach >= 1 && a.reach <= 1024 && a.buckets >= 1 &&
         (int64_t)a.n_tiles * a.heads < (int64_t(1) << 31) &&
         (tile_rows == 32 || tile_rows == 64 || tile_rows == 128) &&
         (splits == 1 || (splits == 2 && tile_rows >= 64) ||
          (splits == 4 && tile_rows == 64 && a.dim <= 64 && !backward)) &&
         dtype >= MLCG_DTYPE_F32 && dtype <= MLCG_DTYPE_BF16;
}

}  // namespace

extern "C" int64_t mlcg_chain_attention_workspace_floats(int64_t beads, int heads,
                                                         int64_t n_tiles, int buckets) {
  if (beads < 0 || heads < 1 || n_tiles < 0 || buckets < 1) return -1;
  return heads * (2 * beads + n_tiles * (kAttnWaves + buckets));
}

extern "C" int mlcg_chain_attention(const void* q, const int64_t* q_strides, const void* k,
                                    const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, int64_t beads, int heads,
                                    int kv_heads, int dim, int dtype, const void* table,
                                    int buckets, const int32_t* bucket_of, int reach, float scale,
                                    const int32_t* tiles, int64_t n_tiles, int tile_rows,
                                    int splits, const uint8_t* keep, const int32_t* positions,
                                    void* out, void* rest, float* lse, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && kv_heads >= 1 && heads >= 1 &&
               heads % kv_heads == 0 && n_tiles >= 0 && n_tiles < (int64_t(1) << 31));
  AttnArgs a{q, k, v, table, out, nullptr, q_strides[0], q_strides[1], k_strides[0],
             k_strides[1], v_strides[0], v_strides[1], beads, bucket_of,
             reinterpret_cast<const int4*>(tiles), keep, positions, lse, (int)n_tiles, heads,
             heads / kv_heads, dim, reach, buckets, scale, rest};
  MLCG_REQUIRE(attn_ok(a, tile_rows, splits, dtype, false));
  if (beads == 0 || n_tiles == 0) return MLCG_OK;
  MLCG_REQUIRE(q && k && v && table && bucket_of && tiles && out);
  const int shape = 10 * (tile_rows / 32) + splits;
  hipStream_t s = mlcg_stream(stream);
  if (dtype == MLCG_DTYPE_F32) return attn_forward<float>(a, shape, out, s);
  if (dtype == MLCG_DTYPE_F16) return attn_forward<_Float16>(a, shape, out, s);
  return attn_forward<__bf16>(a, shape, out, s);
}

extern "C" int mlcg_chain_attention_backward(
    const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
    const void* v, const int64_t* v_strides, int64_t beads, int heads, int kv_heads, int dim,
    int dtype, const void* table, int buckets, const int32_t* bucket_of,
    const int32_t* bucket_order, const int32_t* bucket_first, int reach, float scale,
    const int32_t* tiles, int64_t n_tiles, int tile_rows, int splits, const uint8_t* keep,
    const int32_t* positions, const void* out, const void* rest, const float* lse,
    const void* grad_out, void* grad_q, void* grad_k, void* grad_v, void* grad_table, float* workspace,
    int64_t workspace_floats, void* stream) {
  MLCG_REQUIRE(q_strides && k_strides && v_strides && kv_heads >= 1 && heads >= 1 &&
               heads % kv_heads == 0 && n_tiles >= 1 && n_tiles < (int64_t(1) << 31));
  AttnArgs a{q, k, v, table, out, grad_out, q_strides[0], q_strides[1], k_strides[0],
             k_strides[1], v_strides[0], v_strides[1], beads, bucket_of,
             reinterpret_cast<const int4*>(tiles), keep, positions, const_cast<float*>(lse),
             (int)n_tiles, heads, heads / kv_heads, dim, reach, buckets, scale,
             const_cast<void*>(rest)};
  MLCG_REQUIRE(attn_ok(a, tile_rows, splits, dtype, true) && beads >= 1);
  MLCG_REQUIRE(q && k && v && table && bucket_of && bucket_order && bucket_first && tiles && out &&
               lse && grad_out && grad_q && grad_k && grad_v && grad_table && workspace);
  MLCG_REQUIRE(workspace_floats >=
               mlcg_chain_attention_workspace_floats(beads, heads, n_tiles, buckets));
  const int shape = 10 * (tile_rows / 32) + splits;
  hipStream_t s = mlcg_stream(stream);
  const AttnGrads o{grad_q, grad_k, grad_v, grad_table, workspace, bucket_order, bucket_first};
  if (dtype == MLCG_DTYPE_F32) return attn_backward<float>(a, shape, o, s);
  if (dtype == MLCG_DTYPE_F16) return attn_backward<_Float16>(a, shape, o, s);
  return attn_backward<__bf16>(a, shape, o, s);
}
