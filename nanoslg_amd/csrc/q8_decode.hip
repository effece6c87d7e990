// Entry points of the paged decode over 8-bit pools (the kernels: paged_decode.h).
#include "paged_decode.h"

using namespace nslg;

namespace {

bool code_ok(int32_t code) { return code == NSLG_E4M3 || code == NSLG_INT8; }

template <bool kGrouped>
DecodeShape shape8(int32_t code, int32_t dtype, int32_t head_dim, int32_t units, int32_t num_kv_heads, int64_t tokens,
                   int page_size) {
  return code == NSLG_E4M3 ? shape_of<kGrouped, E4M3>(dtype, head_dim, units, num_kv_heads, tokens, page_size)
                           : shape_of<kGrouped, Int8>(dtype, head_dim, units, num_kv_heads, tokens, page_size);
}

}  // namespace

extern "C" size_t nslg_q8_paged_decode_workspace_size(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                                      int32_t head_dim, int64_t total_pages, int32_t page_size,
                                                      int32_t dtype, int32_t code, int32_t num_groups) {
  if (!shape_ok(batch, num_qo_heads, num_kv_heads, head_dim, total_pages, page_size) || !code_ok(code)) return 0;
  if ((dtype != NSLG_F16 && dtype != NSLG_BF16) || num_groups < 0 || num_groups > kMaxGroups) return 0;
  const int group = num_qo_heads / num_kv_heads;
  if (group > kGroupCols) return 0;
  const int64_t tokens = total_pages * page_size;
  if (num_groups == 0)
    return workspace_bytes_for(shape8<false>(code, dtype, head_dim, batch, num_kv_heads, tokens, page_size).most_chunks,
                               batch, num_qo_heads, head_dim, 1, 0);
  return workspace_bytes_for(
      shape8<true>(code, dtype, head_dim, batch + num_groups, num_kv_heads, tokens, page_size).most_chunks, batch,
      num_qo_heads, head_dim, kGroupCols / group, num_groups);
}

extern "C" int nslg_q8_paged_decode(
    const void* q, int64_t q_stride, const void* k_new, int64_t k_new_stride, const void* v_new, int64_t v_new_stride,
    const int32_t* positions, const float* cos_table, const float* sin_table, int64_t table_stride, int64_t table_rows,
    void* k_pool, void* v_pool, float* k_scale, float* v_scale, int64_t num_pages, int32_t page_size,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len, int64_t total_pages,
    int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, float sm_scale, int32_t dtype,
    int32_t code, const int32_t* seq_group_slot, int32_t num_groups, const int32_t* group_prefix_pages,
    const int32_t* group_members, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
    int64_t layout, nslg_stream_t stream) {
  if (!code_ok(code)) return fail(NSLG_EINVAL, "q8_paged_decode: bad code type %d", code);
  if (!(sm_scale > 0.f) || !(sm_scale < INFINITY))
    return fail(NSLG_EINVAL, "q8_paged_decode: sm_scale must be positive and finite");
  NewRows nr;
  nr.k = k_new;
  nr.v = v_new;
  nr.k_stride = k_new_stride;
  nr.v_stride = v_new_stride;
  nr.pos = positions;
  nr.cos = cos_table;
  nr.sin = sin_table;
  nr.table_stride = table_stride;
  nr.table_rows = table_rows;
  PoolScales sc;
  sc.k = k_scale;
  sc.v = v_scale;
  if (num_groups != 0) {
    auto call = code == NSLG_E4M3 ? &grouped_impl<E4M3> : &grouped_impl<Int8>;
    return call(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices, kv_last_page_len, total_pages,
                batch, num_qo_heads, num_kv_heads, head_dim, sm_scale, dtype, seq_group_slot, num_groups,
                group_prefix_pages, group_members, out, out_stride, workspace, workspace_bytes, stream, nr, layout, sc);
  }
  GroupArgs<false> ga;
  auto call = code == NSLG_E4M3 ? &decode_impl<false, E4M3> : &decode_impl<false, Int8>;
  return call(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices, kv_last_page_len, total_pages,
              batch, num_qo_heads, num_kv_heads, head_dim, sm_scale, dtype, out, out_stride, ga, 0, 1, workspace,
              workspace_bytes, stream, nr, layout, sc);
}
