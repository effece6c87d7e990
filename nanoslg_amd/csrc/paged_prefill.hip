// Entry points of the paged prefill over 16-bit and fp32 pools (the kernels: paged_prefill.h).
#include "paged_prefill.h"

using namespace nslg;

extern "C" size_t nslg_paged_prefill_workspace_size(int32_t batch, int32_t num_qo_heads,
                                                    int32_t head_dim, int64_t total_q,
                                                    int32_t max_q) {
  (void)max_q;
  if (batch <= 0 || num_qo_heads <= 0 || head_dim <= 0 || total_q <= 0) return 256;
  // an upper bound of the runs of keys a call of this shape takes (whatever its KV heads)
  const int64_t rows = total_q * num_qo_heads;
  const int rows_wg = rows_per_wg(head_dim);
  const int64_t s = kCUs / ((rows + rows_wg - 1) / rows_wg);
  if (s < 2) return 256;  // one run: all state is kept on chip
  return split_bytes(rows, (int)(s > kMaxSplits ? kMaxSplits : s), head_dim);
}

extern "C" int nslg_paged_prefill(const void* q, int64_t q_stride, const int32_t* qo_indptr,
                                  int64_t total_q, int32_t max_q, const void* k_pool,
                                  const void* v_pool, int64_t num_pages, int32_t page_size,
                                  const int32_t* kv_indptr, const int32_t* kv_indices,
                                  const int32_t* kv_last_page_len, int32_t batch,
                                  int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                  float sm_scale, int32_t dtype, void* out, int64_t out_stride,
                                  void* workspace, size_t workspace_bytes, nslg_stream_t stream) {
  return prefill_impl<Raw16>(q, q_stride, qo_indptr, nullptr, 0, total_q, max_q, k_pool, v_pool, num_pages, page_size,
                      kv_indptr, kv_indices, kv_last_page_len, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale,
                      dtype, out, out_stride, workspace, workspace_bytes, stream);
}

extern "C" int nslg_paged_prefill_grid(const void* q, int64_t q_stride, const int32_t* qo_indptr,
                                       const int32_t* q_rows, int32_t grid_width, int64_t total_q,
                                       int32_t max_q, const void* k_pool, const void* v_pool,
                                       int64_t num_pages, int32_t page_size, const int32_t* kv_indptr,
                                       const int32_t* kv_indices, const int32_t* kv_last_page_len,
                                       int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                       int32_t head_dim, float sm_scale, int32_t dtype, void* out,
                                       int64_t out_stride, void* workspace, size_t workspace_bytes,
                                       nslg_stream_t stream) {
  if (batch > 0 && !q_rows) return fail(NSLG_EINVAL, "paged_prefill_grid: null q_rows");
  return prefill_impl<Raw16>(q, q_stride, qo_indptr, q_rows, grid_width, total_q, max_q, k_pool, v_pool, num_pages,
                      page_size, kv_indptr, kv_indices, kv_last_page_len, batch, num_qo_heads, num_kv_heads,
                      head_dim, sm_scale, dtype, out, out_stride, workspace, workspace_bytes, stream);
}

extern "C" int nslg_paged_prefill_append(const void* q, int64_t q_stride, const int32_t* qo_indptr,
                                         const int32_t* q_rows, int32_t grid_width, int64_t total_q,
                                         int32_t max_q, const void* k_new, int64_t k_new_stride,
                                         const void* v_new, int64_t v_new_stride, void* k_pool, void* v_pool,
                                         int64_t num_pages, int32_t page_size, const int32_t* kv_indptr,
                                         const int32_t* kv_indices, const int32_t* kv_last_page_len,
                                         int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                         int32_t head_dim, float sm_scale, int32_t dtype, void* out,
                                         int64_t out_stride, void* workspace, size_t workspace_bytes,
                                         nslg_stream_t stream) {
  if (batch > 0 && total_q > 0 && (!k_new || !v_new)) return fail(NSLG_EINVAL, "paged_prefill_append: null k_new/v_new");
  return prefill_impl<Raw16>(q, q_stride, qo_indptr, q_rows, grid_width, total_q, max_q, k_pool, v_pool, num_pages,
                      page_size, kv_indptr, kv_indices, kv_last_page_len, batch, num_qo_heads, num_kv_heads,
                      head_dim, sm_scale, dtype, out, out_stride, workspace, workspace_bytes, stream, k_new, k_new_stride, v_new,
                      v_new_stride);
}
