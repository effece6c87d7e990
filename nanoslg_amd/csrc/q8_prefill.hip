// Entry point of the paged prefill over 8-bit pools (the kernels: paged_prefill.h).
#include "paged_prefill.h"

using namespace nslg;

extern "C" int nslg_q8_paged_prefill(const void* q, int64_t q_stride, const int32_t* qo_indptr, const int32_t* q_rows,
                                     int32_t grid_width, int64_t total_q, int32_t max_q, const void* k_pool,
                                     const void* v_pool, const float* k_scale, const float* v_scale, int64_t num_pages,
                                     int32_t page_size, const int32_t* kv_indptr, const int32_t* kv_indices,
                                     const int32_t* kv_last_page_len, int32_t batch, int32_t num_qo_heads,
                                     int32_t num_kv_heads, int32_t head_dim, float sm_scale, int32_t dtype, int32_t code,
                                     void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
                                     nslg_stream_t stream) {
  if (code != NSLG_E4M3 && code != NSLG_INT8) return fail(NSLG_EINVAL, "q8_paged_prefill: bad code type %d", code);
  PrefillScales sc;
  sc.k = k_scale;
  sc.v = v_scale;
  auto call = code == NSLG_E4M3 ? &prefill_impl<E4M3> : &prefill_impl<Int8>;
  return call(q, q_stride, qo_indptr, q_rows, grid_width, total_q, max_q, k_pool, v_pool, num_pages, page_size, kv_indptr,
              kv_indices, kv_last_page_len, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale, dtype, out, out_stride,
              workspace, workspace_bytes, stream, nullptr, 0, nullptr, 0, sc);
}
