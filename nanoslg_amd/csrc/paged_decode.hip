// Entry points of the paged decode over 16-bit and fp32 pools (the kernels: paged_decode.h).
#include "paged_decode.h"

using namespace nslg;

namespace {

// Workspace bytes of an ungrouped call: for this call, or for it and every call of fewer pages.
size_t plain_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, int64_t total_pages,
                   int32_t page_size, int32_t dtype, bool smaller_too) {
  if (!shape_ok(batch, num_qo_heads, num_kv_heads, head_dim, total_pages, page_size)) return 0;
  if (dtype == NSLG_F32)  // partials of the key splits of the fp32 path (their number grows with the pages)
    return attention_f32_workspace(batch, num_qo_heads, head_dim,
                                   attention_f32_decode_splits(batch, num_kv_heads,
                                                               total_pages * (int64_t)page_size));
  const DecodeShape sh = shape_of<false>(dtype, head_dim, batch, num_kv_heads, total_pages * page_size, page_size);
  return workspace_bytes_for(smaller_too ? sh.most_chunks : sh.max_chunks, batch, num_qo_heads, head_dim, 1, 0);
}

}  // namespace

extern "C" size_t nslg_paged_decode_workspace_size(int32_t batch, int32_t num_qo_heads,
                                                   int32_t num_kv_heads, int32_t head_dim,
                                                   int64_t total_pages, int32_t page_size,
                                                   int32_t dtype) {
  return plain_bytes(batch, num_qo_heads, num_kv_heads, head_dim, total_pages, page_size, dtype, true);
}

extern "C" size_t nslg_paged_decode_grouped_workspace_size(int32_t batch, int32_t num_qo_heads,
                                                           int32_t num_kv_heads, int32_t head_dim,
                                                           int64_t total_pages, int32_t page_size,
                                                           int32_t dtype, int32_t num_groups) {
  if (!shape_ok(batch, num_qo_heads, num_kv_heads, head_dim, total_pages, page_size)) return 0;
  if (num_groups < 1 || num_groups > kMaxGroups) return 0;
  if (dtype == NSLG_F32) return 0;  // grouped decode runs on the 16-bit MFMA path only
  const int group = num_qo_heads / num_kv_heads;
  if (group > kGroupCols) return 0;
  const DecodeShape sh =
      shape_of<true>(dtype, head_dim, batch + num_groups, num_kv_heads, total_pages * page_size, page_size);
  return workspace_bytes_for(sh.most_chunks, batch, num_qo_heads, head_dim, kGroupCols / group, num_groups);
}

extern "C" int nslg_paged_decode(const void* q, int64_t q_stride, const void* k_pool,
                                 const void* v_pool, int64_t num_pages, int32_t page_size,
                                 const int32_t* kv_indptr, const int32_t* kv_indices,
                                 const int32_t* kv_last_page_len, int64_t total_pages,
                                 int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                 int32_t head_dim, float sm_scale, int32_t dtype, void* out,
                                 int64_t out_stride, void* workspace, size_t workspace_bytes,
                                 int64_t layout, nslg_stream_t stream) {
  GroupArgs<false> ga;
  return decode_impl<false>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices,
                            kv_last_page_len, total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale,
                            dtype, out, out_stride, ga, 0, 1, workspace, workspace_bytes, stream, NewRows{},
                            layout);
}

// ---- decode without a caller workspace ---------------------------------------------
// The split-K partials and chunk ranges of nslg_paged_decode_noalloc live in this
// fixed device array instead of a caller's workspace. Every GPU the library runs on
// holds its own copy at its own address until the process ends. Host code never
// passes the array's name to a kernel: its device address is looked up once per
// device (hipGetSymbolAddress, with that device current) and used from then on.
static __device__ __align__(256) unsigned char scratch[NSLG_NOALLOC_SCRATCH_BYTES];

namespace {

std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};

// Device address of `scratch` on the current device (looked up on the first call
// made with that device current).
int scratch_of_current_device(void** out) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    (void)hipGetLastError();
    return fail(NSLG_EINVAL, "paged_decode_noalloc: no current device (or device %d >= %d)", dev, kMaxDevices);
  }
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* ptr = nullptr;
    const hipError_t e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !ptr) {
      (void)hipGetLastError();
      return fail(NSLG_ELAUNCH, "paged_decode_noalloc: hipGetSymbolAddress(scratch) failed on device %d: %s", dev,
                  hipGetErrorString(e));
    }
    g_scratch_ptr[dev] = ptr;
  }
  *out = g_scratch_ptr[dev];
  return NSLG_OK;
}

}  // namespace

extern "C" int nslg_paged_decode_noalloc(const void* q, int64_t q_stride, const void* k_pool,
                                         const void* v_pool, int64_t num_pages, int32_t page_size,
                                         const int32_t* kv_indptr, const int32_t* kv_indices,
                                         const int32_t* kv_last_page_len, int64_t total_pages,
                                         int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                         int32_t head_dim, float sm_scale, int32_t dtype, void* out,
                                         int64_t out_stride, nslg_stream_t stream) {
  // Same scratch layout as nslg_paged_decode's workspace, of what this call needs; nothing in it has
  // to start at zero (every chunk range and partial is written before it is read).
  const size_t need = plain_bytes(batch, num_qo_heads, num_kv_heads, head_dim, total_pages, page_size, dtype, false);
  if (need > (size_t)NSLG_NOALLOC_SCRATCH_BYTES)
    return fail(NSLG_EWORKSPACE,
                "paged_decode_noalloc: this call needs %zu bytes of scratch, more than the %zu-byte static "
                "scratch; call nslg_paged_decode with a workspace",
                need, (size_t)NSLG_NOALLOC_SCRATCH_BYTES);
  void* ws = nullptr;
  const int rc = scratch_of_current_device(&ws);
  if (rc) return rc;
  GroupArgs<false> ga;
  return decode_impl<false>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices,
                            kv_last_page_len, total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale,
                            dtype, out, out_stride, ga, 0, 1, ws, (size_t)NSLG_NOALLOC_SCRATCH_BYTES, stream);
}

extern "C" int nslg_paged_decode_append(const void* q, int64_t q_stride, const void* k_new,
                                        int64_t k_new_stride, const void* v_new, int64_t v_new_stride,
                                        void* k_pool, void* v_pool, int64_t num_pages, int32_t page_size,
                                        const int32_t* kv_indptr, const int32_t* kv_indices,
                                        const int32_t* kv_last_page_len, int64_t total_pages,
                                        int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                        int32_t head_dim, float sm_scale, int32_t dtype, void* out,
                                        int64_t out_stride, void* workspace, size_t workspace_bytes,
                                        int64_t layout, nslg_stream_t stream) {
  if (batch > 0 && (!k_new || !v_new)) return fail(NSLG_EINVAL, "paged_decode_append: null k_new or v_new");
  NewRows nr;
  nr.k = k_new;
  nr.v = v_new;
  nr.k_stride = k_new_stride;
  nr.v_stride = v_new_stride;
  GroupArgs<false> ga;
  return decode_impl<false>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices,
                            kv_last_page_len, total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale,
                            dtype, out, out_stride, ga, 0, 1, workspace, workspace_bytes, stream, nr, layout);
}

extern "C" int nslg_paged_decode_rope_append(
    const void* q, int64_t q_stride, const void* k_new, int64_t k_new_stride, const void* v_new,
    int64_t v_new_stride, const int32_t* positions, const float* cos_table, const float* sin_table,
    int64_t table_stride, int64_t table_rows, void* k_pool, void* v_pool, int64_t num_pages, int32_t page_size,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len, int64_t total_pages,
    int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, float sm_scale, int32_t dtype,
    void* out, int64_t out_stride, void* workspace, size_t workspace_bytes, int64_t layout, nslg_stream_t stream) {
  if (batch > 0 && (!k_new || !v_new || !cos_table))
    return fail(NSLG_EINVAL, "paged_decode_rope_append: null k_new, v_new or tables");
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
  GroupArgs<false> ga;
  return decode_impl<false>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices,
                            kv_last_page_len, total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale,
                            dtype, out, out_stride, ga, 0, 1, workspace, workspace_bytes, stream, nr, layout);
}

extern "C" int nslg_paged_decode_grouped(const void* q, int64_t q_stride, const void* k_pool,
                                         const void* v_pool, int64_t num_pages, int32_t page_size,
                                         const int32_t* kv_indptr, const int32_t* kv_indices,
                                         const int32_t* kv_last_page_len, int64_t total_pages,
                                         int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                         int32_t head_dim, float sm_scale, int32_t dtype,
                                         const int32_t* seq_group_slot, int32_t num_groups,
                                         const int32_t* group_prefix_pages, const int32_t* group_members,
                                         void* out, int64_t out_stride, void* workspace,
                                         size_t workspace_bytes, int64_t layout, nslg_stream_t stream) {
  return grouped_impl<Raw16>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices, kv_last_page_len,
                      total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale, dtype, seq_group_slot,
                      num_groups, group_prefix_pages, group_members, out, out_stride, workspace, workspace_bytes,
                      stream, NewRows{}, layout);
}

extern "C" int nslg_paged_decode_grouped_append(
    const void* q, int64_t q_stride, const void* k_new, int64_t k_new_stride, const void* v_new,
    int64_t v_new_stride, void* k_pool, void* v_pool, int64_t num_pages, int32_t page_size,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len, int64_t total_pages,
    int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, float sm_scale, int32_t dtype,
    const int32_t* seq_group_slot, int32_t num_groups, const int32_t* group_prefix_pages,
    const int32_t* group_members, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
    int64_t layout, nslg_stream_t stream) {
  if (batch > 0 && (!k_new || !v_new)) return fail(NSLG_EINVAL, "paged_decode_grouped_append: null k_new or v_new");
  NewRows nr;
  nr.k = k_new;
  nr.v = v_new;
  nr.k_stride = k_new_stride;
  nr.v_stride = v_new_stride;
  return grouped_impl<Raw16>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices, kv_last_page_len,
                      total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale, dtype, seq_group_slot,
                      num_groups, group_prefix_pages, group_members, out, out_stride, workspace, workspace_bytes,
                      stream, nr, layout);
}

extern "C" int nslg_paged_decode_grouped_rope_append(
    const void* q, int64_t q_stride, const void* k_new, int64_t k_new_stride, const void* v_new,
    int64_t v_new_stride, const int32_t* positions, const float* cos_table, const float* sin_table,
    int64_t table_stride, int64_t table_rows, void* k_pool, void* v_pool, int64_t num_pages, int32_t page_size,
    const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len, int64_t total_pages,
    int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim, float sm_scale, int32_t dtype,
    const int32_t* seq_group_slot, int32_t num_groups, const int32_t* group_prefix_pages,
    const int32_t* group_members, void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
    int64_t layout, nslg_stream_t stream) {
  if (batch > 0 && (!k_new || !v_new || !cos_table))
    return fail(NSLG_EINVAL, "paged_decode_grouped_rope_append: null k_new, v_new or tables");
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
  return grouped_impl<Raw16>(q, q_stride, k_pool, v_pool, num_pages, page_size, kv_indptr, kv_indices, kv_last_page_len,
                      total_pages, batch, num_qo_heads, num_kv_heads, head_dim, sm_scale, dtype, seq_group_slot,
                      num_groups, group_prefix_pages, group_members, out, out_stride, workspace, workspace_bytes,
                      stream, nr, layout);
}
