// Writing an 8-bit KV cache and reading it back.
#include "q8_common.h"

namespace nslg {
namespace {

// ---- append: a forward's rows into their blocks -----------------------------------
// One wave per (block, KV head, K or V) that the forward writes: the block's rows, at most 16 of D elements, are
// read once into registers, their maximum sets the scale, and the codes are written (write_block). Blocks are the
// unit so that no two waves share a scale; a workgroup holds one block's K and V of two heads, and V's waves tell
// K's through LDS what is not finite. 2 bytes read and 1 written per element; bound by the launch and the
// chain of loads (lengths, rows and page id, old scale): 8 x 512 rows of 8 x 128, 25 MB, 9.4 us (with K and V in one
// wave 10.1).
struct Append8Params {
  const uint16_t* k_new;
  const uint16_t* v_new;
  int64_t k_stride;  // elements between rows
  int64_t v_stride;
  int64_t num_rows;  // rows of k_new / v_new
  int64_t total_q;
  const int32_t* qo_indptr;
  const int32_t* q_rows;  // null: ragged rows; else the grid row of each ragged row
  char* k_pool;
  char* v_pool;
  float* k_scale;
  float* v_scale;
  int64_t num_pages;
  int32_t page_size;
  int32_t blocks_per_page;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  int32_t batch;
  int32_t num_kv_heads;
};

struct BlockTask {
  int q0;     // first ragged row of the sequence
  int start;  // position of its first new token
  int len;    // its tokens, new ones included
  int seq;
  int blk;    // the task's block: page * blocks_per_page + block, of the sequence's pages
};

// The g-th block that the forward writes, sequences in batch order. Every wave finds its own,
// the lanes holding the sequences.
__device__ inline bool locate_block(const Append8Params& p, int g, BlockTask& out) {
  const int lane = threadIdx.x & 63;
  const int ps = p.page_size, nb = p.blocks_per_page;
  for (int s0 = 0; s0 < p.batch; s0 += 64) {
    const int s = s0 + lane;
    int q0 = 0, len = 0, start = 0, first = 0, nt = 0;
    if (s < p.batch) {
      q0 = p.qo_indptr[s];
      const int n = p.qo_indptr[s + 1] - q0;
      const int np = p.indptr[s + 1] - p.indptr[s];
      int lpl = p.last_len[s];
      lpl = lpl < 1 ? 1 : (lpl > ps ? ps : lpl);
      len = np > 0 ? (np - 1) * ps + lpl : 0;
      start = max(len - max(n, 0), 0);
      if (n > 0 && len > 0) {
        first = start / ps * nb + start % ps / kBlockToks;
        nt = (len - 1) / ps * nb + (len - 1) % ps / kBlockToks - first + 1;
      }
    }
    int incl = nt;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(incl, off, 64);
      if (lane >= off) incl += y;
    }
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (g >= total) {
      g -= total;
      continue;
    }
    const int src = __ffsll((long long)__ballot(g >= incl - nt && g < incl)) - 1;
    out.seq = s0 + src;
    out.q0 = __builtin_amdgcn_readlane(q0, src);
    out.start = __builtin_amdgcn_readlane(start, src);
    out.len = __builtin_amdgcn_readlane(len, src);
    out.blk = __builtin_amdgcn_readlane(first, src) + g - __builtin_amdgcn_readlane(incl - nt, src);
    return true;
  }
  return false;
}

template <typename T, typename F, int D>
__global__ void __launch_bounds__(256) append_q8_kernel(Append8Params p) {
  __shared__ uint32_t bad[2][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = blockIdx.y * 4 + wave;  // (head, K or V)
  const bool is_v = wave & 1;
  const int h = c >> 1;
  BlockTask t;
  if (!locate_block(p, blockIdx.x, t)) return;  // (this and the next two returns: the whole workgroup)
  const int page = t.blk / p.blocks_per_page, i = t.blk - page * p.blocks_per_page;
  const int pid = p.indices[p.indptr[t.seq] + page];
  const int base = page * p.page_size + kBlockToks * i;  // position of the block's row 0
  const int end = min(t.len, page * p.page_size + min(p.page_size, kBlockToks * (i + 1)));
  const int a = max(t.start - base, 0), cnt = end - base - a;
  // its new rows, contiguous in k_new / v_new
  int64_t r0 = t.q0;
  if (r0 < 0 || r0 >= p.total_q) return;
  if (p.q_rows) r0 = p.q_rows[r0];
  r0 += base + a - t.start;
  if (cnt < 1 || r0 < 0 || r0 + cnt > p.num_rows) return;
  const int64_t stride = is_v ? p.v_stride : p.k_stride;
  BlockRows<D> rows;  // (loaded before the page id is waited for)
  if (h < p.num_kv_heads) {
    const uint16_t* src = (is_v ? p.v_new : p.k_new) + r0 * stride + (int64_t)h * D;
    load_block_rows<D>(rows, a, cnt, [&](int r, int e) { return *reinterpret_cast<const u16x8*>(src + (r - a) * stride + e); });
    if (is_v) bad[wave >> 1][threadIdx.x & 63] = not_finite<T, D>(rows);
  }
  __syncthreads();
  if (h >= p.num_kv_heads || pid < 0 || (int64_t)pid >= p.num_pages) return;
  const int64_t row_bytes = (int64_t)p.num_kv_heads * D;
  const int64_t at = ((int64_t)pid * p.page_size + kBlockToks * i) * row_bytes + (int64_t)h * D;
  const int64_t blk = ((int64_t)pid * p.blocks_per_page + i) * p.num_kv_heads + h;
  if (is_v) {
    write_block<T, F, D, false>(rows, p.v_pool + at, row_bytes, p.v_scale + blk, a, cnt);
    return;
  }
  spoil<D>(rows, bad[wave >> 1][threadIdx.x & 63]);
  write_block<T, F, D, true>(rows, p.k_pool + at, row_bytes, p.k_scale + blk, a, cnt);
}

// ---- gather: the cached tokens as contiguous rows ----------------------------------
// A workgroup takes kGatherToks tokens of a sequence (blockIdx.y: sequence, blockIdx.z: K or V), a thread
// 8 codes of a row at a time: 8 bytes and a scale in, 16 (or 32) bytes out, both whole lines over a wave,
// kGatherUnroll of them in flight (2 or 8: the same). HBM-bound: 16 conversations of 2k to 16k tokens, int8 to fp16,
// 232 MB of codes in and 727 MB out (past the lengths too), 174 us.
constexpr int kGatherToks = 16;
constexpr int kGatherUnroll = 4;
constexpr int64_t kGatherStreamBytes = (int64_t)128 << 20;  // larger outputs go out past the caches: 188 -> 174 us
struct Gather8Params {
  const char* k_pool;
  const char* v_pool;
  const float* k_scale;
  const float* v_scale;
  int64_t num_pages;
  int32_t page_size;
  int32_t blocks_per_page;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  int32_t max_len;
  int32_t num_kv_heads;
  void* k_out;
  void* v_out;
};

struct OutF32 {
  typedef float Elem;
  __device__ static inline float of(float x) { return x; }
};
template <typename T>
struct Out16 {
  typedef unsigned short Elem;
  __device__ static inline unsigned short of(float x) { return T::from_f32(x); }
};

template <typename O, typename F, int D, bool kStream>
__global__ void __launch_bounds__(256) gather_q8_kernel(Gather8Params p) {
  constexpr int kChunks = D / 8;  // of one head's row
  typedef typename O::Elem E;
  typedef E E8 __attribute__((ext_vector_type(8)));
  const int per_row = p.num_kv_heads * kChunks;
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int p0 = p.indptr[b], np = p.indptr[b + 1] - p0;
  int lpl = p.last_len[b];
  lpl = lpl < 1 ? 1 : (lpl > p.page_size ? p.page_size : lpl);
  const int64_t len = np > 0 ? (int64_t)(np - 1) * p.page_size + lpl : 0;
  const int t0 = blockIdx.x * kGatherToks;
  const int items = min(kGatherToks, p.max_len - t0) * per_row;
  E8* dst = reinterpret_cast<E8*>(is_v ? p.v_out : p.k_out) + ((int64_t)b * p.max_len + t0) * per_row;
  const float* scales = is_v ? p.v_scale : p.k_scale;
  const char* pool = is_v ? p.v_pool : p.k_pool;
  for (int j0 = threadIdx.x; j0 < items; j0 += 256 * kGatherUnroll) {
    u32x2 w[kGatherUnroll];
    float s[kGatherUnroll];
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u) {
      const int j = j0 + 256 * u;
      w[u] = u32x2{0u, 0u};
      s[u] = 0.f;
      const int r = j / per_row, t = t0 + r, c = j - r * per_row;
      if (j < items && t < len) {
        const int page = t / p.page_size, slot = t - page * p.page_size;
        int pid = p.indices[p0 + page];
        if (pid < 0 || (int64_t)pid >= p.num_pages) pid = 0;
        s[u] = scales[scale_index(pid, slot, p.blocks_per_page, p.num_kv_heads, c / kChunks)];
        w[u] = *reinterpret_cast<const u32x2*>(pool + (((int64_t)pid * p.page_size + slot) * per_row + c) * 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u) {
      const int j = j0 + 256 * u;
      if (j >= items) break;
      E8 out;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float f[4];
        F::decode4(w[u][k], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * k + e] = O::of(f[e] * s[u]);
      }
      if constexpr (kStream)
        stream_store(dst + j, out);
      else
        dst[j] = out;
    }
  }
}

template <typename T, typename F>
void launch_append(const Append8Params& p, int head_dim, dim3 grid, hipStream_t s) {
  switch (head_dim) {
    case 64: append_q8_kernel<T, F, 64><<<grid, 256, 0, s>>>(p); break;
    case 128: append_q8_kernel<T, F, 128><<<grid, 256, 0, s>>>(p); break;
    default: append_q8_kernel<T, F, 256><<<grid, 256, 0, s>>>(p); break;
  }
}

template <typename O, typename F, int D>
void launch_gather_d(const Gather8Params& p, int64_t out_bytes, dim3 grid, hipStream_t s) {
  if (out_bytes > kGatherStreamBytes)
    gather_q8_kernel<O, F, D, true><<<grid, 256, 0, s>>>(p);
  else
    gather_q8_kernel<O, F, D, false><<<grid, 256, 0, s>>>(p);
}

template <typename O, typename F>
void launch_gather(const Gather8Params& p, int head_dim, int64_t out_bytes, dim3 grid, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_gather_d<O, F, 64>(p, out_bytes, grid, s);
    case 128: return launch_gather_d<O, F, 128>(p, out_bytes, grid, s);
    default: return launch_gather_d<O, F, 256>(p, out_bytes, grid, s);
  }
}

// The checks that every call on an 8-bit cache layer shares.
int check_cache(const char* what, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                int64_t num_pages, int32_t page_size, const int32_t* indptr, const int32_t* indices,
                const int32_t* last_len, int32_t batch, int32_t num_kv_heads, int32_t head_dim, int32_t code) {
  if (num_pages <= 0 || page_size <= 0 || batch < 0 || num_kv_heads <= 0 || head_dim <= 0)
    return fail(NSLG_EINVAL, "%s: bad sizes", what);
  if (code != NSLG_E4M3 && code != NSLG_INT8) return fail(NSLG_EINVAL, "%s: bad code type %d", what, code);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(NSLG_EUNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, head_dim);
  if (num_kv_heads > 65535) return fail(NSLG_EUNSUPPORTED, "%s: %d KV heads", what, num_kv_heads);
  if (num_pages * (int64_t)page_size >= ((int64_t)1 << 31))
    return fail(NSLG_EUNSUPPORTED, "%s: pool has >= 2^31 token slots", what);
  if (batch == 0) return NSLG_OK;
  if (!k_pool || !v_pool || !k_scale || !v_scale || !indptr || !indices || !last_len)
    return fail(NSLG_EINVAL, "%s: null pointer", what);
  if (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15 || ((uintptr_t)k_scale | (uintptr_t)v_scale) & 3)
    return fail(NSLG_EINVAL, "%s: pools must be 16-byte aligned, scales 4-byte", what);
  return NSLG_OK;
}

}  // namespace
}  // namespace nslg

using namespace nslg;

extern "C" int nslg_q8_append_kv(const void* k_new, int64_t k_new_stride, const void* v_new, int64_t v_new_stride,
                                 const int32_t* qo_indptr, const int32_t* q_rows, int32_t grid_width, int64_t total_q,
                                 void* k_pool, void* v_pool, float* k_scale, float* v_scale, int64_t num_pages,
                                 int32_t page_size, const int32_t* kv_indptr, const int32_t* kv_indices,
                                 const int32_t* kv_last_page_len, int32_t batch, int32_t num_kv_heads, int32_t head_dim,
                                 int32_t dtype, int32_t code, nslg_stream_t stream) {
  const int rc = check_cache("q8_append_kv", k_pool, v_pool, k_scale, v_scale, num_pages, page_size, kv_indptr, kv_indices,
                             kv_last_page_len, batch, num_kv_heads, head_dim, code);
  if (rc) return rc;
  if (dtype != NSLG_F16 && dtype != NSLG_BF16)
    return fail(NSLG_EUNSUPPORTED, "q8_append_kv: rows of dtype %d (f16 or bf16)", dtype);
  if (total_q < 0 || total_q > 0x7fffffff) return fail(NSLG_EINVAL, "q8_append_kv: %lld tokens", (long long)total_q);
  if (q_rows && (grid_width < 1 || (int64_t)batch * grid_width > 0x7fffffff || total_q > (int64_t)batch * grid_width))
    return fail(NSLG_EINVAL, "q8_append_kv: grid of %d x %d rows for %lld tokens", batch, grid_width, (long long)total_q);
  if (batch == 0 || total_q == 0) return NSLG_OK;
  if (!k_new || !v_new || !qo_indptr) return fail(NSLG_EINVAL, "q8_append_kv: null pointer");
  const int64_t row = (int64_t)num_kv_heads * head_dim, rows = q_rows ? (int64_t)batch * grid_width : total_q;
  if (rows > 1 && (k_new_stride < row || v_new_stride < row))
    return fail(NSLG_EINVAL, "q8_append_kv: rows overlap (strides %lld, %lld < Hkv*D = %lld)", (long long)k_new_stride,
                (long long)v_new_stride, (long long)row);
  if (((uintptr_t)k_new | (uintptr_t)v_new) & 15 || (k_new_stride * 2) % 16 || (v_new_stride * 2) % 16)
    return fail(NSLG_EINVAL, "q8_append_kv: rows must be 16-byte aligned");
  Append8Params p;
  p.k_new = (const uint16_t*)k_new;
  p.v_new = (const uint16_t*)v_new;
  p.k_stride = k_new_stride;
  p.v_stride = v_new_stride;
  p.num_rows = rows;
  p.total_q = total_q;
  p.qo_indptr = qo_indptr;
  p.q_rows = q_rows;
  p.k_pool = (char*)k_pool;
  p.v_pool = (char*)v_pool;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.blocks_per_page = (page_size + kBlockToks - 1) / kBlockToks;
  p.indptr = kv_indptr;
  p.indices = kv_indices;
  p.last_len = kv_last_page_len;
  p.batch = batch;
  p.num_kv_heads = num_kv_heads;
  // blocks written, at most: a sequence's n tokens touch (n - 1) / 16 + 2 blocks where 16 divides
  // the page, else (n - 1) / page_size + 2 pages
  int64_t blocks = page_size % kBlockToks == 0 ? total_q / kBlockToks + 2 * (int64_t)batch
                                               : (total_q / page_size + 2 * (int64_t)batch) * p.blocks_per_page;
  blocks = blocks < total_q ? blocks : total_q;
  const dim3 grid((unsigned)blocks, (unsigned)((num_kv_heads + 1) / 2));
  hipStream_t s = as_stream(stream);
  if (dtype == NSLG_F16)
    code == NSLG_E4M3 ? launch_append<F16, E4M3>(p, head_dim, grid, s) : launch_append<F16, Int8>(p, head_dim, grid, s);
  else
    code == NSLG_E4M3 ? launch_append<BF16, E4M3>(p, head_dim, grid, s) : launch_append<BF16, Int8>(p, head_dim, grid, s);
  return check_launch("q8_append_kv");
}

extern "C" int nslg_q8_gather_kv(const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                                 int64_t num_pages, int32_t page_size, const int32_t* kv_indptr,
                                 const int32_t* kv_indices, const int32_t* kv_last_page_len, int32_t batch, int32_t max_len,
                                 int32_t num_kv_heads, int32_t head_dim, int32_t code, int32_t dtype, void* k_out,
                                 void* v_out, nslg_stream_t stream) {
  const int rc = check_cache("q8_gather_kv", k_pool, v_pool, k_scale, v_scale, num_pages, page_size, kv_indptr, kv_indices,
                             kv_last_page_len, batch, num_kv_heads, head_dim, code);
  if (rc) return rc;
  if (!elem_bytes(dtype)) return fail(NSLG_EINVAL, "q8_gather_kv: bad dtype %d", dtype);
  if (max_len < 0 || batch > 65535) return fail(NSLG_EINVAL, "q8_gather_kv: %d x %d rows", batch, max_len);
  if (batch == 0 || max_len == 0) return NSLG_OK;
  if (!k_out || !v_out) return fail(NSLG_EINVAL, "q8_gather_kv: null pointer");
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) return fail(NSLG_EINVAL, "q8_gather_kv: outputs must be 16-byte aligned");
  const int64_t work = ((int64_t)max_len + kGatherToks - 1) / kGatherToks;
  Gather8Params p;
  p.k_pool = (const char*)k_pool;
  p.v_pool = (const char*)v_pool;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.blocks_per_page = (page_size + kBlockToks - 1) / kBlockToks;
  p.indptr = kv_indptr;
  p.indices = kv_indices;
  p.last_len = kv_last_page_len;
  p.max_len = max_len;
  p.num_kv_heads = num_kv_heads;
  p.k_out = k_out;
  p.v_out = v_out;
  const int64_t out_bytes = 2 * (int64_t)batch * max_len * num_kv_heads * head_dim * elem_bytes(dtype);
  const dim3 grid((unsigned)work, (unsigned)batch, 2);
  hipStream_t s = as_stream(stream);
  if (dtype == NSLG_F16)
    code == NSLG_E4M3 ? launch_gather<Out16<F16>, E4M3>(p, head_dim, out_bytes, grid, s)
                      : launch_gather<Out16<F16>, Int8>(p, head_dim, out_bytes, grid, s);
  else if (dtype == NSLG_BF16)
    code == NSLG_E4M3 ? launch_gather<Out16<BF16>, E4M3>(p, head_dim, out_bytes, grid, s)
                      : launch_gather<Out16<BF16>, Int8>(p, head_dim, out_bytes, grid, s);
  else
    code == NSLG_E4M3 ? launch_gather<OutF32, E4M3>(p, head_dim, out_bytes, grid, s) : launch_gather<OutF32, Int8>(p, head_dim, out_bytes, grid, s);
  return check_launch("q8_gather_kv");
}
