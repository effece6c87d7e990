// Attention of trees of drafted tokens over a paged cache, for gfx950 (CDNA4).
//
// Sequence b's last n_b tokens are the nodes of its tree; node t sees every token before
// the tree and, of the nodes, those of its mask (its ancestors and itself). Query rows are
// packed GQA-style, row = node * G + g, so one K/V load serves all G query heads of a KV head.
//
// Work. The sequences' tokens are cut into chunks of one length, a multiple of the key tile, that every wave
// finds from the lengths: the smallest one whose chunks fit the call's budget. A workgroup (4 waves)
// takes one (chunk, KV head, tile of query rows): 64 rows, 16 a wave, or 128, 32 a wave. Key tiles go through
// LDS, double buffered, the next tile's loads in flight during the present one's products. Per 32 keys:
//   S^T[key x row] = K Q^T      (MFMA; lane (r, gq) then holds keys 16 t + 4 gq + j of row r)
//   online softmax in fp32, the running maximum raised lazily
//   O^T[d x row] += V^T P^T     (MFMA; 16-bit V^T operands by transposing LDS reads)
// The rows of a sequence of several chunks are left as fp32 partials for tree_merge_kernel.
//
// A key that a row does not see counts nothing, whatever it holds: its score is replaced, and since a
// probability of 0 would not keep a value that is not finite out of a matrix product, such values of the nodes are
// staged as 0 and added row by row to those that see them.
#include "nslg_common.h"

#include <math.h>

namespace nslg {
namespace {

constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
constexpr int kTreeCUs = 256;
constexpr int kTreeMaxNodes = 1024;
constexpr float kTreeSlack = 8.0f;  // how far (log2) scores may rise above the running maximum that P is taken at

struct TreeParams {
  const char* q;
  int64_t q_stride;  // bytes between rows, as out_stride, k_new_stride and v_new_stride
  const int32_t* qo_indptr;
  const int32_t* q_rows;  // null, or the grid row of every ragged row
  int32_t grid_width;
  int64_t total_q;
  const uint32_t* mask;  // [total_q, mask_words]
  int32_t mask_words;
  const char* k_pool;
  const char* v_pool;
  int64_t num_pages;
  int32_t page_size;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
  int32_t batch;
  int32_t num_qo_heads;
  int32_t num_kv_heads;
  int32_t group;
  float scale_log2;
  char* out;
  int64_t out_stride;
  const char* k_new;  // null: the nodes' rows are in the pool
  const char* v_new;
  int64_t k_new_stride;
  int64_t v_new_stride;
  int32_t max_nodes;   // a tree's nodes, at most (more are cut off)
  int32_t max_chunks;  // chunks of the batch, at most; 0: one a sequence, no partials
  int32_t num_work;    // workgroups that attend; the others write the new rows
  int64_t part_rows;   // rows of the partials
  uint64_t* ws_tag;    // the workspace's first word: a decode call's record in the same memory is void
  int4* meta;          // per sequence: first row of its partials, chunks, rows
  float2* part_ml;     // [part_rows]: running maximum (log2 units), sum
  float* part_o;       // [part_rows, D]
};

// Element types: fp32 takes its products on the fp32 matrix instructions.
struct F32 {
  static constexpr int kDtype = NSLG_F32;
};

template <typename T, int D>
struct TreeTile {
  static constexpr bool kF32 = T::kDtype == NSLG_F32;
  static constexpr int kBytes = kF32 ? 4 : 2;
  static constexpr int kSub = kF32 && D == 256 ? 1 : 2;        // 16-key pieces of a block
  static constexpr int kBlocks = kF32 || D == 256 ? 1 : 2;     // blocks of a tile
  static constexpr int kKeys = 16 * kSub * kBlocks;            // keys of a tile: two workgroups fit a CU
  static constexpr int kPitch = D * kBytes + (kF32 ? 16 : 32); // bytes of a tile's row in LDS (no bank conflicts)
};

struct SeqOf {
  int nodes, len;
};

// Sequence s's nodes and tokens (nodes among them).
__device__ inline SeqOf tree_seq(const TreeParams& p, int s) {
  SeqOf x = {0, 0};
  if (s < p.batch) {
    const int np = p.indptr[s + 1] - p.indptr[s];
    int lpl = p.last_len[s];
    lpl = lpl < 1 ? 1 : (lpl > p.page_size ? p.page_size : lpl);
    x.len = np > 0 ? (np - 1) * p.page_size + lpl : 0;
    x.nodes = min(max(p.qo_indptr[s + 1] - p.qo_indptr[s], 0), p.max_nodes);
    if (x.nodes == 0) x.len = 0;
  }
  return x;
}

__device__ inline int64_t tree_row(const TreeParams& p, int t) {
  if (!p.q_rows) return t;
  const int64_t r = p.q_rows[t];
  return r >= 0 && r < (int64_t)p.batch * p.grid_width ? r : -1;
}

// Keys per chunk: ceil(all keys / (budget - batch)) rounded up to whole tiles; a sequence of L keys then
// has at most L / chunk + 1, all of them at most `budget`.
__device__ inline int tree_chunk(const TreeParams& p, int64_t keys, int tile) {
  const int64_t room = p.max_chunks - p.batch;
  if (room <= 0) return 0x7fffffff / tile * tile;
  const int64_t c = (keys + room - 1) / room;
  const int64_t up = (c + tile - 1) / tile * tile;
  return (int)(up < tile ? tile : up);
}

__device__ inline int64_t wave_sum_i64(int64_t x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off, 64);
  return x;
}
__device__ inline int wave_scan_i32(int x) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

// The new rows of K and V into their page slots, one wave a row.
__device__ inline void write_row(char* dst, const char* src, int vecs) {
  for (int i = threadIdx.x & 63; i < vecs; i += 64)
    stream_store(reinterpret_cast<u32x4*>(dst) + i, reinterpret_cast<const u32x4*>(src)[i]);
}

__device__ inline void tree_write_new(const TreeParams& p, int wg, int row_bytes) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)wg * kTreeWaves + (threadIdx.x >> 6);
  if (t >= p.total_q) return;
  // the row's sequence: the last one that starts at or before it
  int b = -1;
  for (int s0 = 0; s0 < p.batch; s0 += 64) {
    const unsigned long long m = __ballot(s0 + lane < p.batch && p.qo_indptr[min(s0 + lane, p.batch)] <= t);
    b += __popcll(m);
    if (m != ~0ull) break;
  }
  if (b < 0 || t >= p.qo_indptr[b + 1]) return;
  const int node = (int)(t - p.qo_indptr[b]);
  const SeqOf sq = tree_seq(p, b);
  const int pos = sq.len - sq.nodes + node;
  const int64_t src = tree_row(p, (int)t);
  if (node >= sq.nodes || pos < 0 || src < 0) return;
  const int pid = p.indices[p.indptr[b] + pos / p.page_size];
  if (pid < 0 || (int64_t)pid >= p.num_pages) return;
  const int64_t at = ((int64_t)pid * p.page_size + pos % p.page_size) * row_bytes;
  write_row(const_cast<char*>(p.k_pool) + at, p.k_new + src * p.k_new_stride, row_bytes / 16);
  write_row(const_cast<char*>(p.v_pool) + at, p.v_new + src * p.v_new_stride, row_bytes / 16);
}

// 16 bytes of V with the elements that are not finite set to 0 (and bad set).
template <typename T>
__device__ inline u32x4 drop_not_finite(u32x4 x, bool& bad) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T::kDtype == NSLG_F32) {
      if ((x[i] & 0x7f800000u) == 0x7f800000u) x[i] = 0, bad = true;
    } else {
      constexpr uint32_t kExp = T::kDtype == NSLG_F16 ? 0x7c00u : 0x7f80u;
      if ((x[i] & kExp) == kExp) x[i] &= 0xffff0000u, bad = true;
      if ((x[i] & (kExp << 16)) == kExp << 16) x[i] &= 0xffffu, bad = true;
    }
  }
  return x;
}

template <typename T, int D, int kCB>
__global__ void __launch_bounds__(kTreeThreads, 2) tree_attention_kernel(TreeParams p) {
  using Tile = TreeTile<T, D>;
  constexpr bool kF32 = Tile::kF32;
  constexpr int kBytes = Tile::kBytes;
  constexpr int kSub = Tile::kSub, kBlocks = Tile::kBlocks, kKeys = Tile::kKeys, kBlockKeys = 16 * kSub;
  constexpr int kPitch = Tile::kPitch;
  constexpr int kRows = 16 * kCB * kTreeWaves;
  constexpr int NT = D / 16;
  constexpr int kSteps = kF32 ? D / 16 : D / 32;            // 16-byte operands of a key or row
  constexpr int kVecs = D * kBytes / 16;                    // 16-byte pieces of a row
  constexpr int kPer = kKeys * kVecs / kTreeThreads;        // pieces of K (and of V) a thread and tile
  constexpr int kStep = kTreeThreads / kVecs;               // keys between a thread's pieces
  constexpr bool kSplitP = T::kDtype == NSLG_BF16;

  __shared__ __attribute__((aligned(16))) char k_lds[2][kKeys * kPitch];
  __shared__ __attribute__((aligned(16))) char v_lds[2][kKeys * kPitch];
  // keys of a tile with a value of V that is not finite (three tiles' words in turn: one is cleared a barrier
  // before the tile that writes it)
  __shared__ uint32_t bad_lds[3][kBlocks];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, gq = lane >> 4;
  const int G = p.group, ps = p.page_size;
  const int row_bytes = p.num_kv_heads * D * kBytes;
  const int w = (int)blockIdx.x;
  if (p.q_rows)
    zero_pad_rows(p.qo_indptr, p.q_rows, p.grid_width, p.batch, p.out, p.out_stride, p.num_qo_heads * D * kBytes,
                  w * kTreeWaves + wave, (int)gridDim.x * kTreeWaves);
  if (w >= p.num_work) {
    tree_write_new(p, w - p.num_work, row_bytes);
    return;
  }
  if (w == 0 && tid == 0 && p.ws_tag) *p.ws_tag = 0;
  if (tid < 3 * kBlocks) bad_lds[tid / kBlocks][tid % kBlocks] = 0;

  // ---- the workgroup's item: KV head (in turn: neighbours of a head share an XCD's L2), then sequence, chunk, row tile
  const int h = w % p.num_kv_heads;
  int k = w / p.num_kv_heads;
  int64_t keys = 0;
  for (int s0 = 0; s0 < p.batch; s0 += 64) keys += tree_seq(p, s0 + lane).len;
  const int chunk = tree_chunk(p, wave_sum_i64(keys), kKeys);
  int b = -1, n_nodes = 0, L = 0, n_chunks = 0, n_tiles = 0;
  int64_t part0 = 0;  // the sequence's first row of the partials (of one KV head)
  for (int s0 = 0; s0 < p.batch; s0 += 64) {
    const SeqOf sq = tree_seq(p, s0 + lane);
    const int rows = sq.nodes * G;
    const int tiles = (rows + kRows - 1) / kRows;
    const int chunks = sq.len > 0 ? (sq.len - 1) / chunk + 1 : 0;
    const int items = tiles * chunks;
    const int incl = wave_scan_i32(items);
    const int parts = chunks > 1 ? chunks * rows : 0;
    const int pincl = wave_scan_i32(parts);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (k >= total) {
      k -= total;
      part0 += __builtin_amdgcn_readlane(pincl, 63);
      continue;
    }
    const int src = __ffsll((long long)__ballot(k < incl)) - 1;
    k -= __builtin_amdgcn_readlane(incl - items, src);
    part0 += __builtin_amdgcn_readlane(pincl - parts, src);
    b = s0 + src;
    n_nodes = __builtin_amdgcn_readlane(sq.nodes, src);
    L = __builtin_amdgcn_readlane(sq.len, src);
    n_chunks = __builtin_amdgcn_readlane(chunks, src);
    n_tiles = __builtin_amdgcn_readlane(tiles, src);
    break;
  }
  if (b < 0) return;  // uniform over the workgroup
  const int c_no = k / n_tiles, tile = k - c_no * n_tiles;  // (the row tiles of a chunk next to each other)
  const int nrows = n_nodes * G;
  const int start = max(L - n_nodes, 0);
  const int q0 = p.qo_indptr[b];
  const int kv_begin = c_no * chunk;
  const int kv_end = min(L - kv_begin, chunk) + kv_begin;
  if (p.meta && h == 0 && k == 0 && tid == 0) p.meta[b] = int4{(int)part0, n_chunks, nrows, 0};
  const int32_t* idx = p.indices + p.indptr[b];

  // ---- the wave's rows
  const int wave_row0 = tile * kRows + 16 * kCB * wave;
  const bool wave_on = wave_row0 < nrows;  // (a wave without rows only helps to stage the tiles)
  u32x4 qb[kCB][kSteps];
  const uint32_t* mrow[kCB];
  bool row_ok[kCB];
#pragma unroll
  for (int cb = 0; cb < kCB; ++cb) {
    const int row = wave_row0 + 16 * cb + r;
    const int t = row / G;
    row_ok[cb] = row < nrows && q0 + t < p.total_q;
    const int64_t at = row_ok[cb] ? tree_row(p, q0 + t) : -1;
    mrow[cb] = p.mask + (int64_t)(row_ok[cb] ? q0 + t : 0) * p.mask_words;
    const char* src = p.q + (at >= 0 ? at : 0) * p.q_stride + ((int64_t)(h * G + row % G) * D) * kBytes + 16 * gq;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qb[cb][s] = at >= 0 ? *reinterpret_cast<const u32x4*>(src + 64 * s) : u32x4{0, 0, 0, 0};
  }
  float thr[kCB], neg_m[kCB];  // the raw score above which the maximum is raised; -maximum (log2 units; 0: none yet)
  f32x4 lsum[kCB], o[kCB][NT];
#pragma unroll
  for (int cb = 0; cb < kCB; ++cb) {
    thr[cb] = -INFINITY;
    neg_m[cb] = 0.f;
    lsum[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NT; ++n) o[cb][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float inv_scale = 1.f / p.scale_log2;

  // ---- tiles: thread tid moves piece tid % kVecs of keys tid / kVecs + kStep i
  const int f_c = 16 * (tid % kVecs), f_key = tid / kVecs;
  const int head_off = h * D * kBytes;
  const bool pow2 = (ps & (ps - 1)) == 0;
  const int ps_shift = __builtin_ctz((unsigned)ps);
  u32x4 kreg[kPer], vreg[kPer];
  int pid[kPer];
  auto page_of = [&](int key) { return pow2 ? key >> ps_shift : key / ps; };
  // where key's K and V rows of this head are: a page slot, or the forward's new row
  auto pool_at = [&](int key, int page) {
    page = page < 0 || (int64_t)page >= p.num_pages ? 0 : page;
    return ((int64_t)page * ps + (key - page_of(key) * ps)) * row_bytes + head_off;
  };
  int64_t new_row0 = q0;  // row of k_new / v_new of node 0 (a tree's rows are contiguous)
  if (p.k_new && p.q_rows) {
    const int64_t at = tree_row(p, q0);
    const int64_t rows = (int64_t)p.batch * p.grid_width;
    new_row0 = at < 0 || at + n_nodes > rows ? 0 : at;
  }
  const bool fresh = p.k_new != nullptr;
  const int64_t new_last = (p.q_rows ? (int64_t)p.batch * p.grid_width : p.total_q) - 1;
  auto new_at = [&](int key) { return min(new_row0 + (key - start), new_last); };
  auto fetch_pages = [&](int key0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) pid[i] = idx[page_of(min(key0 + f_key + kStep * i, kv_end - 1))];
  };
  auto fetch = [&](int key0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int key = min(key0 + f_key + kStep * i, kv_end - 1);
      const char *ks, *vs;
      if (fresh && key >= start) {
        const int64_t at = new_at(key);
        ks = p.k_new + at * p.k_new_stride + head_off;
        vs = p.v_new + at * p.v_new_stride + head_off;
      } else {
        const int64_t at = pool_at(key, pid[i]);
        ks = p.k_pool + at;
        vs = p.v_pool + at;
      }
      kreg[i] = *reinterpret_cast<const u32x4*>(ks + f_c);
      vreg[i] = *reinterpret_cast<const u32x4*>(vs + f_c);
    }
  };
  auto stash = [&](int key0, int stage, int rot) {
    if (key0 + kKeys > start) {  // uniform: a tile with nodes, or the end of the keys
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int key = f_key + kStep * i;
        bool bad = false;
        if (key0 + key >= kv_end) {
          vreg[i] = u32x4{0, 0, 0, 0};
        } else if (key0 + key >= start) {
          vreg[i] = drop_not_finite<T>(vreg[i], bad);
        }
        if (bad) atomicOr(&bad_lds[rot][key / kBlockKeys], 1u << (key % kBlockKeys));
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int key = f_key + kStep * i;
      *reinterpret_cast<u32x4*>(&k_lds[stage][key * kPitch + f_c]) = kreg[i];
      *reinterpret_cast<u32x4*>(&v_lds[stage][key * kPitch + f_c]) = vreg[i];
    }
  };
  // the bits of the block's keys that row cb of the lane sees
  auto visible = [&](int kbase, int cb) -> uint32_t {
    const int rel = kbase - start;
    const int words = p.mask_words;
    uint32_t v;
    if (rel >= 0) {
      const int wi = rel >> 5, sh = rel & 31;
      const uint32_t lo = wi < words ? mrow[cb][wi] : 0u;
      const uint32_t hi = wi + 1 < words ? mrow[cb][wi + 1] : 0u;
      v = sh ? (lo >> sh) | (hi << (32 - sh)) : lo;
    } else {
      v = (1u << -rel) - 1u;  // (rel > -kBlockKeys >= -32: not all of the block lies before the tree)
      v |= mrow[cb][0] << -rel;
    }
    const int left = kv_end - kbase;
    if (left < 32) v &= (1u << left) - 1u;
    return row_ok[cb] ? v : 0u;
  };

  auto compute = [&](int key0, int stage, int rot) {
#pragma unroll
    for (int blk = 0; blk < kBlocks; ++blk) {
      const int kbase = key0 + blk * kBlockKeys;
      if (kbase >= kv_end) break;
      // scores
      f32x4 s[kCB][kSub];
#pragma unroll
      for (int t = 0; t < kSub; ++t) {
        u32x4 ka[kSteps];
        const char* krow = &k_lds[stage][(blk * kBlockKeys + 16 * t + r) * kPitch + 16 * gq];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) ka[i] = *reinterpret_cast<const u32x4*>(krow + 64 * i);
#pragma unroll
        for (int cb = 0; cb < kCB; ++cb) {
          if constexpr (kF32) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
              const f32x4 a = __builtin_bit_cast(f32x4, ka[i]), q = __builtin_bit_cast(f32x4, qb[cb][i]);
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[0], q[0], x, 0, 0, 0);
              y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[1], q[1], y, 0, 0, 0);
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[2], q[2], x, 0, 0, 0);
              y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[3], q[3], y, 0, 0, 0);
            }
            s[cb][t] = x + y;
          } else {
            s[cb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
              s[cb][t] = T::mma_k32(__builtin_bit_cast(u16x8, ka[i]), __builtin_bit_cast(u16x8, qb[cb][i]), s[cb][t]);
          }
        }
      }
      // mask, maximum, probabilities (in place of the scores)
      const bool tail = kbase + kBlockKeys > start;  // uniform; the keys past the end are behind the nodes
      uint32_t vis[kCB];
      u16x8 pb[kCB], pb_lo[kCB];
#pragma unroll
      for (int cb = 0; cb < kCB; ++cb) {
        if (tail) {
          vis[cb] = visible(kbase, cb);
#pragma unroll
          for (int j = 0; j < 4 * kSub; ++j)
            if (!(vis[cb] >> (16 * (j >> 2) + 4 * gq + (j & 3)) & 1)) s[cb][j >> 2][j & 3] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4 * kSub; ++j) top = fmaxf(top, s[cb][j >> 2][j & 3]);
        if (__ballot(top > thr[cb])) {
          const float m_run = thr[cb] == -INFINITY ? -INFINITY : -neg_m[cb];
          const float m_new = fmaxf(m_run, rows_max(top * p.scale_log2));
          const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
          lsum[cb] *= alpha;
#pragma unroll
          for (int n = 0; n < NT; ++n) o[cb][n] *= alpha;
          thr[cb] = (m_new + kTreeSlack) * inv_scale;
          neg_m[cb] = m_new == -INFINITY ? 0.f : -m_new;
        }
#pragma unroll
        for (int j = 0; j < 4 * kSub; ++j) {
          const float x = fast_exp2(fmaf(s[cb][j >> 2][j & 3], p.scale_log2, neg_m[cb]));
          s[cb][j >> 2][j & 3] = x;
          if constexpr (kF32) {
            lsum[cb][j & 3] += x;
          } else {
            // half keeps 11 bits of a probability; bfloat16's 8 are too few for the 2e-3 of the 16-bit caches'
            // attention: the rest goes in as a second term
            pb[cb][j] = T::from_f32(x);
            if constexpr (kSplitP) pb_lo[cb][j] = T::from_f32(x - T::to_f32(pb[cb][j]));
          }
        }
      }
      // O^T += V^T P^T
      if constexpr (kF32) {
#pragma unroll
        for (int t = 0; t < kSub; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const char* vrow = &v_lds[stage][(blk * kBlockKeys + 16 * t + 4 * gq + j) * kPitch + 16 * r];
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              const f32x4 v = *reinterpret_cast<const f32x4*>(vrow + 256 * c);
#pragma unroll
              for (int cb = 0; cb < kCB; ++cb)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  o[cb][4 * c + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], s[cb][t][j], o[cb][4 * c + e], 0, 0, 0);
            }
          }
      } else {
        typedef short i16x4_t __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) i16x4_t* lds_i16x4;
        // lane r of a 16-lane group addresses keys 4 gq + r / 4 (then + 16), columns 16 n + 4 (r % 4) .. + 3, and
        // receives keys 4 gq + 0..3 (+ 16) at d = 16 n + r
        const char* vsrc = &v_lds[stage][(blk * kBlockKeys + 4 * gq + (r >> 2)) * kPitch + 8 * (r & 3)];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vsrc + 32 * n));
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(vsrc + 32 * n + 16 * kPitch));
          const u16x8 va = __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int cb = 0; cb < kCB; ++cb) {
            o[cb][n] = T::mma_k32(va, pb[cb], o[cb][n]);
            if constexpr (kSplitP) o[cb][n] = T::mma_k32(va, pb_lo[cb], o[cb][n]);
          }
        }
        // the rows' sums by an all-ones operand: of the probabilities as they were multiplied
        const u16x8 ones = u16x8(T::from_f32(1.f));
#pragma unroll
        for (int cb = 0; cb < kCB; ++cb) {
          lsum[cb] = T::mma_k32(ones, pb[cb], lsum[cb]);
          if constexpr (kSplitP) lsum[cb] = T::mma_k32(ones, pb_lo[cb], lsum[cb]);
        }
      }
      // nodes whose V is not finite: those elements, for the rows that see the node
      uint32_t bad = tail ? __builtin_amdgcn_readfirstlane(bad_lds[rot][blk]) : 0u;
      while (bad) {
        const int kk = __ffs(bad) - 1;
        bad &= bad - 1;
        const int key = kbase + kk;
        const char* vsrc = fresh ? p.v_new + new_at(key) * p.v_new_stride + head_off
                                 : p.v_pool + pool_at(key, idx[page_of(key)]);
#pragma unroll
        for (int cb = 0; cb < kCB; ++cb) {
          float pr = 0.f;
#pragma unroll
          for (int j = 0; j < 4 * kSub; ++j)
            if (16 * (j >> 2) + (j & 3) == (kk & ~12)) pr = s[cb][j >> 2][j & 3];
          pr = __shfl(pr, 16 * ((kk >> 2) & 3) + r, 64);
          if (!(vis[cb] >> kk & 1)) continue;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (kF32) {
                const float v = reinterpret_cast<const float*>(vsrc)[64 * (n >> 2) + 16 * gq + 4 * i + (n & 3)];
                if (!(fabsf(v) < INFINITY)) o[cb][n][i] += pr * v;
              } else {
                const float v = T::to_f32(reinterpret_cast<const uint16_t*>(vsrc)[16 * n + 4 * gq + i]);
                if (!(fabsf(v) < INFINITY)) o[cb][n][i] += pr * v;
              }
            }
        }
      }
    }
  };

  __syncthreads();  // bad_lds is clear
  fetch_pages(kv_begin);
  fetch(kv_begin);
  fetch_pages(kv_begin + kKeys);
  stash(kv_begin, 0, 0);
  int stage = 0, rot = 0;
  for (int key0 = kv_begin; key0 < kv_end; key0 += kKeys) {
    __syncthreads();  // this tile is staged, the one before is read
    const int next = rot == 2 ? 0 : rot + 1, after = next == 2 ? 0 : next + 1;
    if (tid < kBlocks) bad_lds[after][tid] = 0;
    const bool more = key0 + kKeys < kv_end;
    if (more) {
      fetch(key0 + kKeys);
      fetch_pages(key0 + 2 * kKeys);
    }
    if (wave_on) compute(key0, stage, rot);
    if (more) stash(key0 + kKeys, stage ^ 1, next);
    stage ^= 1;
    rot = next;
  }
  if (!wave_on) return;

  // ---- the rows: normalised into `out`, or the chunk's share as a partial
#pragma unroll
  for (int cb = 0; cb < kCB; ++cb) {
    float l;
    if constexpr (kF32)
      l = rows_sum((lsum[cb][0] + lsum[cb][1]) + (lsum[cb][2] + lsum[cb][3]));
    else
      l = lsum[cb][0];
    if (!row_ok[cb]) continue;
    const int row = wave_row0 + 16 * cb + r;
    float f = 1.f;
    char* dst;
    bool wide = true;  // fp32 elements
    if (n_chunks > 1) {
      const int64_t slot = (part0 + (int64_t)c_no * nrows + row) * p.num_kv_heads + h;
      if (slot >= p.part_rows) continue;
      if (gq == 0) p.part_ml[slot] = float2{thr[cb] == -INFINITY ? -INFINITY : -neg_m[cb], l};
      dst = reinterpret_cast<char*>(p.part_o + slot * D);
    } else {
      const int64_t at = tree_row(p, q0 + row / G);
      if (at < 0) continue;
      f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (a sum that is NaN makes the row NaN)
      dst = p.out + at * p.out_stride + (int64_t)(h * G + row % G) * D * kBytes;
      wide = kF32;
    }
    if constexpr (kF32) {
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(dst + 4 * (64 * c + 16 * gq + 4 * j)) =
              f32x4{o[cb][4 * c][j], o[cb][4 * c + 1][j], o[cb][4 * c + 2][j], o[cb][4 * c + 3][j]} * f;
    } else if (wide) {
#pragma unroll
      for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4*>(dst + 4 * (16 * n + 4 * gq)) = o[cb][n];
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        u16x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = T::from_f32(o[cb][n][i] * f);
        *reinterpret_cast<u16x4*>(dst + 2 * (16 * n + 4 * gq)) = x;
      }
    }
  }
}

// Log-sum-exp merge of the chunks of each (node, query head): D / 4 lanes take a chunk's row, kParts such groups the
// row's chunks in turn.
template <typename T, int D, int kParts>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeParams p) {
  constexpr int kLanes = D / 4;
  constexpr int kRows = 256 / (kLanes * kParts);  // rows a workgroup
  __shared__ f32x4 o_lds[kParts > 1 ? kRows * kParts * kLanes : 1];
  __shared__ float2 ml_lds[kParts > 1 ? kRows * kParts : 1];
  const int part = threadIdx.x / kLanes % kParts, wg_row = threadIdx.x / (kLanes * kParts);
  const int col = threadIdx.x % kLanes;
  const int64_t rows = p.total_q * p.num_qo_heads;
  const int64_t row = (int64_t)blockIdx.x * kRows + wg_row;
  const int t = (int)min(row / p.num_qo_heads, p.total_q - 1);
  const int head = (int)(row - (int64_t)t * p.num_qo_heads);
  // the row's sequence: the last one that starts at or before it (binary search)
  int lo = 0, hi = p.batch;  // qo_indptr[lo] <= t < qo_indptr[hi], if in any
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.qo_indptr[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  const int node = t - p.qo_indptr[lo];
  int4 meta = int4{0, 0, 0, 0};
  const bool in = row < rows && node >= 0 && t < p.qo_indptr[lo + 1] && node < p.max_nodes;
  if (in && p.indptr[lo + 1] > p.indptr[lo]) meta = p.meta[lo];  // (a sequence without tokens has no entry)
  const int chunks = meta.y;
  const int h = head / p.group, g = head - h * p.group;
  const int64_t slot0 = ((int64_t)meta.x + node * p.group + g) * p.num_kv_heads + h;
  const int64_t step = (int64_t)meta.z * p.num_kv_heads;
  const bool on = chunks > 1 && slot0 + (chunks - 1) * step < p.part_rows;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (on) {
    for (int c0 = part; c0 < chunks; c0 += 4 * kParts) {
      float2 ml[4];
      f32x4 o[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t slot = slot0 + min(c0 + u * kParts, chunks - 1) * step;
        ml[u] = p.part_ml[slot];
        o[u] = *reinterpret_cast<const f32x4*>(p.part_o + slot * D + 4 * col);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (c0 + u * kParts < chunks) top = fmaxf(top, ml[u].x);
      const float f0 = l == 0.f ? 0.f : fast_exp2(m - top);
      l *= f0;
      acc *= f0;
      m = top;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (c0 + u * kParts >= chunks || ml[u].y == 0.f) continue;  // 0: no key of the chunk seen
        const float f = fast_exp2(ml[u].x - m);
        l = fmaf(f, ml[u].y, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, o[u][e], acc[e]);
      }
    }
  }
  if constexpr (kParts > 1) {
    const int at = wg_row * kParts + part;
    o_lds[at * kLanes + col] = acc;
    if (col == 0) ml_lds[at] = float2{m, l};
    __syncthreads();
    if (part) return;
    float2 ml[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) ml[i] = ml_lds[wg_row * kParts + i], m = fmaxf(m, ml[i].x);
    l = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const float f = ml[i].y == 0.f ? 0.f : fast_exp2(ml[i].x - m);
      if (ml[i].y == 0.f) continue;
      l = fmaf(f, ml[i].y, l);
      const f32x4 x = o_lds[(wg_row * kParts + i) * kLanes + col];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, x[e], acc[e]);
    }
  }
  if (!on) return;
  const int64_t at = tree_row(p, t);
  if (at < 0) return;
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  acc *= inv;
  char* dst = p.out + at * p.out_stride;
  if constexpr (T::kDtype == NSLG_F32) {
    *reinterpret_cast<f32x4*>(dst + 4 * ((int64_t)head * D + 4 * col)) = acc;
  } else {
    u16x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = T::from_f32(acc[e]);
    *reinterpret_cast<u16x4*>(dst + 2 * ((int64_t)head * D + 4 * col)) = x;
  }
}

// ---- host ------------------------------------------------------------------------------

// Rows of a workgroup: two column blocks a wave where the trees' rows fill them (registers: not at D = 256, nor fp32).
inline int tree_row_blocks(int64_t rows, int head_dim, int dtype) {
  return dtype != NSLG_F32 && head_dim != 256 && rows > 64 ? 2 : 1;
}
inline int tree_tile_keys(int head_dim, int dtype) {
  if (dtype == NSLG_F32) return head_dim == 256 ? 16 : 32;
  return head_dim == 256 ? 32 : 64;
}

// Chunks of a call's sequences, at most: enough for about four workgroups a CU.
int64_t tree_chunks(int64_t batch, int64_t total_keys, int64_t rows, int num_kv_heads, int head_dim, int dtype) {
  const int64_t rows_wg = 64 * tree_row_blocks(rows, head_dim, dtype);
  const int64_t tiles = (rows + rows_wg - 1) / rows_wg;
  int64_t n = 4 * kTreeCUs / (tiles * num_kv_heads);
  const int64_t most = total_keys / tree_tile_keys(head_dim, dtype) + 1;  // (a tile each)
  n = n < 1 ? 1 : (n > most ? most : n);
  return n + batch;
}

size_t tree_bytes(int64_t batch, int64_t part_rows, int head_dim) {
  const size_t meta = ((size_t)batch * 16 + 255) / 256 * 256;
  const size_t ml = ((size_t)part_rows * 8 + 255) / 256 * 256;
  return 512 + meta + ml + (size_t)part_rows * head_dim * 4;
}

template <typename T, int D>
int launch_tree(const TreeParams& p, int64_t rows, int64_t wgs, hipStream_t s) {
  if (tree_row_blocks(rows, D, T::kDtype) == 2) {
    if constexpr (T::kDtype != NSLG_F32 && D != 256)
      tree_attention_kernel<T, D, 2><<<dim3((unsigned)wgs), kTreeThreads, 0, s>>>(p);
  } else {
    tree_attention_kernel<T, D, 1><<<dim3((unsigned)wgs), kTreeThreads, 0, s>>>(p);
  }
  const int rc = check_launch("paged_tree_attention");
  if (rc || p.max_chunks == 0) return rc;
  const int64_t out_rows = p.total_q * p.num_qo_heads;
  const int64_t each = p.max_chunks / p.batch;  // chunks of a sequence, on average
  auto grid = [&](int parts) { return dim3((unsigned)((out_rows + 1024 / (D * parts) - 1) / (1024 / (D * parts)))); };
  if (each >= 8 && D <= 128)
    tree_merge_kernel<T, D, D <= 128 ? 8 : 4><<<grid(D <= 128 ? 8 : 4), 256, 0, s>>>(p);
  else if (each >= 8)
    tree_merge_kernel<T, D, 4><<<grid(4), 256, 0, s>>>(p);
  else
    tree_merge_kernel<T, D, 1><<<grid(1), 256, 0, s>>>(p);
  return check_launch("paged_tree_attention merge");
}

template <typename T>
int launch_tree_dim(const TreeParams& p, int head_dim, int64_t rows, int64_t wgs, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_tree<T, 64>(p, rows, wgs, s);
    case 128: return launch_tree<T, 128>(p, rows, wgs, s);
    default: return launch_tree<T, 256>(p, rows, wgs, s);
  }
}

}  // namespace
}  // namespace nslg

using namespace nslg;

extern "C" size_t nslg_paged_tree_workspace_size(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                                 int32_t head_dim, int64_t total_pages, int32_t page_size,
                                                 int32_t max_q, int32_t dtype) {
  if (batch <= 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || num_qo_heads % num_kv_heads || total_pages <= 0 ||
      page_size <= 0 || max_q <= 0 || max_q > kTreeMaxNodes || !elem_bytes(dtype) ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  const int64_t rows = (int64_t)max_q * (num_qo_heads / num_kv_heads);
  const int64_t n = tree_chunks(batch, total_pages * page_size, rows, num_kv_heads, head_dim, dtype);
  return tree_bytes(batch, n * rows * num_kv_heads, head_dim);
}

extern "C" int nslg_paged_tree_attention(const void* q, int64_t q_stride, const uint32_t* mask, int32_t mask_words,
                                         const int32_t* qo_indptr, const int32_t* q_rows, int32_t grid_width,
                                         int64_t total_q, int32_t max_q, const void* k_new, int64_t k_new_stride,
                                         const void* v_new, int64_t v_new_stride, void* k_pool, void* v_pool,
                                         int64_t num_pages, int32_t page_size, const int32_t* kv_indptr,
                                         const int32_t* kv_indices, const int32_t* kv_last_page_len,
                                         int64_t total_pages, int32_t batch, int32_t num_qo_heads,
                                         int32_t num_kv_heads, int32_t head_dim, float sm_scale, int32_t dtype,
                                         void* out, int64_t out_stride, void* workspace, size_t workspace_bytes,
                                         nslg_stream_t stream) {
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(NSLG_EINVAL, "paged_tree_attention: bad dtype %d", dtype);
  if (batch < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || num_pages <= 0 ||
      total_q < 0 || total_pages < 0)
    return fail(NSLG_EINVAL, "paged_tree_attention: bad sizes");
  if (q_rows && (grid_width < 1 || (int64_t)batch * grid_width > 0x7fffffff || total_q > (int64_t)batch * grid_width))
    return fail(NSLG_EINVAL, "paged_tree_attention: grid of %d x %d rows for %lld nodes", batch, grid_width,
                (long long)total_q);
  if (!(sm_scale > 0.f) || !(sm_scale < INFINITY))
    return fail(NSLG_EINVAL, "paged_tree_attention: sm_scale must be positive and finite");
  if (batch == 0 || (total_q == 0 && !q_rows)) return NSLG_OK;  // (a grid without nodes still has its rows zeroed)
  if (max_q < 0 || (max_q == 0 && total_q > 0) || (int64_t)max_q * batch < total_q)
    return fail(NSLG_EINVAL, "paged_tree_attention: %lld nodes in %d trees of at most %d", (long long)total_q, batch, max_q);
  if (max_q > kTreeMaxNodes)
    return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: trees of up to %d nodes (%d)", kTreeMaxNodes, max_q);
  if (mask_words < (max_q + 31) / 32)
    return fail(NSLG_EINVAL, "paged_tree_attention: masks of %d words for %d nodes", mask_words, max_q);
  if (!q || !qo_indptr || !k_pool || !v_pool || !kv_indptr || !kv_indices || !kv_last_page_len || !out ||
      (!mask && total_q > 0))
    return fail(NSLG_EINVAL, "paged_tree_attention: null pointer");
  if (!k_new != !v_new) return fail(NSLG_EINVAL, "paged_tree_attention: k_new and v_new go together");
  if (num_qo_heads % num_kv_heads)
    return fail(NSLG_EINVAL, "paged_tree_attention: Hq=%d not a multiple of Hkv=%d", num_qo_heads, num_kv_heads);
  const int group = num_qo_heads / num_kv_heads;
  if (group > 16) return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: GQA group %d > 16", group);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: head_dim %d (64, 128 or 256)", head_dim);
  if (q_stride < (int64_t)num_qo_heads * head_dim || out_stride < (int64_t)num_qo_heads * head_dim)
    return fail(NSLG_EINVAL, "paged_tree_attention: row stride smaller than Hq*D");
  if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out) & 15 || (q_stride * eb) % 16 ||
      (out_stride * eb) % 16)
    return fail(NSLG_EINVAL, "paged_tree_attention: q/pool/out must be 16-byte aligned with row strides of 16 bytes");
  if (((uintptr_t)mask | (uintptr_t)qo_indptr | (uintptr_t)q_rows | (uintptr_t)kv_indptr | (uintptr_t)kv_indices |
       (uintptr_t)kv_last_page_len) & 3)
    return fail(NSLG_EINVAL, "paged_tree_attention: masks and tables must be 4-byte aligned");
  if (k_new) {
    if (k_new_stride < (int64_t)num_kv_heads * head_dim || v_new_stride < (int64_t)num_kv_heads * head_dim)
      return fail(NSLG_EINVAL, "paged_tree_attention: k/v row stride smaller than Hkv*D");
    if (((uintptr_t)k_new | (uintptr_t)v_new) & 15 || (k_new_stride * eb) % 16 || (v_new_stride * eb) % 16)
      return fail(NSLG_EINVAL, "paged_tree_attention: k_new/v_new rows must be 16-byte aligned");
  }
  if (num_pages * (int64_t)page_size >= ((int64_t)1 << 31))
    return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: pool has >= 2^31 token slots");
  if ((int64_t)num_kv_heads * head_dim * eb > 0x7fffffff)
    return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: rows of >= 2 GiB");

  const int64_t rows = (int64_t)max_q * group;
  TreeParams p = {};
  p.q = (const char*)q;
  p.q_stride = q_stride * eb;
  p.qo_indptr = qo_indptr;
  p.q_rows = q_rows;
  p.grid_width = grid_width;
  p.total_q = total_q;
  p.mask = mask;
  p.mask_words = mask_words;
  p.k_pool = (const char*)k_pool;
  p.v_pool = (const char*)v_pool;
  p.num_pages = num_pages;
  p.page_size = page_size;
  p.indptr = kv_indptr;
  p.indices = kv_indices;
  p.last_len = kv_last_page_len;
  p.batch = batch;
  p.num_qo_heads = num_qo_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = group;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.out = (char*)out;
  p.out_stride = out_stride * eb;
  p.k_new = (const char*)k_new;
  p.v_new = (const char*)v_new;
  p.k_new_stride = k_new_stride * eb;
  p.v_new_stride = v_new_stride * eb;
  p.max_nodes = max_q;
  int64_t chunks = batch;
  if (workspace && total_q > 0) {
    int64_t n = tree_chunks(batch, total_pages * page_size, rows, num_kv_heads, head_dim, dtype);
    const int64_t each = rows * num_kv_heads;
    while (n > batch && tree_bytes(batch, n * each, head_dim) > workspace_bytes) --n;
    if (n > batch && n < 0x7fffffff && n * each < 0x7fffffff) {
      char* ws = (char*)(((uintptr_t)workspace + 255) / 256 * 256);  // (tree_bytes has room for this)
      p.max_chunks = (int32_t)n;
      p.part_rows = n * each;
      p.ws_tag = (uint64_t*)ws;
      ws += 256;
      p.meta = (int4*)ws;
      ws += ((size_t)batch * 16 + 255) / 256 * 256;
      p.part_ml = (float2*)ws;
      ws += ((size_t)p.part_rows * 8 + 255) / 256 * 256;
      p.part_o = (float*)ws;
      chunks = n;
    }
  }
  const int64_t rows_wg = 64 * tree_row_blocks(rows, head_dim, dtype);
  const int64_t work = total_q > 0 ? chunks * ((rows + rows_wg - 1) / rows_wg) * num_kv_heads : 0;
  int64_t wgs = work + (k_new ? (total_q + kTreeWaves - 1) / kTreeWaves : 0);
  if (wgs == 0) wgs = batch;  // pad rows only
  if (wgs > 0x7fffffff / 8) return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: too many rows");
  p.num_work = (int32_t)work;
  hipStream_t s = as_stream(stream);
  if (dtype == NSLG_F16) return launch_tree_dim<F16>(p, head_dim, rows, wgs, s);
  if (dtype == NSLG_BF16) return launch_tree_dim<BF16>(p, head_dim, rows, wgs, s);
  return launch_tree_dim<F32>(p, head_dim, rows, wgs, s);
}
