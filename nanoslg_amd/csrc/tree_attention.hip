// Attention of trees of drafted tokens over a paged cache, for gfx950 (CDNA4).
//
// Sequence b's last n_b tokens are the nodes of its tree; node t sees every token before the tree and, of the nodes, those of
// its mask (its ancestors and itself):
//   out_t = sum_j exp(s_tj - m_t) v_j / sum_j exp(s_tj - m_t),  s_tj = scale q_t k_j, j over what t sees.
// Query rows are packed GQA-style, row = node * G + g, so that one read of K and V serves the G query heads of a KV head.
//
// Work. A KV head's work is one line of units, (sequence, tile of 128 or 256 rows, 16 KB block of keys), cut into equal spans, one
// a workgroup and CU, so that lengths however uneven leave no CU idle (with chunks of one length, staged
// through registers by 4 waves, 32 trees over 2k-16k tokens took 352 us). A workgroup finds its span from the lengths, walks
// its row tiles, and leaves an fp32 partial (maximum, sum, rows as its lanes hold them) where a row tile's keys begin or end
// outside its span; tree_merge_kernel joins those by their maxima. Without a workspace a workgroup takes a whole row tile.
// (Two workgroups of 8 waves and half the LDS a CU, so that one computes while the other begins a row tile: 64 trees of 16 over
// 100-1000 tokens 54 -> 51 us, but one tree over 8k 33 -> 36 and 16 over 1k-8k 73 -> 77, for twice the partials.)
//
// Within a workgroup, 16 waves (8 for rows of 512 bytes and more), 16 rows a wave; with 128 rows a second group of
// waves takes the other half of every block's keys, joined through LDS at the row tile's end. Blocks of K and V come straight into
// LDS, swizzled so that no read conflicts, three blocks ahead of the one in use. Per 32 keys a wave computes
//   S^T[key x row] = K Q^T      (MFMA; lane (r, gq) then holds keys 16 t + 4 gq + j of row r: V's operand layout,
//                                so that probabilities never leave their registers)
//   online softmax in fp32, the running maximum raised lazily
//   O^T[d x row] += V^T P^T     (MFMA; 16-bit V^T operands by transposing LDS reads; P in two terms)
//
// What bounds it (a call among others; 32/8 heads, D = 128 but in the fourth):
//   32 trees of 32 over 2k-16k, fp16      302 us: 2.2 us a block of 16 KB and 128 rows: its way from HBM (1.8 at a 2 GiB
//                                                 copy's 4.96 TB/s), LDS, products and softmax of waves in step with each
//                                                 other; matrix units busy for 39 %, vector units 63 % (259 us, and 1.4 times
//                                                 the error, with P in one term)
//   8 trees of 24-60 over 256-8k, bf16     55 us: products and softmax of the same waves in turn, 2.9 us a block and 256
//                                                 rows (2.5 at the rate of an 8192^3 product), and about 8 us a row tile (its
//                                                 pages, rows, first block, partial). Over the call the vector units are
//                                                 busy for 50 %, the matrix units 29 %, LDS 20 %, without conflicts
//   4 trees of 128 over 1k-6k, D = 256     62 us: the same, 1.5 us a block and 128 rows (1.3); 4 row tiles a tree read its keys
//   1 tree of 16 over 2k, fp16             18 us: a chain of dependent reads (lengths, pages, keys, partials) and two launches
//   4 chains of 5-9 over 700-3k, fp32      27 us: the same, and products at a ninth of bf16's rate
//
// A key that a row does not see counts nothing, whatever it holds: its score is replaced, and since a
// probability of 0 would not keep a value that is not finite out of a matrix product, such values of the blocks with nodes are
// set to 0 in LDS and added row by row to those that see them. In the blocks before, which every row sees, they go through the
// product, and come out as they went in because no probability there has a term that is 0 or below.
#include "nslg_common.h"

#include <math.h>

#include <type_traits>

namespace nslg {
namespace {

constexpr int kTreeCUs = 256;
constexpr int kTreeMaxNodes = 1024;
constexpr int kTreeWin = 1024;          // pages whose place is in LDS
constexpr int kTreeBlockBytes = 16384;  // K, or V, of a block of keys
constexpr int kTreeSlots = 4;           // blocks in LDS: 128 KB, one workgroup a CU
constexpr int64_t kTreeStream = 256 << 20;  // bytes of K/V, read once, from which on they are loaded past the caches, which they exceed
constexpr int kTreeTurn = 3;            // blocks' time that a workgroup takes to begin a row tile
constexpr float kTreeSlack = 8.0f;  // how far (log2) scores may rise above the running maximum that P is taken at
constexpr float kTreeHalfUp = 7.0f;  // log2 of what half's P are taken times: with the slack 2^15 at most; half's smallest number is then 2^-31
                                     // of a row's largest weight (2^-24 without: 131072 weak keys beside a strong one lost 2e-3)

// Division of 0 .. 2^31 - 1 by a number that the host knows: with 2^l >= d, m = floor(2^(31 + l) / d) + 1 exceeds
// 2^(31 + l) / d by at most 2^l / d of what a quotient's floor allows.
struct Divisor {
  uint32_t m;
  int32_t l;
  int32_t d;
  __host__ static Divisor of(int32_t d) {
    int l = 0;
    while (((int64_t)1 << l) < d) ++l;
    return Divisor{(uint32_t)((((uint64_t)1 << (31 + l)) / (uint64_t)d) + 1), l, d};
  }
  __device__ inline int quotient(int n) const { return (int)(__umulhi(2u * (uint32_t)n, m) >> l); }
};

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
  Divisor page_div;    // by page_size
  Divisor group_div;   // by group
  int32_t max_nodes;   // a tree's nodes, at most (more are cut off)
  int32_t spans;       // workgroups per KV head
  int32_t tile_waves;  // waves of 16 rows of a row tile
  int32_t whole;       // no partials: a workgroup takes a whole row tile
  int32_t one_tile;    // trees are one row tile each: K/V are read once
  int32_t num_work;    // workgroups that attend (spans a KV head); the others write the new rows
  uint64_t* ws_tag;    // the workspace's first word: a decode call's record in the same memory is void
  int4* meta;          // per sequence: its first unit of work, its blocks, units a workgroup, units before a row tile's blocks
  float2* part_ml;     // [num_work, 2, 16 * tile_waves]: running maximum (log2 units), sum
  f32x4* part_o;       // [num_work, 2, tile_waves, D / 16, 64]: a wave's output tiles, as its lanes hold them
};

// Element types: fp32 takes its products on the fp32 matrix instructions.
struct F32 {
  static constexpr int kDtype = NSLG_F32;
};

// A row tile is kRW waves of 16 rows; the workgroup's other waves, a second group, take half of every block's keys. 128
// rows a tile; 256 for trees of more, whose keys are then loaded once (8 trees of 24 to 60 nodes 66 us, in two tiles 77),
// but not with rows of 512 bytes and more, whose registers leave two waves a SIMD.
template <typename T, int D, int kRW>
struct TreeTile {
  static constexpr bool kF32 = T::kDtype == NSLG_F32;
  static constexpr int kBytes = kF32 ? 4 : 2;
  static constexpr int kRowBytes = D * kBytes;
  static constexpr int kWaves = kRowBytes >= 512 ? 8 : 16;
  static constexpr int kRowWaves = kRW;
  static constexpr int kRows = 16 * kRowWaves;
  static constexpr int kThreads = 64 * kWaves;
  static constexpr int kGroups = kWaves / kRowWaves;     // groups of waves that share a block's keys
  static constexpr int kKeys = kTreeBlockBytes / kRowBytes;  // keys of a block
  static constexpr int kGroupKeys = kKeys / kGroups;     // a group's
  static constexpr int kStep = kGroupKeys < 32 ? 16 : 32;    // keys taken at a time
  static constexpr int kSub = kStep / 16;                // in pieces of 16
};

struct SeqOf {
  int nodes, len, q0, page0;  // its nodes and tokens (nodes among them), first ragged row, first entry of its table
};

__device__ inline SeqOf tree_seq(const TreeParams& p, int s) {
  SeqOf x = {0, 0, 0, 0};
  if (s < p.batch) {
    x.page0 = p.indptr[s];
    x.q0 = p.qo_indptr[s];
    const int np = p.indptr[s + 1] - x.page0;
    int lpl = p.last_len[s];
    lpl = lpl < 1 ? 1 : (lpl > p.page_size ? p.page_size : lpl);
    x.len = np > 0 ? (np - 1) * p.page_size + lpl : 0;
    x.nodes = min(max(p.qo_indptr[s + 1] - x.q0, 0), p.max_nodes);
    if (x.nodes == 0) x.len = 0;
  }
  return x;
}

__device__ inline int64_t tree_row(const TreeParams& p, int t) {
  if (!p.q_rows) return t;
  const int64_t r = p.q_rows[t];
  return r >= 0 && r < (int64_t)p.batch * p.grid_width ? r : -1;
}

// Sum over the lanes up to one's own.
__device__ inline int wave_scan_i32(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return x;
}

// The new rows of K and V into their page slots, one wave a row.
__device__ inline void write_row(char* dst, const char* src, int vecs) {
  for (int i = threadIdx.x & 63; i < vecs; i += 64)
    stream_store(reinterpret_cast<u32x4*>(dst) + i, reinterpret_cast<const u32x4*>(src)[i]);
}

__device__ inline void tree_write_new(const TreeParams& p, int64_t t, int row_bytes) {
  const int lane = threadIdx.x & 63;
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

// Where piece `c` (16 bytes) of key `key`'s row lies in its block: permuted so that the operand reads of 16 (V: 8) keys
// fall on distinct banks without padding, which the direct loads into LDS could not write.
template <int kVecs>
__device__ inline int swizzle_k(int key) {
  return kVecs >= 16 ? key & 15 : (key >> 1) & 7;
}
template <typename T, int kVecs>
__device__ inline int swizzle_v(int key) {
  if constexpr (T::kDtype == NSLG_F32) return 0;  // (read as whole rows)
  return kVecs >= 16 ? (key & 7) << 1 : ((key >> 1) & 3) << 1;
}

// A lane's 16 bytes into LDS at dst + 16 * lane (dst uniform).
template <bool kStream>
__device__ inline void load_lds16(const char* src, char* dst) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)dst, 16, 0, kStream ? 2 : 0);
}

// The wave's direct loads but the last `kLeft`, and its LDS reads, are over; then all waves meet.
template <int kLeft>
__device__ inline void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(kLeft) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A lane's share of a row: o[n][i] is d = 16 n + 4 gq + i (fp32: d = 64 (n / 4) + 16 gq + 4 i + n % 4).
template <typename T, int NT>
__device__ inline void store_row(char* dst, int gq, const f32x4 (&o)[NT]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    if constexpr (T::kDtype == NSLG_F32) {
      const int c = n >> 2, i = n & 3;
      *reinterpret_cast<f32x4*>(dst + 4 * (64 * c + 16 * gq + 4 * i)) = f32x4{o[4 * c][i], o[4 * c + 1][i], o[4 * c + 2][i], o[4 * c + 3][i]};
    } else {
      u16x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = T::from_f32(o[n][i]);
      *reinterpret_cast<u16x4*>(dst + 2 * (16 * n + 4 * gq)) = x;
    }
  }
}

template <typename T, int D, int kRW>
__global__ void __launch_bounds__((TreeTile<T, D, kRW>::kThreads), (TreeTile<T, D, kRW>::kWaves / 4)) tree_attention_kernel(TreeParams p) {
  using Tile = TreeTile<T, D, kRW>;
  static_assert(Tile::kGroups <= 2 && (Tile::kF32 ? Tile::kGroupKeys % 16 : Tile::kGroupKeys % 32) == 0);
  constexpr bool kF32 = Tile::kF32;
  constexpr int kBytes = Tile::kBytes, kWaves = Tile::kWaves, kThreads = Tile::kThreads, kGroups = Tile::kGroups;
  constexpr int kSub = Tile::kSub, kStep = Tile::kStep, kGroupKeys = Tile::kGroupKeys, kKeys = Tile::kKeys;
  constexpr int kRowBytes = Tile::kRowBytes, kRowWaves = Tile::kRowWaves, kRows = Tile::kRows, kBlockBytes = kTreeBlockBytes, kSlots = kTreeSlots;
  constexpr int NT = D / 16;
  constexpr int kOps = kRowBytes / 64;                      // 16-byte operands of a key or row, a lane
  constexpr int kVecs = kRowBytes / 16;                     // 16-byte pieces of a row
  constexpr int kPer = kBlockBytes / (16 * kThreads);       // pieces of K (and of V) a thread and block
  constexpr int kSteps = kGroupKeys / kStep;                // steps of a group's keys of a block
  constexpr float kUp = T::kDtype == NSLG_F16 ? kTreeHalfUp : 0.f;

  __shared__ __attribute__((aligned(1024))) char kv_lds[2 * kSlots * kBlockBytes];
  __shared__ float2 ml_lds[kGroups == 2 ? kRows : 1];
  __shared__ int32_t page_lds[kTreeWin];
  __shared__ SeqOf seq_lds[64];   // 64 sequences, and the units before each and up to its end
  __shared__ int2 unit_lds[64];
  __shared__ uint32_t bad_lds[2][kKeys / kStep];  // keys of a step with a value of V that is not finite (blocks in turn)

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row_wave = wave % kRowWaves, group = wave / kRowWaves;
  char* k_lds = kv_lds;
  char* v_lds = kv_lds + kSlots * kBlockBytes;
  // The lane's number, anew: what is derived from it is then not kept in registers from block to block. (Spilled, a
  // register's reload would wait for all of the wave's direct loads.)
  auto fresh_lane = [&]() {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  const int G = p.group, ps = p.page_size;
  const int row_bytes = p.num_kv_heads * kRowBytes;
  const int w = (int)blockIdx.x;
  if (p.q_rows)
    zero_pad_rows(p.qo_indptr, p.q_rows, p.grid_width, p.batch, p.out, p.out_stride, p.num_qo_heads * kRowBytes,
                  w * kWaves + wave, (int)gridDim.x * kWaves);
  if (w >= p.num_work) {
    tree_write_new(p, (int64_t)(w - p.num_work) * kWaves + wave, row_bytes);
    return;
  }
  if (w == 0 && tid == 0 && p.ws_tag) *p.ws_tag = 0;

  // ---- the workgroup's span of work. A KV head's work is one line of units: sequence after sequence, row tile after
  // row tile, block of keys after block; workgroup j of the head takes `span` of them from j * span on (KV heads in turn:
  // a head's neighbours share an XCD's L2). What begins or ends inside a row tile's keys leaves a partial. A row tile's blocks
  // lie behind `turn` units without any, the time that it takes a workgroup to begin another row tile (8 trees of 24-60 nodes
  // 66 -> 62 us, 4 fp32 chains 34.6 -> 31.8, caches cold; 2 and 4 units do as well, 6 less); where spans are as short as
  // that, every one lies in one or two row tiles, and a longer span only costs. Without partials a unit is a row tile with all its keys.
  const int h = w % p.num_kv_heads;
  const int j = w / p.num_kv_heads;
  auto blocks_of = [&](const SeqOf& x) { return (x.len + kKeys - 1) / kKeys; };
  auto tiles_of = [&](const SeqOf& x) { return x.len > 0 ? (x.nodes * G + kRows - 1) / kRows : 0; };
  int turn = 0;
  auto units_of = [&](const SeqOf& x) { return tiles_of(x) * (p.whole ? 1 : blocks_of(x) + turn); };
  int group0 = 0, before = 0;  // the first of the sequences in seq_lds, the units before it
  int total;
  bool stream;
  {
    const SeqOf s = tree_seq(p, lane);
    int u = units_of(s), tiles = tiles_of(s);
    int incl = wave_scan_i32(u), incl_tiles = wave_scan_i32(p.whole ? tiles * blocks_of(s) : tiles);
    total = __builtin_amdgcn_readlane(incl, 63);
    int all_tiles = __builtin_amdgcn_readlane(incl_tiles, 63);  // (whole: blocks)
    for (int s0 = 64; s0 < p.batch; s0 += 64) {
      const SeqOf x = tree_seq(p, s0 + lane);
      total += wave_sum_i32(units_of(x));
      all_tiles += wave_sum_i32(p.whole ? tiles_of(x) * blocks_of(x) : tiles_of(x));
    }
    total = __builtin_amdgcn_readfirstlane(total);
    // (by the lengths: a page may be far larger than what a sequence has of it)
    stream = p.one_tile && (int64_t)__builtin_amdgcn_readfirstlane(p.whole ? all_tiles : total) * p.num_kv_heads * 2 * kTreeBlockBytes > kTreeStream;
    if (!p.whole && total >= kTreeTurn * p.spans) {  // uniform
      turn = kTreeTurn;
      total += turn * __builtin_amdgcn_readfirstlane(all_tiles);
      u += turn * tiles;
      incl += turn * incl_tiles;
    }
    if (wave == 0) seq_lds[lane] = s, unit_lds[lane] = int2{incl - u, incl};
  }
  const int span = p.whole ? 1 : max(__builtin_amdgcn_readfirstlane((total + p.spans - 1) / p.spans), 1);
  int pos = __builtin_amdgcn_readfirstlane((int)min((int64_t)j * span, (int64_t)total));
  const int pos_end = __builtin_amdgcn_readfirstlane(min(total - pos, span) + pos);
  if (w == 0 && wave == 0 && p.meta) {
    int at = 0;
    for (int s0 = 0; s0 < p.batch; s0 += 64) {
      const SeqOf x = tree_seq(p, s0 + lane);
      const int u = units_of(x);
      const int sum = wave_scan_i32(u);
      if (s0 + lane < p.batch) p.meta[s0 + lane] = int4{at + sum - u, blocks_of(x), span, turn};
      at += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  __syncthreads();
  while (pos < pos_end) {
    while (pos - before >= unit_lds[63].y) {  // uniform: beyond these sequences
      before = __builtin_amdgcn_readfirstlane(before + unit_lds[63].y);
      group0 += 64;
      const SeqOf s = tree_seq(p, group0 + lane);
      const int u = units_of(s);
      const int incl = wave_scan_i32(u);
      __syncthreads();
      if (wave == 0) seq_lds[lane] = s, unit_lds[lane] = int2{incl - u, incl};
      __syncthreads();
    }
    const int src = __ffsll((long long)__ballot(pos - before < unit_lds[lane].y)) - 1;
    const SeqOf seq = seq_lds[src];

    const int first_unit = __builtin_amdgcn_readfirstlane(before + unit_lds[src].x);
    const int n_nodes = __builtin_amdgcn_readfirstlane(seq.nodes), L = __builtin_amdgcn_readfirstlane(seq.len);
    const int q0 = __builtin_amdgcn_readfirstlane(seq.q0);
    const int32_t* idx = p.indices + __builtin_amdgcn_readfirstlane(seq.page0);
    const int all_blk = (L + kKeys - 1) / kKeys;
    int tile = 0, blk0 = pos - first_unit, n_blk = all_blk;
    if (p.whole) {
      tile = blk0;
      blk0 = 0;
      ++pos;
    } else {
      const int per = all_blk + turn;
      if (blk0 >= per) {
        tile = blk0 / per;
        blk0 -= tile * per;
      }
      const int units = min(pos_end - pos, per - blk0);
      pos += units;
      n_blk = blk0 + units - turn;  // where the blocks end
      blk0 = max(blk0 - turn, 0);
      n_blk -= blk0;
      if (n_blk <= 0) continue;  // uniform
    }
    const bool to_end = blk0 + n_blk == all_blk;
    const bool partial = blk0 > 0 || !to_end;
    const int nrows = n_nodes * G;
    const int start = max(L - n_nodes, 0);
    const int kv_begin = blk0 * kKeys;
    const int kv_end = to_end ? L : kv_begin + n_blk * kKeys;

    // ---- the wave's rows: lane's row r of them, its row of q and out (-1: none), its node and its bytes' offset there
    const int wave_row0 = tile * kRows + 16 * row_wave;
    const bool wave_on = wave_row0 < nrows;  // (a wave without rows only helps to load)
    struct Row {
      int64_t at;
      int node, off;
      bool ok;
    };
    auto row_of = [&](int r) {
      const int row = wave_row0 + r;
      Row x;
      x.node = p.group_div.quotient(row);
      x.ok = row < nrows && q0 + x.node < p.total_q;
      x.at = x.ok ? tree_row(p, q0 + x.node) : -1;
      x.off = (h * G + row - x.node * G) * kRowBytes;
      return x;
    };
    // ---- blocks of keys: wave-wide loads of 1 KB straight into LDS. Load u of a block fills bytes 1024 u .. + 1023, lane l
    // the 16 at 16 l: piece l % kVecs of key u * (64 / kVecs) + l / kVecs, where the swizzle has put piece (l % kVecs) ^
    // swizzle(key) of the row.
    const int head_off = h * kRowBytes;
    auto page_of = [&](int key) { return p.page_div.quotient(key); };
    auto checked = [&](int page) { return page < 0 || (int64_t)page >= p.num_pages ? 0 : page; };
    const bool fresh = p.k_new != nullptr;
    int64_t new_row0 = q0;  // row of k_new / v_new of node 0 (a tree's rows are contiguous)
    if (fresh && p.q_rows) {
      const int64_t at = tree_row(p, q0);
      new_row0 = at < 0 ? 0 : at;
    }
    const int64_t new_last = (p.q_rows ? (int64_t)p.batch * p.grid_width : p.total_q) - 1;
    auto new_at = [&](int key) { return min(new_row0 + (key - start), new_last); };
    // page_lds[i]: what is added to a key of page win + i to make its slot
    int win = 0, win_blk = 0;  // the window's first page; the first block that reaches past it
    auto load_pages = [&](int key) {
      win = page_of(key);
      const int last = page_of(kv_end - 1);
      for (int i = tid; i < kTreeWin && win + i <= last; i += kThreads) page_lds[i] = (checked(idx[win + i]) - (win + i)) * ps;
      win_blk = last < win + kTreeWin ? 0x7fffffff : ((win + kTreeWin) * ps - kv_begin) / kKeys;
    };
    auto key_of = [&](int ln) { return wave * (64 / kVecs) + ln / kVecs; };  // of a lane's first piece
    constexpr int kKeyStep = kWaves * (64 / kVecs);  // keys between a lane's pieces
    constexpr int kTurn = kPer == 1 ? 0 : kKeyStep % 16;  // (the swizzles repeat after 16 keys)
    static_assert(kTurn == 0 || (kTurn == 8 && kPer == 2 && kF32), "a lane's second piece is swizzled as key + 8, fp32 V not at all");
    auto issue = [&](int blk) {
      char* ks = k_lds + (blk & (kSlots - 1)) * kBlockBytes + 1024 * wave;
      char* vs = v_lds + (blk & (kSlots - 1)) * kBlockBytes + 1024 * wave;
      const int key0 = kv_begin + blk * kKeys;
      const bool nodes = fresh && key0 + kKeys > start;  // uniform: some of the block's rows are not in the pool
      const int ln = fresh_lane();
      const int l_key = key_of(ln), l_piece = ln % kVecs;
      const int v_piece = head_off + 16 * (l_piece ^ swizzle_v<T, kVecs>(l_key));
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int k_piece = head_off + 16 * (l_piece ^ swizzle_k<kVecs>(l_key + kTurn * i));
        const int kabs = min(key0 + l_key + kKeyStep * i, kv_end - 1);
        const uint32_t slot = (uint32_t)(kabs + page_lds[page_of(kabs) - win]);
        const char* kp = p.k_pool + k_piece + (uint64_t)slot * (uint32_t)row_bytes;
        const char* vp = p.v_pool + v_piece + (uint64_t)slot * (uint32_t)row_bytes;
        if (nodes && kabs >= start) {
          const int64_t at = new_at(kabs);
          kp = p.k_new + at * p.k_new_stride + k_piece;
          vp = p.v_new + at * p.v_new_stride + v_piece;
        }
        if (stream) {  // uniform
          load_lds16<true>(kp, ks + 1024 * kWaves * i);
          load_lds16<true>(vp, vs + 1024 * kWaves * i);
        } else {
          load_lds16<false>(kp, ks + 1024 * kWaves * i);
          load_lds16<false>(vp, vs + 1024 * kWaves * i);
        }
      }
    };
    // The first pages and the row of q are under way together, then q's own rows while the first blocks are sent for.
    constexpr int kWinPer = kTreeWin / kThreads;
    int32_t first_pages[kWinPer];
    const int last_page = page_of(kv_end - 1);
    win = page_of(kv_begin);
    win_blk = last_page < win + kTreeWin ? 0x7fffffff : ((win + kTreeWin) * ps - kv_begin) / kKeys;
#pragma unroll
    for (int i = 0; i < kWinPer; ++i) first_pages[i] = win + tid + kThreads * i <= last_page ? idx[win + tid + kThreads * i] : 0;
    const Row q_row = row_of(lane & 15);
#pragma unroll
    for (int i = 0; i < kWinPer; ++i) {
      const int at = tid + kThreads * i;
      if (win + at <= last_page) page_lds[at] = (checked(first_pages[i]) - (win + at)) * ps;
    }
    u32x4 qb[kOps];
    {
      const char* src = p.q + (q_row.at >= 0 ? q_row.at * p.q_stride + q_row.off : 0) + 16 * (lane >> 4);
#pragma unroll
      for (int s = 0; s < kOps; ++s) qb[s] = q_row.at >= 0 ? *reinterpret_cast<const u32x4*>(src + 64 * s) : u32x4{0, 0, 0, 0};
    }
    if (tid < 2 * (kKeys / kStep)) bad_lds[tid / (kKeys / kStep)][tid % (kKeys / kStep)] = 0;
    __syncthreads();
    static_assert(kSlots * kKeys <= kTreeWin);  // the blocks on the way, even of single-token pages
#pragma unroll 1
    for (int i = 0; i < min(n_blk, kSlots - 1); ++i) issue(i);

    // the raw score above which the maximum is raised; kUp - maximum (log2 units; 0: none yet), the exponents' offset
    float thr = -INFINITY, neg_m = 0.f;
    f32x4 lsum = {0.f, 0.f, 0.f, 0.f}, o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float inv_scale = 1.f / p.scale_log2;

    // the bits of a step's keys (kbase on) that row r sees
    auto visible = [&](int kbase, int r) -> uint32_t {
      const Row x = row_of(r);
      const uint32_t* mrow = p.mask + (int64_t)(x.ok ? q0 + x.node : 0) * p.mask_words;
      const int rel = kbase - start;
      const int words = p.mask_words;
      uint32_t v;
      if (rel >= 0) {
        const int wi = rel >> 5, sh = rel & 31;
        const uint32_t lo = wi < words ? mrow[wi] : 0u;
        const uint32_t hi = wi + 1 < words ? mrow[wi + 1] : 0u;
        v = sh ? (lo >> sh) | (hi << (32 - sh)) : lo;
      } else if (rel > -32) {
        v = (1u << -rel) - 1u;
        v |= mrow[0] << -rel;
      } else {
        v = ~0u;
      }
      const int left = kv_end - kbase;
      if (left < 32) v &= left > 0 ? (1u << left) - 1u : 0u;
      return x.ok ? v : 0u;
    };

    const int share = group * (kGroupKeys * kRowBytes);  // the group's share of a block
    // One step of a block: scores, mask (`tail`: a block with nodes, or past the end), probabilities, product with V.
    auto step = [&](int blk, int u, auto tail) {
      constexpr bool kTail = decltype(tail)::value;
      const int kbase = kv_begin + blk * kKeys + group * kGroupKeys + u * kStep;
      const char* ksrc = k_lds + (blk & (kSlots - 1)) * kBlockBytes + u * kStep * kRowBytes;
      const char* vsrc = v_lds + (blk & (kSlots - 1)) * kBlockBytes + u * kStep * kRowBytes;
      const int ln = fresh_lane(), r = ln & 15, gq = ln >> 4;
      // LDS offsets of the lane's operands: K at operand i is k_at ^ 64 i, V of output tile n (16 bits) v_at ^ 32 n
      const int k_at = share + r * kRowBytes + 16 * (gq ^ swizzle_k<kVecs>(r));
      const int v_key = kF32 ? 4 * gq : 4 * gq + (r >> 2);
      const int v_at = share + v_key * kRowBytes + (kF32 ? 16 * r : 16 * swizzle_v<T, kVecs>(v_key) + 8 * (r & 3));
      f32x4 s[kSub];
      u32x4 ka[kSub][kOps];
#pragma unroll
      for (int t = 0; t < kSub; ++t)
#pragma unroll
        for (int i = 0; i < kOps; ++i) ka[t][i] = *reinterpret_cast<const u32x4*>(ksrc + 16 * t * kRowBytes + (k_at ^ (64 * i)));
      if constexpr (kF32) {
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < kOps; ++i) {
            const f32x4 a = __builtin_bit_cast(f32x4, ka[t][i]), q = __builtin_bit_cast(f32x4, qb[i]);
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[0], q[0], x, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[1], q[1], y, 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[2], q[2], x, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[3], q[3], y, 0, 0, 0);
          }
          s[t] = x + y;
        }
      } else {
#pragma unroll
        for (int t = 0; t < kSub; ++t) s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kOps; ++i)
#pragma unroll
          for (int t = 0; t < kSub; ++t) s[t] = T::mma_k32(__builtin_bit_cast(u16x8, ka[t][i]), __builtin_bit_cast(u16x8, qb[i]), s[t]);
      }
      // V's operand of output tile n (16 bits): lane r of a 16-lane group addresses keys 4 gq + r / 4 (then + 16), columns 16 n
      // + 4 (r % 4) .. + 3, and receives keys 4 gq + 0..3 (+ 16) at d = 16 n + r. Read ahead of the softmax, which covers
      // their way (read one by one as they are used, the reads took most of the time).
      typedef short i16x4_t __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) i16x4_t* lds_i16x4;
      u16x8 va[kF32 ? 1 : NT];
      if constexpr (!kF32) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const char* at = vsrc + (v_at ^ (32 * n));
          const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)at);
          const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4)(at + 16 * kRowBytes));
          va[n] = __builtin_bit_cast(u16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      // A later block's loads go out here: at the block's start the waves waited to get rid of theirs, all at once, before any
      // product (265 us with 32 trees of 32 nodes over 2k-16k tokens and P in one term, 308 from there).
      if (u == 0 && blk + kSlots - 1 < n_blk) issue(blk + kSlots - 1);
      __builtin_amdgcn_sched_barrier(0);
      uint32_t vis = 0;
      if constexpr (kTail) {
        vis = visible(kbase, r);
#pragma unroll
        for (int j = 0; j < 4 * kSub; ++j)
          if (!(vis >> (16 * (j >> 2) + 4 * gq + (j & 3)) & 1)) s[j >> 2][j & 3] = -INFINITY;
      }
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4 * kSub; ++j) top = fmaxf(top, s[j >> 2][j & 3]);
      if (__ballot(top > thr)) {
        const float m_run = thr == -INFINITY ? -INFINITY : -neg_m;
        const float m_new = fmaxf(m_run, rows_max(top * p.scale_log2) - kUp);
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
        lsum *= alpha;
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n] *= alpha;
        thr = (m_new + (kUp + kTreeSlack)) * inv_scale;
        neg_m = m_new == -INFINITY ? 0.f : -m_new;
      }
      u16x8 pb, pb_lo;
      typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      float minus_one = -1.f;  // (known to the compiler, it would make three instructions of a half's rest)
      asm("" : "+s"(minus_one));
#pragma unroll
      for (int j = 0; j < 4 * kSub; ++j) {
        const float x = fast_exp2(fmaf(s[j >> 2][j & 3], p.scale_log2, neg_m));
        s[j >> 2][j & 3] = x;
        // (the rows' sums take the probabilities before they are rounded, a lane's keys at a time; as a product with a row of ones
        // they cost a matrix instruction in 13 to 17: 250 us with 32 trees over 2k-16k tokens and P in one term, then 243)
        lsum[j & 3] += x;
      }
      // A probability goes into the product in two terms: 16 bits of bfloat16, 21 of half (one term, of 11, was seen in the outputs:
      // 1.4 times the error of probabilities in fp32). The first is cut off, so that neither is negative, and
      // over blocks that every row sees no term of a probability above 0 is 0: what is infinite in V stays that.
      if constexpr (!kF32) {
        u32x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 4 * kSub; j += 2) {
          const float x = s[j >> 2][j & 3], y = s[j >> 2][(j & 3) + 1];
          if constexpr (T::kDtype == NSLG_BF16) {
            const uint32_t xh = __float_as_uint(x) & 0xffff0000u, yh = __float_as_uint(y) & 0xffff0000u;
            hi[j >> 1] = xh >> 16 | yh;
            // (2^-23 of the probability more than the rest)
            lo[j >> 1] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)fmaf(x, 0x1.000002p+0f, -__uint_as_float(xh)),
                                                             (__bf16)fmaf(y, 0x1.000002p+0f, -__uint_as_float(yh))});
          } else {
            // (half's smallest number, 2^-31 of the row's largest weight, or more)
            constexpr _Float16 kLeast = kTail ? (_Float16)0.f : (_Float16)0x1p-24f;
            const f16x2 least = {kLeast, kLeast};
            uint32_t pair = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
            if constexpr (!kTail) pair = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(f16x2, pair), least));
            asm("" : "+v"(pair));  // (the rests take them from here, not from conversions of their own)
            const f16x2 h = __builtin_bit_cast(f16x2, pair);
            f16x2 rest = {(_Float16)fmaf((float)h[0], minus_one, x), (_Float16)fmaf((float)h[1], minus_one, y)};
            if constexpr (!kTail) rest = __builtin_elementwise_max(rest, least);
            hi[j >> 1] = pair;
            lo[j >> 1] = __builtin_bit_cast(uint32_t, rest);
          }
        }
        pb = __builtin_bit_cast(u16x8, hi), pb_lo = __builtin_bit_cast(u16x8, lo);
      }
      // O^T += V^T P^T
      if constexpr (kF32) {
#pragma unroll
        for (int t = 0; t < kSub; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              const f32x4 v = *reinterpret_cast<const f32x4*>(vsrc + (16 * t + j) * kRowBytes + v_at + 256 * c);
#pragma unroll
              for (int e = 0; e < 4; ++e) o[4 * c + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], s[t][j], o[4 * c + e], 0, 0, 0);
            }
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n] = T::mma_k32(va[n], pb, o[n]);
          o[n] = T::mma_k32(va[n], pb_lo, o[n]);
        }
      }
      // nodes whose V is not finite: those elements, for the rows that see the node
      if constexpr (kTail) {
        uint32_t bad = __builtin_amdgcn_readfirstlane(bad_lds[blk & 1][group * kSteps + u]);
        while (__builtin_expect(bad != 0, 0)) {
          const int kk = __ffs(bad) - 1;
          bad &= bad - 1;
          const int key = kbase + kk;
          const char* vrow = (fresh && key >= start ? p.v_new + new_at(key) * p.v_new_stride
                                    : p.v_pool + ((int64_t)checked(idx[page_of(key)]) * ps + (key - page_of(key) * ps)) * row_bytes) +
                             head_off;
          float pr = 0.f;
#pragma unroll
          for (int j = 0; j < 4 * kSub; ++j)
            if (16 * (j >> 2) + (j & 3) == (kk & ~12)) pr = s[j >> 2][j & 3];
          pr = __shfl(pr, 16 * ((kk >> 2) & 3) + r, 64);
          if (!(vis >> kk & 1)) continue;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v;
              if constexpr (kF32)
                v = reinterpret_cast<const float*>(vrow)[64 * (n >> 2) + 16 * gq + 4 * i + (n & 3)];
              else
                v = T::to_f32(reinterpret_cast<const uint16_t*>(vrow)[16 * n + 4 * gq + i]);
              if (!(fabsf(v) < INFINITY)) o[n][i] += pr * v;
            }
        }
      }
    };
    // Values of a block's V that are not finite, and those past the end, become 0 in LDS.
    auto tidy = [&](int blk) {
      char* vs = v_lds + (blk & (kSlots - 1)) * kBlockBytes;
      const int ln = fresh_lane();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int key = key_of(ln) + kKeyStep * i;
        const int kabs = kv_begin + blk * kKeys + key;
        u32x4* at = reinterpret_cast<u32x4*>(vs + 1024 * (wave + kWaves * i) + 16 * ln);
        if (kabs >= kv_end) {
          *at = u32x4{0, 0, 0, 0};
        } else {
          bool bad = false;
          const u32x4 x = drop_not_finite<T>(*at, bad);
          if (bad) {
            *at = x;
            atomicOr(&bad_lds[blk & 1][key / kStep], 1u << (key % kStep));
          }
        }
      }
    };

    // A block has landed for all waves once each has waited for its loads and all have met; then the block before it has
    // been read, and the loads of block i + kSlots - 1 take its slot.
    auto block = [&](int blk, auto tail) {
      if (blk + kSlots - 2 < n_blk)
        wait_and_meet<2 * kPer * (kSlots - 2)>();
      else
        wait_and_meet<0>();
      if (blk + kSlots - 1 < n_blk) {
        if (blk + kSlots - 1 >= win_blk) {  // uniform
          load_pages(kv_begin + (blk + kSlots - 1) * kKeys);
          __syncthreads();
        }
        if (!wave_on) issue(blk + kSlots - 1);  // (the others in the course of their step)
      }
      if constexpr (decltype(tail)::value) {
        tidy(blk);
        __syncthreads();
        if (tid < kKeys / kStep) bad_lds[(blk + 1) & 1][tid] = 0;
      }
      if (wave_on) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u) step(blk, u, tail);
      }
    };
    const int n_plain = min(max(start - kv_begin, 0) / kKeys, n_blk);  // blocks that lie before the tree
    // q is waited for here: within the loop the wait for it would be one for every direct load on its way. (No time was
    // measured for that, but the loads would be one block ahead, not three.)
#pragma unroll
    for (int s = 0; s < kOps; ++s) asm volatile("" : "+v"(qb[s]));
    int blk = 0;
    for (; blk < n_plain; ++blk) block(blk, std::false_type());
    for (; blk < n_blk; ++blk) block(blk, std::true_type());

    // ---- the second group's rows to the first's, lane by lane, through the blocks' LDS
    const int r = lane & 15, gq = lane >> 4;
    float l = rows_sum((lsum[0] + lsum[1]) + (lsum[2] + lsum[3]));
    float m = thr == -INFINITY ? -INFINITY : -neg_m;
    if constexpr (kGroups == 2) {
      wait_and_meet<0>();
      f32x4* buf = reinterpret_cast<f32x4*>(kv_lds) + row_wave * (64 * NT) + lane;
      static_assert(kRowWaves * 64 * NT * 16 <= 2 * kSlots * kBlockBytes);
      if (group && wave_on) {
#pragma unroll
        for (int n = 0; n < NT; ++n) buf[64 * n] = o[n];
        if (gq == 0) ml_lds[16 * row_wave + r] = float2{m, l};
      }
      wait_and_meet<0>();
      if (!group && wave_on) {
        const float2 other = ml_lds[16 * row_wave + r];
        const float top = fmaxf(m, other.x);
        const float f0 = l == 0.f ? 0.f : fast_exp2(m - top);  // 0: no key of the group seen
        const float f1 = other.y == 0.f ? 0.f : fast_exp2(other.x - top);
        l = fmaf(f0, l, f1 * other.y);
        m = top;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const f32x4 x = buf[64 * n];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] = fmaf(f0, o[n][e], f1 * x[e]);
        }
      }
    }

    // ---- the rows: normalised into `out`, or the span's share as a partial
    if (partial && wave_on && group == 0) {
      // (a workgroup has at most one that began before its span and one that goes on behind it)
      const int64_t slot = ((int64_t)2 * w + (blk0 == 0)) * kRowWaves + row_wave;
      if (gq == 0) p.part_ml[16 * slot + r] = float2{m, l};
#pragma unroll
      for (int n = 0; n < NT; ++n) p.part_o[(slot * NT + n) * 64 + lane] = o[n];
    } else if (!partial && wave_on && group == 0) {
      const Row x = row_of(r);
      const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (a sum that is NaN makes the row NaN)
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n] *= f;
      if (x.at >= 0) store_row<T, NT>(p.out + x.at * p.out_stride + x.off, gq, o);
    }
    if (pos < pos_end) __syncthreads();  // the next row tile's loads overwrite what the other waves may still read
  }
}

// Log-sum-exp merge of the parts of 16 rows (a row wave's) of one KV head. Waves 0 .. kTileWaves - 1 of a workgroup share
// the output tiles, kSplit such sets the parts, four at a time each; the sets' sums go through LDS.
template <typename T, int D, int kSplit>
__global__ void __launch_bounds__(256 * kSplit) tree_merge_kernel(TreeParams p, int row_waves) {
  constexpr int NT = D / 16, kN = T::kDtype == NSLG_F32 ? 4 : NT / 4;  // (fp32 rows are stored four tiles at a time)
  constexpr int kTileWaves = NT / kN;
  __shared__ f32x4 o_lds[kSplit > 1 ? kSplit - 1 : 1][kSplit > 1 ? NT * 64 : 1];
  __shared__ float2 ml_lds[kSplit][16];
  const int lane = threadIdx.x & 63, r = lane & 15, gq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int tw = wave % kTileWaves, set = wave / kTileWaves;
  const int h = blockIdx.x % p.num_kv_heads;
  const int k = blockIdx.x / p.num_kv_heads;
  const int b = k / row_waves, rw = k - b * row_waves;
  const int G = p.group;
  const int4 meta = p.meta[b];
  const int q0 = p.qo_indptr[b];
  const int nodes = min(max(p.qo_indptr[b + 1] - q0, 0), p.max_nodes);
  if (16 * rw >= nodes * G || meta.y <= 0) return;
  const int tile = rw / p.tile_waves;
  const int first = meta.x + tile * (meta.y + meta.w) + meta.w;  // the row tile's first block's unit
  const int j0 = first / meta.z;
  const int parts = (first + meta.y - 1) / meta.z - j0 + 1;
  if (parts < 2 || j0 + parts > p.spans) return;  // uniform over the workgroup
  // the partial of the rows' part i: the first part goes on behind its workgroup's span, the others began before theirs
  auto slot_of = [&](int i) {
    return ((int64_t)2 * ((j0 + i) * p.num_kv_heads + h) + (i == 0)) * p.tile_waves + rw - tile * p.tile_waves;
  };
  float m = -INFINITY, l = 0.f;
  f32x4 o[kN];
#pragma unroll
  for (int n = 0; n < kN; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto join = [&](float m1, float l1, const f32x4 (&x)[kN]) {
    if (l1 == 0.f) return;  // no key of the part seen
    const float top = fmaxf(m, m1);
    const float f0 = l == 0.f ? 0.f : fast_exp2(m - top), f1 = fast_exp2(m1 - top);
    l = fmaf(f0, l, f1 * l1);
    m = top;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = fmaf(f0, o[n][e], f1 * x[n][e]);
  };
  const int each = (parts + kSplit - 1) / kSplit;
  const int end = min(parts, (set + 1) * each);
  if (set < kSplit) {
    for (int i0 = set * each; i0 < end; i0 += 4) {
      float2 ml[4];
      f32x4 x[4][kN];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t slot = slot_of(min(i0 + u, end - 1));
        ml[u] = p.part_ml[16 * slot + r];
#pragma unroll
        for (int n = 0; n < kN; ++n) x[u][n] = p.part_o[(slot * NT + tw * kN + n) * 64 + lane];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u < end) join(ml[u].x, ml[u].y, x[u]);
    }
  }
  if constexpr (kSplit > 1) {
    if (set > 0 && set < kSplit) {
#pragma unroll
      for (int n = 0; n < kN; ++n) o_lds[set - 1][(tw * kN + n) * 64 + lane] = o[n];
      if (tw == 0 && gq == 0) ml_lds[set][r] = float2{m, l};
    }
    __syncthreads();
    if (set) return;
#pragma unroll
    for (int i = 1; i < kSplit; ++i) {
      f32x4 x[kN];
#pragma unroll
      for (int n = 0; n < kN; ++n) x[n] = o_lds[i - 1][(tw * kN + n) * 64 + lane];
      join(ml_lds[i][r].x, ml_lds[i][r].y, x);
    }
  } else {
    if (set) return;
  }
  const int row = 16 * rw + r;
  const int node = p.group_div.quotient(row);
  if (row >= nodes * G || q0 + node >= p.total_q) return;
  const int64_t at = tree_row(p, q0 + node);
  if (at < 0) return;
  const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int n = 0; n < kN; ++n) o[n] *= f;
  constexpr int kBytes = T::kDtype == NSLG_F32 ? 4 : 2;
  char* dst = p.out + at * p.out_stride + (int64_t)(h * G + row - node * G) * D * kBytes;
  store_row<T, kN>(dst + tw * 16 * kN * kBytes, gq, o);
}

// ---- host ------------------------------------------------------------------------------

inline int64_t tree_rows(int64_t rows, int head_dim, int dtype) {
  return rows > 128 && head_dim * elem_bytes(dtype) < 512 ? 256 : 128;
}
inline int64_t tree_tiles(int64_t rows, int head_dim, int dtype) {
  const int64_t n = tree_rows(rows, head_dim, dtype);
  return (rows + n - 1) / n;
}

// Workgroups per KV head: one a CU, which its blocks in LDS fill.
int64_t tree_spans(int64_t batch, int64_t total_keys, int64_t rows, int num_kv_heads, int head_dim, int dtype) {
  int64_t n = kTreeCUs / num_kv_heads;
  const int64_t most = (total_keys * head_dim * elem_bytes(dtype) / kTreeBlockBytes + batch) * tree_tiles(rows, head_dim, dtype);
  n = n > most ? most : n;
  return n < 1 ? 1 : n;
}

// The workspace of n such workgroups: the first word, the sequences' entries, two partials of a row tile each.
size_t tree_bytes(int64_t batch, int64_t n, int num_kv_heads, int64_t tile_rows, int head_dim) {
  const size_t rows = (size_t)n * num_kv_heads * 2 * tile_rows;
  return 512 + ((size_t)batch * 16 + 255) / 256 * 256 + (rows * 8 + 255) / 256 * 256 + rows * head_dim * 4;
}

template <typename T, int D>
int launch_tree(TreeParams p, hipStream_t s) {
  constexpr int kWaves = TreeTile<T, D, 8>::kWaves;
  int64_t wgs = p.num_work + (p.k_new ? (p.total_q + kWaves - 1) / kWaves : 0);
  if (wgs == 0) wgs = p.batch;  // pad rows only
  if (wgs > 0x7fffffff / 16) return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: too many rows");
  const dim3 grid((unsigned)wgs);
  if (p.tile_waves == 8) {
    tree_attention_kernel<T, D, 8><<<grid, 64 * kWaves, 0, s>>>(p);
  } else if constexpr (kWaves == 16) {
    tree_attention_kernel<T, D, 16><<<grid, 64 * kWaves, 0, s>>>(p);
  }
  const int rc = check_launch("paged_tree_attention");
  if (rc || p.whole) return rc;
  const int row_waves = (p.max_nodes * p.group + 15) / 16;
  const int64_t merges = (int64_t)p.batch * row_waves * p.num_kv_heads;
  if (merges > 0x7fffffff) return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: too many rows");
  // Several sets of waves where a sequence has many parts on average (one sequence, 16 nodes over 2k tokens, 17 parts:
  // 12 -> 5 us; 32 trees of 2 to 3 parts: 12 and 15).
  if (p.spans >= 8 * p.batch)
    tree_merge_kernel<T, D, 4><<<dim3((unsigned)merges), 1024, 0, s>>>(p, row_waves);
  else
    tree_merge_kernel<T, D, 1><<<dim3((unsigned)merges), 256, 0, s>>>(p, row_waves);
  return check_launch("paged_tree_attention merge");
}

template <typename T>
int launch_tree_dim(const TreeParams& p, int head_dim, hipStream_t s) {
  switch (head_dim) {
    case 64: return launch_tree<T, 64>(p, s);
    case 128: return launch_tree<T, 128>(p, s);
    default: return launch_tree<T, 256>(p, s);
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
  const int64_t n = tree_spans(batch, total_pages * page_size, rows, num_kv_heads, head_dim, dtype);
  return tree_bytes(batch, n, num_kv_heads, tree_rows(rows, head_dim, dtype), head_dim);
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
  p.page_div = Divisor::of(page_size);
  p.group_div = Divisor::of(group);
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.out = (char*)out;
  p.out_stride = out_stride * eb;
  p.k_new = (const char*)k_new;
  p.v_new = (const char*)v_new;
  p.k_new_stride = k_new_stride * eb;
  p.v_new_stride = v_new_stride * eb;
  p.max_nodes = max_q;
  const int64_t tile_rows = tree_rows(rows, head_dim, dtype);
  p.tile_waves = (int32_t)(tile_rows / 16);
  int64_t spans = batch * tree_tiles(rows, head_dim, dtype);
  p.whole = 1;
  if (workspace && total_q > 0) {
    int64_t n = tree_spans(batch, total_pages * page_size, rows, num_kv_heads, head_dim, dtype);
    while (n > 0 && tree_bytes(batch, n, num_kv_heads, tile_rows, head_dim) > workspace_bytes) --n;
    if (n > 0) {
      char* ws = (char*)(((uintptr_t)workspace + 255) / 256 * 256);  // (tree_bytes has room for this)
      const size_t part_rows = (size_t)n * num_kv_heads * 2 * tile_rows;
      p.whole = 0;
      p.ws_tag = (uint64_t*)ws;
      ws += 256;
      p.meta = (int4*)ws;
      ws += ((size_t)batch * 16 + 255) / 256 * 256;
      p.part_ml = (float2*)ws;
      ws += (part_rows * 8 + 255) / 256 * 256;
      p.part_o = (f32x4*)ws;
      spans = n;
    }
  }
  if (spans * num_kv_heads > 0x7fffffff / 8) return fail(NSLG_EUNSUPPORTED, "paged_tree_attention: too many rows");
  p.spans = (int32_t)spans;
  const int64_t work = total_q > 0 ? spans * num_kv_heads : 0;
  p.num_work = (int32_t)work;
  p.one_tile = tree_tiles(rows, head_dim, dtype) == 1;
  hipStream_t s = as_stream(stream);
  if (dtype == NSLG_F16) return launch_tree_dim<F16>(p, head_dim, s);
  if (dtype == NSLG_BF16) return launch_tree_dim<BF16>(p, head_dim, s);
  return launch_tree_dim<F32>(p, head_dim, s);
}
