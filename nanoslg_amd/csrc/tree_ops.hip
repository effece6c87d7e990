// What a step of speculative decoding needs besides its attention, for gfx950: the trees' ancestor masks and positions, the
// verification of the drafted tokens, and the move of the accepted nodes' K/V.
#include "nslg_common.h"

namespace nslg {
namespace {

constexpr int kTreeMaxNodes = 1024;

// ---- masks and positions ---------------------------------------------------------------
// One workgroup per tree: the parents in LDS, a thread a node. A node's ancestors have falling indices, so its
// words are built from the last to the first in one register. 3.4 us for 16 trees of 20 to 32 nodes, 3.6 for 256 of 100 to 256
// (1.8 MB): a launch and three dependent reads.
struct TreePlanParams {
  const int32_t* parents;
  const int32_t* qo_indptr;
  const int32_t* start;
  const int32_t* q_rows;
  int32_t grid_width;
  int64_t total_q;
  int32_t max_q;
  int32_t batch;
  uint32_t* mask;
  int32_t mask_words;
  int32_t* positions;
};

__global__ void __launch_bounds__(256) tree_plan_kernel(TreePlanParams p) {
  __shared__ int parent[kTreeMaxNodes];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int q0 = p.qo_indptr[b];
  const int n = (int)min((int64_t)min(max(p.qo_indptr[b + 1] - q0, 0), p.max_q), p.total_q - q0);
  for (int j = tid; j < n; j += 256) parent[j] = p.parents[q0 + j];
  const int64_t row0 = (int64_t)b * p.grid_width;
  int64_t at0 = 0;  // the grid row of node 0
  if (p.q_rows) {
    at0 = n > 0 ? (int64_t)p.q_rows[q0] : row0;
    for (int c = tid; c < p.grid_width; c += 256)
      if (row0 + c < at0 || row0 + c >= at0 + n) p.positions[row0 + c] = 0;
  }
  __syncthreads();
  const int start = p.start[b];
  for (int j = tid; j < n; j += 256) {
    uint32_t* row = p.mask + (int64_t)(q0 + j) * p.mask_words;
    int a = j, depth = 0;
    for (int w = p.mask_words - 1; w >= 0; --w) {
      uint32_t bits = 0;
      while (a >= 0 && a >> 5 == w) {
        bits |= 1u << (a & 31);
        const int up = parent[a];
        a = up < a ? up : -1;  // (an ancestor that does not lie before its child: a root)
        depth += a >= 0;
      }
      row[w] = bits;
    }
    const int64_t at = p.q_rows ? p.q_rows[q0 + j] : q0 + j;
    if (!p.q_rows || (at >= 0 && at < (int64_t)p.batch * p.grid_width)) p.positions[at] = start + depth;
  }
}

// ---- verification ----------------------------------------------------------------------
// At a node with target row p and draft row q, what is left of p once drawn children were rejected is, up to a factor,
// max(p - c q, 0): taking max(r / W - q, 0), W the sum of r, from r = max(p - c q, 0) leaves max(p - (c + W) q, 0) / W. So a
// rejection needs the sum of that at the new c and nothing else, and those sums, kept by pieces of kVerPiece tokens, are also
// what the next token is found from: its piece from their running sum, then the token inside it.
//
// Bound by latency, then by how fast a workgroup reads a row (0.5 MB at 128k tokens in fp32; one alone took 25 us of it). So
// `slices` workgroups take a sequence: each walks down from the root (64 nodes at a time, with the probabilities that
// their tests take already loaded) to the first sum that is wanted, and sums its slice of the row. The last one to be done goes
// on alone: in most trees it only has the next token to find. Sums and tests are in 64 bits: the order of adding
// decides no token.
//
// One tree of 26 nodes over 128k fp32 tokens 9.6 us, 64 drawn chains of 4 to 8 over them 18.6 (66 MB: 13 at a copy's
// rate), 16 drawn trees of 32 over 32k bf16 tokens 29.5: what the last workgroup rejects one after the other.
struct VerifyParams {
  const int32_t* tokens;
  const int32_t* parents;
  const int32_t* qo_indptr;
  const int32_t* q_rows;
  int64_t total_q;
  int32_t max_q;
  int32_t batch;
  int64_t rows;  // rows of the probabilities
  const char* target;
  int64_t target_stride;  // bytes
  const char* draft;
  int64_t draft_stride;
  int32_t vocab;
  const float* u_accept;
  const float* u_next;
  int32_t* path;
  int32_t* count;
  int32_t* next;
  int32_t slices;    // workgroups a sequence
  int32_t* arrived;  // [batch]: those done, 0 between calls (slices > 1)
  double* sums;      // [batch, pieces]
};

constexpr int kVerThreads = 1024;
constexpr int kVerWaves = kVerThreads / 64;
constexpr int kVerPiece = 256;       // tokens of a piece: a wave, four each
constexpr int kVerMaxPieces = 4096;  // (32 KB of LDS)
constexpr int kVerBatch = 8;         // pieces that a wave loads at a time

template <typename T>
__device__ inline float prob_of(const char* row, int i) {
  if constexpr (T::kDtype == NSLG_F32)
    return reinterpret_cast<const float*>(row)[i];
  else
    return T::to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
}

struct VF32 {
  static constexpr int kDtype = NSLG_F32;
};

// Tokens i .. i + 3 of a row, 4 elements aligned.
template <typename T>
__device__ inline void load4(const char* row, int i, float (&x)[4]) {
  if constexpr (T::kDtype == NSLG_F32) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(row + 4 * (int64_t)i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = v[e];
  } else {
    const u16x4 v = *reinterpret_cast<const u16x4*>(row + 2 * (int64_t)i);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = T::to_f32(v[e]);
  }
}

// The weight that is left of p at c: p - c q, not below 0; what is no number counts nothing.
template <bool kDraft>
__device__ inline double weight(float p, float q, double c) {
  double x = (double)p;
  if constexpr (kDraft)
    if (c != 0.0) x -= c * (double)q;
  return x > 0.0 && x < INFINITY ? x : 0.0;
}

__device__ inline double f64_of(unsigned lo, unsigned hi) { return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo); }
__device__ inline unsigned lo_of(double v) { return (unsigned)__builtin_bit_cast(uint64_t, v); }
__device__ inline unsigned hi_of(double v) { return (unsigned)(__builtin_bit_cast(uint64_t, v) >> 32); }
template <int kCtrl>
__device__ inline double dpp_f64(double x) {
  return f64_of(__builtin_amdgcn_mov_dpp(lo_of(x), kCtrl, 0xf, 0xf, false), __builtin_amdgcn_mov_dpp(hi_of(x), kCtrl, 0xf, 0xf, false));
}
// Two sums a step on their way: of x in even rows of 16 lanes and of y in odd ones; of x in the lower half of the wave and
// of y in the upper.
__device__ inline double join16_f64(double x, double y) {
  const auto a = __builtin_amdgcn_permlane16_swap(lo_of(x), lo_of(y), false, false), c = __builtin_amdgcn_permlane16_swap(hi_of(x), hi_of(y), false, false);
  return f64_of(a[0], c[0]) + f64_of(a[1], c[1]);
}
__device__ inline double join32_f64(double x, double y) {
  const auto a = __builtin_amdgcn_permlane32_swap(lo_of(x), lo_of(y), false, false), c = __builtin_amdgcn_permlane32_swap(hi_of(x), hi_of(y), false, false);
  return f64_of(a[0], c[0]) + f64_of(a[1], c[1]);
}

// Sum over the wave's lanes: rotations within 16 lanes, then the row swaps.
__device__ inline double wave_sum_f64(double x) {
  x += dpp_f64<0x128>(x);  // row_ror:8
  x += dpp_f64<0x124>(x);  // row_ror:4
  x += dpp_f64<0x122>(x);  // row_ror:2
  x += dpp_f64<0x121>(x);  // row_ror:1
  x = join16_f64(x, x);
  return join32_f64(x, x);
}

// Eight sums over the wave's lanes, each step joining two of them (10 additions where eight sums by themselves take 48): the lanes
// of each eight have the sum of x[sum8_of(lane)].
__device__ inline int sum8_of(int lane) { return (lane >> 1 & 4) | (lane >> 3 & 2) | (lane >> 5 & 1); }
__device__ inline double wave_sum8_f64(const double (&x)[8]) {
  const double a = join16_f64(join32_f64(x[0], x[1]), join32_f64(x[2], x[3]));
  const double b = join16_f64(join32_f64(x[4], x[5]), join32_f64(x[6], x[7]));
  const bool upper = threadIdx.x & 8;
  double s = (upper ? b : a) + dpp_f64<0x128>(upper ? a : b);  // row_ror:8
  s += dpp_f64<0xb1>(s);                                       // quad_perm 1 0 3 2
  s += dpp_f64<0x4e>(s);                                       // quad_perm 2 3 0 1
  return s + dpp_f64<0x141>(s);                                // row_half_mirror
}
__device__ inline double wave_scan_f64(double x) {  // sum over the lanes up to one's own
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __shfl_up(x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}

template <typename T, bool kDraft>
__global__ void __launch_bounds__(kVerThreads) tree_verify_kernel(VerifyParams p) {
  __shared__ double piece[kVerMaxPieces];
  __shared__ int rejected[kDraft ? 1 : kTreeMaxNodes];  // tokens rejected at the present node
  __shared__ int path_lds[kTreeMaxNodes];
  __shared__ int s_done, s_row, s_rejects, s_next;
  __shared__ double s_c;

  const int b = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int q0 = p.qo_indptr[b];
  const int n = (int)min((int64_t)min(max(p.qo_indptr[b + 1] - q0, 0), p.max_q), p.total_q - q0);
  int32_t* path = p.path + (int64_t)b * p.max_q;
  if (n <= 0) {  // no tree: nothing accepted, no token
    if (slice == 0) {
      for (int i = tid; i < p.max_q; i += kVerThreads) path[i] = -1;
      if (tid == 0) p.count[b] = 0, p.next[b] = -1;
    }
    return;
  }
  auto row_of = [&](int node) -> int64_t {
    const int64_t at = p.q_rows ? p.q_rows[q0 + node] : q0 + node;
    return at < 0 ? 0 : (at >= p.rows ? p.rows - 1 : at);
  };
  // The state of the walk (wave 0, uniform): node, next child to look at, accepted nodes, rejections at the node (tokens
  // given), c and the sum W of what is left (tokens drawn).
  int cur = 0, from = 1, count = 1, rejects = 0;
  double c = 0.0, W = 1.0;
  // the lane's node of the 64 from `loaded` on: parent, token, number, the probabilities of its test
  int loaded = -1, up = -2, x = -1;
  float u = 0.f;
  bool tried = false;
  double pj = 0.0, qj = 1.0;
  // Down to the first sum that is wanted, or to the end.
  auto walk = [&]() {
    bool wanted = false;
    while (from < n && !wanted) {
      const int base = from & ~63;
      const int j = base + lane;
      if (base != loaded) {
        loaded = base;
        up = j < n ? p.parents[q0 + j] : -2;
        x = j < n ? p.tokens[q0 + j] : -1;
        u = j < n ? p.u_accept[q0 + j] : 0.f;
        tried = up >= 0 && up < j && x >= 0 && x < p.vocab;
        if (tried) {
          const int64_t at = row_of(up);
          pj = (double)prob_of<T>(p.target + at * p.target_stride, x);
          if constexpr (kDraft) qj = (double)prob_of<T>(p.draft + at * p.draft_stride, x);
        }
      }
      while (!wanted) {
        const unsigned long long m = __ballot(j >= from && j < n && up == cur);
        if (m == 0) {
          from = base + 64;
          break;
        }
        const int src = __ffsll((long long)m) - 1;
        from = base + src + 1;
        const bool ok_token = __shfl((int)tried, src, 64);
        const int xs = __shfl(x, src, 64);
        double left = __shfl(pj, src, 64);
        const double q = __shfl(qj, src, 64);
        const double us = (double)__shfl(u, src, 64);
        if constexpr (kDraft) {
          if (c != 0.0) left -= c * q;
        } else {
          bool again = false;
          for (int i = lane; i < rejects; i += 64) again |= rejected[i] == xs;
          if (__ballot(again)) left = 0.0;
        }
        left = ok_token && left > 0.0 && left < INFINITY ? left : 0.0;
        if (left > 0.0 && us * W * q < left) {  // accepted
          cur = base + src;
          if (lane == 0) path_lds[count] = cur;
          ++count;
          c = 0.0, W = 1.0, rejects = 0;
          continue;
        }
        if constexpr (kDraft) {
          if (W > 0.0) c += W, wanted = true;
        } else {
          W -= left;
          if (left > 0.0) {
            if (lane == 0) rejected[rejects] = xs;
            ++rejects;
            // (one wave's LDS operations complete in order; the fence is for the compiler)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          }
        }
      }
    }
    if (lane == 0) s_done = !wanted, s_row = cur, s_c = c, s_rejects = rejects;
  };
  // The sums of pieces g0 .. g1 - 1 of what is left of a row, the workgroup's waves kVerBatch pieces at a time.
  auto sum_pieces = [&](int row, double cc, int gone, int g0, int g1) {
    const int64_t at = row_of(row);
    const char* prow = p.target + at * p.target_stride;
    const char* qrow = kDraft ? p.draft + at * p.draft_stride : nullptr;
    const bool need_q = kDraft && cc != 0.0;
    const bool wide = ((uintptr_t)prow | (uintptr_t)(need_q ? qrow : prow)) % (T::kDtype == NSLG_F32 ? 16 : 8) == 0;
    for (int g = g0 + wave * kVerBatch; g < g1; g += kVerWaves * kVerBatch) {
      // (a lane takes four tokens in a row of each piece: one load where the rows allow it)
      float pv[kVerBatch][4], qv[kVerBatch][4];
#pragma unroll
      for (int k = 0; k < kVerBatch; ++k) {
        const int i = (g + k) * kVerPiece + 4 * lane;
        if (wide && i + 4 <= p.vocab) {
          load4<T>(prow, i, pv[k]);
          if (need_q) load4<T>(qrow, i, qv[k]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pv[k][e] = prob_of<T>(prow, min(i + e, p.vocab - 1));
            if (need_q) qv[k][e] = prob_of<T>(qrow, min(i + e, p.vocab - 1));
          }
        }
      }
      double x[kVerBatch];
#pragma unroll
      for (int k = 0; k < kVerBatch; ++k) {
        x[k] = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = (g + k) * kVerPiece + 4 * lane + e;
          double v = i < p.vocab ? weight<kDraft>(pv[k][e], need_q ? qv[k][e] : 0.f, cc) : 0.0;
          if constexpr (!kDraft)
            for (int z = 0; z < gone; ++z) v = rejected[z] == i ? 0.0 : v;
          x[k] += v;
        }
      }
      static_assert(kVerBatch == 8);
      const double sum = wave_sum8_f64(x);
      const int k = sum8_of(lane);
      if (lane % 8 == 0 && g + k < g1) piece[g + k] = sum;
    }
  };
  const int pieces = (p.vocab + kVerPiece - 1) / kVerPiece;

  if (tid == 0) path_lds[0] = 0;
  if (wave == 0) walk();
  __syncthreads();
  const int each = ((pieces + p.slices - 1) / p.slices + kVerBatch - 1) / kVerBatch * kVerBatch;
  const int g0 = min(slice * each, pieces), g1 = min(g0 + each, pieces);
  sum_pieces(s_row, s_c, s_rejects, g0, g1);
  __syncthreads();
  if (p.slices > 1) {
    // The sums go past the caches of the workgroup's XCD (stores and loads at the device's scope), and each wave's are there
    // before the workgroup counts itself in: the last one sees them all. (A fence at that scope in each workgroup, which
    // writes the XCD's cache back, took 64 sequences from 27 to 144 us.)
    double* sums = p.sums + (int64_t)b * pieces;
    for (int g = g0 + tid; g < g1; g += kVerThreads) __hip_atomic_store(&sums[g], piece[g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) s_next = __hip_atomic_fetch_add(&p.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_next != p.slices - 1) return;
    if (tid == 0) __hip_atomic_store(&p.arrived[b], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int g = tid; g < pieces; g += kVerThreads)
      piece[g] = __hip_atomic_load(&sums[g], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  }
  // The sequence's last workgroup. The pieces are those of row s_row at s_c; a lane takes `run` of them in turn.
  const int run = (pieces + 63) / 64;
  while (true) {
    const int done = s_done, row = s_row, gone = s_rejects;
    const double at_c = s_c;
    double mine = 0.0;
    if (wave == 0) {
      for (int g = lane * run; g < min((lane + 1) * run, pieces); ++g) mine += piece[g];
      W = wave_sum_f64(mine);
    }
    __syncthreads();  // the state is read
    if (!done) {
      if (wave == 0) walk();
      __syncthreads();
      if (s_row != row || s_c != at_c) {
        sum_pieces(s_row, s_c, s_rejects, 0, pieces);
        __syncthreads();
      }
      continue;
    }
    // the next token
    int found = -1;
    if (wave == 0) {
      if (W > 0.0) {
        const double goal = (double)p.u_next[b] * W;
        const int64_t at = row_of(row);
        const char* prow = p.target + at * p.target_stride;
        const char* qrow = kDraft ? p.draft + at * p.draft_stride : nullptr;
        const double incl = wave_scan_f64(mine);
        // the lane whose pieces the goal lies in (the last one with any weight where a rounding leaves it unreached)
        const unsigned long long hit = __ballot(incl > goal && mine > 0.0), some = __ballot(mine > 0.0);
        const int src = hit ? __ffsll((long long)hit) - 1 : 63 - __clzll((long long)some);
        double base = __shfl(incl - mine, src, 64);
        int g = -1;
        double g_base = 0.0;
        for (int k = src * run; k < min((src + 1) * run, pieces); ++k) {
          const double x = piece[k];
          if (x > 0.0) g = k, g_base = base;
          base += x;
          if (x > 0.0 && base > goal) break;
        }
        auto left_of = [&](int i) -> double {
          if (i >= p.vocab) return 0.0;
          if constexpr (!kDraft)
            for (int z = 0; z < gone; ++z)
              if (rejected[z] == i) return 0.0;
          return weight<kDraft>(prob_of<T>(prow, i), kDraft && at_c != 0.0 ? prob_of<T>(qrow, i) : 0.f, at_c);
        };
        double v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = left_of(g * kVerPiece + 64 * e + lane);
        int last = -1;
        for (int e = 0; e < 4 && found < 0; ++e) {
          const double sum = wave_scan_f64(v[e]);
          const unsigned long long at_goal = __ballot(g_base + sum > goal && v[e] > 0.0), any = __ballot(v[e] > 0.0);
          if (any) last = g * kVerPiece + 64 * e + 63 - __clzll((long long)any);
          if (at_goal) found = g * kVerPiece + 64 * e + __ffsll((long long)at_goal) - 1;
          g_base += __shfl(sum, 63, 64);
        }
        if (found < 0) found = last;
      }
      if (lane == 0) s_next = found;
    }
    __syncthreads();
    if (s_next >= 0 || (at_c == 0.0 && gone == 0)) break;
    // rejections have left nothing of the row: from the row as it is
    if (tid == 0) s_c = 0.0, s_rejects = 0;
    __syncthreads();
    sum_pieces(row, 0.0, 0, 0, pieces);
    __syncthreads();
  }
  if (wave == 0) {
    for (int i = lane; i < p.max_q; i += 64) path[i] = i < count ? path_lds[i] : -1;
    if (lane == 0) p.count[b] = count, p.next[b] = s_next;
  }
}

// ---- the accepted nodes' K/V -------------------------------------------------------------
// A path's nodes have rising indices, so node path[i] >= i: reading eight of them ahead of the eight writes and
// going up overwrites nothing that is still to be read. Workgroup: (layer and K | V, sequence); a thread keeps its
// 16-byte word of the rows. One sequence in 32 layers 3.9 us, 64 in 16 layers 8.1: the reads' latency.
struct MoveParams {
  char* k_pool;
  char* v_pool;
  int64_t num_pages;
  int32_t page_size;
  int64_t row_bytes;
  const int32_t* path;
  int32_t path_stride;
  const int32_t* count;
  const int32_t* qo_indptr;
  const int32_t* indptr;
  const int32_t* indices;
  const int32_t* last_len;
};

template <typename V>
__global__ void __launch_bounds__(256) tree_move_kernel(MoveParams p) {
  __shared__ int64_t src_lds[8], dst_lds[8];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int layer = blockIdx.x >> 1;
  const int n = max(p.qo_indptr[b + 1] - p.qo_indptr[b], 0);
  const int count = p.count[b];
  if (count > min(n, p.path_stride)) return;
  const int32_t* path = p.path + (int64_t)b * p.path_stride;
  // a path: rising nodes of the tree
  bool ok = true;
  for (int i = tid; i < count; i += 256) {
    const int a = path[i];
    ok &= a >= 0 && a < n && (i == 0 || a > path[i - 1]);
  }
  if (__syncthreads_or(!ok)) return;
  const int np = p.indptr[b + 1] - p.indptr[b];
  int lpl = p.last_len[b];
  lpl = lpl < 1 ? 1 : (lpl > p.page_size ? p.page_size : lpl);
  const int len = np > 0 ? (np - 1) * p.page_size + lpl : 0;
  const int start = len - n;
  if (start < 0) return;
  const int32_t* idx = p.indices + p.indptr[b];
  char* pool = (blockIdx.x & 1 ? p.v_pool : p.k_pool) + (int64_t)layer * p.num_pages * p.page_size * p.row_bytes;
  auto slot = [&](int node) -> int64_t {
    const int pos = start + node;
    const int pid = idx[pos / p.page_size];
    return pid < 0 || (int64_t)pid >= p.num_pages ? -1 : (int64_t)pid * p.page_size + pos % p.page_size;
  };
  const int vecs = (int)(p.row_bytes / (int64_t)sizeof(V));
  for (int i0 = 0; i0 < count; i0 += 8) {
    if (tid < 8) {
      const int i = i0 + tid;
      int64_t s = -1, d = -1;
      if (i < count && path[i] != i) s = slot(path[i]), d = slot(i);
      src_lds[tid] = s < 0 || d < 0 ? -1 : s;
      dst_lds[tid] = d;
    }
    __syncthreads();
    for (int w = tid; w < vecs; w += 256) {
      V x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (src_lds[u] >= 0) x[u] = reinterpret_cast<const V*>(pool + src_lds[u] * p.row_bytes)[w];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (src_lds[u] >= 0) reinterpret_cast<V*>(pool + dst_lds[u] * p.row_bytes)[w] = x[u];
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace nslg

using namespace nslg;

extern "C" int nslg_tree_plan(const int32_t* parents, const int32_t* qo_indptr, const int32_t* start,
                              const int32_t* q_rows, int32_t grid_width, int64_t total_q, int32_t max_q, int32_t batch,
                              uint32_t* mask, int32_t mask_words, int32_t* positions, nslg_stream_t stream) {
  if (batch < 0 || total_q < 0 || max_q < 0 || (int64_t)max_q * batch < total_q)
    return fail(NSLG_EINVAL, "tree_plan: %lld nodes in %d trees of at most %d", (long long)total_q, batch, max_q);
  if (max_q > kTreeMaxNodes) return fail(NSLG_EUNSUPPORTED, "tree_plan: trees of up to %d nodes (%d)", kTreeMaxNodes, max_q);
  if (q_rows && (grid_width < 1 || (int64_t)batch * grid_width > 0x7fffffff || total_q > (int64_t)batch * grid_width))
    return fail(NSLG_EINVAL, "tree_plan: grid of %d x %d rows for %lld nodes", batch, grid_width, (long long)total_q);
  if (batch == 0 || (total_q == 0 && !q_rows)) return NSLG_OK;
  if (mask_words < (max_q + 31) / 32) return fail(NSLG_EINVAL, "tree_plan: masks of %d words for %d nodes", mask_words, max_q);
  if (!qo_indptr || !start || !positions || (total_q > 0 && (!parents || !mask)))
    return fail(NSLG_EINVAL, "tree_plan: null pointer");
  TreePlanParams p = {parents, qo_indptr, start, q_rows, grid_width, total_q, max_q, batch, mask, mask_words, positions};
  tree_plan_kernel<<<dim3((unsigned)batch), 256, 0, as_stream(stream)>>>(p);
  return check_launch("tree_plan");
}

// Workgroups a sequence: of 16 pieces (4096 tokens) each at least, and as many as the CUs take at once, one each (twice as
// many: 64 chains over 128k tokens 25.5 us, now 18.6).
static int verify_slices(int32_t batch, int32_t vocab) {
  const int by_row = (vocab + 16 * kVerPiece - 1) / (16 * kVerPiece);
  const int by_cus = 256 / batch;
  const int n = by_row < by_cus ? by_row : by_cus;
  return n < 1 ? 1 : n;
}
// The counters (slices > 1: at most 128 sequences) before the sums, at an offset that does not depend on the call: a
// later one of another batch finds its counters zero.
constexpr int kVerHead = 1024;
static size_t verify_bytes(int32_t batch, int32_t vocab) {
  return kVerHead + (size_t)batch * ((vocab + kVerPiece - 1) / kVerPiece) * 8;
}

extern "C" size_t nslg_verify_tree_workspace_size(int32_t batch, int32_t vocab) {
  if (batch <= 0 || vocab <= 0 || vocab > kVerMaxPieces * kVerPiece || verify_slices(batch, vocab) == 1) return 0;
  return verify_bytes(batch, vocab);
}

extern "C" int nslg_verify_tree(const int32_t* tokens, const int32_t* parents, const int32_t* qo_indptr,
                                const int32_t* q_rows, int64_t total_q, int32_t max_q, int32_t batch,
                                const void* target_probs, int64_t target_stride, const void* draft_probs,
                                int64_t draft_stride, int64_t num_rows, int32_t vocab, int32_t dtype,
                                const float* u_accept, const float* u_next, int32_t* path, int32_t* count,
                                int32_t* next_token, void* workspace, size_t workspace_bytes, nslg_stream_t stream) {
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(NSLG_EINVAL, "verify_tree: bad dtype %d", dtype);
  if (batch < 0 || total_q < 0 || max_q < 0 || (int64_t)max_q * batch < total_q)
    return fail(NSLG_EINVAL, "verify_tree: %lld nodes in %d trees of at most %d", (long long)total_q, batch, max_q);
  if (max_q > kTreeMaxNodes)
    return fail(NSLG_EUNSUPPORTED, "verify_tree: trees of up to %d nodes (%d)", kTreeMaxNodes, max_q);
  if (vocab < 1 || num_rows < 0 || (num_rows < 1 && total_q > 0) || (!q_rows && num_rows < total_q))
    return fail(NSLG_EINVAL, "verify_tree: %lld rows of %d probabilities for %lld nodes", (long long)num_rows, vocab,
                (long long)total_q);
  if (batch == 0) return NSLG_OK;
  if (vocab > kVerMaxPieces * kVerPiece)
    return fail(NSLG_EUNSUPPORTED, "verify_tree: vocabularies of up to %d tokens (%d)", kVerMaxPieces * kVerPiece, vocab);
  if (!qo_indptr || !count || !next_token || !u_next || (max_q > 0 && !path) ||
      (total_q > 0 && (!tokens || !parents || !target_probs || !u_accept)))
    return fail(NSLG_EINVAL, "verify_tree: null pointer");
  if (target_stride < vocab || (draft_probs && draft_stride < vocab))
    return fail(NSLG_EINVAL, "verify_tree: row stride smaller than the vocabulary");
  if (((uintptr_t)target_probs | (uintptr_t)draft_probs) % eb) return fail(NSLG_EINVAL, "verify_tree: unaligned rows");
  if (batch > 65535) return fail(NSLG_EUNSUPPORTED, "verify_tree: batches of up to 65535 (%d)", batch);
  if ((uintptr_t)workspace & 7) return fail(NSLG_EINVAL, "verify_tree: the workspace must be 8-byte aligned");
  VerifyParams p = {tokens, parents, qo_indptr, q_rows, total_q, max_q, batch, num_rows,
                    (const char*)target_probs, target_stride * eb, (const char*)draft_probs, draft_stride * eb, vocab,
                    u_accept, u_next, path, count, next_token, 1, nullptr, nullptr};
  if (workspace && workspace_bytes >= verify_bytes(batch, vocab)) {
    p.slices = verify_slices(batch, vocab);
    p.arrived = (int32_t*)workspace;
    p.sums = (double*)((char*)workspace + kVerHead);
  }
  hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)p.slices, (unsigned)batch);
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (draft_probs)
      tree_verify_kernel<T, true><<<grid, kVerThreads, 0, s>>>(p);
    else
      tree_verify_kernel<T, false><<<grid, kVerThreads, 0, s>>>(p);
  };
  if (dtype == NSLG_F16)
    launch(F16());
  else if (dtype == NSLG_BF16)
    launch(BF16());
  else
    launch(VF32());
  return check_launch("verify_tree");
}

extern "C" int nslg_move_accepted(void* k_pool, void* v_pool, int32_t num_layers, int64_t num_pages, int32_t page_size,
                                  int32_t num_kv_heads, int32_t head_dim, int32_t dtype, const int32_t* path,
                                  int32_t path_stride, const int32_t* count, const int32_t* qo_indptr,
                                  const int32_t* kv_indptr, const int32_t* kv_indices, const int32_t* kv_last_page_len,
                                  int32_t batch, nslg_stream_t stream) {
  const int eb = elem_bytes(dtype);
  if (!eb) return fail(NSLG_EINVAL, "move_accepted: bad dtype %d", dtype);
  if (num_layers <= 0 || num_pages <= 0 || page_size <= 0 || num_kv_heads <= 0 || head_dim <= 0 || batch < 0 || path_stride < 0)
    return fail(NSLG_EINVAL, "move_accepted: bad sizes");
  if (batch == 0 || path_stride == 0) return NSLG_OK;
  if (!k_pool || !v_pool || !path || !count || !qo_indptr || !kv_indptr || !kv_indices || !kv_last_page_len)
    return fail(NSLG_EINVAL, "move_accepted: null pointer");
  if (batch > 65535) return fail(NSLG_EUNSUPPORTED, "move_accepted: batches of up to 65535 (%d)", batch);
  if (num_layers > (1 << 24)) return fail(NSLG_EUNSUPPORTED, "move_accepted: too many layers");
  if (num_pages * (int64_t)page_size >= ((int64_t)1 << 31))
    return fail(NSLG_EUNSUPPORTED, "move_accepted: pool has >= 2^31 token slots");
  const int64_t row_bytes = (int64_t)num_kv_heads * head_dim * eb;
  MoveParams p = {(char*)k_pool, (char*)v_pool, num_pages, page_size, row_bytes, path, path_stride, count,
                  qo_indptr, kv_indptr, kv_indices, kv_last_page_len};
  const dim3 grid((unsigned)(2 * num_layers), (unsigned)batch);
  hipStream_t s = as_stream(stream);
  const uintptr_t all = (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)row_bytes;
  if (all % 16 == 0)
    tree_move_kernel<u32x4><<<grid, 256, 0, s>>>(p);
  else if (all % 4 == 0)
    tree_move_kernel<uint32_t><<<grid, 256, 0, s>>>(p);
  else
    tree_move_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
  return check_launch("move_accepted");
}
