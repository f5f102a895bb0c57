// Everything around the MXFP4 products: group tables, the hi/lo split of bf16
// activations into the product's row order, and the combine of the routed FFN.
#include <limits.h>

#include "common.cuh"
#include "mxfp4.cuh"

namespace dsmoe {
namespace mx {
namespace {

// Inclusive scan over the block (blockDim.x == kMaxGroups): sum or maximum.
template <bool MAX>
__device__ __forceinline__ int block_scan(int v, int* buf) {
  const int i = threadIdx.x;
  buf[i] = v;
  __syncthreads();
  for (int o = 1; o < kMaxGroups; o <<= 1) {
    const int a = i >= o ? buf[i - o] : (MAX ? INT_MIN : 0);
    __syncthreads();
    buf[i] = MAX ? max(buf[i], a) : buf[i] + a;
    __syncthreads();
  }
  const int r = buf[i];
  __syncthreads();
  return r;
}

// Offsets are clamped to [0, rows] and made non-decreasing, so that segments
// never overlap or leave the rows whatever the offsets hold; a table that
// needed it is reported in *status.
__global__ void __launch_bounds__(kMaxGroups) segments_kernel(const int32_t* __restrict__ offsets, int n, int rows,
                                                              int tile, int32_t* __restrict__ counts,
                                                              int32_t* __restrict__ row_start,
                                                              int32_t* __restrict__ tile_start,
                                                              int32_t* __restrict__ next, int* __restrict__ status) {
  __shared__ int buf[kMaxGroups];
  launch_dependents();
  const int i = threadIdx.x;
  if (i < 2) next[i] = 0;
  const int lo = i < n ? offsets[i] : 0, hi = i < n ? offsets[i + 1] : 0;
  if (i < n && (lo < 0 || hi < lo || hi > rows)) atomicCAS(status, 0, kDevBadCount);
  const int first = min(max(offsets[0], 0), rows);
  const int end = max(first, block_scan<true>(min(max(hi, 0), rows), buf));
  // start = the previous group's end
  buf[i] = end;
  __syncthreads();
  const int start = i ? buf[i - 1] : first;
  __syncthreads();
  const int c = i < n ? end - start : 0;
  const int nt = (c + tile - 1) / tile;
  const int tiles = block_scan<false>(nt, buf);
  if (i < n) {
    counts[i] = c;
    row_start[i] = start;
    tile_start[i] = tiles - nt;
    if (i == n - 1) tile_start[n] = tiles;
  }
}

// Stable counting sort of the (token, k) pairs by expert, by one cluster of
// CTAs: each warp owns a contiguous range of pairs, counts it, and after the
// scans over warps, CTAs (through shared memory) and groups walks it again in
// order; lanes of one step that hold the same expert are ranked by lane. The
// row of a pair therefore depends on the routing only. 32768 pairs: 15.5 us,
// latency of the chain of scans; one CTA took 63.
constexpr int kPlanWarps = 32;
constexpr int kPlanCtas = 8;

__device__ __forceinline__ int load_peer(const int* p, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(1024) route_plan_kernel(const int64_t* __restrict__ idx, int T, int top_k,
                                                          int n_routed, int shared, int tile,
                                                          int32_t* __restrict__ counts, int32_t* __restrict__ row_start,
                                                          int32_t* __restrict__ tile_start, int32_t* __restrict__ next,
                                                          int32_t* __restrict__ pos) {
  extern __shared__ int hist[];  // [kPlanWarps][n_routed]
  __shared__ int s_total[kMaxGroups];  // this CTA's pairs per expert
  __shared__ int s_sum[2][kMaxGroups / 32];
  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = gridDim.x, me = blockIdx.x;  // the grid is one cluster
  const int pairs = T * top_k;
  const int per = ((pairs + kPlanWarps * ctas - 1) / (kPlanWarps * ctas) + 31) & ~31;
  const int p0 = min(pairs, (me * kPlanWarps + warp) * per), p1 = min(pairs, p0 + per);
  for (int i = threadIdx.x; i < kPlanWarps * n_routed; i += 1024) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * n_routed;
  // expert of pair p, -1 past the warp's pairs or for an id outside; batches of
  // 8 x 32 pairs are loaded together
  constexpr int B = 8;
  auto expert = [&](int p) {
    if (p >= p1) return -1;
    const int64_t e = __ldg(idx + p);
    return e >= 0 && e < n_routed ? static_cast<int>(e) : -1;
  };
  for (int p = p0; p < p1; p += 32 * B) {
    int e[B];
#pragma unroll
    for (int j = 0; j < B; ++j) e[j] = expert(p + 32 * j + lane);
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (e[j] >= 0) atomicAdd(&mine[e[j]], 1);
  }
  __syncthreads();
  // per expert: the pairs of earlier warps, then of earlier CTAs
  const int g = threadIdx.x;  // group
  const int ex = g - shared;  // its expert
  const bool routed = ex >= 0 && ex < n_routed;
  int own = 0;
  if (routed) {
    for (int w = 0; w < kPlanWarps; ++w) {
      int* h = &hist[w * n_routed + ex];
      const int n = *h;
      *h = own;
      own += n;
    }
    s_total[ex] = own;
  }
  int c = g < shared ? T : own, before = 0;
  if (ctas > 1) {
    cluster_sync();
    if (routed) {
      c = 0;
      for (int r = 0; r < ctas; ++r) {
        const int n = r == me ? own : load_peer(&s_total[ex], r);
        if (r < me) before += n;
        c += n;
      }
    }
    cluster_sync();  // no CTA leaves, or reuses s_total, while it is read
  }
  // scans of rows and token tiles over the groups (the first kMaxGroups threads)
  const int nt = (c + tile - 1) / tile;
  int rows = c, tiles = nt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, rows, o), b = __shfl_up_sync(0xffffffffu, tiles, o);
    if (lane >= o) rows += a, tiles += b;
  }
  if (lane == 31 && warp < kMaxGroups / 32) s_sum[0][warp] = rows, s_sum[1][warp] = tiles;
  __syncthreads();
  for (int w = 0; w < min(warp, kMaxGroups / 32); ++w) rows += s_sum[0][w], tiles += s_sum[1][w];
  const int groups = n_routed + shared;
  if (g < groups) {
    const int start = rows - c;
    if (me == 0) {
      counts[g] = c;
      row_start[g] = start;
      tile_start[g] = tiles - nt;
      if (g == groups - 1) tile_start[groups] = tiles;
    }
    if (routed)
      for (int w = 0; w < kPlanWarps; ++w) hist[w * n_routed + ex] += start + before;
  }
  if (me == 0 && threadIdx.x < 2) next[threadIdx.x] = 0;
  __syncthreads();
  for (int p = p0; p < p1; p += 32 * B) {  // warp-uniform
    int e[B];
#pragma unroll
    for (int j = 0; j < B; ++j) e[j] = expert(p + 32 * j + lane);
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int q = p + 32 * j + lane;
      const unsigned same = __match_any_sync(0xffffffffu, e[j]);
      const int rank = __popc(same & ((1u << lane) - 1));
      const int base = e[j] >= 0 ? mine[e[j]] : 0;
      __syncwarp();
      if (e[j] >= 0 && rank == 0) mine[e[j]] = base + __popc(same);
      __syncwarp();
      if (q < p1) pos[q] = e[j] >= 0 ? base + rank : -1;
    }
  }
}

// Where row r of a product's rows keeps its scale word of K block kb: hi
// columns, and lo columns where hi and lo are side by side (lo_word < 0: not).
struct SfSpot {
  long long hi, lo;  // word indexes at kb = 0; a K block further is `step` words on
};
template <int TILE>
__device__ __forceinline__ SfSpot sf_spot(int tile0, int count, int local, int KB) {
  const int t = local / TILE, c = local - t * TILE;
  const int n = side_by_side(TILE, min(TILE, count - t * TILE));
  const long long base = static_cast<long long>(tile0 + t) * KB * tile_atoms(TILE) * 128;
  auto word = [](int col) { return (col >> 7) * 128 + (col & 31) * 4 + ((col >> 5) & 3); };
  return {base + word(c), n ? base + word(c + n) : -1};
}

// Split kernels: blocks of kSplitThreads, 16 columns of a row per thread.
constexpr int kSplitThreads = 128;
constexpr int kSplitCols = kSplitThreads * 16;

// This thread's 16 columns of a row (zero past its end): block y of the grid
// has columns kSplitCols * y and up.
__device__ __forceinline__ Cols load_cols(const __nv_bfloat16* row, int K) {
  const int col = blockIdx.y * kSplitCols + threadIdx.x * 16;
  Cols c{};
  if (col < K) {
    const uint4* p = reinterpret_cast<const uint4*>(row + col);
    c.a = __ldg(p);
    c.b = __ldg(p + 1);
  }
  return c;
}

// Splits the row and stores it, with its scale words, at n rows. 2 threads
// share a 32-number block, 8 a K block's scale word.
__device__ __forceinline__ void split_row(const Cols& q, int K, int P, int n, const int* s_row, const SfSpot* s_spot,
                                          int atoms, uint8_t* __restrict__ xq, uint8_t* __restrict__ sf) {
  const int tid = threadIdx.x;
  const int col = blockIdx.y * kSplitCols + tid * 16;
  const bool in = col < K;  // K is a multiple of 128: 8 threads of a K block are in or out together
  uint32_t hw[4], lw[4], word;
  split_cols(q, hw, lw, word);
  if (!in) return;
  uint32_t* s32 = reinterpret_cast<uint32_t*>(sf) + static_cast<long long>(col >> 7) * atoms * 128;
  const size_t lo_rows = static_cast<size_t>(P) * K;
  for (int r = 0; r < n; ++r) {
    const int row = s_row[r];
    if (row < 0) continue;
    uint8_t* dst = xq + static_cast<size_t>(row) * K + col;
    *reinterpret_cast<uint4*>(dst) = make_uint4(hw[0], hw[1], hw[2], hw[3]);
    *reinterpret_cast<uint4*>(dst + lo_rows) = make_uint4(lw[0], lw[1], lw[2], lw[3]);
    if ((tid & 7) == 0) {
      const SfSpot at = s_spot[r];
      s32[at.hi] = word;
      if (at.lo >= 0) s32[at.lo] = word;
    }
  }
}

constexpr int MAXR = 9;  // rows of a token: the shared expert's and top_k <= 8

// One block: kSplitCols columns of R rows (tokens), their loads in flight together.
// The place of a row is found by one thread each: for a routing the group is
// known from idx, for segments it is searched in a shared-memory copy of their
// starts (nine dependent global loads took twice as long as the split itself:
// 322 us for 32768 rows of 7168; 165 us now, 5.7 TB/s of what is read and written).
template <int TILE, int R>
__global__ void __launch_bounds__(kSplitThreads) split_kernel(const __nv_bfloat16* __restrict__ x, long long row_stride, int T,
                                                    int K, const Groups g, const int64_t* __restrict__ idx,
                                                    const int32_t* pos, int top_k, int shared, int P,
                                                    uint8_t* __restrict__ xq, uint8_t* __restrict__ sf,
                                                    __nv_bfloat16* __restrict__ zero_out, int M) {
  const int t0 = blockIdx.x * R;
  const int tid = threadIdx.x;
  const int KB = K / 128;
  launch_dependents();
  Cols q[R];
#pragma unroll
  for (int r = 0; r < R; ++r) q[r] = t0 + r < T ? load_cols(x + (t0 + r) * row_stride, K) : Cols{};
  dependency_wait();
  __shared__ int s_row[R * MAXR];
  __shared__ SfSpot s_spot[R * MAXR];
  __shared__ int s_start[kMaxGroups];
  if (!pos && g.counts) {
    for (int i = tid; i < g.n; i += kSplitThreads) s_start[i] = load_dep(g.row_start + i);
    __syncthreads();
  }
  const int n = pos ? top_k + shared : 1;
  if (tid < R * n) {
    const int r = tid / n, j = tid - r * n, t = t0 + r;
    int row = -1, grp = 0, count = g.rows, local = t, tile0 = 0;
    if (t < T) {
      row = t;
      if (pos && j >= shared) {
        const size_t pair = static_cast<size_t>(t) * top_k + j - shared;
        row = load_dep(pos + pair);
        if (row >= 0) grp = static_cast<int>(__ldg(idx + pair)) + shared;  // row < 0: an id outside
      } else if (g.counts && !pos) {
        int lo = 0, hi = g.n;  // last group that starts at or before the row
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_start[mid] <= row) lo = mid; else hi = mid;
        }
        grp = lo;
      }
      if (g.counts && row >= 0) {
        count = load_dep(g.counts + grp);
        local = row - load_dep(g.row_start + grp);
        tile0 = load_dep(g.tile_start + grp);
        if (local < 0 || local >= count) row = -1;  // a row outside every segment
      }
    }
    s_row[tid] = row;
    if (row >= 0) s_spot[tid] = sf_spot<TILE>(tile0, count, local, KB);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (t0 + r >= T) break;
    if (!pos && s_row[r] < 0) {
      if (zero_out && blockIdx.y == 0)
        for (int c = tid; c < M / 8; c += kSplitThreads)
          reinterpret_cast<uint4*>(zero_out + static_cast<size_t>(t0 + r) * M)[c] = make_uint4(0, 0, 0, 0);
      continue;
    }
    split_row(q[r], K, P, n, s_row + r * n, s_spot + r * n, tile_atoms(TILE), xq, sf);
  }
}

// Tables and split for a few rows: every block builds the group tables for
// itself in shared memory (~1 us) instead of waiting for a kernel that does;
// block 0 also writes them out.
struct SmallTables {
  int cnt[kMaxGroups], start[kMaxGroups], tile[kMaxGroups];
  int sum[2][kSplitThreads / 32];
};
constexpr int kGroupsPerThread = kMaxGroups / kSplitThreads;

// Exclusive scan of the token tiles (and with ROWS of the rows) of t.cnt;
// thread tid has groups kGroupsPerThread * tid and up.
template <int TILE, bool ROWS>
__device__ __forceinline__ void scan_tables(SmallTables& t) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int c[kGroupsPerThread], rows = 0, tiles = 0;
#pragma unroll
  for (int j = 0; j < kGroupsPerThread; ++j) {
    c[j] = t.cnt[kGroupsPerThread * tid + j];
    rows += c[j];
    tiles += (c[j] + TILE - 1) / TILE;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, rows, o), b = __shfl_up_sync(0xffffffffu, tiles, o);
    if (lane >= o) rows += a, tiles += b;
  }
  if (lane == 31) t.sum[0][warp] = rows, t.sum[1][warp] = tiles;
  __syncthreads();
  for (int w = 0; w < warp; ++w) rows += t.sum[0][w], tiles += t.sum[1][w];
#pragma unroll
  for (int j = kGroupsPerThread - 1; j >= 0; --j) {
    rows -= c[j];
    tiles -= (c[j] + TILE - 1) / TILE;
    if (ROWS) t.start[kGroupsPerThread * tid + j] = rows;
    t.tile[kGroupsPerThread * tid + j] = tiles;
  }
  __syncthreads();
}

template <int TILE>
__device__ __forceinline__ void write_tables(const SmallTables& t, int G, int32_t* counts, int32_t* row_start,
                                             int32_t* tile_start, int32_t* next) {
  if (blockIdx.x != 0 || blockIdx.y != 0) return;
  if (threadIdx.x < 2) next[threadIdx.x] = 0;
  for (int g = threadIdx.x; g <= G; g += kSplitThreads) {
    if (g < G) counts[g] = t.cnt[g], row_start[g] = t.start[g], tile_start[g] = t.tile[g];
    else tile_start[g] = t.tile[G - 1] + (t.cnt[G - 1] + TILE - 1) / TILE;
  }
}

template <int TILE>
__global__ void __launch_bounds__(kSplitThreads)
route_split_kernel(const __nv_bfloat16* __restrict__ x, long long row_stride, int T, int K,
                   const int64_t* __restrict__ idx, int top_k, int n_routed, int shared, int P,
                   int32_t* __restrict__ counts, int32_t* __restrict__ row_start, int32_t* __restrict__ tile_start,
                   int32_t* __restrict__ next, int32_t* __restrict__ pos, uint8_t* __restrict__ xq,
                   uint8_t* __restrict__ sf) {
  constexpr int NT = kSplitThreads;
  __shared__ SmallTables tab;
  __shared__ int s_e[kRoutePairs];
  __shared__ int s_row[MAXR];
  __shared__ SfSpot s_spot[MAXR];
  launch_dependents();
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pairs = T * top_k;
  const Cols q = load_cols(x + t * row_stride, K);
  for (int p = tid; p < pairs; p += NT) {
    const int64_t v = __ldg(idx + p);
    s_e[p] = v >= 0 && v < n_routed ? static_cast<int>(v) + shared : -1;
  }
  for (int g = tid; g < kMaxGroups; g += NT) tab.cnt[g] = 0;
  __syncthreads();
  for (int p = tid; p < pairs; p += NT)
    if (s_e[p] >= 0) atomicAdd(&tab.cnt[s_e[p]], 1);
  if (shared && tid == 0) tab.cnt[0] = T;
  __syncthreads();
  scan_tables<TILE, true>(tab);
  write_tables<TILE>(tab, n_routed + shared, counts, row_start, tile_start, next);
  // A warp places a pair of the token: earlier pairs of the same expert first.
  const int n = top_k + shared;
  for (int k = warp; k < top_k; k += NT / 32) {
    const int p = t * top_k + k, mine = s_e[p];
    int rank = 0;
    for (int b = 0; b < p; b += 32) rank += __popc(__ballot_sync(0xffffffffu, b + lane < p && s_e[b + lane] == mine));
    if (lane == 0) {
      const int row = mine >= 0 ? tab.start[mine] + rank : -1;
      s_row[shared + k] = row;
      if (mine >= 0) s_spot[shared + k] = sf_spot<TILE>(tab.tile[mine], tab.cnt[mine], rank, K / 128);
      if (blockIdx.y == 0) pos[p] = row;
    }
  }
  if (shared && tid == 0) {
    s_row[0] = t;
    s_spot[0] = sf_spot<TILE>(0, T, t, K / 128);
  }
  __syncthreads();
  split_row(q, K, P, n, s_row, s_spot, tile_atoms(TILE), xq, sf);
}

// segments_kernel and split_kernel in one; offsets are clamped the same way.
template <int TILE>
__global__ void __launch_bounds__(kSplitThreads)
segments_split_kernel(const __nv_bfloat16* __restrict__ x, long long row_stride, int rows, int K,
                      const int32_t* __restrict__ offsets, int E, int32_t* __restrict__ counts,
                      int32_t* __restrict__ row_start, int32_t* __restrict__ tile_start, int32_t* __restrict__ next,
                      int* __restrict__ status, uint8_t* __restrict__ xq, uint8_t* __restrict__ sf,
                      __nv_bfloat16* __restrict__ zero_out, int M) {
  constexpr int GT = kGroupsPerThread;
  __shared__ SmallTables tab;
  __shared__ int s_row[1];
  __shared__ SfSpot s_spot[1];
  launch_dependents();
  const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Cols q = load_cols(x + t * row_stride, K);
  // Ends: the running maximum of the clamped offsets.
  const int first = min(max(__ldg(offsets), 0), rows);
  int end[GT], top = first;
#pragma unroll
  for (int j = 0; j < GT; ++j) {
    const int g = GT * tid + j;
    if (g < E) {
      const int lo = __ldg(offsets + g), hi = __ldg(offsets + g + 1);
      if (blockIdx.x == 0 && blockIdx.y == 0 && (lo < 0 || hi < lo || hi > rows)) atomicCAS(status, 0, kDevBadCount);
      top = max(top, min(max(hi, 0), rows));
    }
    end[j] = top;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, top, o);
    if (lane >= o) top = max(top, a);
  }
  if (lane == 31) tab.sum[0][warp] = top;
  int before = __shfl_up_sync(0xffffffffu, top, 1);
  if (lane == 0) before = first;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before = max(before, tab.sum[0][w]);
#pragma unroll
  for (int j = 0; j < GT; ++j) {
    const int start = j ? max(before, end[j - 1]) : before;
    tab.start[GT * tid + j] = start;
    tab.cnt[GT * tid + j] = max(before, end[j]) - start;
  }
  __syncthreads();  // also: tab.sum is free again
  scan_tables<TILE, false>(tab);
  write_tables<TILE>(tab, E, counts, row_start, tile_start, next);
  if (tid == 0) {
    int lo = 0, hi = E;  // last group that starts at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tab.start[mid] <= t) lo = mid; else hi = mid;
    }
    const int local = t - tab.start[lo];
    const bool in = local >= 0 && local < tab.cnt[lo];
    s_row[0] = in ? t : -1;
    if (in) s_spot[0] = sf_spot<TILE>(tab.tile[lo], tab.cnt[lo], local, K / 128);
  }
  __syncthreads();
  if (s_row[0] < 0) {
    if (zero_out && blockIdx.y == 0)
      for (int c = tid; c < M / 8; c += kSplitThreads)
        reinterpret_cast<uint4*>(zero_out + static_cast<size_t>(t) * M)[c] = make_uint4(0, 0, 0, 0);
    return;
  }
  split_row(q, K, rows, 1, s_row, s_spot, tile_atoms(TILE), xq, sf);
}

// Bound by memory: the token's rows are loaded together and summed in fp32 in
// top-k order. 4096 tokens x 9 rows of 7168: 88 us, 6.7 TB/s.
__global__ void __launch_bounds__(256) combine_kernel(const __nv_bfloat16* y, int T, int H,
                                                      const int32_t* pos, const float* __restrict__ w,
                                                      int top_k, int shared, float scale,
                                                      __nv_bfloat16* __restrict__ out) {
  constexpr int MAXK = 8;
  const int t = blockIdx.x;
  __shared__ int s_row[MAXK];
  __shared__ float s_w[MAXK];
  dependency_wait();
  if (threadIdx.x < top_k) {
    s_row[threadIdx.x] = load_dep(pos + static_cast<size_t>(t) * top_k + threadIdx.x);
    s_w[threadIdx.x] = scale * w[static_cast<size_t>(t) * top_k + threadIdx.x];
  }
  __syncthreads();
  for (int c = blockIdx.y * 256 + threadIdx.x; c < H / 8; c += gridDim.y * 256) {
    uint4 v[MAXK + 1];
#pragma unroll
    for (int k = 0; k < MAXK; ++k)
      if (k < top_k && s_row[k] >= 0) v[k] = load_dep(reinterpret_cast<const uint4*>(y + static_cast<size_t>(s_row[k]) * H) + c);
    if (shared) v[MAXK] = load_dep(reinterpret_cast<const uint4*>(y + static_cast<size_t>(t) * H) + c);
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    auto add = [&](const uint4& q, float f) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 p = __bfloat1622float2(h[i]);
        acc[2 * i] = fmaf(f, p.x, acc[2 * i]);
        acc[2 * i + 1] = fmaf(f, p.y, acc[2 * i + 1]);
      }
    };
#pragma unroll
    for (int k = 0; k < MAXK; ++k)
      if (k < top_k && s_row[k] >= 0) add(v[k], s_w[k]);
    if (shared) add(v[MAXK], 1.f);
    uint4 o;
    __nv_bfloat162* ob = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) ob[i] = __floats2bfloat162_rn(acc[2 * i], acc[2 * i + 1]);
    reinterpret_cast<uint4*>(out + static_cast<size_t>(t) * H)[c] = o;
  }
}

}  // namespace

cudaError_t launch_segments(const int32_t* offsets, int n, int rows, int tile, int32_t* counts, int32_t* row_start,
                            int32_t* tile_start, int32_t* next, int* status, cudaStream_t s) {
  segments_kernel<<<1, kMaxGroups, 0, s>>>(offsets, n, rows, tile, counts, row_start, tile_start, next, status);
  return cudaGetLastError();
}

cudaError_t launch_route_plan(const int64_t* idx, int T, int top_k, int n_routed, int shared, int tile,
                              int32_t* counts, int32_t* row_start, int32_t* tile_start, int32_t* next, int32_t* pos,
                              cudaStream_t s) {
  const int smem = kPlanWarps * n_routed * 4;
  if (smem > 40 * 1024) {  // static shared memory counts against the default limit too
    // Always the largest: the limit is the function's, and another thread may be
    // between its own setting and its launch.
    const cudaError_t e = cudaFuncSetAttribute(route_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               kPlanWarps * kMaxGroups * 4);
    if (e != cudaSuccess) return e;
  }
  // A CTA's warps take 32 pairs a step: a few steps each before more CTAs help.
  const int ctas = T * top_k >= 4096 ? kPlanCtas : 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = ctas;
  cfg.blockDim = 1024;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, route_plan_kernel, idx, T, top_k, n_routed, shared, tile, counts, row_start, tile_start,
                            next, pos);
}

cudaError_t launch_split(const __nv_bfloat16* x, long long row_stride, int T, int K, const Groups& g, int tile,
                         const int64_t* idx, const int32_t* pos, int top_k, int shared, int P, uint8_t* xq, uint8_t* sf,
                         __nv_bfloat16* zero_out, int M, cudaStream_t s) {
  constexpr int R = 4;
  const bool many = T >= 1024;  // fewer rows: one per block, to reach every SM
  const dim3 grid(many ? (T + R - 1) / R : T, (K + kSplitCols - 1) / kSplitCols);
  auto go = [&](auto one, auto several) {
    return launch_chained(g.counts != nullptr, many ? several : one, grid, kSplitThreads, 0, s, x, row_stride, T, K, g, idx, pos,
                          top_k, shared, P, xq, sf, zero_out, M);
  };
  switch (tile) {
    case 32: return go(split_kernel<32, 1>, split_kernel<32, R>);
    case 64: return go(split_kernel<64, 1>, split_kernel<64, R>);
    case 128: return go(split_kernel<128, 1>, split_kernel<128, R>);
    case 160: return go(split_kernel<160, 1>, split_kernel<160, R>);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_route_split(const __nv_bfloat16* x, long long row_stride, int T, int K, const int64_t* idx, int top_k,
                               int n_routed, int shared, int tile, int P, int32_t* counts, int32_t* row_start,
                               int32_t* tile_start, int32_t* next, int32_t* pos, uint8_t* xq, uint8_t* sf,
                               cudaStream_t s) {
  if (T * top_k > kRoutePairs || n_routed + shared > kMaxGroups) return cudaErrorInvalidValue;
  const dim3 grid(T, (K + kSplitCols - 1) / kSplitCols);
  auto go = [&](auto kern) {
    return launch_chained(false, kern, grid, kSplitThreads, 0, s, x, row_stride, T, K, idx, top_k, n_routed, shared, P,
                          counts, row_start, tile_start, next, pos, xq, sf);
  };
  switch (tile) {
    case 32: return go(route_split_kernel<32>);
    case 64: return go(route_split_kernel<64>);
    case 160: return go(route_split_kernel<160>);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_segments_split(const __nv_bfloat16* x, long long row_stride, int rows, int K, const int32_t* offsets,
                                  int n, int tile, int32_t* counts, int32_t* row_start, int32_t* tile_start,
                                  int32_t* next, int* status, uint8_t* xq, uint8_t* sf, __nv_bfloat16* zero_out, int M,
                                  cudaStream_t s) {
  const dim3 grid(rows, (K + kSplitCols - 1) / kSplitCols);
  auto go = [&](auto kern) {
    return launch_chained(false, kern, grid, kSplitThreads, 0, s, x, row_stride, rows, K, offsets, n, counts, row_start,
                          tile_start, next, status, xq, sf, zero_out, M);
  };
  switch (tile) {
    case 32: return go(segments_split_kernel<32>);
    case 64: return go(segments_split_kernel<64>);
    case 160: return go(segments_split_kernel<160>);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_combine(bool chained, const __nv_bfloat16* y, int T, int H, const int32_t* pos, const float* w,
                           int top_k, int shared, float scale, __nv_bfloat16* out, cudaStream_t s) {
  // Few tokens: a block per 2048 columns; many: one per token.
  const dim3 grid(T, T < 512 ? (H + 2047) / 2048 : 1);
  return launch_chained(chained, combine_kernel, grid, 256, 0, s, y, T, H, pos, w, top_k, shared, scale, out);
}

}  // namespace mx
}  // namespace dsmoe
