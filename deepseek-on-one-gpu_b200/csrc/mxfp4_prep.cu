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
                                                              int* __restrict__ status) {
  __shared__ int buf[kMaxGroups];
  const int i = threadIdx.x;
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

// Stable counting sort of the (token, k) pairs by expert, by one block: warp w
// owns a contiguous range of pairs, counts it, and after the scans walks it
// again in order; lanes of one step that hold the same expert are ranked by
// lane. The row of a pair therefore depends on the routing only.
constexpr int kPlanWarps = 32;

__global__ void __launch_bounds__(1024) route_plan_kernel(const int64_t* __restrict__ idx, int T, int top_k,
                                                          int n_routed, int shared, int tile,
                                                          int32_t* __restrict__ counts, int32_t* __restrict__ row_start,
                                                          int32_t* __restrict__ tile_start, int32_t* __restrict__ pos) {
  extern __shared__ int hist[];  // [kPlanWarps][n_routed]
  __shared__ int buf[kMaxGroups];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pairs = T * top_k;
  const int per = ((pairs + kPlanWarps - 1) / kPlanWarps + 31) & ~31;
  const int p0 = min(pairs, warp * per), p1 = min(pairs, p0 + per);
  for (int i = threadIdx.x; i < kPlanWarps * n_routed; i += 1024) hist[i] = 0;
  __syncthreads();
  int* mine = hist + warp * n_routed;
  for (int p = p0 + lane; p < p1; p += 32) {
    const int64_t e = idx[p];
    if (e >= 0 && e < n_routed) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  // group totals and, per warp, the rows of earlier warps
  const int groups = n_routed + shared;
  const int g = threadIdx.x;
  int c = 0;
  if (g < groups) {
    if (g < shared) {
      c = T;
    } else {
      for (int w = 0; w < kPlanWarps; ++w) {
        int* h = &hist[w * n_routed + g - shared];
        const int n = *h;
        *h = c;
        c += n;
      }
    }
  }
  // Scans over the first kMaxGroups threads; the others keep the barriers.
  const int nt = (c + tile - 1) / tile;
  int rows = c, tiles = nt;
  for (int pass = 0; pass < 2; ++pass) {
    int& v = pass ? tiles : rows;
    if (g < kMaxGroups) buf[g] = v;
    __syncthreads();
    for (int o = 1; o < kMaxGroups; o <<= 1) {
      const int a = g < kMaxGroups && g >= o ? buf[g - o] : 0;
      __syncthreads();
      if (g < kMaxGroups) buf[g] += a;
      __syncthreads();
    }
    if (g < kMaxGroups) v = buf[g];
    __syncthreads();
  }
  if (g < groups) {
    const int start = rows - c;
    counts[g] = c;
    row_start[g] = start;
    tile_start[g] = tiles - nt;
    if (g == groups - 1) tile_start[groups] = tiles;
    if (g >= shared)
      for (int w = 0; w < kPlanWarps; ++w) hist[w * n_routed + g - shared] += start;
  }
  __syncthreads();
  for (int b = p0; b < p1; b += 32) {  // warp-uniform
    const int p = b + lane;
    int e = -1;
    if (p < p1) {
      const int64_t v = idx[p];
      if (v >= 0 && v < n_routed) e = static_cast<int>(v);
    }
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1));
    const int base = e >= 0 ? mine[e] : 0;
    __syncwarp();
    if (e >= 0 && rank == 0) mine[e] = base + __popc(same);
    __syncwarp();
    if (p < p1) pos[p] = e >= 0 ? base + rank : -1;
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
  const int n32 = side_by_side(TILE, min(TILE, count - t * TILE));
  const long long base = static_cast<long long>(tile0 + t) * KB * tile_atoms(TILE) * 128;
  auto word = [](int col) { return (col >> 7) * 128 + (col & 31) * 4 + ((col >> 5) & 3); };
  return {base + word(c), n32 ? base + word(c + n32) : -1};
}

// One block: 2048 columns of one row. 4 threads share a 32-number block, 16 a
// K block's scale word.
template <int TILE>
__global__ void __launch_bounds__(256) split_kernel(const __nv_bfloat16* __restrict__ x, long long row_stride, int T,
                                                    int K, const Groups g, const int32_t* __restrict__ pos, int top_k,
                                                    int shared, int P, uint8_t* __restrict__ xq,
                                                    uint8_t* __restrict__ sf, __nv_bfloat16* __restrict__ zero_out,
                                                    int M) {
  constexpr int MAXR = 9;
  const int t = blockIdx.x;
  const int tid = threadIdx.x;
  const int KB = K / 128;
  __shared__ int s_row[MAXR];
  __shared__ SfSpot s_spot[MAXR];
  const int n = pos ? top_k + shared : 1;
  if (tid < n) {
    int row, grp = 0, count, local, tile0 = 0;
    if (pos) row = tid < shared ? t : pos[static_cast<size_t>(t) * top_k + tid - shared];
    else row = t;
    if (row >= 0 && g.counts) {
      int lo = 0, hi = g.n;  // last group that starts at or before the row
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (g.row_start[mid] <= row) lo = mid; else hi = mid;
      }
      grp = lo;
      count = g.counts[grp];
      local = row - g.row_start[grp];
      tile0 = g.tile_start[grp];
      if (local < 0 || local >= count) row = -1;
    } else {
      count = g.rows;
      local = row;
    }
    s_row[tid] = row;
    if (row >= 0) s_spot[tid] = sf_spot<TILE>(tile0, count, local, KB);
  }
  __syncthreads();
  if (!pos && s_row[0] < 0) {  // a row outside every segment
    if (zero_out && blockIdx.y == 0)
      for (int c = tid; c < M / 8; c += 256)
        reinterpret_cast<uint4*>(zero_out + static_cast<size_t>(t) * M)[c] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int col = blockIdx.y * 2048 + tid * 8;
  const bool in = col < K;  // K is a multiple of 128: 16 threads of a K block are in or out together
  uint4 q = make_uint4(0, 0, 0, 0);
  if (in) q = __ldg(reinterpret_cast<const uint4*>(x + t * row_stride + col));
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t amax = 0;  // |bf16| bit patterns order like the numbers
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = max(amax, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const uint32_t ef = amax >> 7;
  const uint32_t byte = ef == 255 ? 255u : (ef > 7 ? ef - 7 : 0u);
  const float inv = ef == 255 ? 0.f : __uint_as_float((254u - byte) << 23);
  uint32_t hw[2] = {0, 0}, lw[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = __uint_as_float(w[i] << 16) * inv, b = __uint_as_float(w[i] & 0xffff0000u) * inv;
    const uint32_t h2 = f32x2_to_e4m3x2(a, b);
    const uint32_t l2 = f32x2_to_e4m3x2(a - e4m3_to_f32(h2 & 0xff), b - e4m3_to_f32(h2 >> 8));
    hw[i >> 1] |= h2 << (16 * (i & 1));
    lw[i >> 1] |= l2 << (16 * (i & 1));
  }
  // scale word of the K block: bytes from threads 0, 4, 8, 12 of its 16
  uint32_t word = byte << (8 * ((tid >> 2) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if (!in) return;
  const long long step = static_cast<long long>(col >> 7) * tile_atoms(TILE) * 128;
  for (int r = 0; r < n; ++r) {
    const int row = s_row[r];
    if (row < 0) continue;
    const size_t off = static_cast<size_t>(row) * K + col;
    *reinterpret_cast<uint2*>(xq + off) = make_uint2(hw[0], hw[1]);
    *reinterpret_cast<uint2*>(xq + static_cast<size_t>(P) * K + off) = make_uint2(lw[0], lw[1]);
    if ((tid & 15) == 0) {
      uint32_t* s32 = reinterpret_cast<uint32_t*>(sf);
      s32[s_spot[r].hi + step] = word;
      if (s_spot[r].lo >= 0) s32[s_spot[r].lo + step] = word;
    }
  }
}

__global__ void __launch_bounds__(256) combine_kernel(const __nv_bfloat16* __restrict__ y, int T, int H,
                                                      const int32_t* __restrict__ pos, const float* __restrict__ w,
                                                      int top_k, int shared, float scale,
                                                      __nv_bfloat16* __restrict__ out) {
  constexpr int MAXK = 8;
  const int t = blockIdx.x;
  __shared__ int s_row[MAXK];
  __shared__ float s_w[MAXK];
  if (threadIdx.x < top_k) {
    s_row[threadIdx.x] = pos[static_cast<size_t>(t) * top_k + threadIdx.x];
    s_w[threadIdx.x] = scale * w[static_cast<size_t>(t) * top_k + threadIdx.x];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < H / 8; c += 256) {
    uint4 v[MAXK + 1];
#pragma unroll
    for (int k = 0; k < MAXK; ++k)
      if (k < top_k && s_row[k] >= 0) v[k] = __ldg(reinterpret_cast<const uint4*>(y + static_cast<size_t>(s_row[k]) * H) + c);
    if (shared) v[MAXK] = __ldg(reinterpret_cast<const uint4*>(y + static_cast<size_t>(t) * H) + c);
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
                            int32_t* tile_start, int* status, cudaStream_t s) {
  segments_kernel<<<1, kMaxGroups, 0, s>>>(offsets, n, rows, tile, counts, row_start, tile_start, status);
  return cudaGetLastError();
}

cudaError_t launch_route_plan(const int64_t* idx, int T, int top_k, int n_routed, int shared, int tile,
                              int32_t* counts, int32_t* row_start, int32_t* tile_start, int32_t* pos, cudaStream_t s) {
  const int smem = kPlanWarps * n_routed * 4;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(route_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  route_plan_kernel<<<1, 1024, smem, s>>>(idx, T, top_k, n_routed, shared, tile, counts, row_start, tile_start, pos);
  return cudaGetLastError();
}

cudaError_t launch_split(const __nv_bfloat16* x, long long row_stride, int T, int K, const Groups& g, int tile,
                         const int32_t* pos, int top_k, int shared, int P, uint8_t* xq, uint8_t* sf,
                         __nv_bfloat16* zero_out, int M, cudaStream_t s) {
  const dim3 grid(T, (K + 2047) / 2048);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, s>>>(x, row_stride, T, K, g, pos, top_k, shared, P, xq, sf, zero_out, M);
  };
  switch (tile) {
    case 32: go(split_kernel<32>); break;
    case 64: go(split_kernel<64>); break;
    case 160: go(split_kernel<160>); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_combine(const __nv_bfloat16* y, int T, int H, const int32_t* pos, const float* w, int top_k,
                           int shared, float scale, __nv_bfloat16* out, cudaStream_t s) {
  combine_kernel<<<T, 256, 0, s>>>(y, T, H, pos, w, top_k, shared, scale, out);
  return cudaGetLastError();
}

}  // namespace mx
}  // namespace dsmoe
