// Internal interface of the MXFP4 operators (mxfp4_quant.cu, mxfp4_prep.cu,
// mxfp4_gemm.cu, mxfp4_api.cu).
//
// MXFP4: a row of K numbers is K e2m1 codes (two per byte, the even element
// in the low nibble) and one e8m0 scale byte b = 2^(b - 127) per 32
// consecutive numbers; byte 255 is NaN.
//
// The tensor core takes bf16 activations as two e4m3 terms that share one
// power-of-two scale per 32 numbers: with 2^7 <= amax * 2^-e < 2^8,
//   hi = e4m3(x * 2^-e),  lo = e4m3(x * 2^-e - hi).
// hi keeps 4 of a bf16's 8 significant bits and the remainder fits lo's 4
// exactly, as long as its last bit is not below e4m3's smallest step 2^-9:
// numbers down to 2^-9 of the block's amax are exact, smaller ones are off by
// at most 2^-10 * 2^e <= 2^-17 of the amax.
//
// Scale factors are stored as the 512-byte atoms tcgen05.cp takes: rows
// 32j + l (j < 4, l < 32) of a 128-row tile and one K block of 128 numbers;
// bytes l * 16 + j * 4 .. + 3 hold row 32j + l's four scales of that block.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace dsmoe {
namespace mx {

constexpr int kMaxGroups = 512;
constexpr int kWorkWarps = 16;  // epilogue warps, and those that prepare rows in the kernel
constexpr int kRawRows = 32;   // most bf16 rows that a single-group product splits itself
constexpr int kMaxSplit = 8;  // CTAs of a cluster that share one tile's K

// Token tiles of the product kernels: columns of one work unit, and 512-byte
// scale atoms per token tile and K block.
constexpr int tile_atoms(int bn) { return bn > 64 ? 2 : 1; }

// bf16 activations: columns n of a tile that run hi and lo side by side in one
// MMA of N = 2 n (hi columns then lo columns), or 0 where hi and lo are two
// MMAs. Side by side the MMA is twice as wide, which pays while a narrow one
// does not fill the tensor pipe; the accumulators then take 4 columns of TMEM
// per token, which caps it at 96. n follows the rows in the tile in steps of 8:
// every column beyond costs energy, and a long run is held back by the power
// limit.
__host__ __device__ constexpr int side_by_side(int bn, int ncols) {
  const int n = (ncols + 7) & ~7;
  return bn <= 64 || n <= 96 ? n : 0;
}

enum { kTypeBf16 = 0, kTypeF16 = 1, kTypeF32 = 2, kTypeE4m3 = 3 };

// Group tables of a product: group g has counts[g] rows from row_start[g] on
// and owns token tiles [tile_start[g], tile_start[g + 1]).
struct Groups {
  const int32_t* counts;      // NULL: one group of `rows` rows
  const int32_t* row_start;
  const int32_t* tile_start;
  int n;
  int rows;
};

// What the tables of a few rows are made from: a product with a small tile
// builds them for itself (`tiles` up to 64), so that it can start on its
// weights while the kernel that splits the rows still runs.
struct TableSource {
  const int64_t* idx;      // a routing's pairs, or
  const int32_t* offsets;  // segments of g.rows rows, or neither
  int pairs, n_routed, shared, tokens;
};

struct GemmArgs {
  Groups g;
  TableSource own;
  int M;                 // features of one weight matrix
  int K;
  int P;                 // first lo row of the split activations
  int ksplit;            // parts of K per tile, a cluster's CTAs (1 unless g.counts == NULL)
  int unit0;             // with ksplit > 1, the first unit of this launch: one per CTA from there on
  // Scale atoms of the weights, a unit's two A tiles together: [group][pair of
  // tiles][K/128][2][512], SwiGLU [group][tile][K/128][gate, up][512].
  const uint8_t* sfa;
  const uint8_t* sfb;    // scale atoms of the rows [tile][K/128][tile_atoms][512]
  __nv_bfloat16* y;      // [row][M]
  int32_t* next;         // counter of handed-out units, 0 before the launch; NULL: units in fixed turns
  // The rows themselves, where the kernel prepares them: bf16 numbers, rows
  // raw_stride apart, or the scale bytes of dense MXFP4 rows.
  const void* raw;
  long long raw_stride;
  uint8_t* hq;           // SwiGLU: split rows [2][P][M] and their atoms
  uint8_t* hsf;
  int* status;
};

// Four scaled numbers (f16 pairs) -> their hi and lo e4m3 terms, the first in
// the lowest byte. f16 holds what the two terms can (8 significant bits down
// to 2^-9, |x| <= 256), and its pairs take half the instructions of fp32: one
// number at a time, the split of activations was issue-bound at 28
// instructions per number.
__device__ __forceinline__ void split4(uint32_t x01, uint32_t x23, uint32_t& hi, uint32_t& lo) {
  asm("{\n\t.reg .b16 a, b;\n\t.reg .b32 f, g;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 a, %2;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 b, %3;\n\t"
      "mov.b32 %0, {a, b};\n\t"
      "cvt.rn.f16x2.e4m3x2 f, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 g, b;\n\t"
      "sub.rn.f16x2 f, %2, f;\n\t"
      "sub.rn.f16x2 g, %3, g;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 a, f;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 b, g;\n\t"
      "mov.b32 %1, {a, b};\n\t}"
      : "=&r"(hi), "=r"(lo)
      : "r"(x01), "r"(x23));
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 bf16 numbers, two threads (lanes l and l ^ 1) per 32-number block and eight
// (an aligned group of lanes) per K block of 128, to their two e4m3 terms and the
// K block's scale word. Every lane of the warp takes part.
struct Cols {
  uint4 a, b;
};
__device__ __forceinline__ void split_cols(const Cols& q, uint32_t* hw, uint32_t* lw, uint32_t& word) {
  const uint32_t w[8] = {q.a.x, q.a.y, q.a.z, q.a.w, q.b.x, q.b.y, q.b.z, q.b.w};
  // |bf16| bit patterns order like the numbers; two at a time
  uint32_t m2 = w[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m2 = __vmaxu2(m2, w[i] & 0x7fff7fffu);
  m2 = __vmaxu2(m2, __shfl_xor_sync(0xffffffffu, m2, 1));
  const uint32_t amax = max(m2 & 0xffffu, m2 >> 16);
  const uint32_t ef = amax >> 7;
  const uint32_t byte = ef == 255 ? 255u : (ef > 7 ? ef - 7 : 0u);
  // 2^(127 - byte); the product is exact (or below all that the terms hold)
  const __nv_bfloat162 inv = __bfloat162bfloat162(__ushort_as_bfloat16(ef == 255 ? 0 : (254u - byte) << 7));
  uint32_t x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __bfloat1622float2(__hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), inv));
    x[i] = f16_pair(f.x, f.y);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) split4(x[2 * i], x[2 * i + 1], hw[i], lw[i]);
  // bytes from lanes 0, 2, 4, 6 of the K block's 8
  word = byte << (8 * ((threadIdx.x >> 1) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 2);
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
}

// The kernels of one call are chained by programmatic dependent launches: the
// first one is launched normally, so everything enqueued before the call is
// done when it starts; a later one may start while its predecessor runs and
// waits (dependency_wait) before it touches anything an earlier one of the
// chain reads or writes. Under dsmoe_set_gemm_sm_limit a product and the combine
// are launched normally: waiting on the SMs left free, they would keep another
// stream's kernels off them.
__device__ __forceinline__ void dependency_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("fence.proxy.async.global;" ::: "memory");  // its data may be read by TMA next
}
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Loads of what an earlier kernel of the chain wrote. Not __ldg, and not
// through a const __restrict__ pointer: the compiler takes such data as fixed
// for the whole kernel and may read it before the wait.
__device__ __forceinline__ int32_t load_dep(const int32_t* p) {
  int32_t v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 load_dep(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

template <class... P, class... A>
cudaError_t launch_chained(bool chained, void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s,
                           A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = chained ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

// -------------------------------------------------------- mxfp4_quant.cu
cudaError_t launch_quantize(const void* x, int type, long long rows, int K, long long row_stride, const float* scale_inv,
                            long long rows_per_mat, uint8_t* codes, uint8_t* scales, cudaStream_t s);
cudaError_t launch_dequantize(const uint8_t* codes, const uint8_t* scales, long long blocks, int type, void* out,
                              cudaStream_t s);
// Scales [mats][N][K/32] -> atoms [mats][ceil(N/tile)][K/128][atoms][512].
cudaError_t launch_tile_scales(const uint8_t* scales, int mats, int N, int K, int tile, int atoms, uint8_t* out,
                               cudaStream_t s);

// --------------------------------------------------------- mxfp4_prep.cu
// Segments of rows sorted by expert from offsets[n + 1].
// The kernels that make group tables also clear next[2].
cudaError_t launch_segments(const int32_t* offsets, int n, int rows, int tile, int32_t* counts, int32_t* row_start,
                            int32_t* tile_start, int32_t* next, int* status, cudaStream_t s);
// Segments from a routing: pos[T][top_k] is the row of each (token, k), in
// token order inside an expert, -1 for an id outside [0, n_routed).
cudaError_t launch_route_plan(const int64_t* idx, int T, int top_k, int n_routed, int shared, int tile,
                              int32_t* counts, int32_t* row_start, int32_t* tile_start, int32_t* next, int32_t* pos,
                              cudaStream_t s);
// bf16 rows [T][K] -> hi/lo rows and scale atoms. pos == NULL: row t is row t
// of g (zero_out, optional: rows of y outside every segment are cleared);
// else token t goes to the rows pos names for its ids idx (and to row t of group
// 0 with shared).
// Chained to the kernel that made the tables, if g has any.
cudaError_t launch_split(const __nv_bfloat16* x, long long row_stride, int T, int K, const Groups& g, int tile,
                         const int64_t* idx, const int32_t* pos, int top_k, int shared, int P, uint8_t* xq, uint8_t* sf,
                         __nv_bfloat16* zero_out, int M, cudaStream_t s);
// launch_route_plan and launch_split in one kernel, for up to kRoutePairs pairs.
constexpr int kRoutePairs = 1024;
cudaError_t launch_route_split(const __nv_bfloat16* x, long long row_stride, int T, int K, const int64_t* idx, int top_k,
                               int n_routed, int shared, int tile, int P, int32_t* counts, int32_t* row_start,
                               int32_t* tile_start, int32_t* next, int32_t* pos, uint8_t* xq, uint8_t* sf,
                               cudaStream_t s);
// launch_segments and launch_split in one kernel, for few rows.
constexpr int kSegmentRows = 1024;
cudaError_t launch_segments_split(const __nv_bfloat16* x, long long row_stride, int rows, int K, const int32_t* offsets,
                                  int n, int tile, int32_t* counts, int32_t* row_start, int32_t* tile_start,
                                  int32_t* next, int* status, uint8_t* xq, uint8_t* sf, __nv_bfloat16* zero_out, int M,
                                  cudaStream_t s);
// out[t] = bf16(shared row + scale * sum_k w[t][k] y[pos[t][k]]), summed in fp32
cudaError_t launch_combine(bool chained, const __nv_bfloat16* y, int T, int H, const int32_t* pos, const float* w,
                           int top_k, int shared, float scale, __nv_bfloat16* out, cudaStream_t s);

// --------------------------------------------------------- mxfp4_gemm.cu
// K split of a single-group product of `units` (feature tile pair, token tile)
// pairs on the current device.
int pick_ksplit(bool fp4, int tile, int units, int kblocks);
// x: rows in boxes of the token tile, x32 and x8: of 32 and 8.
cudaError_t launch_gemm(bool chained, bool fp4, bool swiglu, const CUtensorMap& w0, const CUtensorMap& w1,
                        const CUtensorMap& x, const CUtensorMap& x32, const CUtensorMap& x8, const GemmArgs& a,
                        int tile, int grid, cudaStream_t s);

}  // namespace mx
}  // namespace dsmoe
