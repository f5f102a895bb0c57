// C ABI of the MXFP4 operators: argument checks, workspace plans, TMA
// descriptors and launch sequences. See include/dsmoe.h.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/dsmoe.h"
#include "kernels.h"
#include "mxfp4.cuh"

using namespace dsmoe;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return set_last_error(code, buf);
}

#define MX_CUDA(call)                                                                     \
  do {                                                                                    \
    cudaError_t e_ = (call);                                                              \
    if (e_ != cudaSuccess) return fail(DSMOE_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_)); \
  } while (0)

constexpr int kMaxK = 32768;          // row offsets inside a K block stay in int
constexpr int kMaxN = 1 << 18;
constexpr long long kMaxRows = 1 << 22;  // rows of a product, copies for several experts included

bool aligned(const void* p, size_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }
size_t up(size_t v) { return (v + 255) / 256 * 256; }
int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Token tile and K split of a single-group product: the pair with the least
// estimated time in SM cycles. Per K block a tile of n columns takes 8 n cycles
// of MMA (16 of N = n, or 8 of N = 2 n with hi and lo side by side), 4-bit rows
// 2 n, with a floor of 64 cycles an MMA, and small tiles pay `drag` for moving
// more operand bytes per MMA. Around the K loop a tile costs ~1500 cycles plus
// its epilogue, a split as much again for the sums. Against every choice
// measured (T x N x K, us for tiles 32 / 64 / 128 / 160, the estimate's choice
// starred): 128x7168x2048 *10.7 / 12.8 / - / 15.5; 256x7168x2048 16.0 / *13.0 /
// - / 20.3; 512x2048x7168 23.9 / *22.0 / 24.4 / 27.1; 1024x7168x2048 42.8 / 33.3 /
// *32.6 / 36.7; 4096x7168x2048 - / 102 / 98.9 / *91.9.
struct Choice {
  int tile, ksplit, units;
};
Choice estimate(bool fp4, int rows, int K, int N) {
  static const int bf16_tiles[] = {16, 32, 64, 128, 160}, fp4_tiles[] = {64, 160};
  const int* tiles = fp4 ? fp4_tiles : bf16_tiles;
  const int n_tiles = fp4 ? 2 : 5, kb = K / 128, sms = sm_count();
  Choice best{};
  double least = 0;
  const int first = !fp4 && rows > 16 ? 1 : 0;
  for (int i = first; i < n_tiles; ++i) {
    const int tile = tiles[i], n = rows < tile ? ceil_div(rows, 16) * 16 : tile;
    const int pair = fp4 ? 0 : mx::side_by_side(tile, n);
    const int per_kb = fp4 ? 4 * (n < 128 ? 64 : n / 2) : pair ? 8 * (pair < 64 ? 64 : pair) : 16 * (n < 128 ? 64 : n / 2);
    const double drag = fp4 ? 1.0 : tile <= 64 ? 1.2 : tile == 128 ? 1.07 : 1.0;
    const long long units = static_cast<long long>(ceil_div(rows, tile)) * ceil_div(N, 256);
    const int split = units < sms ? mx::pick_ksplit(fp4, tile, static_cast<int>(units), kb) : 1;
    const long long waves = split > 1 ? 1 : (units + sms - 1) / sms;
    double t = waves * (ceil_div(kb, split) * drag * per_kb + 1500 + 25.0 * n);
    if (split > 1) t += 1500 + 40.0 * n;
    if (i == first || t < least) {
      least = t;
      best = {tile, split, static_cast<int>(units)};
    }
    if (rows <= tile) break;  // a larger tile holds no more rows and fewer stages
  }
  return best;
}

// The choice depends on sizes and the device only; the last ones asked for are
// remembered (a decode loop asks for the same few, twice per call, and the
// occupancy queries behind an estimate cost as much as a launch).
Choice choose(bool fp4, int rows, int K, int N) {
  struct Entry {
    int dev, rows, K, N;
    bool fp4;
    Choice c;
  };
  static thread_local Entry memo[64] = {};  // rows == 0: empty
  int dev = 0;
  cudaGetDevice(&dev);
  const uint32_t h = (rows * 2654435761u) ^ (K * 40503u) ^ (N * 69069u) ^ (fp4 ? 977u : 0u);
  Entry& e = memo[(h >> 16 ^ h) & 63];
  if (e.rows != rows || e.K != K || e.N != N || e.fp4 != fp4 || e.dev != dev)
    e = {dev, rows, K, N, fp4, estimate(fp4, rows, K, N)};
  return e.c;
}

// Token tile where `rows` rows spread over `groups` experts: one that most
// experts' rows fit. Routed FFN, 256 experts of 7168 x 2048 (ms for tiles 64 /
// 160): T=768 1.26 / 1.38, T=1536 (48 rows per expert) 1.64 / 1.72, T=2048 2.13 /
// 1.93; below 16 rows per expert tile 32 leaves room for more stages.
int grouped_tile(long long rows, int groups) {
  const long long mean = (rows + groups - 1) / groups;
  return mean <= 16 ? 32 : mean <= 48 ? 64 : 160;
}

struct Plan {
  size_t counts = 0, row_start = 0, tile_start = 0, next = 0, pos = 0, xq = 0, sf = 0, hq = 0, hsf = 0, y = 0, total = 0;
  int tile = 32, P = 0, ksplit = 1, units = 0;
  long long tiles = 0;
  bool raw = false;  // the product prepares its rows: the workspace is asked for, but not used
  size_t take(size_t bytes) {
    const size_t at = total;
    total = up(total + bytes);
    return at;
  }
  void tables(int groups) {
    counts = take(4 * static_cast<size_t>(groups));
    row_start = take(4 * static_cast<size_t>(groups));
    tile_start = take(4 * (static_cast<size_t>(groups) + 1));
    next = take(8);
  }
  size_t atoms(int K) const { return static_cast<size_t>(tiles) * (K / 128) * mx::tile_atoms(tile) * 512; }
  void set(const Choice& c, int rows) {
    tile = c.tile;
    ksplit = c.ksplit;
    units = c.units;
    tiles = ceil_div(rows, tile);
    P = rows;
  }
};

// Rows that a product splits itself. One launch less is worth 5 us of host time
// and 1-2 us between the kernels, but 17 to 32 rows are split faster ahead (us in a
// captured graph, itself / ahead: 17 x 7168 x 2048 8.8 / 8.5, 32 x 2048 x 7168 11.2 /
// 10.5, 32 x 7168 x 18432 22.9 / 20.7; calls one by one take 11.5 / 17 at least):
// so only where a call's launches take longer than its kernels.
bool splits_itself(int T, int K, int N) {
  return T <= 16 || (T <= mx::kRawRows && static_cast<long long>(N) * K <= 1 << 26);
}

Plan plan_linear(int T, int K, int N) {
  Plan w;
  w.set(choose(false, T, K, N), T);
  w.raw = splits_itself(T, K, N);  // tile 16 or 32
  w.xq = w.take(w.raw ? 1 : 2 * static_cast<size_t>(T) * K);
  if (!w.raw) w.sf = w.take(w.atoms(K));
  return w;
}

Plan plan_matmul(int T, int K, int N) {
  Plan w;
  w.set(choose(true, T, K, N), T);
  w.raw = w.tile == 64;
  w.sf = w.take(w.raw ? 1 : w.atoms(K));
  return w;
}

Plan plan_grouped(int R, int K, int E) {
  Plan w;
  w.tile = grouped_tile(R, E);
  w.P = R;
  w.tiles = R / w.tile + (R < E ? R : E);
  w.tables(E);
  w.xq = w.take(2 * static_cast<size_t>(R) * K);
  w.sf = w.take(w.atoms(K));
  return w;
}

Plan plan_moe(int T, int H, int F, int E, int shared, int top_k) {
  Plan w;
  const long long pairs = static_cast<long long>(T) * top_k;
  const long long rows = pairs + (shared ? T : 0);
  w.tile = grouped_tile(pairs, E);
  w.P = static_cast<int>(rows);
  w.tiles = rows / w.tile + (pairs < E ? pairs : E) + (shared ? 1 : 0);
  w.tables(E + shared);
  w.pos = w.take(4 * static_cast<size_t>(pairs));
  w.xq = w.take(2 * static_cast<size_t>(rows) * H);
  w.sf = w.take(w.atoms(H));
  w.hq = w.take(2 * static_cast<size_t>(rows) * F);
  w.hsf = w.take(w.atoms(F));
  w.y = w.take(2 * static_cast<size_t>(rows) * H);
  return w;
}

template <class T>
T* at(void* base, size_t off) {
  return reinterpret_cast<T*>(static_cast<uint8_t*>(base) + off);
}

int check_shape(const char* what, long long rows, int K, int N) {
  if (K < 128 || K % 128 || K > kMaxK)
    return fail(DSMOE_ERR_UNSUPPORTED, "%s: in features (%d) must be a multiple of 128 up to %d", what, K, kMaxK);
  if (N < 8 || N % 8 || N > kMaxN)
    return fail(DSMOE_ERR_UNSUPPORTED, "%s: out features (%d) must be a multiple of 8 up to %d", what, N, kMaxN);
  if (rows < 0) return fail(DSMOE_ERR_INVALID, "%s: negative row count", what);
  if (rows > kMaxRows) return fail(DSMOE_ERR_UNSUPPORTED, "%s: more than %lld rows", what, kMaxRows);
  return DSMOE_OK;
}

int check_ws(const char* what, const void* ws, size_t have, size_t need) {
  if (!aligned(ws, 256)) return fail(DSMOE_ERR_INVALID, "%s: workspace NULL or not 256-byte aligned", what);
  if (have < need) return fail(DSMOE_ERR_WORKSPACE, "%s: workspace %zu bytes, need %zu", what, have, need);
  return DSMOE_OK;
}

int check_weight(const char* what, const void* codes, const void* atoms) {
  if (!aligned(codes, 32) || !aligned(atoms, 16))
    return fail(DSMOE_ERR_INVALID, "%s: weight codes must be 32-byte and scale atoms 16-byte aligned", what);
  return DSMOE_OK;
}

// A product with bf16 activations (split rows xq) or, with fp4, MXFP4 rows.
// With a.raw bf16 rows need no map.
int run_gemm(bool fp4, bool swiglu, const void* w0, const void* w1, int mats, const uint8_t* x, mx::GemmArgs& a,
             int tile, long long max_units, cudaStream_t s) {
  CUtensorMap m_w0, m_w1, m_x, m_x32, m_x8;
  const uint64_t wrows = static_cast<uint64_t>(mats) * a.M;
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int r;
  if (fp4) {
    const uint64_t kb = a.K / 2;
    if ((r = make_tma_map(&m_w0, u8, kb, w0, kb, wrows, 128, 128))) return r;
    m_w1 = m_w0;
    if ((r = make_tma_map(&m_x, u8, kb, x, kb, a.P, 128, tile))) return r;
    m_x32 = m_x8 = m_x;
  } else {
    const auto u4 = CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B;
    if ((r = make_tma_map(&m_w0, u4, a.K / 2, w0, a.K, wrows, 128, 128))) return r;
    m_w1 = m_w0;
    if (w1 != w0 && (r = make_tma_map(&m_w1, u4, a.K / 2, w1, a.K, wrows, 128, 128))) return r;
    const uint64_t rows = 2 * static_cast<uint64_t>(a.P);
    m_x = m_x32 = m_x8 = m_w0;
    if (!a.raw && (r = make_tma_map(&m_x32, u8, a.K, x, a.K, rows, 128, 32))) return r;
    if (!a.raw && (r = make_tma_map(&m_x8, u8, a.K, x, a.K, rows, 128, 8))) return r;
    if (tile > 64 &&  // smaller ones never load as one box
        (r = make_tma_map(&m_x, u8, a.K, x, a.K, rows, 128, tile))) return r;
  }
  // Persistent CTAs, or clusters of one tile each, one unit per CTA. All clusters fit
  // the device (pick_ksplit); where fewer SMs may be used they come in several
  // launches of as many whole clusters as fit, at least one: the split, and so the
  // order of the sums, stays.
  const int sms = gemm_grid();
  const long long most = a.ksplit == 1 ? sms : sms < a.ksplit ? a.ksplit : sms / a.ksplit * a.ksplit;
  const long long end = a.ksplit == 1 ? 1 : max_units;
  for (long long u = 0; u < end; u += most) {
    a.unit0 = static_cast<int>(u);
    const int grid = static_cast<int>(max_units - u < most ? max_units - u : most);
    MX_CUDA(mx::launch_gemm(!gemm_limited(), fp4, swiglu, m_w0, m_w1, m_x, m_x32, m_x8, a, tile, grid, s));
  }
  return DSMOE_OK;
}

mx::Groups tables(const Plan& L, void* ws, int n) {
  return {at<int32_t>(ws, L.counts), at<int32_t>(ws, L.row_start), at<int32_t>(ws, L.tile_start), n, 0};
}

}  // namespace

extern "C" {

int dsmoe_mxfp4_quantize(const void* x, int32_t dtype, int64_t rows, int32_t cols, int64_t row_stride,
                         const float* scale_inv, int64_t rows_per_matrix, void* codes, void* scales,
                         dsmoe_stream_t stream) {
  if (dtype < DSMOE_BF16 || dtype > DSMOE_E4M3) return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: unknown dtype %d", dtype);
  if (cols < 32 || cols % 32) return fail(DSMOE_ERR_UNSUPPORTED, "mxfp4_quantize: cols (%d) must be a multiple of 32", cols);
  if (rows < 0) return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: negative row count");
  if (rows == 0) return DSMOE_OK;
  if (rows > (0xffffffe0ll * 8) / cols) return fail(DSMOE_ERR_UNSUPPORTED, "mxfp4_quantize: more than 2^35 numbers");
  const int size = dtype == DSMOE_F32 ? 4 : dtype == DSMOE_E4M3 ? 1 : 2;
  if (!aligned(x, 16) || !aligned(codes, 8) || !scales)
    return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: pointer NULL, x not 16-byte or codes not 8-byte aligned");
  if (rows > 1 && (row_stride < cols || row_stride * size % 16))
    return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: rows must not overlap and must start on 16 bytes");
  if (dtype == DSMOE_E4M3) {
    if (!aligned(scale_inv, 4)) return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: e4m3 needs its block scales");
    if (rows_per_matrix < 1 || rows % rows_per_matrix)
      return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: rows_per_matrix must divide rows");
  } else if (scale_inv) {
    return fail(DSMOE_ERR_INVALID, "mxfp4_quantize: block scales go with e4m3 only");
  } else {
    rows_per_matrix = rows;
  }
  MX_CUDA(mx::launch_quantize(x, dtype, rows, cols, row_stride, scale_inv, rows_per_matrix,
                              static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
                              reinterpret_cast<cudaStream_t>(stream)));
  return DSMOE_OK;
}

int dsmoe_mxfp4_dequantize(const void* codes, const void* scales, int64_t blocks, int32_t dtype, void* out,
                           dsmoe_stream_t stream) {
  if (dtype < DSMOE_BF16 || dtype > DSMOE_F32) return fail(DSMOE_ERR_INVALID, "mxfp4_dequantize: bf16, fp16 or fp32 output");
  if (blocks < 0) return fail(DSMOE_ERR_INVALID, "mxfp4_dequantize: negative block count");
  if (blocks == 0) return DSMOE_OK;
  if (!aligned(codes, 4) || !scales || !aligned(out, 16))
    return fail(DSMOE_ERR_INVALID, "mxfp4_dequantize: pointer NULL or unaligned");
  MX_CUDA(mx::launch_dequantize(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), blocks, dtype,
                                out, reinterpret_cast<cudaStream_t>(stream)));
  return DSMOE_OK;
}

size_t dsmoe_mxfp4_scale_atoms_bytes(int32_t matrices, int32_t out_features, int32_t in_features) {
  if (matrices < 1 || check_shape("mxfp4_scale_atoms", 0, in_features, out_features)) return 0;
  return static_cast<size_t>(matrices) * ceil_div(out_features, 256) * (in_features / 128) * 1024;
}

int dsmoe_mxfp4_scale_atoms(const void* scales, int32_t matrices, int32_t out_features, int32_t in_features,
                            void* atoms, dsmoe_stream_t stream) {
  int r = check_shape("mxfp4_scale_atoms", 0, in_features, out_features);
  if (r) return r;
  if (matrices < 1 || !aligned(scales, 4) || !aligned(atoms, 16))
    return fail(DSMOE_ERR_INVALID, "mxfp4_scale_atoms: no matrix, or pointer NULL or unaligned");
  MX_CUDA(mx::launch_tile_scales(static_cast<const uint8_t*>(scales), matrices, out_features, in_features, 256, 2,
                                 static_cast<uint8_t*>(atoms), reinterpret_cast<cudaStream_t>(stream)));
  return DSMOE_OK;
}

size_t dsmoe_mxfp4_linear_workspace_size(int32_t tokens, int32_t in_features, int32_t out_features) {
  if (check_shape("mxfp4_linear", tokens, in_features, out_features) || tokens == 0) return 0;
  return plan_linear(tokens, in_features, out_features).total;
}

int dsmoe_mxfp4_linear(const void* x, int64_t row_stride, int32_t tokens, int32_t in_features, int32_t out_features,
                       const void* codes, const void* atoms, void* out, void* workspace, size_t workspace_bytes,
                       int32_t* device_status, dsmoe_stream_t stream) {
  int r = check_shape("mxfp4_linear", tokens, in_features, out_features);
  if (r) return r;
  if (tokens == 0) return DSMOE_OK;
  if ((r = check_weight("mxfp4_linear", codes, atoms))) return r;
  if (!aligned(x, 16) || !aligned(out, 16) || !aligned(device_status, 4))
    return fail(DSMOE_ERR_INVALID, "mxfp4_linear: pointer NULL or not 16-byte aligned");
  if (tokens > 1 && (row_stride < in_features || row_stride % 8))
    return fail(DSMOE_ERR_INVALID, "mxfp4_linear: rows must not overlap and must start on 16 bytes");
  const Plan L = plan_linear(tokens, in_features, out_features);
  if ((r = check_ws("mxfp4_linear", workspace, workspace_bytes, L.total))) return r;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  mx::GemmArgs a{};
  a.g.n = 1;
  a.g.rows = tokens;
  a.M = out_features;
  a.K = in_features;
  a.P = L.P;
  a.ksplit = L.ksplit;
  a.sfa = static_cast<const uint8_t*>(atoms);
  a.sfb = at<uint8_t>(workspace, L.sf);
  a.y = static_cast<__nv_bfloat16*>(out);
  a.status = device_status;
  if (L.raw) {
    a.raw = x;
    a.raw_stride = row_stride;
  } else {
    MX_CUDA(mx::launch_split(static_cast<const __nv_bfloat16*>(x), row_stride, tokens, in_features, a.g, L.tile, nullptr,
                             nullptr, 0, 0, L.P, at<uint8_t>(workspace, L.xq), at<uint8_t>(workspace, L.sf), nullptr, 0,
                             s));
  }
  return run_gemm(false, false, codes, codes, 1, at<uint8_t>(workspace, L.xq), a, L.tile,
                  static_cast<long long>(L.units) * L.ksplit, s);
}

size_t dsmoe_mxfp4_matmul_workspace_size(int32_t tokens, int32_t in_features, int32_t out_features) {
  if (check_shape("mxfp4_matmul", tokens, in_features, out_features) || tokens == 0) return 0;
  return plan_matmul(tokens, in_features, out_features).total;
}

int dsmoe_mxfp4_matmul(const void* x_codes, const void* x_scales, int32_t tokens, int32_t in_features,
                       int32_t out_features, const void* codes, const void* atoms, void* out, void* workspace,
                       size_t workspace_bytes, int32_t* device_status, dsmoe_stream_t stream) {
  int r = check_shape("mxfp4_matmul", tokens, in_features, out_features);
  if (r) return r;
  if (tokens == 0) return DSMOE_OK;
  if ((r = check_weight("mxfp4_matmul", codes, atoms))) return r;
  if (!aligned(x_codes, 16) || !aligned(x_scales, 4) || !aligned(out, 16) || !aligned(device_status, 4))
    return fail(DSMOE_ERR_INVALID, "mxfp4_matmul: pointer NULL or unaligned");
  const Plan L = plan_matmul(tokens, in_features, out_features);
  if ((r = check_ws("mxfp4_matmul", workspace, workspace_bytes, L.total))) return r;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  mx::GemmArgs a{};
  a.g.n = 1;
  a.g.rows = tokens;
  a.M = out_features;
  a.K = in_features;
  a.P = tokens;
  a.ksplit = L.ksplit;
  a.sfa = static_cast<const uint8_t*>(atoms);
  a.sfb = at<uint8_t>(workspace, L.sf);
  a.y = static_cast<__nv_bfloat16*>(out);
  a.status = device_status;
  if (L.raw)
    a.raw = x_scales;
  else
    MX_CUDA(mx::launch_tile_scales(static_cast<const uint8_t*>(x_scales), 1, tokens, in_features, L.tile,
                                   mx::tile_atoms(L.tile), at<uint8_t>(workspace, L.sf), s));
  return run_gemm(true, false, codes, codes, 1, static_cast<const uint8_t*>(x_codes), a, L.tile,
                  static_cast<long long>(L.units) * L.ksplit, s);
}

size_t dsmoe_mxfp4_grouped_linear_workspace_size(int32_t rows, int32_t in_features, int32_t out_features,
                                                 int32_t n_experts) {
  if (check_shape("mxfp4_grouped_linear", rows, in_features, out_features) || rows == 0 || n_experts < 1 ||
      n_experts > mx::kMaxGroups)
    return 0;
  return plan_grouped(rows, in_features, n_experts).total;
}

int dsmoe_mxfp4_grouped_linear(const void* x, int64_t row_stride, int32_t rows, int32_t in_features,
                               int32_t out_features, int32_t n_experts, const int32_t* offsets, const void* codes,
                               const void* atoms, void* out, int32_t clear_rest, void* workspace,
                               size_t workspace_bytes, int32_t* device_status, dsmoe_stream_t stream) {
  int r = check_shape("mxfp4_grouped_linear", rows, in_features, out_features);
  if (r) return r;
  if (n_experts < 1 || n_experts > mx::kMaxGroups)
    return fail(DSMOE_ERR_UNSUPPORTED, "mxfp4_grouped_linear: 1 to %d experts", mx::kMaxGroups);
  if (rows == 0) return DSMOE_OK;
  if ((r = check_weight("mxfp4_grouped_linear", codes, atoms))) return r;
  if (!aligned(x, 16) || !aligned(out, 16) || !aligned(device_status, 4) || !aligned(offsets, 4))
    return fail(DSMOE_ERR_INVALID, "mxfp4_grouped_linear: pointer NULL or unaligned");
  if (rows > 1 && (row_stride < in_features || row_stride % 8))
    return fail(DSMOE_ERR_INVALID, "mxfp4_grouped_linear: rows must not overlap and must start on 16 bytes");
  const Plan L = plan_grouped(rows, in_features, n_experts);
  if ((r = check_ws("mxfp4_grouped_linear", workspace, workspace_bytes, L.total))) return r;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  mx::GemmArgs a{};
  a.g = tables(L, workspace, n_experts);
  a.M = out_features;
  a.K = in_features;
  a.P = L.P;
  a.ksplit = 1;
  a.sfa = static_cast<const uint8_t*>(atoms);
  a.sfb = at<uint8_t>(workspace, L.sf);
  a.y = static_cast<__nv_bfloat16*>(out);
  a.next = at<int32_t>(workspace, L.next);
  a.status = device_status;
  const __nv_bfloat16* rx = static_cast<const __nv_bfloat16*>(x);
  int32_t *counts = at<int32_t>(workspace, L.counts), *row_start = at<int32_t>(workspace, L.row_start),
          *tile_start = at<int32_t>(workspace, L.tile_start);
  uint8_t *xq = at<uint8_t>(workspace, L.xq), *sf = at<uint8_t>(workspace, L.sf);
  __nv_bfloat16* clear = clear_rest ? a.y : nullptr;
  if (rows <= mx::kSegmentRows) {
    a.g.rows = rows;
    a.own.offsets = offsets;
    MX_CUDA(mx::launch_segments_split(rx, row_stride, rows, in_features, offsets, n_experts, L.tile, counts, row_start,
                                      tile_start, a.next, device_status, xq, sf, clear, out_features, s));
  } else {
    MX_CUDA(mx::launch_segments(offsets, n_experts, rows, L.tile, counts, row_start, tile_start, a.next, device_status, s));
    MX_CUDA(mx::launch_split(rx, row_stride, rows, in_features, a.g, L.tile, nullptr, nullptr, 0, 0, L.P, xq, sf, clear,
                             out_features, s));
  }
  return run_gemm(false, false, codes, codes, n_experts, xq, a, L.tile,
                  L.tiles * ceil_div(out_features, 256), s);
}

static int check_moe(int32_t tokens, int32_t hidden, int32_t inter, int32_t n_routed, int32_t shared, int32_t top_k) {
  int r = check_shape("mxfp4_moe", static_cast<long long>(tokens) * (top_k + (shared ? 1 : 0)), hidden, hidden);
  if (r) return r;
  if (inter < 128 || inter % 128 || inter > kMaxK)
    return fail(DSMOE_ERR_UNSUPPORTED, "mxfp4_moe: inter (%d) must be a multiple of 128 up to %d", inter, kMaxK);
  if (shared != 0 && shared != 1) return fail(DSMOE_ERR_INVALID, "mxfp4_moe: shared must be 0 or 1");
  if (n_routed < 1 || n_routed + shared > mx::kMaxGroups)
    return fail(DSMOE_ERR_UNSUPPORTED, "mxfp4_moe: 1 to %d experts", mx::kMaxGroups);
  if (top_k < 1 || top_k > 8) return fail(DSMOE_ERR_UNSUPPORTED, "mxfp4_moe: top_k (%d) must be in [1, 8]", top_k);
  return DSMOE_OK;
}

size_t dsmoe_mxfp4_moe_workspace_size(int32_t tokens, int32_t hidden, int32_t inter, int32_t n_routed, int32_t shared,
                                      int32_t top_k) {
  if (check_moe(tokens, hidden, inter, n_routed, shared, top_k) || tokens == 0) return 0;
  return plan_moe(tokens, hidden, inter, n_routed, shared, top_k).total;
}

int dsmoe_mxfp4_moe(const void* hidden, int64_t row_stride, int32_t tokens, const dsmoe_mxfp4_experts_t* w,
                    const int64_t* topk_idx, const float* topk_w, int32_t top_k, float scale, void* out,
                    void* workspace, size_t workspace_bytes, int32_t* device_status, dsmoe_stream_t stream) {
  if (!w) return fail(DSMOE_ERR_INVALID, "mxfp4_moe: weights is NULL");
  const int H = w->hidden, F = w->inter, E = w->n_routed, shared = w->shared;
  int r = check_moe(tokens, H, F, E, shared, top_k);
  if (r) return r;
  if (!std::isfinite(scale)) return fail(DSMOE_ERR_INVALID, "mxfp4_moe: scale must be finite");
  if (tokens == 0) return DSMOE_OK;
  if ((r = check_weight("mxfp4_moe", w->gate_codes, w->gate_up_atoms)) ||
      (r = check_weight("mxfp4_moe", w->up_codes, w->gate_up_atoms)) ||
      (r = check_weight("mxfp4_moe", w->down_codes, w->down_atoms)))
    return r;
  if (!aligned(hidden, 16) || !aligned(out, 16) || !aligned(topk_idx, 8) || !aligned(topk_w, 4) ||
      !aligned(device_status, 4))
    return fail(DSMOE_ERR_INVALID, "mxfp4_moe: pointer NULL or unaligned");
  if (tokens > 1 && (row_stride < H || row_stride % 8))
    return fail(DSMOE_ERR_INVALID, "mxfp4_moe: rows must not overlap and must start on 16 bytes");
  const Plan L = plan_moe(tokens, H, F, E, shared, top_k);
  if ((r = check_ws("mxfp4_moe", workspace, workspace_bytes, L.total))) return r;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int G = E + shared;
  int32_t* pos = at<int32_t>(workspace, L.pos);
  mx::GemmArgs a{};
  a.g = tables(L, workspace, G);
  a.M = F;
  a.K = H;
  a.P = L.P;
  a.ksplit = 1;
  a.sfa = static_cast<const uint8_t*>(w->gate_up_atoms);
  a.sfb = at<uint8_t>(workspace, L.sf);
  a.hq = at<uint8_t>(workspace, L.hq);
  a.hsf = at<uint8_t>(workspace, L.hsf);
  a.next = at<int32_t>(workspace, L.next);
  a.status = device_status;
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(hidden);
  int32_t *counts = at<int32_t>(workspace, L.counts), *row_start = at<int32_t>(workspace, L.row_start),
          *tile_start = at<int32_t>(workspace, L.tile_start);
  uint8_t *xq = at<uint8_t>(workspace, L.xq), *sf = at<uint8_t>(workspace, L.sf);
  if (tokens * top_k <= mx::kRoutePairs) {
    a.own = {topk_idx, nullptr, tokens * top_k, E, shared, tokens};
    MX_CUDA(mx::launch_route_split(x, row_stride, tokens, H, topk_idx, top_k, E, shared, L.tile, L.P, counts, row_start,
                                   tile_start, a.next, pos, xq, sf, s));
  } else {
    MX_CUDA(mx::launch_route_plan(topk_idx, tokens, top_k, E, shared, L.tile, counts, row_start, tile_start, a.next, pos,
                                  s));
    MX_CUDA(mx::launch_split(x, row_stride, tokens, H, a.g, L.tile, topk_idx, pos, top_k, shared, L.P, xq, sf, nullptr, 0, s));
  }
  if ((r = run_gemm(false, true, w->gate_codes, w->up_codes, G, xq, a, L.tile,
                    L.tiles * (F / 128), s)))
    return r;
  a.M = H;
  a.K = F;
  a.sfa = static_cast<const uint8_t*>(w->down_atoms);
  a.sfb = at<uint8_t>(workspace, L.hsf);
  ++a.next;
  a.y = at<__nv_bfloat16>(workspace, L.y);
  if ((r = run_gemm(false, false, w->down_codes, w->down_codes, G, at<uint8_t>(workspace, L.hq), a, L.tile,
                    L.tiles * ceil_div(H, 256), s)))
    return r;
  MX_CUDA(mx::launch_combine(!gemm_limited(), a.y, tokens, H, pos, topk_w, top_k, shared, scale, static_cast<__nv_bfloat16*>(out), s));
  return DSMOE_OK;
}

size_t dsmoe_mxfp4_moe_forward_workspace_size(const dsmoe_moe_config_t* cfg, int32_t tokens) {
  if (!cfg || tokens <= 0 || check_moe(tokens, cfg->hidden, cfg->inter, cfg->n_routed, 1, cfg->top_k)) return 0;
  const size_t route = route_scratch_bytes(cfg, tokens);
  return route ? route + dsmoe_mxfp4_moe_workspace_size(tokens, cfg->hidden, cfg->inter, cfg->n_routed, 1, cfg->top_k) : 0;
}

int dsmoe_mxfp4_moe_forward(const dsmoe_moe_config_t* cfg, const void* gate_weight, const float* score_bias,
                            const dsmoe_mxfp4_experts_t* w, const void* hidden, int32_t tokens, void* out,
                            int64_t* topk_idx, float* topk_w, void* workspace, size_t workspace_bytes,
                            int32_t* device_status, dsmoe_stream_t stream) {
  if (!cfg || !w) return fail(DSMOE_ERR_INVALID, "mxfp4_moe_forward: config or weights is NULL");
  if (tokens < 0) return fail(DSMOE_ERR_INVALID, "mxfp4_moe_forward: negative token count");
  if (w->hidden != cfg->hidden || w->inter != cfg->inter || w->n_routed != cfg->n_routed || w->shared != 1)
    return fail(DSMOE_ERR_INVALID, "mxfp4_moe_forward: weights do not go with the config (shared expert included)");
  int r = check_moe(tokens, cfg->hidden, cfg->inter, cfg->n_routed, 1, cfg->top_k);
  if (r) return r;
  if (tokens == 0) return DSMOE_OK;
  const size_t route = route_scratch_bytes(cfg, tokens);
  if (route == 0) return DSMOE_ERR_UNSUPPORTED;  // the router's check left its message
  if (!aligned(topk_idx, 8) || !aligned(topk_w, 4) || !aligned(device_status, 4))
    return fail(DSMOE_ERR_INVALID, "mxfp4_moe_forward: pointer NULL or unaligned");
  if ((r = check_ws("mxfp4_moe_forward", workspace, workspace_bytes,
                    dsmoe_mxfp4_moe_forward_workspace_size(cfg, tokens))))
    return r;
  if ((r = route_private(cfg, hidden, gate_weight, score_bias, tokens, topk_idx, topk_w, workspace, device_status,
                         reinterpret_cast<cudaStream_t>(stream))))
    return r;
  const float scale = cfg->router_mode == DSMOE_ROUTER_V3 ? 1.0f : cfg->routed_scaling_factor;
  return dsmoe_mxfp4_moe(hidden, cfg->hidden, tokens, w, topk_idx, topk_w, cfg->top_k, scale, out,
                         at<uint8_t>(workspace, route), workspace_bytes - route, device_status, stream);
}

}  // extern "C"
