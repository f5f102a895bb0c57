// MXFP4 quantisation, its inverse, and the scale layout of the products.
//
// Quantise (one pass): for each block of 32 numbers along a row, with
// a = max|v| and e = max(floor(log2 a) - 2, -127),
//   scale byte = e + 127,  code = e2m1(v * 2^-e), nearest even, saturating
// at 6. floor(log2 a) is a's fp32 exponent field, v * 2^-e is exact, so the
// codes are those of exact arithmetic. A block that holds an infinity or a
// NaN gets scale 255 (NaN) and codes 0; a zero block gets scale byte 0.
// For a checkpoint's e4m3 weight with one fp32 scale per 128x128 block,
// v = w * scale has up to 28 significant bits: it is rounded to odd at 24
// (truncated, last bit set if anything was cut off), which keeps the fp32
// exponent and every later rounding to 2 bits equal to that of the exact
// product.
//
// Bound by memory. A thread holds N numbers: 8 of fp32 (two 16-byte loads), 16
// of bf16 and fp16, a block of e4m3, so that index arithmetic, shuffles and scale
// bytes are shared by as many numbers as the registers allow; codes leave in 4-
// to 16-byte words, contiguous over the warp. Row and matrix indexes come from
// multiplications (FastDiv): two integer divisions per thread cost more than
// the quantisation. 7169 x 18432 in fp32: 90 us, 6.7 TB/s; 32 x 2048 x 7168 in
// e4m3: 135 us, 5.3 TB/s (16 numbers per thread, each rounded to odd: 225 us, at
// 70% of the issue slots).
#include "common.cuh"
#include "kernels.h"
#include "mxfp4.cuh"

#include <cuda_fp16.h>

#include <type_traits>

namespace dsmoe {
namespace mx {
namespace {

// n / d for 32-bit n by one multiplication with 2^64 / d rounded up.
struct FastDiv {
  uint32_t d, lo, hi;
  explicit FastDiv(uint32_t div) : d(div) {
    const uint64_t m = div > 1 ? ~0ull / div + 1 : 0;
    lo = static_cast<uint32_t>(m);
    hi = static_cast<uint32_t>(m >> 32);
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    if (d == 1) return n;
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * hi + __umulhi(n, lo)) >> 32);
  }
};

template <class T> struct Form { static constexpr int N = 16; };  // numbers per thread
template <> struct Form<float> { static constexpr int N = 8; };

__device__ __forceinline__ void load(const __nv_bfloat16* p, float* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + j);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[8 * j + 2 * i] = __uint_as_float(w[i] << 16);
      v[8 * j + 2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void load(const __half* p, float* v) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + j);
    const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[8 * j + 2 * i] = f.x;
      v[8 * j + 2 * i + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void load(const float* p, float* v) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
// 16 e4m3 numbers as f16 pairs (exact).
__device__ __forceinline__ void load(const __nv_fp8_e4m3* p, __half2* v) {
  const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t h;
    const uint16_t two = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
    v[i] = *reinterpret_cast<__half2*>(&h);
  }
}

// Of the two fp32 neighbours of an inexact product the one whose last bit is
// set (rounding to odd).
__device__ __forceinline__ float odd(float a, float b) { return __float_as_uint(a) & 1 ? a : b; }
__device__ __forceinline__ float mul_odd(float w, float s) { return odd(__fmul_rd(w, s), __fmul_ru(w, s)); }
// The lower and the upper neighbours of a pair's products by s.
__device__ __forceinline__ void mul_both(float2 w, float s, float* a, float* b) {
  asm("{\n\t.reg .b64 pw, ps, pa, pb;\n\t"
      "mov.b64 pw, {%4, %5};\n\t"
      "mov.b64 ps, {%6, %6};\n\t"
      "mul.rm.f32x2 pa, pw, ps;\n\t"
      "mul.rp.f32x2 pb, pw, ps;\n\t"
      "mov.b64 {%0, %1}, pa;\n\t"
      "mov.b64 {%2, %3}, pb;\n\t}"
      : "=f"(a[0]), "=f"(a[1]), "=f"(b[0]), "=f"(b[1])
      : "f"(w.x), "f"(w.y), "f"(s));
}

// 8 numbers to e2m1 codes, the first in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Scale byte of a block whose largest magnitude has the bit pattern `amax`.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const uint32_t ef = amax >> 23;
  return ef == 255 ? 255u : (ef > 2 ? ef - 2 : 0u);
}

// `units` = rows * K / N, fewer than 2^32 - 32. ROWS: rows are not back to back.
template <class T, bool ROWS>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, uint32_t units, FastDiv per_row,
                                                       long long row_stride, uint8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ scales) {
  constexpr int N = Form<T>::N;
  // A block's 32 / N threads are in or out together; the loop bound is
  // warp-aligned for the shuffles.
  const uint64_t bound = (static_cast<uint64_t>(units) + 31) & ~31ull;
  for (uint64_t u64 = blockIdx.x * 256u + threadIdx.x; u64 < bound; u64 += gridDim.x * 256u) {
    const uint32_t u = static_cast<uint32_t>(u64);
    const bool in = u64 < units;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    if (in) {
      if constexpr (ROWS) {
        const uint32_t row = per_row(u), c = u - row * per_row.d;
        load(x + row * row_stride + c * N, v);
      } else {
        load(x + static_cast<size_t>(u) * N, v);
      }
    }
    uint32_t amax = 0;  // bit patterns of |v| order like the numbers, NaN above infinity
#pragma unroll
    for (int i = 0; i < N; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 32 / N; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const uint32_t byte = scale_byte(amax);
    const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
    uint32_t w[N / 8];
#pragma unroll
    for (int j = 0; j < N / 8; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * j + i] *= inv;
      w[j] = byte == 255 ? 0 : e2m1x8(v + 8 * j);
    }
    if (in) {
      if constexpr (N == 16) reinterpret_cast<uint2*>(codes)[u] = make_uint2(w[0], w[1]);
      else reinterpret_cast<uint32_t*>(codes)[u] = w[0];
      if (u % (32 / N) == 0) scales[u / (32 / N)] = static_cast<uint8_t>(byte);
    }
  }
}

// The checkpoint's e4m3 with block scales, a block of 32 per thread. It has one
// scale_inv s (128 is a multiple of 32), so its largest product is that of its
// largest number, and s 2^-e is exact: one rounded product per number. Products
// beyond fp32 have their exponent taken 16 lower; a block of zeros keeps s as it
// is, since s times its 2^127 may not be finite. A product lies between its two
// fp32 neighbours: where both round to the same codes these are the exact
// product's; only the rare others (next to a tie) are rounded to odd.
__global__ void __launch_bounds__(256) quantize_fp8_kernel(const __nv_fp8_e4m3* __restrict__ x, uint32_t blocks,
                                                           FastDiv per_row, long long row_stride,
                                                           const float* __restrict__ scale_inv, FastDiv rows_per_mat,
                                                           uint32_t sc_rows, uint32_t sc_cols,
                                                           uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  for (uint64_t b = blockIdx.x * 256u + threadIdx.x; b < blocks; b += gridDim.x * 256u) {
    const uint32_t u = static_cast<uint32_t>(b);
    const uint32_t row = per_row(u), c = u - row * per_row.d;
    const __nv_fp8_e4m3* p = x + row * row_stride + c * 32;
    __half2 v[16];
    load(p, v);
    load(p + 16, v + 8);
    const uint32_t mat = rows_per_mat(row), r = row - mat * rows_per_mat.d;
    const float s = __ldg(scale_inv + (static_cast<size_t>(mat) * sc_rows + r / 128) * sc_cols + c / 4);
    __half2 m = __habs2(v[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) m = __hmax2_nan(m, __habs2(v[i]));
    const float wmax = __half2float(__hmax_nan(__low2half(m), __high2half(m)));
    const bool large = fabsf(s) >= 0x1p64f;
    const uint32_t amax = __float_as_uint(mul_odd(wmax, large ? s * 0x1p-16f : s)) & 0x7fffffffu;
    uint32_t byte = scale_byte(amax);
    if (large && amax && byte != 255) byte = min(byte + 16, 254u);  // from 2^55 on: far from scale_byte's lower end
    float sc = s;
    if (amax) sc *= __uint_as_float(byte < 254 ? (254u - byte) << 23 : 0x00400000u);  // 2^(127 - byte)
    uint32_t w[4], differ = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) mul_both(__half22float2(v[4 * j + i]), sc, lo + 2 * i, hi + 2 * i);
      w[j] = e2m1x8(lo);
      differ |= w[j] ^ e2m1x8(hi);
    }
    if (differ) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float q[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(v[4 * j + i]);
          q[2 * i] = mul_odd(f.x, sc);
          q[2 * i + 1] = mul_odd(f.y, sc);
        }
        w[j] = e2m1x8(q);
      }
    }
    if (byte == 255) w[0] = w[1] = w[2] = w[3] = 0;
    reinterpret_cast<uint2*>(codes)[2 * static_cast<size_t>(u)] = make_uint2(w[0], w[1]);
    reinterpret_cast<uint2*>(codes)[2 * static_cast<size_t>(u) + 1] = make_uint2(w[2], w[3]);
    scales[u] = static_cast<uint8_t>(byte);
  }
}

// 8 codes as four f16 pairs (exact).
__device__ __forceinline__ void e2m1_read(uint32_t w, __half2* h) {
  uint32_t* o = reinterpret_cast<uint32_t*>(h);
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}

__device__ __forceinline__ float e8m0(uint32_t b) {
  return __uint_as_float(b == 255 ? 0x7fffffffu : (b ? b << 23 : 0x00400000u));
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  uint4 q;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = q;
}
__device__ __forceinline__ void store8(__half* p, const float* v) {
  uint4 q;
  __half2* h = reinterpret_cast<__half2*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = q;
}
__device__ __forceinline__ void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// A thread takes 8 codes at a time, 4 such groups a block's width apart with
// their loads together. code * 2^(b - 127) is exact in fp32 and bf16. Bound by
// the stores: 470 M numbers to bf16 in 178 us, 6.7 TB/s.
template <class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, uint64_t units,
                                                         T* __restrict__ out) {
  constexpr int G = 4;
  for (uint64_t u0 = blockIdx.x * (256ull * G) + threadIdx.x; u0 < units; u0 += gridDim.x * (256ull * G)) {
    uint32_t w[G], b[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint64_t u = u0 + 256 * g;
      w[g] = u < units ? __ldg(codes + u) : 0;
      b[g] = u < units ? __ldg(scales + (u >> 2)) : 0;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint64_t u = u0 + 256 * g;
      if (u >= units) break;
      const float s = e8m0(b[g]);
      __half2 h[4];
      e2m1_read(w[g], h);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x * s;
        v[2 * i + 1] = f.y * s;
      }
      store8(out + u * 8, v);
    }
  }
}

// Scales to atoms. One block: one atom's 128 rows and up to KC K blocks, read
// along the rows (4 KC contiguous bytes each), turned in shared
// memory and written as whole atoms. Words of an atom that belong to no row are
// zero. 256 matrices of 7168 x 2048 (118 MB in and out): 74 us; read word by
// word in atom order every sector came in eight times, 148 us.
template <int KC>
__global__ void __launch_bounds__(256) tile_scales_kernel(const uint32_t* __restrict__ scales, int N, int KB, int tile,
                                                          int tiles, int atoms, uint32_t* __restrict__ out) {
  constexpr int RW = 32 / KC;  // rows of a warp's load
  __shared__ uint32_t s[KC][129];
  launch_dependents();
  const int atom = blockIdx.x % atoms, t = blockIdx.x / atoms % tiles, m = blockIdx.x / atoms / tiles;
  const int kb0 = blockIdx.y * KC, nkb = min(KC, KB - kb0);
  const int kb = threadIdx.x % KC, r0 = threadIdx.x / KC;
#pragma unroll 4
  for (int r = r0; r < 128; r += 8 * RW) {
    const int in_tile = atom * 128 + r, row = t * tile + in_tile;
    uint32_t v = 0;
    if (in_tile < tile && row < N && kb < nkb) v = __ldg(scales + (static_cast<size_t>(m) * N + row) * KB + kb0 + kb);
    s[kb][(r & 31) * 4 + (r >> 5)] = v;
  }
  __syncthreads();
  uint32_t* dst = out + ((static_cast<size_t>(m) * tiles + t) * KB + kb0) * atoms * 128 + atom * 128;
  for (int i = threadIdx.x; i < nkb * 128; i += 256) dst[static_cast<size_t>(i >> 7) * atoms * 128 + (i & 127)] = s[i >> 7][i & 127];
}

// Blocks for `units`, up to `most`; the kernels stride over the rest. Quantise:
// 64 per SM (a few waves hide one another's ends, and constants are made once for
// several steps; 16 per SM 4% slower, no limit 12%). Dequantise: no limit (16 per
// SM 18% slower).
uint64_t quant_blocks() { return 64ull * sm_count(); }
int grid_for(uint64_t units, int per_block, uint64_t most) {
  const uint64_t b = (units + per_block - 1) / per_block;
  return static_cast<int>(b < most ? (b ? b : 1) : most);
}

}  // namespace

cudaError_t launch_quantize(const void* x, int type, long long rows, int K, long long row_stride,
                            const float* scale_inv, long long rows_per_mat, uint8_t* codes, uint8_t* scales,
                            cudaStream_t s) {
  if (type == kTypeE4m3) {
    const FastDiv per_row(K / 32), rpm(static_cast<uint32_t>(rows_per_mat));
    const uint64_t blocks = static_cast<uint64_t>(rows) * per_row.d;
    quantize_fp8_kernel<<<grid_for(blocks, 256, quant_blocks()), 256, 0, s>>>(
        static_cast<const __nv_fp8_e4m3*>(x), static_cast<uint32_t>(blocks), per_row, row_stride, scale_inv, rpm,
        static_cast<uint32_t>((rows_per_mat + 127) / 128), (K + 127) / 128, codes, scales);
    return cudaGetLastError();
  }
  auto go = [&](auto* p, auto with_rows) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    constexpr bool ROWS = decltype(with_rows)::value;
    const FastDiv per_row(K / Form<T>::N);
    const uint64_t units = static_cast<uint64_t>(rows) * per_row.d;
    quantize_kernel<T, ROWS><<<grid_for(units, 256, quant_blocks()), 256, 0, s>>>(
        p, static_cast<uint32_t>(units), per_row, row_stride, codes, scales);
  };
  auto either = [&](auto* p) {
    if (rows == 1 || row_stride == K) go(p, std::false_type{});
    else go(p, std::true_type{});
  };
  switch (type) {
    case kTypeBf16: either(static_cast<const __nv_bfloat16*>(x)); break;
    case kTypeF16: either(static_cast<const __half*>(x)); break;
    case kTypeF32: either(static_cast<const float*>(x)); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_dequantize(const uint8_t* codes, const uint8_t* scales, long long blocks, int type, void* out,
                              cudaStream_t s) {
  const uint64_t units = static_cast<uint64_t>(blocks) * 4;
  const int grid = grid_for(units, 1024, 0x7fffffff);
  const uint32_t* c = reinterpret_cast<const uint32_t*>(codes);
  switch (type) {
    case kTypeBf16: dequantize_kernel<<<grid, 256, 0, s>>>(c, scales, units, static_cast<__nv_bfloat16*>(out)); break;
    case kTypeF16: dequantize_kernel<<<grid, 256, 0, s>>>(c, scales, units, static_cast<__half*>(out)); break;
    case kTypeF32: dequantize_kernel<<<grid, 256, 0, s>>>(c, scales, units, static_cast<float*>(out)); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_tile_scales(const uint8_t* scales, int mats, int N, int K, int tile, int atoms, uint8_t* out,
                               cudaStream_t s) {
  const int KB = K / 128, tiles = (N + tile - 1) / tile;
  const long long blocks = static_cast<long long>(mats) * tiles * atoms;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  auto go = [&](auto kern, int kc) {
    kern<<<dim3(static_cast<unsigned>(blocks), (KB + kc - 1) / kc), 256, 0, s>>>(
        reinterpret_cast<const uint32_t*>(scales), N, KB, tile, tiles, atoms, reinterpret_cast<uint32_t*>(out));
    return cudaGetLastError();
  };
  // Few atoms: shorter runs on more SMs.
  return blocks * ((KB + 31) / 32) < 592 ? go(tile_scales_kernel<8>, 8) : go(tile_scales_kernel<32>, 32);
}

}  // namespace mx
}  // namespace dsmoe
