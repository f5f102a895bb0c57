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
// Bound by memory: 4 threads share a block, each holding 8 numbers from one
// or two 16-byte loads; codes leave as 4 bytes per thread (128 contiguous
// bytes per warp).
#include "common.cuh"
#include "mxfp4.cuh"

#include <cuda_fp16.h>

namespace dsmoe {
namespace mx {
namespace {

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* v) {
  const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const __half* p, float* v) {
  const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
  const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float* v) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_fp8_e4m3* p, float* v) {
  const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = e4m3_to_f32(((i < 4 ? q.x : q.y) >> (8 * (i & 3))) & 0xff);
}

// w * s rounded to odd.
__device__ __forceinline__ float mul_odd(float w, float s) {
  const float p = __fmul_rz(w, s);
  const float r = __fmaf_rn(w, s, -p);
  return r != 0.f ? __uint_as_float(__float_as_uint(p) | 1u) : p;
}

__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// One thread: 8 numbers. `units` = rows * K / 8, fewer than 2^32.
template <class T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ x, uint32_t units, uint32_t per_row,
                                                       long long row_stride, const float* __restrict__ scale_inv,
                                                       uint32_t rows_per_mat, uint32_t sc_rows, uint32_t sc_cols,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  // per_row is a multiple of 4, so the 4 threads of a block are in or out
  // together; the loop bound is warp-aligned for the shuffles.
  const uint32_t bound = (units + 31) & ~31u;
  for (uint64_t u64 = blockIdx.x * 256u + threadIdx.x; u64 < bound; u64 += gridDim.x * 256u) {
    const uint32_t u = static_cast<uint32_t>(u64);
    const bool in = u < units;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (in) {
      const uint32_t row = u / per_row, c = u - row * per_row;
      load8(x + row * row_stride + c * 8, v);
      if constexpr (sizeof(T) == 1) {
        const uint32_t mat = row / rows_per_mat, r = row - mat * rows_per_mat;
        const float s = __ldg(scale_inv + (static_cast<size_t>(mat) * sc_rows + r / 128) * sc_cols + c / 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = mul_odd(v[i], s);
      }
    }
    uint32_t amax = 0;  // bit patterns of |v| order like the numbers, NaN above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const uint32_t ef = amax >> 23;
    const bool bad = ef == 255;
    const uint32_t byte = bad ? 255u : (ef > 2 ? ef - 2 : 0u);
    const float inv = __uint_as_float((254u - byte) << 23);  // 2^(127 - byte)
    uint32_t w = 0;
    if (!bad) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= e2m1x2(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
    }
    if (in) {
      reinterpret_cast<uint32_t*>(codes)[u] = w;
      if ((u & 3) == 0) scales[u >> 2] = static_cast<uint8_t>(byte);
    }
  }
}

__device__ __forceinline__ float2 e2m1_pair(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(byte));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
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

// One thread: 8 codes. code * 2^(b - 127) is exact in fp32 and bf16.
template <class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, uint64_t units,
                                                         T* __restrict__ out) {
  for (uint64_t u = blockIdx.x * 256ull + threadIdx.x; u < units; u += gridDim.x * 256ull) {
    const uint32_t w = __ldg(codes + u);
    const float s = e8m0(__ldg(scales + (u >> 2)));
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e2m1_pair((w >> (8 * i)) & 0xff);
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
    store8(out + u * 8, v);
  }
}

// One thread: the four scales of one row and K block (one word of an atom).
// Words of an atom that belong to no row are zero.
__global__ void __launch_bounds__(256) tile_scales_kernel(const uint32_t* __restrict__ scales, int mats, int N, int KB,
                                                          int tile, int atoms, uint32_t* __restrict__ out) {
  launch_dependents();
  const int tiles = (N + tile - 1) / tile;
  const uint64_t words = static_cast<uint64_t>(mats) * tiles * KB * atoms * 128;
  for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < words; i += gridDim.x * 256ull) {
    const int w = i & 127;
    uint64_t r = i >> 7;
    const int atom = r % atoms;
    r /= atoms;
    const int kb = r % KB;
    r /= KB;
    const int t = r % tiles;
    const int m = static_cast<int>(r / tiles);
    const int in_tile = atom * 128 + (w & 3) * 32 + (w >> 2);
    const int row = t * tile + in_tile;
    out[i] = in_tile < tile && row < N ? __ldg(scales + (static_cast<size_t>(m) * N + row) * KB + kb) : 0u;
  }
}

int grid_for(uint64_t units, int per_block) {
  const uint64_t b = (units + per_block - 1) / per_block;
  return static_cast<int>(b < 148 * 16 ? (b ? b : 1) : 148 * 16);
}

}  // namespace

cudaError_t launch_quantize(const void* x, int type, long long rows, int K, long long row_stride,
                            const float* scale_inv, long long rows_per_mat, uint8_t* codes, uint8_t* scales,
                            cudaStream_t s) {
  const uint32_t per_row = K / 8;
  const uint64_t units = static_cast<uint64_t>(rows) * per_row;
  const int grid = grid_for(units, 256);
  const uint32_t scr = static_cast<uint32_t>((rows_per_mat + 127) / 128), scc = (K + 127) / 128;
  const uint32_t rpm = static_cast<uint32_t>(rows_per_mat);
  auto go = [&](auto* p) {
    quantize_kernel<<<grid, 256, 0, s>>>(p, static_cast<uint32_t>(units), per_row, row_stride, scale_inv, rpm, scr, scc,
                                         codes, scales);
  };
  switch (type) {
    case kTypeBf16: go(static_cast<const __nv_bfloat16*>(x)); break;
    case kTypeF16: go(static_cast<const __half*>(x)); break;
    case kTypeF32: go(static_cast<const float*>(x)); break;
    case kTypeE4m3: go(static_cast<const __nv_fp8_e4m3*>(x)); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

cudaError_t launch_dequantize(const uint8_t* codes, const uint8_t* scales, long long blocks, int type, void* out,
                              cudaStream_t s) {
  const uint64_t units = static_cast<uint64_t>(blocks) * 4;
  const int grid = grid_for(units, 256);
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
  const int KB = K / 128;
  const uint64_t words = static_cast<uint64_t>(mats) * ((N + tile - 1) / tile) * KB * atoms * 128;
  tile_scales_kernel<<<grid_for(words, 256), 256, 0, s>>>(reinterpret_cast<const uint32_t*>(scales), mats, N, KB, tile,
                                                          atoms, reinterpret_cast<uint32_t*>(out));
  return cudaGetLastError();
}

}  // namespace mx
}  // namespace dsmoe
