// fp8_quant.cu -- block-scaled e4m3 codes of activations (one scale per 1 x
// 128 block) and weights (128 x 128), and their values.
//
// A block's scale is the smallest power of two s = 2^k with amax / s <= 448
// (e4m3's largest value), amax over the block's finite elements, k clamped to
// [-117, 119] and s = 1 for a block of zeros; a code is x / s rounded to
// nearest even.  A power of two costs no precision (e4m3 keeps its three bits
// after the leading one; up to one octave of its range goes unused) and makes
// everything after the rounding exact: x / s, and code * s in bf16 as in f32
// (k >= -117 keeps the smallest code above bf16's and f32's subnormals, k <=
// 119 keeps 448 * s finite).  NaN and infinities become the NaN code: e4m3
// has no infinity, and a saturated one would hide an overflow.
//
// Both kernels are bound by HBM: they read and write each element once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.h"
#include "sm100.cuh"

namespace nrp {
namespace {

// log2 of the scale of a block whose largest finite magnitude is `amax`.
__device__ __forceinline__ int scale_exp(float amax) {
  if (!(amax > 0.f)) return 0;
  if (amax < 1.17549435e-38f) return -117;  // subnormal: the clamp's value
  const uint32_t u = __float_as_uint(amax);
  // amax = 1.f * 2^e; 448 = 1.75 * 2^8
  const int e = static_cast<int>(u >> 23) - 127;
  const int k = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(k, -117), 119);
}

__device__ __forceinline__ float exp2_int(int k) {  // 2^k, k in [-126, 127]
  return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

// |x| where x is finite, else 0: what amax looks at.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.40282347e38f ? a : 0.f;
}

// Two codes (low byte first) of x0 * inv, x1 * inv.
__device__ __forceinline__ uint32_t codes2(float x0, float x1, float inv) {
  // an infinity times a finite power of two stays one; inf - inf is the NaN
  // the conversion needs, and finite - finite * 0 changes nothing
  const float a = fabsf(x0) <= 3.40282347e38f ? x0 * inv : __uint_as_float(0x7fc00000u);
  const float b = fabsf(x1) <= 3.40282347e38f ? x1 * inv : __uint_as_float(0x7fc00000u);
  return static_cast<uint32_t>(
      __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3));
}

// 16 consecutive elements as f32.
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p) + q);
      v[4 * q] = f.x;
      v[4 * q + 1] = f.y;
      v[4 * q + 2] = f.z;
      v[4 * q + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p) + q);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
        v[8 * q + 2 * e] = f.x;
        v[8 * q + 2 * e + 1] = f.y;
      }
    }
  }
}

__device__ __forceinline__ uint4 codes16(const float (&v)[16], float inv) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    w[q] = codes2(v[4 * q], v[4 * q + 1], inv) |
           (codes2(v[4 * q + 2], v[4 * q + 3], inv) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 1 x 128 blocks: eight lanes of 16 elements each hold a block; a lane group
// walks the blocks of the matrix (row-major) a grid-stride apart.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int cb,
                         uint8_t* __restrict__ codes, float* __restrict__ scales) {
  pdl_launch_dependents();
  pdl_wait();
  const int sub = threadIdx.x & 7;
  const int64_t total = rows * cb;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 32;
  // the warp's four groups stay together for the shuffles
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 5) * 4;
       base < total; base += step) {
    const int64_t blk = base + ((threadIdx.x & 31) >> 3);
    const int64_t row = blk / cb;
    const int col = static_cast<int>(blk - row * cb) * kQBlock + sub * 16;
    const bool in = blk < total && col < cols;
    float v[16];
    float amax = 0.f;
    if (in) {
      load16(x + row * cols + col, v);
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, finite_abs(v[e]));
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const int k = scale_exp(amax);
    if (in)
      *reinterpret_cast<uint4*>(codes + row * cols + col) = codes16(v, exp2_int(-k));
    if (blk < total && sub == 0) scales[blk] = exp2_int(k);
  }
}

// 128 x 128 blocks, one per CTA: a thread holds 16 elements of four rows.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_tiles_kernel(const T* __restrict__ x, int64_t rows, int cols, int cb,
                          uint8_t* __restrict__ codes, float* __restrict__ scales) {
  __shared__ float part[8];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t rb = blockIdx.x / cb;
  const int col = static_cast<int>(blockIdx.x - rb * cb) * kQBlock + (threadIdx.x & 7) * 16;
  float v[4][16];
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = rb * 128 + p * 32 + (threadIdx.x >> 3);
    if (row < rows && col < cols) {
      load16(x + row * cols + col, v[p]);
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, finite_abs(v[p][e]));
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) amax = fmaxf(amax, part[w]);
  const int k = scale_exp(amax);
  const float inv = exp2_int(-k);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = rb * 128 + p * 32 + (threadIdx.x >> 3);
    if (row < rows && col < cols)
      *reinterpret_cast<uint4*>(codes + row * cols + col) = codes16(v[p], inv);
  }
  if (threadIdx.x == 0) scales[blockIdx.x] = exp2_int(k);
}

// 16 codes per thread and step; row_shift 0 or 7 maps a row to its scale row.
template <typename T>
__global__ void __launch_bounds__(256)
    dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                      int64_t rows, int cols, int cb, int row_shift, T* __restrict__ x) {
  pdl_launch_dependents();
  pdl_wait();
  const int units = cols / 16;
  const int64_t total = rows * units;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / units;
    const int col = static_cast<int>(i - row * units) * 16;
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(codes + row * cols + col));
    const float s = __ldg(scales + (row >> row_shift) * cb + (col >> 7));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    float v[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>((w[e >> 1] >> (16 * (e & 1))) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * e] = f.x * s;
      v[2 * e + 1] = f.y * s;
    }
    T* o = x + row * cols + col;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<float4*>(o)[e] =
            make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        reinterpret_cast<uint4*>(o)[e] =
            make_uint4(pack_bf16x2(v[8 * e], v[8 * e + 1]), pack_bf16x2(v[8 * e + 2], v[8 * e + 3]),
                       pack_bf16x2(v[8 * e + 4], v[8 * e + 5]),
                       pack_bf16x2(v[8 * e + 6], v[8 * e + 7]));
    }
  }
}

template <typename T>
cudaError_t quantize(const void* x, int64_t rows, int cols, int block_rows, uint8_t* codes,
                     float* scales, int num_sms, cudaStream_t stream) {
  const int cb = static_cast<int>(qblocks(cols));
  const T* p = static_cast<const T*>(x);
  if (block_rows == 1) {
    const int64_t want = (rows * cb + 31) / 32;
    const int grid = static_cast<int>(want < 8 * num_sms ? want : 8 * num_sms);
    return launch_pdl(quantize_rows_kernel<T>, dim3(grid), dim3(256), 0, stream, p, rows, cols, cb,
                      codes, scales);
  }
  const int64_t blocks = qblocks(rows) * cb;
  if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
  return launch_pdl(quantize_tiles_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                    stream, p, rows, cols, cb, codes, scales);
}

}  // namespace

cudaError_t launch_fp8_quantize(bool bf16, const void* x, int64_t rows, int cols, int block_rows,
                                uint8_t* codes, float* scales, int num_sms, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  return bf16 ? quantize<__nv_bfloat16>(x, rows, cols, block_rows, codes, scales, num_sms, stream)
              : quantize<float>(x, rows, cols, block_rows, codes, scales, num_sms, stream);
}

cudaError_t launch_fp8_dequantize(bool bf16, const uint8_t* codes, const float* scales,
                                  int64_t rows, int cols, int block_rows, void* x, int num_sms,
                                  cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  const int cb = static_cast<int>(qblocks(cols)), shift = block_rows == 128 ? 7 : 0;
  const int64_t want = (rows * (cols / 16) + 255) / 256;
  const dim3 grid(static_cast<unsigned>(want < 8 * num_sms ? want : 8 * num_sms));
  return bf16 ? launch_pdl(dequantize_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, codes,
                           scales, rows, cols, cb, shift, static_cast<__nv_bfloat16*>(x))
              : launch_pdl(dequantize_kernel<float>, grid, dim3(256), 0, stream, codes, scales,
                           rows, cols, cb, shift, static_cast<float*>(x));
}

}  // namespace nrp
