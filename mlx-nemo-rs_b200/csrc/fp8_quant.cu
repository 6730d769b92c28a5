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
// All are bound by HBM: they read and write each element once.  Measured: 16000
// x 4096 bf16 by rows 32 us (6.2 TB/s, a plain copy's rate), 4096 x 1024 f32 by
// 128 x 128 blocks 4.3 us (4.9 TB/s with the launch in it: 256 CTAs hold a block
// each in registers between its maximum and its codes); values of 16000 x 4096 codes
// in bf16 42 us (4.7 TB/s: one unit of 16 codes in flight per thread).
#include "fp8.h"
#include "fp8_quant.cuh"

namespace nrp {
namespace {

template <typename T>
__device__ __forceinline__ void load_raw(const T* p, uint4* raw) {
#pragma unroll
  for (int q = 0; q < kRawWords<T>; ++q) raw[q] = __ldg(reinterpret_cast<const uint4*>(p) + q);
}
template <typename T>
__device__ __forceinline__ void zero_raw(uint4* raw) {
#pragma unroll
  for (int q = 0; q < kRawWords<T>; ++q) raw[q] = make_uint4(0u, 0u, 0u, 0u);
}

// 1 x 128 blocks: eight lanes of 16 elements each hold a block; a lane group
// walks the blocks of the matrix (row-major) a grid-stride apart, kFly of them
// in flight.  kWhole: cols % 128 == 0, so that the blocks are one after another
// in memory.
template <typename T, bool kWhole, int kFly>
__global__ void __launch_bounds__(256)
    quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int cols, int cb,
                         uint8_t* __restrict__ codes, float* __restrict__ scales) {
  pdl_launch_dependents();
  pdl_wait();
  const int sub = threadIdx.x & 7;
  const int64_t total = rows * cb;
  const int64_t step = static_cast<int64_t>(gridDim.x) * 32;
  // element of block blk that the lane starts at, or -1
  auto place = [&](int64_t blk) -> int64_t {
    if (blk >= total) return -1;
    if (kWhole) return blk * kQBlock + sub * 16;
    const int64_t row = blk / cb;
    const int col = static_cast<int>(blk - row * cb) * kQBlock + sub * 16;
    return col < cols ? row * cols + col : -1;
  };
  // the warp's four groups stay together for the shuffles
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 5) * 4;
       base < total; base += kFly * step) {
    const int64_t first = base + ((threadIdx.x & 31) >> 3);
    uint4 raw[kFly][kRawWords<T>];
    int64_t at[kFly];
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      at[i] = place(first + i * step);
      if (at[i] >= 0) load_raw(x + at[i], raw[i]);
      else zero_raw<T>(raw[i]);
    }
#pragma unroll
    for (int i = 0; i < kFly; ++i) {
      float scale;
      const uint4 q = quantize_block<T>(raw[i], scale);
      if (at[i] >= 0) {
        *reinterpret_cast<uint4*>(codes + at[i]) = q;
        if (sub == 0) scales[first + i * step] = scale;
      }
    }
  }
}

// 128 x 128 blocks, one per CTA: a thread holds 16 elements of four rows.
template <typename T>
__global__ void __launch_bounds__(256)
    quantize_tiles_kernel(const T* __restrict__ x, int64_t rows, int cols, int cb,
                          uint8_t* __restrict__ codes, float* __restrict__ scales) {
  __shared__ uint32_t part[8];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t rb = blockIdx.x / cb;
  const int col = static_cast<int>(blockIdx.x - rb * cb) * kQBlock + (threadIdx.x & 7) * 16;
  uint4 raw[4][kRawWords<T>];
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = rb * 128 + p * 32 + (threadIdx.x >> 3);
    if (row < rows && col < cols) load_raw(x + row * cols + col, raw[p]);
    else zero_raw<T>(raw[p]);
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) m = max(m, amax_bits<T>(raw[p]));
  auto over_cta = [&](uint32_t v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) v = max(v, part[w]);
    return v;
  };
  m = over_cta(m);
  const bool finite = m < kInfBits;
  if (!finite) {  // the whole CTA
    m = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) m = max(m, finite_amax_bits<T>(raw[p]));
    __syncthreads();
    m = over_cta(m);
  }
  const int k = scale_exp(m);
  const float inv = exp2_int(-k);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t row = rb * 128 + p * 32 + (threadIdx.x >> 3);
    if (row < rows && col < cols)
      *reinterpret_cast<uint4*>(codes + row * cols + col) = codes16<T>(raw[p], inv, finite);
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
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
    if (sizeof(T) == 4 || is_power_of_two(s)) {  // f32 holds the product
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] *= s;
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = code_times(v[e], s);
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
    // two blocks in flight once every lane group has some (16000 x 4096 bf16:
    // 32.0 us, one 36.0, four 33.8); before that one (896 x 1024 takes 0.7 us less)
    const int64_t want = (rows * cb + 31) / 32, most = 8 * num_sms;
    const bool two = want >= 2 * most;
    const dim3 grid(static_cast<unsigned>(want < most ? want : most));
    auto* kernel = cols % kQBlock ? (two ? quantize_rows_kernel<T, false, 2>
                                         : quantize_rows_kernel<T, false, 1>)
                                  : (two ? quantize_rows_kernel<T, true, 2>
                                         : quantize_rows_kernel<T, true, 1>);
    return launch_pdl(kernel, grid, dim3(256), 0, stream, p, rows, cols, cb, codes, scales);
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
