// fp8_quant.cuh -- the e4m3 quantiser's arithmetic, shared by the kernels
// that make codes (fp8_quant.cu says why the scales are powers of two).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "sm100.cuh"

namespace nrp {

// log2 of the scale of a block whose largest magnitude has the f32 bits
// `amax` (finite, not negative).
__device__ __forceinline__ int scale_exp(uint32_t amax) {
  // amax = 1.f * 2^e; 448 = 1.75 * 2^8.  Subnormals (e = -127) clamp.
  const int e = static_cast<int>(amax >> 23) - 127;
  const int k = e - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax == 0u ? 0 : min(max(k, -117), 119);
}

__device__ __forceinline__ float exp2_int(int k) {  // 2^k, k in [-126, 127]
  return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

constexpr uint32_t kInfBits = 0x7f800000u;

// 16 consecutive elements of type T, as 16-byte words, in f32.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4* raw, float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < (sizeof(T) == 4 ? 4 : 2); ++q) {
    const uint32_t w[4] = {raw[q].x, raw[q].y, raw[q].z, raw[q].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) {
        v[4 * q + e] = __uint_as_float(w[e]);
      } else {
        v[8 * q + 2 * e] = __uint_as_float(w[e] << 16);
        v[8 * q + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      }
    }
  }
}
// 16-byte words of 16 elements.
template <typename T>
constexpr int kRawWords = sizeof(T) == 4 ? 4 : 2;

// The f32 bits of the largest magnitude of 16 elements; at least kInfBits when
// one of them is not finite (bit patterns of magnitudes order like values).
template <typename T>
__device__ __forceinline__ uint32_t amax_bits(const uint4* raw) {
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      m = max(m, max(max(raw[q].x & 0x7fffffffu, raw[q].y & 0x7fffffffu),
                     max(raw[q].z & 0x7fffffffu, raw[q].w & 0x7fffffffu)));
    return m;
  } else {
    // two at a time; max.NaN keeps a NaN (as 0x7fff)
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t w[4] = {raw[q].x, raw[q].y, raw[q].z, raw[q].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[e] & 0x7fff7fffu));
    }
    return max(m << 16, m & 0xffff0000u);
  }
}
// The same over the finite elements only.
template <typename T>
__device__ __forceinline__ uint32_t finite_amax_bits(const uint4* raw) {
  float v[16];
  unpack16<T>(raw, v);
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t u = __float_as_uint(v[e]) & 0x7fffffffu;
    m = max(m, u < kInfBits ? u : 0u);
  }
  return m;
}

__device__ __forceinline__ uint32_t codes2(float a, float b) {
  return static_cast<uint32_t>(
      __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3));
}
// Codes of 16 elements times inv; finite: none of them is NaN or infinite (the
// conversion saturates an infinity, which shall be NaN).
template <typename T>
__device__ __forceinline__ uint4 codes16(const uint4* raw, float inv, bool finite) {
  float v[16];
  unpack16<T>(raw, v);
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] *= inv;
  if (!finite) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (fabsf(v[e]) == __uint_as_float(kInfBits)) v[e] = __uint_as_float(0x7fc00000u);
  }
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    w[q] = codes2(v[4 * q], v[4 * q + 1]) | (codes2(v[4 * q + 2], v[4 * q + 3]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// code * scale on its way to bf16: cut off to f32, with the last bit set where that
// loses some of the product's up to 28 bits, so that the rounding to bf16 is the only
// one (rounded to f32 first, one product in 2^17 lands on a tie that it is not).
__device__ __forceinline__ float code_times(float code, float scale) {
  const float v = __fmul_rz(code, scale);
  return __fmul_ru(code, scale) == __fmul_rd(code, scale)
             ? v
             : __uint_as_float(__float_as_uint(v) | 1u);
}
// A power of two, whose products with codes f32 holds.
__device__ __forceinline__ bool is_power_of_two(float scale) {
  return (__float_as_uint(scale) & 0x807fffffu) == 0;
}

// A 1 x 128 block held by eight lanes (a quarter of a warp), 16 elements each
// (zeros off its end): the lane's codes and, in all eight, the scale.
template <typename T>
__device__ __forceinline__ uint4 quantize_block(const uint4* raw, float& scale) {
  uint32_t m = amax_bits<T>(raw);
#pragma unroll
  for (int o = 4; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const bool finite = m < kInfBits;
  if (!finite) {  // all eight lanes or none
    const uint32_t group = 0xffu << (threadIdx.x & 24);
    m = finite_amax_bits<T>(raw);
#pragma unroll
    for (int o = 4; o; o >>= 1) m = max(m, __shfl_xor_sync(group, m, o));
  }
  const int k = scale_exp(m);
  scale = exp2_int(k);
  return codes16<T>(raw, exp2_int(-k), finite);
}

}  // namespace nrp
