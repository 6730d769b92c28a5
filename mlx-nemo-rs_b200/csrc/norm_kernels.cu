// norm_kernels.cu -- LayerNorm over the last dimension, forward and backward:
//
//   mean = sum x / C, rstd = (sum (x - mean)^2 / C + eps)^-1/2
//   u = (x - mean) * rstd, y = u * gamma + beta
//   g = dy * gamma, dx = rstd * (g - mean_C(g) - u * mean_C(g * u))
//   dgamma = sum_rows dy * u, dbeta = sum_rows dy
//
// in f32, each output rounded once.  The variance is summed about the mean
// (two passes over the registers), so a large mean costs no precision.  The
// backward pass takes x as it was or as the e4m3 checkpoint (codes and one
// scale per 128 columns), with the saved mean and rstd of the exact row.
//
// Bound by HBM.  Up to 1024 columns (2048 forward) a warp holds a row in
// registers, 8 consecutive elements per lane and 256-column chunk (16-byte
// loads), or one element per lane and 32-column chunk where the columns or
// pointers do not allow those.  Wider rows take a CTA each and read x again
// from L1/L2.  The backward's persistent warps add dgamma and dbeta up in
// registers over their rows, the CTA over its warps in shared memory, and a
// second kernel sums the CTAs' partial rows: fixed order, no atomics.
#include <algorithm>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.h"
#include "sm100.cuh"

namespace nrp {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ float code_value(uint8_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}

// kV consecutive elements as f32 (kV 8: 16-byte loads; or 1).
template <int kV>
__device__ __forceinline__ void load_v(const float* p, float* v) {
  if constexpr (kV == 8) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    v[0] = *p;
  }
}
template <int kV>
__device__ __forceinline__ void load_v(const __nv_bfloat16* p, float* v) {
  if constexpr (kV == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(w[e] << 16);
      v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  } else {
    v[0] = __bfloat162float(*p);
  }
}
// codes: the caller multiplies by the block's scale
template <int kV>
__device__ __forceinline__ void load_v(const uint8_t* p, float* v) {
  if constexpr (kV == 8) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    const uint32_t w[2] = {q.x, q.y};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>((w[e >> 1] >> (16 * (e & 1))) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
  } else {
    v[0] = code_value(*p);
  }
}
template <int kV>
__device__ __forceinline__ void store_v(float* p, const float* v) {
  if constexpr (kV == 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *p = v[0];
  }
}
template <int kV>
__device__ __forceinline__ void store_v(__nv_bfloat16* p, const float* v) {
  if constexpr (kV == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                              pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  else
    *p = __float2bfloat16_rn(v[0]);
}

// ------------------------------------------------------------- forward
// One warp per row of at most kCh * 32 * kV columns.
template <typename T, int kV, int kCh>
__global__ void __launch_bounds__(256)
    norm_fwd_kernel(const T* x, int64_t rows, int cols, const float* __restrict__ gamma,
                    const float* __restrict__ beta, float eps, T* y, float* __restrict__ mean_out,
                    float* __restrict__ rstd_out) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  pdl_launch_dependents();
  if (row >= rows) return;
  pdl_wait();
  const T* xr = x + row * cols;
  float v[kCh][kV];
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    const int col = (c * 32 + lane) * kV;
    if (col < cols) {
      load_v<kV>(xr + col, v[c]);
#pragma unroll
      for (int e = 0; e < kV; ++e) s += v[c][e];
    }
  }
  const float mean = warp_sum(s) / static_cast<float>(cols);
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < kCh; ++c)
    if ((c * 32 + lane) * kV < cols) {
#pragma unroll
      for (int e = 0; e < kV; ++e) {
        v[c][e] -= mean;
        q = fmaf(v[c][e], v[c][e], q);
      }
    }
  const float rstd = 1.f / sqrtf(warp_sum(q) / static_cast<float>(cols) + eps);
  T* yr = y + row * cols;
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    const int col = (c * 32 + lane) * kV;
    if (col < cols) {
      float g[kV], b[kV], o[kV];
      load_v<kV>(gamma + col, g);
      load_v<kV>(beta + col, b);
#pragma unroll
      for (int e = 0; e < kV; ++e) o[e] = fmaf(v[c][e] * rstd, g[e], b[e]);
      store_v<kV>(yr + col, o);
    }
  }
  if (lane == 0 && mean_out) {
    mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// Sum of one value per thread over the CTA's 8 warps, to every thread.
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += part[w];
  __syncthreads();
  return s;
}

// Any width: one CTA per row, x read three times.
template <typename T>
__global__ void __launch_bounds__(256)
    norm_fwd_wide_kernel(const T* x, int64_t rows, int cols, const float* __restrict__ gamma,
                         const float* __restrict__ beta, float eps, T* y,
                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float part[8];
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * cols;
    float s = 0.f;
    for (int c = threadIdx.x; c < cols; c += 256) s += get(xr + c);
    const float mean = block_sum(s, part) / static_cast<float>(cols);
    float q = 0.f;
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float d = get(xr + c) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(block_sum(q, part) / static_cast<float>(cols) + eps);
    for (int c = threadIdx.x; c < cols; c += 256)
      put(y + row * cols + c, fmaf((get(xr + c) - mean) * rstd, gamma[c], beta[c]));
    if (threadIdx.x == 0 && mean_out) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

// ------------------------------------------------------------ backward
// CTAs of a backward pass that add up dgamma and dbeta: two per SM, and no
// more than there are groups of 8 rows.
constexpr int kNormParts = 296;
int norm_parts(int64_t rows) {
  return static_cast<int>(std::min<int64_t>((rows + 7) / 8, kNormParts));
}

// Persistent warps, a row each of at most kCh * 32 * kV columns.  TX: T, or
// uint8_t (codes).  partials [gridDim.x][2][cols], or null.
template <typename T, typename TX, int kV, int kCh>
__global__ void __launch_bounds__(256, 2)
    norm_bwd_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                    const T* __restrict__ dy, const float* __restrict__ mean,
                    const float* __restrict__ rstd, const float* __restrict__ gamma, int64_t rows,
                    int cols, T* __restrict__ dx, float* __restrict__ partials) {
  constexpr bool kCodes = sizeof(TX) == 1;
  __shared__ float red[8][32 * kV];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();
  const int cb = (cols + kQBlock - 1) / kQBlock;
  const float inv_c = 1.f / static_cast<float>(cols);
  float ag[kCh][kV], ab[kCh][kV];
#pragma unroll
  for (int c = 0; c < kCh; ++c)
#pragma unroll
    for (int e = 0; e < kV; ++e) ag[c][e] = ab[c][e] = 0.f;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp; row < rows;
       row += static_cast<int64_t>(gridDim.x) * 8) {
    const float mu = mean[row], rs = rstd[row];
    float u[kCh][kV], g[kCh][kV];
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int col = (c * 32 + lane) * kV;
      if (col < cols) {
        load_v<kV>(x + row * cols + col, u[c]);
        load_v<kV>(dy + row * cols + col, g[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int col = (c * 32 + lane) * kV;
      if (col < cols) {
        float gm[kV];
        load_v<kV>(gamma + col, gm);
        const float sx = kCodes ? xs[row * cb + (col >> 7)] : 1.f;
#pragma unroll
        for (int e = 0; e < kV; ++e) {
          const float xv = kCodes ? u[c][e] * sx : u[c][e];
          u[c][e] = (xv - mu) * rs;
          ag[c][e] = fmaf(g[c][e], u[c][e], ag[c][e]);
          ab[c][e] += g[c][e];
          g[c][e] *= gm[e];
          c1 += g[c][e];
          c2 = fmaf(g[c][e], u[c][e], c2);
        }
      }
    }
    c1 = warp_sum(c1) * inv_c;
    c2 = warp_sum(c2) * inv_c;
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int col = (c * 32 + lane) * kV;
      if (col < cols) {
        float o[kV];
#pragma unroll
        for (int e = 0; e < kV; ++e) o[e] = rs * (g[c][e] - c1 - u[c][e] * c2);
        store_v<kV>(dx + row * cols + col, o);
      }
    }
  }
  if (!partials) return;
  float* out = partials + static_cast<int64_t>(blockIdx.x) * 2 * cols;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
#pragma unroll
      for (int e = 0; e < kV; ++e) red[warp][lane * kV + e] = h ? ab[c][e] : ag[c][e];
      __syncthreads();
      if (threadIdx.x < 32 * kV) {
        const int col = c * 32 * kV + threadIdx.x;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += red[w][threadIdx.x];
        if (col < cols) out[h * cols + col] = s;
      }
      __syncthreads();
    }
}

// Any width, dx: one CTA per row, x and dy read twice.
template <typename T, typename TX>
__global__ void __launch_bounds__(256)
    norm_bwd_wide_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                         const T* __restrict__ dy, const float* __restrict__ mean,
                         const float* __restrict__ rstd, const float* __restrict__ gamma,
                         int64_t rows, int cols, T* __restrict__ dx) {
  constexpr bool kCodes = sizeof(TX) == 1;
  __shared__ float part[8];
  pdl_launch_dependents();
  pdl_wait();
  const int cb = (cols + kQBlock - 1) / kQBlock;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mu = mean[row], rs = rstd[row];
    auto u_at = [&](int c) {
      float v;
      load_v<1>(x + row * cols + c, &v);
      if (kCodes) v *= xs[row * cb + (c >> 7)];
      return (v - mu) * rs;
    };
    float c1 = 0.f, c2 = 0.f;
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float g = get(dy + row * cols + c) * gamma[c];
      c1 += g;
      c2 = fmaf(g, u_at(c), c2);
    }
    c1 = block_sum(c1, part) / static_cast<float>(cols);
    c2 = block_sum(c2, part) / static_cast<float>(cols);
    for (int c = threadIdx.x; c < cols; c += 256)
      put(dx + row * cols + c, rs * (get(dy + row * cols + c) * gamma[c] - c1 - u_at(c) * c2));
  }
}

// Any width, the partial column sums: CTA (x, y) takes 32 columns and every
// gridDim.y-th group of 8 rows.
template <typename T, typename TX>
__global__ void __launch_bounds__(256)
    norm_bwd_cols_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                         const T* __restrict__ dy, const float* __restrict__ mean,
                         const float* __restrict__ rstd, int64_t rows, int cols,
                         float* __restrict__ partials) {
  constexpr bool kCodes = sizeof(TX) == 1;
  __shared__ float red[2][8][32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const int cb = (cols + kQBlock - 1) / kQBlock;
  float ag = 0.f, ab = 0.f;
  if (col < cols)
    for (int64_t row = static_cast<int64_t>(blockIdx.y) * 8 + warp; row < rows;
         row += static_cast<int64_t>(gridDim.y) * 8) {
      float v;
      load_v<1>(x + row * cols + col, &v);
      if (kCodes) v *= xs[row * cb + (col >> 7)];
      const float d = get(dy + row * cols + col);
      ag = fmaf(d, (v - mean[row]) * rstd[row], ag);
      ab += d;
    }
  red[0][warp][lane] = ag;
  red[1][warp][lane] = ab;
  __syncthreads();
  if (warp < 2 && col < cols) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[warp][w][lane];
    partials[(static_cast<int64_t>(blockIdx.y) * 2 + warp) * cols + col] = s;
  }
}

// dgamma | dbeta = the sum of the partial rows.
__global__ void __launch_bounds__(256)
    norm_bwd_sum_kernel(const float* __restrict__ partials, int parts, int cols,
                        float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[8][32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < 2 * cols) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 8) s += partials[static_cast<int64_t>(p) * 2 * cols + i];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < 2 * cols) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[w][lane];
    if (i < cols) dgamma[i] = s;
    else dbeta[i - cols] = s;
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct FwdArgs {
  int64_t rows;
  int cols;
  const float *gamma, *beta;
  float eps;
  float *mean, *rstd;
};

template <typename T, int kV, int kCh>
cudaError_t fwd_rows(const T* x, T* y, const FwdArgs& a, cudaStream_t stream) {
  const int64_t grid = (a.rows + 7) / 8;
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  return launch_pdl(norm_fwd_kernel<T, kV, kCh>, dim3(static_cast<unsigned>(grid)), dim3(256), 0,
                    stream, x, a.rows, a.cols, a.gamma, a.beta, a.eps, y, a.mean, a.rstd);
}

template <typename T>
cudaError_t fwd(const T* x, T* y, const FwdArgs& a, int num_sms, cudaStream_t stream) {
  const bool vec = a.cols % 8 == 0 && aligned16(x) && aligned16(y) && aligned16(a.gamma) &&
                   aligned16(a.beta);
  if (vec && a.cols <= 256) return fwd_rows<T, 8, 1>(x, y, a, stream);
  if (vec && a.cols <= 512) return fwd_rows<T, 8, 2>(x, y, a, stream);
  if (vec && a.cols <= 1024) return fwd_rows<T, 8, 4>(x, y, a, stream);
  if (vec && a.cols <= 2048) return fwd_rows<T, 8, 8>(x, y, a, stream);
  if (!vec && a.cols <= 256) return fwd_rows<T, 1, 8>(x, y, a, stream);
  if (!vec && a.cols <= 1024) return fwd_rows<T, 1, 32>(x, y, a, stream);
  const int grid = static_cast<int>(std::min<int64_t>(a.rows, 8 * num_sms));
  return launch_pdl(norm_fwd_wide_kernel<T>, dim3(grid), dim3(256), 0, stream, x, a.rows, a.cols,
                    a.gamma, a.beta, a.eps, y, a.mean, a.rstd);
}

struct BwdArgs {
  const float *xs, *mean, *rstd, *gamma;
  int64_t rows;
  int cols;
  float *dgamma, *dbeta, *partials;
};

template <typename T, typename TX, int kV, int kCh>
cudaError_t bwd_rows(const TX* x, const T* dy, T* dx, const BwdArgs& a, cudaStream_t stream) {
  return launch_pdl(norm_bwd_kernel<T, TX, kV, kCh>, dim3(norm_parts(a.rows)), dim3(256), 0,
                    stream, x, a.xs, dy, a.mean, a.rstd, a.gamma, a.rows, a.cols, dx, a.partials);
}

template <typename T, typename TX>
cudaError_t bwd(const TX* x, const T* dy, T* dx, const BwdArgs& a, cudaStream_t stream) {
  const bool vec = a.cols % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) &&
                   aligned16(a.gamma);
  cudaError_t e;
  if (vec && a.cols <= 256) e = bwd_rows<T, TX, 8, 1>(x, dy, dx, a, stream);
  else if (vec && a.cols <= 512) e = bwd_rows<T, TX, 8, 2>(x, dy, dx, a, stream);
  else if (vec && a.cols <= 1024) e = bwd_rows<T, TX, 8, 4>(x, dy, dx, a, stream);
  else if (!vec && a.cols <= 256) e = bwd_rows<T, TX, 1, 8>(x, dy, dx, a, stream);
  else if (!vec && a.cols <= 1024) e = bwd_rows<T, TX, 1, 32>(x, dy, dx, a, stream);
  else {
    const int grid = static_cast<int>(std::min<int64_t>(a.rows, 8 * 148));
    e = launch_pdl(norm_bwd_wide_kernel<T, TX>, dim3(grid), dim3(256), 0, stream, x, a.xs, dy,
                   a.mean, a.rstd, a.gamma, a.rows, a.cols, dx);
    if (e == cudaSuccess && a.partials)
      e = launch_pdl(norm_bwd_cols_kernel<T, TX>, dim3((a.cols + 31) / 32, norm_parts(a.rows)),
                     dim3(256), 0, stream, x, a.xs, dy, a.mean, a.rstd, a.rows, a.cols, a.partials);
  }
  if (e != cudaSuccess || !a.partials) return e;
  return launch_pdl(norm_bwd_sum_kernel, dim3((2 * a.cols + 31) / 32), dim3(256), 0, stream,
                    static_cast<const float*>(a.partials), norm_parts(a.rows), a.cols, a.dgamma,
                    a.dbeta);
}

template <typename T>
cudaError_t bwd_typed(const void* x, const float* xs, const void* dy, void* dx, const BwdArgs& a,
                      cudaStream_t stream) {
  if (xs)
    return bwd<T, uint8_t>(static_cast<const uint8_t*>(x), static_cast<const T*>(dy),
                           static_cast<T*>(dx), a, stream);
  return bwd<T, T>(static_cast<const T*>(x), static_cast<const T*>(dy), static_cast<T*>(dx), a,
                   stream);
}

}  // namespace

cudaError_t launch_norm_fwd(bool bf16, const void* x, int64_t rows, int cols, const float* gamma,
                            const float* beta, float eps, void* y, float* mean, float* rstd,
                            int num_sms, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  const FwdArgs a{rows, cols, gamma, beta, eps, mean, rstd};
  return bf16 ? fwd(static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(y), a,
                    num_sms, stream)
              : fwd(static_cast<const float*>(x), static_cast<float*>(y), a, num_sms, stream);
}

int64_t norm_bwd_partials(int64_t rows, int cols) {
  return static_cast<int64_t>(norm_parts(rows)) * 2 * cols;
}

cudaError_t launch_norm_bwd(bool bf16, const void* x, const float* xs, const void* dy,
                            const float* mean, const float* rstd, const float* gamma,
                            int64_t rows, int cols, void* dx, float* dgamma, float* dbeta,
                            float* partials, cudaStream_t stream) {
  if (rows <= 0) {
    if (!dgamma) return cudaSuccess;
    if (cudaError_t e = cudaMemsetAsync(dgamma, 0, 4 * static_cast<size_t>(cols), stream)) return e;
    return cudaMemsetAsync(dbeta, 0, 4 * static_cast<size_t>(cols), stream);
  }
  const BwdArgs a{xs, mean, rstd, gamma, rows, cols, dgamma, dbeta, dgamma ? partials : nullptr};
  return bf16 ? bwd_typed<__nv_bfloat16>(x, xs, dy, dx, a, stream)
              : bwd_typed<float>(x, xs, dy, dx, a, stream);
}

}  // namespace nrp
