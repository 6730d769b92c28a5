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
// Bound by HBM.  Forward, up to 2048 columns: a warp holds a row in registers,
// 8 consecutive elements per lane and 256-column chunk (16-byte loads), or
// one element per lane and 32-column chunk where the columns or pointers do
// not allow those.  Backward: strips of 256 columns, see there; the sums over
// rows are added up in registers, over the CTA's groups in shared memory, and
// over CTAs through distributed shared memory (few rows: one cluster) or a
// second kernel over partial rows in the caller's workspace: fixed order, no
// atomics.  Wider rows take a CTA each and read their inputs again from L1/L2.
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
// A group of W = ceil(cols / 256) warps takes kRows rows at a time, each warp
// a strip of 256 columns, a lane eight of them (consecutive, 16-byte loads,
// or 32 apart where the columns or pointers do not allow those).  dgamma and
// dbeta then cost a lane 16 registers whatever the width, and a warp has
// kRows rows' loads in flight.  The rows' two sums cross the warps of a group
// through shared memory (double buffered: one barrier per batch of rows).
constexpr int kRows = 4;
constexpr int kStripWarps = 8;         // W at most: 2048 columns
constexpr int kStripCols = 256 * kStripWarps;
constexpr int kFewRows = 1024;         // up to here one cluster takes all rows
constexpr int kFewThreads = 512;       // threads of its CTAs
constexpr int kManyThreads = 256;
constexpr int kManyParts = 2 * 148;    // CTAs of the persistent grid at most

int strip_warps(int cols) { return (cols + 255) / 256; }
int strip_groups(int cols, int threads) { return std::max(1, threads / 32 / strip_warps(cols)); }

// Partial rows of dgamma | dbeta that go through the workspace (0: none).
int norm_parts(int64_t rows, int cols) {
  if (cols > kStripCols) return static_cast<int>(std::min<int64_t>((rows + 7) / 8, 296));
  if (rows <= kFewRows) return 0;
  const int per = strip_groups(cols, kManyThreads) * kRows;
  return static_cast<int>(std::min<int64_t>((rows + per - 1) / per, kManyParts));
}

// The sums over the warp of kN = 4 or 8 values per lane, halving the values
// and the lanes that hold each: lane l ends with the sum of value l / (32 / kN).
template <int kN>
__device__ __forceinline__ float warp_sums(const float (&v)[kN], int lane) {
  float a[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) a[i] = v[i];
#pragma unroll
  for (int n = kN / 2, o = 16; n >= 1; n /= 2, o /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const bool hi = lane & o;
      a[i] = (hi ? a[i + n] : a[i]) + __shfl_xor_sync(0xffffffffu, hi ? a[i] : a[i + n], o);
    }
#pragma unroll
  for (int o = 16 / kN; o >= 1; o /= 2) a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
  return a[0];
}

// A lane's eight elements of a row as they lie in memory, and as f32.
template <typename T, bool kVec>
struct Strip {
  static constexpr int kWords = static_cast<int>(sizeof(T)) * 2;  // 8 elements
  uint32_t w[kVec ? kWords : 8];
  // p: the row's first element; col: the lane's first column
  __device__ __forceinline__ void load(const T* p, int col, int cols) {
    if constexpr (kVec) {
      if (col < cols) {
        const uint32_t* q = reinterpret_cast<const uint32_t*>(p + col);
        if constexpr (kWords == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(q);
          w[0] = v.x, w[1] = v.y;
        } else {
#pragma unroll
          for (int i = 0; i < kWords / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(q)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = 0.f;
        if (col + 32 * e < cols) load_v<1>(p + col + 32 * e, &v);
        w[e] = __float_as_uint(v);
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 4); ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (!kVec || sizeof(T) == 4) return __uint_as_float(w[e]);
    else if constexpr (sizeof(T) == 2)
      return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>((w[e >> 2] >> (16 * ((e >> 1) & 1))) & 0xffffu),
          __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      return e & 1 ? f.y : f.x;
    }
  }
};
template <typename T, bool kVec>
__device__ __forceinline__ void store_strip(T* p, int col, int cols, const float* v) {
  if constexpr (kVec) {
    if (col < cols) store_v<8>(p + col, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + 32 * e < cols) put(p + col + 32 * e, v[e]);
  }
}

// blockDim.x = 32 * W * groups.  partials [gridDim.x][2][cols], or null: the
// grid is one cluster, and dgamma and dbeta (null: not wanted) are written.
template <typename T, typename TX, bool kVec, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == kManyThreads ? 2 : 1)
    norm_bwd_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                    const T* __restrict__ dy, const float* __restrict__ mean,
                    const float* __restrict__ rstd, const float* __restrict__ gamma, int64_t rows,
                    int cols, int W, T* __restrict__ dx, float* __restrict__ partials,
                    float* __restrict__ dgamma, float* __restrict__ dbeta) {
  constexpr bool kCodes = sizeof(TX) == 1;
  extern __shared__ float col_sums[];  // [groups][2][cols]
  __shared__ __align__(16) float red[2][kThreads / 32][2 * kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int strip = warp % W, grp = warp / W, groups = static_cast<int>(blockDim.x) / 32 / W;
  const int col = strip * 256 + (kVec ? lane * 8 : lane);
  pdl_launch_dependents();
  pdl_wait();
  const int cb = (cols + kQBlock - 1) / kQBlock;
  const float inv_c = 1.f / static_cast<float>(cols);
  float ag[8], ab[8], gm[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    ag[e] = ab[e] = 0.f;
    const int c = col + (kVec ? e : 32 * e);
    gm[e] = c < cols ? gamma[c] : 0.f;
  }
  int buf = 0;
  for (int64_t row0 = (static_cast<int64_t>(blockIdx.x) * groups + grp) * kRows; row0 < rows;
       row0 += static_cast<int64_t>(gridDim.x) * groups * kRows, buf ^= 1) {
    Strip<TX, kVec> rx[kRows];
    Strip<T, kVec> ry[kRows];
    float mu[kRows], rs[kRows], sx[kRows][kCodes && !kVec ? 2 : 1];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = row0 + r;
      mu[r] = rs[r] = sx[r][0] = 0.f;
      if (kCodes && !kVec) sx[r][kCodes && !kVec ? 1 : 0] = 0.f;
      if (row < rows) {
        rx[r].load(x + row * cols, col, cols);
        ry[r].load(dy + row * cols, col, cols);
        mu[r] = mean[row];
        rs[r] = rstd[row];
        if (kCodes) {
          // a lane's columns lie in one block (kVec), or in two
          if (col < cols) sx[r][0] = xs[row * cb + (col >> 7)];
          if (!kVec && col + 128 < cols) sx[r][kVec ? 0 : 1] = xs[row * cb + (col >> 7) + 1];
        }
      } else {
        rx[r].zero();
        ry[r].zero();
      }
    }
    auto u_of = [&](int r, int e) {
      const float v = rx[r].get(e);
      return (kCodes ? fmaf(v, sx[r][kVec ? 0 : e >> 2], -mu[r]) : v - mu[r]) * rs[r];
    };
    float part[2 * kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float u = u_of(r, e), d = ry[r].get(e), g = d * gm[e];
        ag[e] = fmaf(d, u, ag[e]);
        ab[e] += d;
        c1 += g;
        c2 = fmaf(g, u, c2);
      }
      part[r] = c1;
      part[kRows + r] = c2;
    }
    // lanes past the columns hold x = 0 and dy = 0: nothing but zeros added
    const float mine = warp_sums(part, lane);
    constexpr int kHold = 16 / kRows;  // lanes that hold each sum
    float c1[kRows], c2[kRows];
    if (W == 1) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        c1[r] = __shfl_sync(0xffffffffu, mine, kHold * r) * inv_c;
        c2[r] = __shfl_sync(0xffffffffu, mine, kHold * (kRows + r)) * inv_c;
      }
    } else {
      if (lane % kHold == 0) red[buf][warp][lane / kHold] = mine;
      named_bar_sync(1 + grp, 32 * W);
      float s[2 * kRows];
#pragma unroll
      for (int i = 0; i < 2 * kRows; ++i) s[i] = 0.f;
      for (int w = 0; w < W; ++w) {
        const float4* q = reinterpret_cast<const float4*>(red[buf][grp * W + w]);
#pragma unroll
        for (int i = 0; i < kRows / 2; ++i) {
          const float4 v = q[i];
          s[4 * i] += v.x, s[4 * i + 1] += v.y, s[4 * i + 2] += v.z, s[4 * i + 3] += v.w;
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        c1[r] = s[r] * inv_c;
        c2[r] = s[kRows + r] * inv_c;
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (row0 + r >= rows) break;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        o[e] = rs[r] * (ry[r].get(e) * gm[e] - c1[r] - u_of(r, e) * c2[r]);
      store_strip<T, kVec>(dx + (row0 + r) * cols, col, cols, o);
    }
  }
  if (!partials && !dgamma) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int c = col + (kVec ? e : 32 * e);
    if (c < cols) {
      col_sums[2 * grp * cols + c] = ag[e];
      col_sums[(2 * grp + 1) * cols + c] = ab[e];
    }
  }
  __syncthreads();
  if (groups > 1) {
    for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) {
      float s = col_sums[c];
      for (int q = 1; q < groups; ++q) s += col_sums[2 * q * cols + c];
      col_sums[c] = s;
    }
    __syncthreads();
  }
  if (partials) {
    float* out = partials + static_cast<int64_t>(blockIdx.x) * 2 * cols;
    for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) out[c] = col_sums[c];
  } else {
    cluster_sync();
    const int ranks = gridDim.x;
    for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < 2 * cols; c += ranks * blockDim.x) {
      const float s = cluster_sum1(smem_u32(col_sums + c), ranks);
      if (c < cols) dgamma[c] = s;
      else dbeta[c - cols] = s;
    }
    cluster_sync();  // no CTA leaves while another reads its sums
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

template <typename T, typename TX, bool kVec, int kThreads>
cudaError_t bwd_strips(const TX* x, const T* dy, T* dx, const BwdArgs& a, cudaStream_t stream) {
  const int W = strip_warps(a.cols), groups = strip_groups(a.cols, kThreads);
  const int per = groups * kRows;
  const int64_t batches = (a.rows + per - 1) / per;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute la[2];
  la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (kThreads == kFewThreads && a.dgamma) {  // one cluster
    unsigned c = 1;
    while (c < 8 && c < batches) c *= 2;
    cfg.gridDim = dim3(c);
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = c;
    la[1].val.clusterDim.y = 1;
    la[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  } else {
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(batches, kManyParts)));
  }
  cfg.blockDim = dim3(32 * W * groups);
  // groups * W <= 16 warps of 256 columns: 32 KB at most
  cfg.dynamicSmemBytes = a.dgamma ? 8 * static_cast<size_t>(groups) * a.cols : 0;
  cfg.stream = stream;
  cfg.attrs = la;
  float* partials = kThreads == kFewThreads ? nullptr : a.partials;
  return cudaLaunchKernelEx(&cfg, norm_bwd_kernel<T, TX, kVec, kThreads>, x, a.xs, dy, a.mean,
                            a.rstd, a.gamma, a.rows, a.cols, W, dx, partials, a.dgamma, a.dbeta);
}

template <typename T, typename TX>
cudaError_t bwd(const TX* x, const T* dy, T* dx, const BwdArgs& a, cudaStream_t stream) {
  const bool vec = a.cols % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx);
  const int parts = norm_parts(a.rows, a.cols);
  cudaError_t e;
  if (a.cols <= kStripCols) {
    if (parts == 0)
      return vec ? bwd_strips<T, TX, true, kFewThreads>(x, dy, dx, a, stream)
                 : bwd_strips<T, TX, false, kFewThreads>(x, dy, dx, a, stream);
    e = vec ? bwd_strips<T, TX, true, kManyThreads>(x, dy, dx, a, stream)
            : bwd_strips<T, TX, false, kManyThreads>(x, dy, dx, a, stream);
  } else {
    const int grid = static_cast<int>(std::min<int64_t>(a.rows, 8 * 148));
    e = launch_pdl(norm_bwd_wide_kernel<T, TX>, dim3(grid), dim3(256), 0, stream, x, a.xs, dy,
                   a.mean, a.rstd, a.gamma, a.rows, a.cols, dx);
    if (e == cudaSuccess && a.dgamma)
      e = launch_pdl(norm_bwd_cols_kernel<T, TX>, dim3((a.cols + 31) / 32, parts), dim3(256), 0,
                     stream, x, a.xs, dy, a.mean, a.rstd, a.rows, a.cols, a.partials);
  }
  if (e != cudaSuccess || !a.dgamma) return e;
  return launch_pdl(norm_bwd_sum_kernel, dim3((2 * a.cols + 31) / 32), dim3(256), 0, stream,
                    static_cast<const float*>(a.partials), parts, a.cols, a.dgamma, a.dbeta);
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
  return static_cast<int64_t>(norm_parts(rows, cols)) * 2 * cols;
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
