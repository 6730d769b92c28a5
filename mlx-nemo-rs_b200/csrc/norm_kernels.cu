// norm_kernels.cu -- LayerNorm over the last dimension, forward and backward:
//
//   mean = sum x / C, rstd = (sum (x - mean)^2 / C + eps)^-1/2
//   u = (x - mean) * rstd, y = u * gamma + beta
//   g = dy * gamma, dx = rstd * (g - mean_C(g) - u * mean_C(g * u))
//   dgamma = sum_rows dy * u, dbeta = sum_rows dy
//
// in f32, each output rounded once.  The variance is summed about the mean (two
// passes over the registers), so a large mean costs it no digits; a row whose sums
// overflow f32 is taken again in smaller units.  The backward pass takes x as it
// was or as the e4m3 checkpoint (codes and one scale per 128 columns), with the
// saved mean and rstd of the exact row.
//
// Bound by HBM.  Up to 4096 columns, both passes take strips of 256 columns.
// The backward's sums over rows are added up in registers, over the CTA's
// groups in shared memory, and over CTAs through distributed shared memory (few
// rows: one cluster) or a second kernel over partial rows in the caller's
// workspace: fixed order, no atomics.  Wider rows take a CTA each and read their
// inputs again from L1/L2.
//
// Measured: forward, 50000 x 1024 bf16 37 us (5.5 TB/s; a plain copy of that
// size runs at 6.2), 14 x 512 f32 2.6 us; backward of 50000 x 1024 from bf16 dy
// and codes 50 us with its second kernel (5.1 TB/s; instruction issue, at 60%,
// comes close to being the bound), 749 x 512 bf16 6.2 us in two launches.
#include <algorithm>
#include <cfloat>
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
// a code: the caller multiplies by the block's scale
__device__ __forceinline__ float code_value(uint32_t c) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c), __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}
__device__ __forceinline__ float get(const uint8_t* p) { return code_value(*p); }

// Eight consecutive elements, 16-byte aligned.
__device__ __forceinline__ void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                            pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// A lane's eight elements of a row as they lie in memory, and as f32.
template <typename T, bool kVec, int kL = 32>
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
        // as it is: a conversion here would wait for the load (30000 x 777 bf16
        // backward: 49 us, 93 with it)
        w[e] = 0u;
        if (col + kL * e < cols) {
          if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(p[col + kL * e]);
          else if constexpr (sizeof(T) == 2)
            w[e] = reinterpret_cast<const uint16_t*>(p)[col + kL * e];
          else w[e] = p[col + kL * e];
        }
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(w) / 4); ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
    else if constexpr (!kVec) {
      if constexpr (sizeof(T) == 2) return __uint_as_float(w[e] << 16);
      else return code_value(w[e]);
    } else if constexpr (sizeof(T) == 2)
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
template <typename T, bool kVec, int kL = 32>
__device__ __forceinline__ void store_strip(T* p, int col, int cols, const float* v) {
  if constexpr (kVec) {
    if (col < cols) store8(p + col, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + kL * e < cols) put(p + col + kL * e, v[e]);
  }
}

// Packed pairs of f32 (one instruction for two elements).
struct F2 {
  float a, b;
};
__device__ __forceinline__ F2 mul2(F2 x, F2 y) {
  F2 r;
  asm("{\n .reg .b64 rx, ry;\n mov.b64 rx, {%2, %3};\n mov.b64 ry, {%4, %5};\n"
      " mul.rn.f32x2 rx, rx, ry;\n mov.b64 {%0, %1}, rx;\n}"
      : "=f"(r.a), "=f"(r.b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b));
  return r;
}
__device__ __forceinline__ F2 add2(F2 x, F2 y) {
  F2 r;
  add_f32x2(r.a, r.b, x.a, x.b, y.a, y.b);
  return r;
}
__device__ __forceinline__ F2 fma2(F2 x, F2 y, F2 z) {
  F2 r;
  asm("{\n .reg .b64 rx, ry, rz;\n mov.b64 rx, {%2, %3};\n mov.b64 ry, {%4, %5};\n"
      " mov.b64 rz, {%6, %7};\n fma.rn.f32x2 rx, rx, ry, rz;\n mov.b64 {%0, %1}, rx;\n}"
      : "=f"(r.a), "=f"(r.b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b), "f"(z.a), "f"(z.b));
  return r;
}
__device__ __forceinline__ F2 both(float v) { return {v, v}; }

// gamma or beta at a strip's eight columns of a lane (zeros off the end); kVec:
// all of them are inside or none.
template <bool kVec, int kL = 32>
__device__ __forceinline__ void lane_columns(const float* __restrict__ p, int col, int cols,
                                             F2 (&v)[4]) {
  if (kVec && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (col < cols) {
      a = reinterpret_cast<const float4*>(p + col)[0];
      b = reinterpret_cast<const float4*>(p + col)[1];
    }
    v[0] = {a.x, a.y}, v[1] = {a.z, a.w}, v[2] = {b.x, b.y}, v[3] = {b.z, b.w};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c0 = col + (kVec ? 2 * e : 2 * kL * e), c1 = c0 + (kVec ? 1 : kL);
    v[e] = {c0 < cols ? p[c0] : 0.f, c1 < cols ? p[c1] : 0.f};
  }
}

// ------------------------------------------------------------- forward
// A group of W = ceil(cols / 256) warps takes kR rows at a time, each warp a
// strip of 256 columns, a lane eight of them, with the next rows' loads in
// flight.  gamma and beta then stay in 16 registers of a lane: a
// warp that takes whole rows reads 8 bytes of them from L1 for every element
// (50000 x 1024 bf16: 44 us at best).  A strip's mean and sum of squares about
// it are joined through shared memory, one barrier per batch (double
// buffered): with n_w columns each,
//   mean = sum n_w mean_w / C,  M2 = sum M2_w + n_w (mean_w - mean)^2.
constexpr int kStripCols = 2048;  // W at most 8, in CTAs of 256 threads
constexpr int kWideCols = 4096;   // W at most 16, in CTAs of 512
int strip_warps(int cols) { return (cols + 255) / 256; }
int strip_groups(int cols, int threads) { return std::max(1, threads / 32 / strip_warps(cols)); }

// W rounded up to a power of two (lanes of a row when the strips are joined).
__device__ __forceinline__ int strips_pow2(int W) { return W <= 1 ? 1 : 1 << (32 - __clz(W - 1)); }

// The sums over each kL lanes of kN = 2, 4 or 8 <= kL values per lane, halving the
// values and the lanes that hold each: lane l of them ends with the sum of value
// l / (kL / kN).
template <int kL = 32, int kN>
__device__ __forceinline__ float warp_sums(const float (&v)[kN], int lane) {
  float a[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) a[i] = v[i];
#pragma unroll
  for (int n = kN / 2, o = kL / 2; n >= 1; n /= 2, o /= 2)
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const bool hi = lane & o;
      a[i] = (hi ? a[i + n] : a[i]) + __shfl_xor_sync(0xffffffffu, hi ? a[i] : a[i + n], o);
    }
#pragma unroll
  for (int o = kL / 2 / kN; o >= 1; o /= 2) a[0] += __shfl_xor_sync(0xffffffffu, a[0], o);
  return a[0];
}

// Rows whose sum or sum of squares overflows f32 (a spread of about 2^64) are taken
// again times 2^-84: the squares of any f32 values are then in range, over 2^31
// columns too.
constexpr float kFar = 0x1p-84f, kFarInv = 0x1p84f;
__device__ __forceinline__ bool variance_overflows(float v) { return !(v <= FLT_MAX); }
// 1 / sqrt(variance + eps) of a row, times 2^84, from the variance v of the row times
// 2^-84.
__device__ __forceinline__ float far_rstd(float v, float eps) {
  if (v >= 0x1p-120f) return 1.f / sqrtf(v + eps * kFar * kFar);
  return kFarInv / sqrtf(v * kFarInv * kFarInv + eps);  // next to no spread: the sum overflowed
}

// The row's mean from that of the row times 2^-84, which may have been rounded past
// the largest value.
__device__ __forceinline__ float far_mean(float m) {
  return fabsf(m) <= FLT_MAX * kFar * 1.001f ? fminf(fmaxf(m * kFarInv, -FLT_MAX), FLT_MAX)
                                             : m * kFarInv;
}

constexpr int kFwdThreads = 256;
// CTAs per SM of a kernel that takes kR rows at a time (kR W <= 32).
template <int kR, int kThreads>
constexpr int kFwdCtas = kThreads > kFwdThreads ? 1 : kR == 4 ? 2 : 3;

template <typename T, bool kVec, int kR, int kThreads>
__global__ void __launch_bounds__(kThreads, kFwdCtas<kR, kThreads>)
    norm_fwd_kernel(const T* x, int64_t rows, int cols, int W, const float* __restrict__ gamma,
                    const float* __restrict__ beta, float eps, T* y, float* __restrict__ mean_out,
                    float* __restrict__ rstd_out) {
  __shared__ float2 red[2][kThreads / 32][kR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int strip = warp % W, grp = warp / W, groups = static_cast<int>(blockDim.x) / 32 / W;
  const int col = strip * 256 + (kVec ? lane * 8 : lane);
  pdl_launch_dependents();
  pdl_wait();
  const float inv_n = 1.f / static_cast<float>(min(256, cols - strip * 256));
  const int Wp = strips_pow2(W), at_w = lane % Wp, at_r = lane / Wp;
  const float at_n = at_w < W ? static_cast<float>(min(256, cols - at_w * 256)) : 0.f;
  const float inv_c = 1.f / static_cast<float>(cols);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * groups * kR;
  int64_t row0 = (static_cast<int64_t>(blockIdx.x) * groups + grp) * kR;
  Strip<T, kVec> next[kR];
  auto load = [&](int64_t r0) {
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (r0 + r < rows) next[r].load(x + (r0 + r) * cols, col, cols);
      else next[r].zero();
    }
  };
  load(row0);
  // columns of the lane's pair e
  auto c0 = [&](int e) { return col + (kVec ? 2 * e : 64 * e); };
  auto c1 = [&](int e) { return c0(e) + (kVec ? 1 : 32); };
  F2 gm[4], bt[4];
  lane_columns<kVec>(gamma, col, cols, gm);
  lane_columns<kVec>(beta, col, cols, bt);
  int buf = 0;
  for (; row0 < rows; row0 += stride) {
    F2 v[kR][4];
    float part[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      F2 s = both(0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[r][e] = {next[r].get(2 * e), next[r].get(2 * e + 1)};
        s = add2(s, v[r][e]);  // columns past the end are zeros
      }
      part[r] = s.a + s.b;
    }
    // (y may be x: these rows are in registers, and the next are others)
    load(row0 + stride);
    constexpr int kHold = 32 / kR;  // lanes that hold each sum
    const int per = W == 1 ? kHold : Wp;  // ... and each row's when the strips are joined
    float mean[kR], rstd[kR];
    // From the lane's sums of the rows: the rows' means and, in lane l, the variance of
    // row l / per.
    auto stats = [&]() {
      // lane l: the strip's mean of row l / kHold, then its sum of squares
      const float mean_w = warp_sums(part, lane) * inv_n;
#pragma unroll
      for (int r = 0; r < kR; ++r) mean[r] = __shfl_sync(0xffffffffu, mean_w, kHold * r);
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        F2 q = both(0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          F2 d = add2(v[r][e], both(-mean[r]));
          if (!kVec) d = {c0(e) < cols ? d.a : 0.f, c1(e) < cols ? d.b : 0.f};
          q = fma2(d, d, q);
        }
        part[r] = !kVec || col < cols ? q.a + q.b : 0.f;  // (the others hold -mean)
      }
      const float m2_w = warp_sums(part, lane);
      if (W == 1) return m2_w * inv_c;
      if (lane % kHold == 0) red[buf][warp][lane / kHold] = make_float2(mean_w, m2_w);
      named_bar_sync(1 + grp, 32 * W);
      // lane (r, w) takes strip w's share of row r
      const bool mine = at_w < W && at_r < kR;
      const float2 p = mine ? red[buf][grp * W + at_w][at_r] : make_float2(0.f, 0.f);
      float m = p.x * at_n * inv_c;
      for (int o = Wp / 2; o; o /= 2) m += __shfl_xor_sync(0xffffffffu, m, o);
      const float d = p.x - m;
      float t = fmaf(d * d, at_n, p.y);
      for (int o = Wp / 2; o; o /= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
#pragma unroll
      for (int r = 0; r < kR; ++r) mean[r] = __shfl_sync(0xffffffffu, m, Wp * r);
      buf ^= 1;
      return t * inv_c;
    };
    const float var = stats() + eps;
    float rs = 1.f / sqrtf(var);
    // (alike in a group's warps, which hold the same sums)
    const uint32_t far = __ballot_sync(0xffffffffu, variance_overflows(var));
    if (far) {
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const F2 f = both(far >> (per * r) & 1 ? kFar : 1.f);
        F2 s = both(0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[r][e] = mul2(v[r][e], f);
          s = add2(s, v[r][e]);
        }
        part[r] = s.a + s.b;
      }
      const float far_var = stats();
      if (far >> lane & 1) rs = far_rstd(far_var, eps);
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) rstd[r] = __shfl_sync(0xffffffffu, rs, per * r);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (row0 + r >= rows) break;
      float o[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const F2 u = mul2(add2(v[r][e], both(-mean[r])), both(rstd[r]));
        const F2 f = fma2(u, gm[e], bt[e]);
        o[2 * e] = f.a;
        o[2 * e + 1] = f.b;
      }
      store_strip<T, kVec>(y + (row0 + r) * cols, col, cols, o);
      if (mean_out && strip == 0 && lane == 0) {
        const bool up = far >> (per * r) & 1;
        mean_out[row0 + r] = up ? far_mean(mean[r]) : mean[r];
        rstd_out[row0 + r] = up ? rstd[r] * kFar : rstd[r];
      }
    }
  }
}

// A row whose variance overflows, by a warp, x read three times.
template <typename T>
__device__ __noinline__ void far_row(const T* x, int cols, const float* gamma, const float* beta,
                                     float eps, T* y, float* mean_out, float* rstd_out) {
  const int lane = threadIdx.x & 31;
  const float inv_c = 1.f / static_cast<float>(cols);
  float s = 0.f, q = 0.f;
  for (int c = lane; c < cols; c += 32) s = fmaf(get(x + c), kFar, s);
  const float mean = warp_sum(s) * inv_c;
  for (int c = lane; c < cols; c += 32) {
    const float d = fmaf(get(x + c), kFar, -mean);
    q = fmaf(d, d, q);
  }
  const float rstd = far_rstd(warp_sum(q) * inv_c, eps);
  for (int c = lane; c < cols; c += 32)
    put(y + c, fmaf(fmaf(get(x + c), kFar, -mean) * rstd, gamma[c], beta[c]));
  if (lane == 0 && mean_out) {
    *mean_out = far_mean(mean);
    *rstd_out = rstd * kFar;
  }
}

// Columns or pointers that do not allow 16-byte loads: a warp's whole row, of at
// most kCh strips, a lane's elements 32 apart.
constexpr int kRowThreads = 128;
// CTAs per SM by strips: 64, 48 and 40 registers.
template <int kCh>
constexpr int kRowCtas = kCh == 4 ? 8 : kCh == 2 ? 10 : 12;
template <typename T, int kCh>
__global__ void __launch_bounds__(kRowThreads, kRowCtas<kCh>)
    norm_fwd_rows_kernel(const T* x, int64_t rows, int cols, const float* __restrict__ gamma,
                         const float* __restrict__ beta, float eps, T* y,
                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  const int lane = threadIdx.x & 31;
  const int64_t row =
      static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  pdl_launch_dependents();
  if (row >= rows) return;
  pdl_wait();
  const float inv_c = 1.f / static_cast<float>(cols);
  // column of the lane's element e of strip c
  auto col_of = [&](int c, int e) { return c * 256 + lane + 32 * e; };
  Strip<T, false> v[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) v[c].load(x + row * cols, col_of(c, 0), cols);
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < kCh; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[c].get(e);  // columns past the end are zeros
  const float mean = warp_sum(s) * inv_c;
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < kCh; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = v[c].get(e) - mean;
      if (col_of(c, e) < cols) q = fmaf(d, d, q);
    }
  const float var = warp_sum(q) * inv_c + eps;
  if (variance_overflows(var)) {  // (the whole warp)
    far_row(x + row * cols, cols, gamma, beta, eps, y + row * cols,
            mean_out ? mean_out + row : nullptr, mean_out ? rstd_out + row : nullptr);
    return;
  }
  const float rstd = 1.f / sqrtf(var);
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = col_of(c, e);
      o[e] = i < cols ? fmaf((v[c].get(e) - mean) * rstd, gamma[i], beta[i]) : 0.f;
    }
    store_strip<T, false>(y + row * cols, col_of(c, 0), cols, o);
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

// A thread's consecutive elements of a wide row, 8 where its address allows 16-byte
// loads (4000 x 8192 bf16: forward 36 us, 60 by single elements; backward 88, 206).
template <bool kVec>
constexpr int kPiece = kVec ? 8 : 1;
template <typename T, bool kVec>
struct Piece {
  float v[kPiece<kVec>];
  __device__ __forceinline__ explicit Piece(const T* p) {
    if constexpr (kVec) {
      Strip<T, true> s;
      s.load(p, 0, 1);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s.get(e);
    } else {
      v[0] = get(p);
    }
  }
};
template <bool kVec, typename T>
__device__ __forceinline__ void put_piece(T* p, const float* v) {
  if constexpr (kVec) store8(p, v);
  else put(p, v[0]);
}

// Any width: one CTA per row, x read three times.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256)
    norm_fwd_wide_kernel(const T* x, int64_t rows, int cols, const float* __restrict__ gamma,
                         const float* __restrict__ beta, float eps, T* y,
                         float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  constexpr int kE = kPiece<kVec>;
  __shared__ float part[8];
  pdl_launch_dependents();
  pdl_wait();
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * cols;
    float mean, rstd, f = 1.f;  // (f 1: the fma with it is an addition)
    while (true) {
      float s = 0.f;
      for (int c = threadIdx.x * kE; c < cols; c += 256 * kE) {
        const Piece<T, kVec> p(xr + c);
#pragma unroll
        for (int e = 0; e < kE; ++e) s = fmaf(p.v[e], f, s);
      }
      mean = block_sum(s, part) / static_cast<float>(cols);
      float q = 0.f;
      for (int c = threadIdx.x * kE; c < cols; c += 256 * kE) {
        const Piece<T, kVec> p(xr + c);
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float d = fmaf(p.v[e], f, -mean);
          q = fmaf(d, d, q);
        }
      }
      const float var = block_sum(q, part) / static_cast<float>(cols);
      rstd = f == 1.f ? 1.f / sqrtf(var + eps) : far_rstd(var, eps);
      if (f != 1.f || !variance_overflows(var + eps)) break;  // (the whole CTA)
      f = kFar;
    }
    for (int c = threadIdx.x * kE; c < cols; c += 256 * kE) {
      Piece<T, kVec> p(xr + c);
      const Piece<float, kVec> gm(gamma + c), bt(beta + c);
#pragma unroll
      for (int e = 0; e < kE; ++e)
        p.v[e] = fmaf(fmaf(p.v[e], f, -mean) * rstd, gm.v[e], bt.v[e]);
      put_piece<kVec>(y + row * cols + c, p.v);
    }
    if (threadIdx.x == 0 && mean_out) {
      mean_out[row] = f == 1.f ? mean : far_mean(mean);
      rstd_out[row] = rstd * f;
    }
  }
}

// ------------------------------------------------------------ backward
// Groups of W warps and strips of columns as in the forward pass: dgamma and
// dbeta cost a lane 16 registers whatever the width.  The rows' two sums cross
// the warps of a group through shared memory.
// A batch is kR rows: 2, or 4 where the rows wait in shared memory (bf16 dy,
// 16-byte copies, W <= 4: 2 kR W <= 32 lanes when the strips are joined).
constexpr int kRingWarps = 4;
// Up to this many elements (of whole strips) one cluster takes all rows, in one
// launch: the same time on the device, 2.3 us less on the host (bf16 128 x 512
// 5.3 us and 4.7 against 5.2 and 7.0 in two launches, 256 x 512 6.3 against 5.7,
// 64 x 2048 7.2 against 5.3; f32 64 x 512 6.6 against 5.3).
constexpr int64_t kFewElements = 1 << 16;
constexpr int kFewThreads = 512;       // threads of its CTAs
constexpr int kManyThreads = 256;
// Rows of up to 128 columns take half a warp each (30000 x 64 bf16: 8.7 us, 12.2 with
// a warp to a row; x 77 10.5 against 14.4).
constexpr int kNarrowLanes = 16, kNarrow = 8 * kNarrowLanes;
// CTAs of the persistent grid, two to an SM, at most: the workspace is asked for
// without a device and has room for those of 148 SMs.
constexpr int kManyParts = 2 * 148;

// The most partial rows of dgamma | dbeta that go through the workspace (0: none).
int norm_parts(int64_t rows, int cols) {
  if (cols > kWideCols) return static_cast<int>(std::min<int64_t>((rows + 7) / 8, kManyParts));
  if (cols > kStripCols) return static_cast<int>(std::min<int64_t>(rows, kManyParts / 2));
  if (rows <= kFewElements / (256 * strip_warps(cols))) return 0;
  const int per = strip_groups(cols, kManyThreads) * 2;
  return static_cast<int>(std::min<int64_t>((rows + per - 1) / per, kManyParts));
}

// kR rows of a lane's strip.
template <typename T, typename TX, bool kVec, int kR, int kL>
struct Batch {
  static constexpr int kScales = sizeof(TX) == 1 ? (kVec ? 1 : 2) : 0;
  Strip<TX, kVec, kL> x[kR];
  Strip<T, kVec, kL> dy[kR];
  float mu[kR], rs[kR], sx[kR][kScales ? kScales : 1];
  __device__ __forceinline__ void load(const TX* px, const float* xs, const T* pdy,
                                       const float* mean, const float* rstd, int64_t row0,
                                       int64_t rows, int cols, int cb, int col) {
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int64_t row = row0 + r;
      mu[r] = rs[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kScales; ++i) sx[r][i] = 0.f;
      if (row < rows) {
        x[r].load(px + row * cols, col, cols);
        dy[r].load(pdy + row * cols, col, cols);
        // (lanes past the columns keep u = 0, whatever the row's mean times rstd)
        if (!kVec || col < cols) mu[r] = mean[row];
        rs[r] = rstd[row];
        // a lane's columns lie in one block (kVec), or in two
#pragma unroll
        for (int i = 0; i < kScales; ++i)
          if (col + 128 * i < cols) sx[r][i] = xs[row * cb + (col >> 7) + i];
      } else {
        x[r].zero();
        dy[r].zero();
      }
    }
  }
};

// The ring of the rows on their way: kDepth batches, each thread its own columns
// in its own places ([piece][thread], no barrier), a warp the rows' mean, rstd
// and scales in 16 floats.  It frees the registers that the next batch takes
// otherwise for four rows at a time, which share the reductions, the barrier and
// the addresses: those are two thirds of the instructions (50000 x 1024, bf16
// dy and codes: 59.5 us with two rows in registers and their next on the way, 56.5
// with two rows and this ring, 49.2 with four; 50.3 three batches deep).  f32 runs
// at the rate of a copy with two rows in registers (100 us; 161 with this ring).
template <typename T, typename TX, int kR>
struct Ring {
  static constexpr int kDepth = 2;
  static constexpr int kBytes = kR * 8 * static_cast<int>(sizeof(T) + sizeof(TX));  // per thread
  static constexpr int kSlot = kManyThreads * kBytes + kManyThreads / 32 * 64;
};
template <int kN>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool read) {
  const int n = read ? kN : 0;  // else zeros
  if constexpr (kN == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kN),
                 "r"(n)
                 : "memory");
}
// Eight elements of a row into thread-strided pieces of up to 16 bytes.
template <typename E>
__device__ __forceinline__ uint32_t copy_strip(uint32_t at, int threads, const E* p, bool read) {
  constexpr int kAll = 8 * static_cast<int>(sizeof(E)), kPiece = kAll < 16 ? kAll : 16;
#pragma unroll
  for (int i = 0; i < kAll / kPiece; ++i) {
    copy_async<kPiece>(at + threadIdx.x * kPiece, reinterpret_cast<const uint8_t*>(p) + i * kPiece,
                       read);
    at += threads * kPiece;
  }
  return at;
}
template <typename E>
__device__ __forceinline__ const uint8_t* take_strip(const uint8_t* at, int threads,
                                                     Strip<E, true>& s) {
  constexpr int kAll = 8 * static_cast<int>(sizeof(E)), kPiece = kAll < 16 ? kAll : 16;
#pragma unroll
  for (int i = 0; i < kAll / kPiece; ++i) {
    if constexpr (kPiece == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(at + threadIdx.x * 8);
      s.w[0] = v.x, s.w[1] = v.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(at + threadIdx.x * 16);
      s.w[4 * i] = v.x, s.w[4 * i + 1] = v.y, s.w[4 * i + 2] = v.z, s.w[4 * i + 3] = v.w;
    }
    at += threads * kPiece;
  }
  return at;
}

// blockDim.x = 32 * W * groups.  partials [gridDim.x][2][cols], or null: the
// grid is one cluster, and dgamma and dbeta (null: not wanted) are written.
// kL < 32 (W is 1): each kL lanes take rows of their own, of 8 kL columns at most.
template <typename T, typename TX, bool kVec, int kThreads, int kR, int kL>
__global__ void __launch_bounds__(kThreads, kThreads == kManyThreads ? 2 : 1)
    norm_bwd_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                    const T* __restrict__ dy, const float* __restrict__ mean,
                    const float* __restrict__ rstd, const float* __restrict__ gamma, int64_t rows,
                    int cols, int W, T* __restrict__ dx, float* __restrict__ partials,
                    float* __restrict__ dgamma, float* __restrict__ dbeta) {
  constexpr bool kCodes = sizeof(TX) == 1, kRing = kR == 4;
  // the ring of rows, then [groups][2][cols] column sums
  extern __shared__ __align__(16) uint8_t norm_smem[];
  float* col_sums = reinterpret_cast<float*>(norm_smem);
  __shared__ float red[2][kThreads / 32][2 * kR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int strip = warp % W, grp = warp / W, groups = static_cast<int>(blockDim.x) / 32 / W;
  const int sub = lane % kL;
  const int col = strip * 256 + (kVec ? sub * 8 : sub);
  pdl_launch_dependents();
  pdl_wait();
  const int cb = (cols + kQBlock - 1) / kQBlock;
  const float inv_c = 1.f / static_cast<float>(cols);
  const int Wp = strips_pow2(W), at_w = lane % Wp, at_i = lane / Wp;
  constexpr int kBatch = kR * (32 / kL);  // rows of a group
  const int64_t stride = static_cast<int64_t>(gridDim.x) * groups * kBatch;
  int64_t first = (static_cast<int64_t>(blockIdx.x) * groups + grp) * kBatch;
  const int own = lane / kL * kR;  // the lane's rows among them
  using Rg = Ring<T, TX, kR>;
  const uint32_t ring = smem_u32(norm_smem);
  const bool in = col < cols;
  auto issue = [&](int slot, int64_t r0) {
    uint32_t at = ring + slot * Rg::kSlot;
    // lanes 0..3: mean, 4..7: rstd, then the scales of the strip's two blocks
    const int64_t row = r0 + (lane & 3);
    const int blk = strip * 2 + ((lane >> 2) & 1);
    const float* src = lane < 4 ? mean + row : lane < 8 ? rstd + row : xs + row * cb + blk;
    const bool read = row < rows && (lane < 8 || blk < cb);
    if (lane < (kCodes ? 16 : 8))
      copy_async<4>(at + kThreads * Rg::kBytes + warp * 64 + lane * 4, read ? src : mean, read);
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const bool get = in && r0 + r < rows;
      const int64_t off = get ? (r0 + r) * cols + col : 0;
      at = copy_strip(at, kThreads, x + off, get);
      at = copy_strip(at, kThreads, dy + off, get);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int slot = 0;
  [[maybe_unused]] Batch<T, TX, kVec, kR, kL> next;
  if constexpr (kRing) {
#pragma unroll
    for (int d = 0; d < Rg::kDepth - 1; ++d) issue(d, first + d * stride);
  } else {
    next.load(x, xs, dy, mean, rstd, first + own, rows, cols, cb, col);
  }
  F2 ag[4], ab[4], gm[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) ag[e] = ab[e] = both(0.f);
  lane_columns<kVec, kL>(gamma, col, cols, gm);
  // columns of the lane's pair e
  auto col0 = [&](int e) { return col + (kVec ? 2 * e : 2 * kL * e); };
  auto col1 = [&](int e) { return col0(e) + (kVec ? 1 : kL); };
  int buf = 0;
  for (; first < rows; first += stride, buf ^= 1) {
    const int64_t row0 = first + own;
    Batch<T, TX, kVec, kR, kL> now;
    if constexpr (kRing) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Rg::kDepth - 2) : "memory");
      __syncwarp();  // the warp's floats are there; the slot before has been read
      issue(slot == 0 ? Rg::kDepth - 1 : slot - 1, first + (Rg::kDepth - 1) * stride);
      const uint8_t* at = norm_smem + slot * Rg::kSlot;
      const float* of_warp = reinterpret_cast<const float*>(at + kThreads * Rg::kBytes) + warp * 16;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        now.mu[r] = in ? of_warp[r] : 0.f;
        now.rs[r] = of_warp[4 + r];
        if constexpr (kCodes) now.sx[r][0] = of_warp[8 + r + 4 * (lane >> 4)];
        at = take_strip(at, kThreads, now.x[r]);
        at = take_strip(at, kThreads, now.dy[r]);
      }
      slot = slot == Rg::kDepth - 1 ? 0 : slot + 1;
    } else {
      now = next;
      next.load(x, xs, dy, mean, rstd, row0 + stride, rows, cols, cb, col);
    }
    F2 u[kR][4], g[kR][4];
    float part[2 * kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      F2 c1 = both(0.f), c2 = both(0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const F2 xv = {now.x[r].get(2 * e), now.x[r].get(2 * e + 1)};
        const F2 d = {now.dy[r].get(2 * e), now.dy[r].get(2 * e + 1)};
        // (code * scale - mean) * rstd, the product exact in the fma
        const F2 c = kCodes ? fma2(xv, both(now.sx[r][kVec || kL < 32 ? 0 : e >> 1]),
                                   both(-now.mu[r]))
                            : add2(xv, both(-now.mu[r]));
        u[r][e] = mul2(c, both(now.rs[r]));
        if (!kVec) u[r][e] = {col0(e) < cols ? u[r][e].a : 0.f, col1(e) < cols ? u[r][e].b : 0.f};
        ag[e] = fma2(d, u[r][e], ag[e]);
        ab[e] = add2(ab[e], d);
        g[r][e] = mul2(d, gm[e]);
        c1 = add2(c1, g[r][e]);
        c2 = fma2(g[r][e], u[r][e], c2);
      }
      part[r] = c1.a + c1.b;
      part[kR + r] = c2.a + c2.b;
    }
    // columns past the end hold u = 0 and dy = 0: nothing but zeros added
    const float mine = warp_sums<kL>(part, lane);
    constexpr int kHold = kL / 2 / kR;  // lanes that hold each sum
    float s[2 * kR];
    if (kL < 32 || W == 1) {
#pragma unroll
      for (int i = 0; i < 2 * kR; ++i) s[i] = __shfl_sync(0xffffffffu, mine, kHold * i, kL);
    } else {
      if (lane % kHold == 0) red[buf][warp][lane / kHold] = mine;
      named_bar_sync(1 + grp, 32 * W);
      // lane (i, w) takes strip w's share of sum i
      float t = at_w < W && at_i < 2 * kR ? red[buf][grp * W + at_w][at_i] : 0.f;
      for (int o = Wp / 2; o; o /= 2) t += __shfl_xor_sync(0xffffffffu, t, o);
#pragma unroll
      for (int i = 0; i < 2 * kR; ++i) s[i] = __shfl_sync(0xffffffffu, t, Wp * i);
    }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      if (row0 + r >= rows) break;
      // dx = rstd g - rstd mean(g) - u rstd mean(g u)
      const float rs = now.rs[r];
      const F2 k0 = both(-rs * (s[r] * inv_c)), k2 = both(-rs * (s[kR + r] * inv_c));
      float o[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const F2 v = fma2(u[r][e], k2, fma2(g[r][e], both(rs), k0));
        o[2 * e] = v.a;
        o[2 * e + 1] = v.b;
      }
      store_strip<T, kVec, kL>(dx + (row0 + r) * cols, col, cols, o);
    }
  }
  if constexpr (kRing) asm volatile("cp.async.wait_all;" ::: "memory");
  if (!partials && !dgamma) return;
  if constexpr (kRing) __syncthreads();  // the sums take its place
  // the lanes' rows apart hold the same columns
#pragma unroll
  for (int o = 16; o >= kL; o /= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ag[e] = add2(ag[e], {__shfl_xor_sync(0xffffffffu, ag[e].a, o),
                           __shfl_xor_sync(0xffffffffu, ag[e].b, o)});
      ab[e] = add2(ab[e], {__shfl_xor_sync(0xffffffffu, ab[e].a, o),
                           __shfl_xor_sync(0xffffffffu, ab[e].b, o)});
    }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float* to = col_sums + 2 * grp * cols;
    if (lane >= kL) break;
    if (col0(e) < cols) to[col0(e)] = ag[e].a, to[cols + col0(e)] = ab[e].a;
    if (col1(e) < cols) to[col1(e)] = ag[e].b, to[cols + col1(e)] = ab[e].b;
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
template <typename T, typename TX, bool kVec>
__global__ void __launch_bounds__(256)
    norm_bwd_wide_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                         const T* __restrict__ dy, const float* __restrict__ mean,
                         const float* __restrict__ rstd, const float* __restrict__ gamma,
                         int64_t rows, int cols, T* __restrict__ dx) {
  constexpr int kE = kPiece<kVec>;
  __shared__ float part[8];
  pdl_launch_dependents();
  pdl_wait();
  const int cb = (cols + kQBlock - 1) / kQBlock;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mu = mean[row], rs = rstd[row];
    // (a piece lies in one block)
    auto scale = [&](int c) { return sizeof(TX) == 1 ? xs[row * cb + (c >> 7)] : 1.f; };
    float c1 = 0.f, c2 = 0.f;
    for (int c = threadIdx.x * kE; c < cols; c += 256 * kE) {
      const Piece<TX, kVec> px(x + row * cols + c);
      const Piece<T, kVec> pd(dy + row * cols + c);
      const Piece<float, kVec> gm(gamma + c);
      const float k = scale(c);
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        const float g = pd.v[e] * gm.v[e];
        c1 += g;
        c2 = fmaf(g, fmaf(px.v[e], k, -mu) * rs, c2);
      }
    }
    c1 = block_sum(c1, part) / static_cast<float>(cols);
    c2 = block_sum(c2, part) / static_cast<float>(cols);
    for (int c = threadIdx.x * kE; c < cols; c += 256 * kE) {
      const Piece<TX, kVec> px(x + row * cols + c);
      Piece<T, kVec> pd(dy + row * cols + c);
      const Piece<float, kVec> gm(gamma + c);
      const float k = scale(c);
#pragma unroll
      for (int e = 0; e < kE; ++e)
        pd.v[e] = rs * (pd.v[e] * gm.v[e] - c1 - fmaf(px.v[e], k, -mu) * rs * c2);
      put_piece<kVec>(dx + row * cols + c, pd.v);
    }
  }
}

// Any width, the partial column sums: CTA (x, y) takes 32 pieces of columns and
// every gridDim.y-th group of 8 rows.
template <typename T, typename TX, bool kVec>
__global__ void __launch_bounds__(256)
    norm_bwd_cols_kernel(const TX* __restrict__ x, const float* __restrict__ xs,
                         const T* __restrict__ dy, const float* __restrict__ mean,
                         const float* __restrict__ rstd, int64_t rows, int cols,
                         float* __restrict__ partials) {
  constexpr int kE = kPiece<kVec>;
  __shared__ float red[2][8][32 * kE];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + lane) * kE;
  const int cb = (cols + kQBlock - 1) / kQBlock;
  float ag[kE], ab[kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) ag[e] = ab[e] = 0.f;
  if (col < cols)
    for (int64_t row = static_cast<int64_t>(blockIdx.y) * 8 + warp; row < rows;
         row += static_cast<int64_t>(gridDim.y) * 8) {
      const Piece<TX, kVec> px(x + row * cols + col);
      const Piece<T, kVec> pd(dy + row * cols + col);
      const float k = sizeof(TX) == 1 ? xs[row * cb + (col >> 7)] : 1.f;
      const float mu = mean[row], rs = rstd[row];
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        ag[e] = fmaf(pd.v[e], fmaf(px.v[e], k, -mu) * rs, ag[e]);
        ab[e] += pd.v[e];
      }
    }
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    red[0][warp][32 * e + lane] = ag[e];
    red[1][warp][32 * e + lane] = ab[e];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * kE; i += 256) {
    const int which = i / (32 * kE), at = i % (32 * kE);
    const int c = (blockIdx.x * 32 + at % 32) * kE + at / 32;
    if (c >= cols) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += red[which][w][at];
    partials[(static_cast<int64_t>(blockIdx.y) * 2 + which) * cols + c] = s;
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
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int64_t all = 2 * static_cast<int64_t>(cols);
  float s = 0.f;
  if (i < all) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 8) s += partials[p * all + i];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && i < all) {
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

template <typename T, bool kVec, int kR, int kThreads = kFwdThreads>
cudaError_t fwd_strips(const T* x, T* y, const FwdArgs& a, int num_sms, cudaStream_t stream) {
  const int W = strip_warps(a.cols), groups = strip_groups(a.cols, kThreads);
  const int per = groups * kR;
  const int64_t grid =
      std::min<int64_t>((a.rows + per - 1) / per, kFwdCtas<kR, kThreads> * num_sms);
  return launch_pdl(norm_fwd_kernel<T, kVec, kR, kThreads>, dim3(static_cast<unsigned>(grid)),
                    dim3(32 * W * groups), 0, stream, x, a.rows, a.cols, W, a.gamma, a.beta, a.eps,
                    y, a.mean, a.rstd);
}

template <typename T, int kCh>
cudaError_t fwd_rows(const T* x, T* y, const FwdArgs& a, cudaStream_t stream) {
  const int64_t grid = (a.rows + kRowThreads / 32 - 1) / (kRowThreads / 32);
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  return launch_pdl(norm_fwd_rows_kernel<T, kCh>, dim3(static_cast<unsigned>(grid)),
                    dim3(kRowThreads), 0, stream, x, a.rows, a.cols, a.gamma, a.beta, a.eps, y,
                    a.mean, a.rstd);
}

template <typename T>
cudaError_t fwd(const T* x, T* y, const FwdArgs& a, int num_sms, cudaStream_t stream) {
  const bool vec = a.cols % 8 == 0 && aligned16(x) && aligned16(y);
  // f32 strips of several warps are faster with two rows and three CTAs per SM
  // (50000 x 1024: 67 us, 77 with four and two), the others with four and two
  if (vec && a.cols <= kStripCols)
    return sizeof(T) == 4 && a.cols > 256 ? fwd_strips<T, true, 2>(x, y, a, num_sms, stream)
                                          : fwd_strips<T, true, 4>(x, y, a, num_sms, stream);
  if (a.cols <= 256) return fwd_rows<T, 1>(x, y, a, stream);
  if (a.cols <= 512) return fwd_rows<T, 2>(x, y, a, stream);
  if (a.cols <= 1024) return fwd_rows<T, 4>(x, y, a, stream);
  // long rows as strips all the same (30000 x 1999 bf16: 65 us, 106 with a warp to a
  // row, which 30000 x 333 favours: 13.7 against 16.0)
  if (a.cols <= kStripCols) return fwd_strips<T, false, 4>(x, y, a, num_sms, stream);
  // (4000 x 4096 bf16: 18.6 us, 28.9 by the kernel below)
  if (a.cols <= kWideCols)
    return vec ? fwd_strips<T, true, 2, 512>(x, y, a, num_sms, stream)
               : fwd_strips<T, false, 2, 512>(x, y, a, num_sms, stream);
  const int grid = static_cast<int>(std::min<int64_t>(a.rows, 8 * num_sms));
  const bool all = vec && aligned16(a.gamma) && aligned16(a.beta);
  return launch_pdl(all ? norm_fwd_wide_kernel<T, true> : norm_fwd_wide_kernel<T, false>,
                    dim3(grid), dim3(256), 0, stream, x, a.rows, a.cols, a.gamma, a.beta, a.eps, y,
                    a.mean, a.rstd);
}

struct BwdArgs {
  const float *xs, *mean, *rstd, *gamma;
  int64_t rows;
  int cols;
  float *dgamma, *dbeta, *partials;
  int num_sms;
};

// parts: the CTAs, which is the partial rows written.
template <typename T, typename TX, bool kVec, int kThreads, int kR, int kL = 32>
cudaError_t bwd_strips(const TX* x, const T* dy, T* dx, const BwdArgs& a, int& parts,
                       cudaStream_t stream) {
  const int W = strip_warps(a.cols), groups = strip_groups(a.cols, kThreads);
  const int per = groups * kR * (32 / kL);
  const int64_t batches = (a.rows + per - 1) / per;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute la[2];
  la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  constexpr bool kOne = kThreads == kFewThreads && kR > 1;  // one cluster (kR 1: wide rows)
  if (kOne && a.dgamma) {
    unsigned c = 1;
    while (c < 8 && c < batches) c *= 2;
    cfg.gridDim = dim3(c);
    la[1].id = cudaLaunchAttributeClusterDimension;
    la[1].val.clusterDim.x = c;
    la[1].val.clusterDim.y = 1;
    la[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  } else {
    const int many = std::min(kManyParts, 2 * a.num_sms);
    const int most = kThreads == kManyThreads ? many : many / 2;
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(batches, most)));
  }
  cfg.blockDim = dim3(32 * W * groups);
  parts = static_cast<int>(cfg.gridDim.x);
  // groups * W <= 16 warps of 256 columns: 32 KB of sums at most
  auto* kernel = norm_bwd_kernel<T, TX, kVec, kThreads, kR, kL>;
  const size_t sums = a.dgamma ? 8 * static_cast<size_t>(groups) * a.cols : 0;
  cfg.dynamicSmemBytes = sums;
  if constexpr (kR == 4) {
    static std::atomic<uint64_t> attr{0};
    constexpr int kSmem = std::max(Ring<T, TX, kR>::kDepth * Ring<T, TX, kR>::kSlot, 16384);
    if (cudaError_t e = smem_attr_once(kernel, kSmem, attr)) return e;
    cfg.dynamicSmemBytes = kSmem;
  }
  cfg.stream = stream;
  cfg.attrs = la;
  float* partials = kOne ? nullptr : a.partials;
  return cudaLaunchKernelEx(&cfg, kernel, x, a.xs, dy, a.mean, a.rstd, a.gamma, a.rows, a.cols, W,
                            dx, partials, a.dgamma, a.dbeta);
}

template <typename T, typename TX>
cudaError_t bwd(const TX* x, const T* dy, T* dx, const BwdArgs& a, cudaStream_t stream) {
  const bool vec = a.cols % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx);
  int parts = norm_parts(a.rows, a.cols);
  cudaError_t e;
  if (a.cols <= kStripCols) {
    if (parts == 0)
      return vec ? bwd_strips<T, TX, true, kFewThreads, 2>(x, dy, dx, a, parts, stream)
                 : bwd_strips<T, TX, false, kFewThreads, 2>(x, dy, dx, a, parts, stream);
    constexpr int kBest = sizeof(T) == 2 ? 4 : 2;
    if (a.cols <= kNarrow)
      e = vec ? bwd_strips<T, TX, true, kManyThreads, 2, kNarrowLanes>(x, dy, dx, a, parts, stream)
              : bwd_strips<T, TX, false, kManyThreads, 2, kNarrowLanes>(x, dy, dx, a, parts,
                                                                        stream);
    else if (vec && strip_warps(a.cols) <= kRingWarps)
      e = bwd_strips<T, TX, true, kManyThreads, kBest>(x, dy, dx, a, parts, stream);
    else
      e = vec ? bwd_strips<T, TX, true, kManyThreads, 2>(x, dy, dx, a, parts, stream)
              : bwd_strips<T, TX, false, kManyThreads, 2>(x, dy, dx, a, parts, stream);
  } else if (a.cols <= kWideCols) {
    // (4000 x 4096 bf16: 31.5 us, 103 by the kernels below)
    e = vec ? bwd_strips<T, TX, true, kFewThreads, 1>(x, dy, dx, a, parts, stream)
            : bwd_strips<T, TX, false, kFewThreads, 1>(x, dy, dx, a, parts, stream);
  } else {
    const int grid = static_cast<int>(std::min<int64_t>(a.rows, 8 * a.num_sms));
    const bool all = vec && aligned16(a.gamma);
    e = launch_pdl(all ? norm_bwd_wide_kernel<T, TX, true> : norm_bwd_wide_kernel<T, TX, false>,
                   dim3(grid), dim3(256), 0, stream, x, a.xs, dy, a.mean, a.rstd, a.gamma, a.rows,
                   a.cols, dx);
    const int across = 32 * (vec ? kPiece<true> : kPiece<false>);
    if (e == cudaSuccess && a.dgamma)
      e = launch_pdl(vec ? norm_bwd_cols_kernel<T, TX, true> : norm_bwd_cols_kernel<T, TX, false>,
                     dim3((a.cols + across - 1) / across, parts), dim3(256), 0, stream, x, a.xs, dy,
                     a.mean, a.rstd, a.rows, a.cols, a.partials);
  }
  if (e != cudaSuccess || !a.dgamma) return e;
  const auto grid = static_cast<unsigned>((2 * static_cast<int64_t>(a.cols) + 31) / 32);
  return launch_pdl(norm_bwd_sum_kernel, dim3(grid), dim3(256), 0, stream,
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
                            float* partials, int num_sms, cudaStream_t stream) {
  if (rows <= 0) {
    if (!dgamma) return cudaSuccess;
    if (cudaError_t e = cudaMemsetAsync(dgamma, 0, 4 * static_cast<size_t>(cols), stream)) return e;
    return cudaMemsetAsync(dbeta, 0, 4 * static_cast<size_t>(cols), stream);
  }
  const BwdArgs a{xs,   mean,   rstd,  gamma,    rows,
                  cols, dgamma, dbeta, dgamma ? partials : nullptr, num_sms};
  return bf16 ? bwd_typed<__nv_bfloat16>(x, xs, dy, dx, a, stream)
              : bwd_typed<float>(x, xs, dy, dx, a, stream);
}

}  // namespace nrp
