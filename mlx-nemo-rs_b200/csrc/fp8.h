// fp8.h -- launchers of the 8-bit floating-point (e4m3) linears, their
// gradients and the LayerNorm's forward and backward pass (internal, not the
// C ABI).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm.h"

namespace nrp {

// Columns of a scale block; rows are 1 (activations) or 128 (weights).
constexpr int kQBlock = 128;
inline int64_t qblocks(int64_t n) { return (n + kQBlock - 1) / kQBlock; }

// codes [rows, cols] e4m3 and scales f32 [ceil(rows / block_rows),
// ceil(cols / 128)] of x (f32 or bf16) [rows, cols]; cols % 16 == 0, x and
// codes 16-byte aligned, block_rows 1 or 128.
cudaError_t launch_fp8_quantize(bool bf16, const void* x, int64_t rows, int cols, int block_rows,
                                uint8_t* codes, float* scales, int num_sms, cudaStream_t stream);
// x = codes * scales, rounded once to x's type.
cudaError_t launch_fp8_dequantize(bool bf16, const uint8_t* codes, const float* scales,
                                  int64_t rows, int cols, int block_rows, void* x, int num_sms,
                                  cudaStream_t stream);

// y[M, NO] (f32 or bf16) = sum over 128-blocks b of the reduction of
//   xs[m, b] * ws[.] * sum_{r in b} xq[m, r] * w(r, n)  (+ bias[n])
// xq e4m3 [M, R] with scales [M, ceil(R/128)].  trans == false: w(r, n) =
// wq[n, r], wq [NO, R], ws [ceil(NO/128), ceil(R/128)] (the forward
// product); true: w(r, n) = wq[r, n], wq [R, NO], ws [ceil(R/128),
// ceil(NO/128)] (the input's gradient).  R % 16 == 0; trans: NO % 16 == 0.
cudaError_t launch_gemm_fp8(bool bf16_out, bool trans, const uint8_t* xq, const float* xs, int M,
                            int R, const uint8_t* wq, const float* ws, int NO, const void* bias,
                            void* y, int num_sms, int* err, cudaStream_t stream);

// The forward product for few rows, x quantised on the way: y[M, N] = q(x) .
// w^T (+ bias).  x (f32 or bf16 as y, 16-byte aligned) is quantised into xq, xs;
// x null: xq, xs are inputs.  fp8_small_supported: M <= kFp8SmallMaxM and K up
// to what M rows of codes leave room for in shared memory.
constexpr int kFp8SmallMaxM = 32;
// fp8_small_quantizes: M rows are better quantised by it than ahead of it.
bool fp8_small_supported(int M, int K);
bool fp8_small_quantizes(int M);
cudaError_t launch_fp8_small(bool bf16, const void* x, uint8_t* xq, float* xs, int M, int K,
                             const uint8_t* wq, const float* ws, int N, const void* bias, void* y,
                             int num_sms, cudaStream_t stream);

// dw[N, K] (f32 or bf16) = sum_m dy[m, n] * x~[m, k], x~ = xq * xs rounded
// to bf16 (exact for power-of-two scales); db[n] = sum_m dy[m, n] in dw's
// type (db may be null).  dy bf16 [M, N], N % 8 == 0, K % 16 == 0.
cudaError_t launch_fp8_weight_grad(bool bf16_out, const void* dy, const uint8_t* xq,
                                   const float* xs, int M, int N, int K, void* dw, void* db,
                                   int num_sms, int* err, cudaStream_t stream);

// y = (x - mean) * rstd * gamma + beta over rows of cols; mean and rstd
// (f32 [rows]) written when non-null.  y may be x.
cudaError_t launch_norm_fwd(bool bf16, const void* x, int64_t rows, int cols, const float* gamma,
                            const float* beta, float eps, void* y, float* mean, float* rstd,
                            int num_sms, cudaStream_t stream);
// dx, dgamma, dbeta.  x: f32 or bf16 as dy, or e4m3 codes when xs is
// non-null.  dgamma and dbeta may both be null; otherwise partials holds
// norm_bwd_partials(rows, cols) floats.
int64_t norm_bwd_partials(int64_t rows, int cols);
cudaError_t launch_norm_bwd(bool bf16, const void* x, const float* xs, const void* dy,
                            const float* mean, const float* rstd, const float* gamma,
                            int64_t rows, int cols, void* dx, float* dgamma, float* dbeta,
                            float* partials, int num_sms, cudaStream_t stream);

}  // namespace nrp
