// fp8_api.cpp -- C ABI of the 8-bit floating-point linears, their gradients
// and the LayerNorm's forward and backward pass (include/nemo_relpos.h).
#include <cuda_runtime.h>

#include <initializer_list>

#include "../../include/nemo_relpos.h"
#include "fp8.h"
#include "handles.h"
#include "internal.h"

using nrp::failf;
using nrp::ProfScope;

namespace {

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// cudaSuccess -> NRP_OK; else the error, also taken out of the runtime's
// last-error slot.
int status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return NRP_OK;
  cudaGetLastError();
  return failf(e == cudaErrorMemoryAllocation ? NRP_ERR_NOMEM : NRP_ERR_CUDA, "%s: %s", what,
               cudaGetErrorString(e));
}

int check_dtype(int dtype) {
  if (dtype == NRP_DTYPE_F32 || dtype == NRP_DTYPE_BF16) return NRP_OK;
  return failf(NRP_ERR_UNSUPPORTED, "dtype %d", dtype);
}

// The largest row and column counts of a product and columns of a LayerNorm: the
// kernels round them up to whole tiles and look a few tiles ahead in 32-bit indices.
constexpr int kMaxSize = INT32_MAX - 4095;
int check_sizes(const char* what, std::initializer_list<int> sizes) {
  for (int n : sizes)
    if (n > kMaxSize) return failf(NRP_ERR_UNSUPPORTED, "%s: size %d (at most %d)", what, n, kMaxSize);
  return NRP_OK;
}

// A matrix of codes: 16-byte rows (TMA and 16-byte loads), 16-byte aligned.
// Those of one without rows are not looked at.
int check_codes(const char* name, const void* codes, const void* scales, int64_t cols,
                bool empty = false) {
  if (!empty && (!codes || !scales))
    return failf(NRP_ERR_INVALID, "%s: null codes or scales", name);
  if (cols % 16)
    return failf(NRP_ERR_UNSUPPORTED, "%s: %lld columns (codes need a multiple of 16)", name,
                 static_cast<long long>(cols));
  if (!empty && (!aligned(codes, 16) || !aligned(scales, 4)))
    return failf(NRP_ERR_INVALID, "%s: codes must be 16-byte and scales 4-byte aligned", name);
  return NRP_OK;
}

int64_t elem(int dtype) { return dtype == NRP_DTYPE_BF16 ? 2 : 4; }
int64_t scale_bytes(int64_t rows, int64_t cols, int block_rows) {
  return 4 * (block_rows == 1 ? rows : nrp::qblocks(rows)) * nrp::qblocks(cols);
}

// An argument's bytes and the alignment that its loads and stores need.
struct Span {
  const char* name;
  const void* p;
  int64_t bytes;
  int64_t align;
};
// Every argument is aligned, and no output overlaps another argument (the
// kernels read inputs while they write outputs).
int check_spans(const char* what, std::initializer_list<Span> outputs,
                std::initializer_list<Span> inputs) {
  for (const auto& list : {outputs, inputs})
    for (const Span& s : list)
      if (s.bytes > 0 && !aligned(s.p, static_cast<size_t>(s.align)))
        return failf(NRP_ERR_INVALID, "%s: %s must be %lld-byte aligned", what, s.name,
                     static_cast<long long>(s.align));
  auto meet = [](const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x && y && a.bytes > 0 && b.bytes > 0 && x < y + static_cast<uintptr_t>(b.bytes) &&
           y < x + static_cast<uintptr_t>(a.bytes);
  };
  for (const Span* o = outputs.begin(); o != outputs.end(); ++o) {
    for (const Span* q = o + 1; q != outputs.end(); ++q)
      if (meet(*o, *q))
        return failf(NRP_ERR_INVALID, "%s: %s and %s overlap", what, o->name, q->name);
    for (const Span& i : inputs)
      if (meet(*o, i))
        return failf(NRP_ERR_INVALID, "%s: %s and %s overlap", what, o->name, i.name);
  }
  return NRP_OK;
}

// The arguments of a product [M, R] x weight [wr, wc].
int check_product(const char* what, int dtype, const void* x, const uint8_t* xq, const float* xs,
                  int64_t M, int64_t R, const uint8_t* wq, const float* ws, int64_t wr, int64_t wc,
                  const void* bias, const void* y, int64_t NO) {
  const int64_t es = elem(dtype), n = M * R, sb = scale_bytes(M, R, 1);
  const Span out{"the output", y, M * NO * es, es};
  const Span w{"the weight's codes", wq, wr * wc, 16};
  const Span wsc{"the weight's scales", ws, scale_bytes(wr, wc, 128), 4};
  const Span b{"bias", bias, NO * es, es};
  if (!x) return check_spans(what, {out}, {{"codes", xq, n, 16}, {"scales", xs, sb, 4}, w, wsc, b});
  return check_spans(what, {out, {"codes", xq, n, 16}, {"scales", xs, sb, 4}},
                     {{"the input", x, n * es, 16}, w, wsc, b});
}

// Quantises x (when given) into xq, xs and multiplies by the weight.
int product(nrp_context* ctx, cudaStream_t st, bool trans, int dtype, const void* x, uint8_t* xq,
            float* xs, int M, int R, const uint8_t* wq, const float* ws, int NO, const void* bias,
            void* y) {
  const bool bf16 = dtype == NRP_DTYPE_BF16;
  const bool small = !trans && nrp::fp8_small_supported(M, R);
  if (x && !(small && nrp::fp8_small_quantizes(M))) {
    ProfScope ps(ctx, NRP_KERNEL_FP8_QUANT, st);
    if (int rc = status(nrp::launch_fp8_quantize(bf16, x, M, R, 1, xq, xs, ctx->num_sms, st),
                        "fp8 quantize"))
      return rc;
    x = nullptr;
  }
  if (small) {
    ProfScope ps(ctx, NRP_KERNEL_FP8_SMALL, st);
    return status(nrp::launch_fp8_small(bf16, x, xq, xs, M, R, wq, ws, NO, bias, y, ctx->num_sms,
                                        st),
                  "fp8 linear");
  }
  ProfScope ps(ctx, NRP_KERNEL_GEMM_FP8, st);
  return status(nrp::launch_gemm_fp8(bf16, trans, xq, xs, M, R, wq, ws, NO, bias, y, ctx->num_sms,
                                     ctx->d_err, st),
                "fp8 linear");
}

}  // namespace

extern "C" {

int nrp_fp8_quantize(nrp_context* ctx, void* stream, int dtype, const void* x, int64_t rows,
                     int cols, int block_rows, uint8_t* codes, float* scales) {
  if (!ctx || (rows && !x) || rows < 0 || cols <= 0)
    return failf(NRP_ERR_INVALID, "invalid quantize arguments");
  if (int rc = check_dtype(dtype)) return rc;
  if (block_rows != 1 && block_rows != 128)
    return failf(NRP_ERR_UNSUPPORTED, "block_rows %d (supported: 1, 128)", block_rows);
  if (int rc = check_codes("quantize", codes, scales, cols, rows == 0)) return rc;
  if (int rc = check_spans("quantize",
                           {{"codes", codes, rows * cols, 16},
                            {"scales", scales, scale_bytes(rows, cols, block_rows), 4}},
                           {{"the input", x, rows * cols * elem(dtype), 16}}))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope ps(ctx, NRP_KERNEL_FP8_QUANT, st);
  return status(nrp::launch_fp8_quantize(dtype == NRP_DTYPE_BF16, x, rows, cols, block_rows, codes,
                                         scales, ctx->num_sms, st),
                "fp8 quantize");
}

int nrp_fp8_dequantize(nrp_context* ctx, void* stream, const uint8_t* codes, const float* scales,
                       int64_t rows, int cols, int block_rows, int dtype, void* x) {
  if (!ctx || (rows && !x) || rows < 0 || cols <= 0)
    return failf(NRP_ERR_INVALID, "invalid dequantize arguments");
  if (int rc = check_dtype(dtype)) return rc;
  if (block_rows != 1 && block_rows != 128)
    return failf(NRP_ERR_UNSUPPORTED, "block_rows %d (supported: 1, 128)", block_rows);
  if (int rc = check_codes("dequantize", codes, scales, cols, rows == 0)) return rc;
  if (int rc = check_spans("dequantize", {{"the output", x, rows * cols * elem(dtype), 16}},
                           {{"codes", codes, rows * cols, 16},
                            {"scales", scales, scale_bytes(rows, cols, block_rows), 4}}))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope ps(ctx, NRP_KERNEL_FP8_QUANT, st);
  return status(nrp::launch_fp8_dequantize(dtype == NRP_DTYPE_BF16, codes, scales, rows, cols,
                                           block_rows, x, ctx->num_sms, st),
                "fp8 dequantize");
}

int nrp_fp8_linear(nrp_context* ctx, void* stream, int dtype, const void* x, uint8_t* xq,
                   float* xs, int M, int K, const uint8_t* wq, const float* ws, int N,
                   const void* bias, void* y) {
  if (!ctx || (M && !y) || M < 0 || K <= 0 || N <= 0)
    return failf(NRP_ERR_INVALID, "invalid fp8 linear arguments");
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_sizes("fp8 linear", {M, K, N})) return rc;
  if (int rc = check_codes("fp8 linear: input", xq, xs, K, M == 0)) return rc;
  if (int rc = check_codes("fp8 linear: weight", wq, ws, K)) return rc;
  if (int rc = check_product("fp8 linear", dtype, x, xq, xs, M, K, wq, ws, N, K, bias, y, N))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  return product(ctx, static_cast<cudaStream_t>(stream), false, dtype, x, xq, xs, M, K, wq, ws, N,
                 bias, y);
}

int nrp_fp8_linear_input_grad(nrp_context* ctx, void* stream, int dtype, const void* dy,
                              uint8_t* gq, float* gs, int M, int N, const uint8_t* wq,
                              const float* ws, int K, void* dx) {
  if (!ctx || (M && !dx) || M < 0 || K <= 0 || N <= 0)
    return failf(NRP_ERR_INVALID, "invalid fp8 input gradient arguments");
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_sizes("fp8 input gradient", {M, N, K})) return rc;
  if (int rc = check_codes("fp8 input gradient: output gradient", gq, gs, N, M == 0)) return rc;
  if (int rc = check_codes("fp8 input gradient: weight", wq, ws, K)) return rc;
  if (int rc = check_product("fp8 input gradient", dtype, dy, gq, gs, M, N, wq, ws, N, K, nullptr,
                             dx, K))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  return product(ctx, static_cast<cudaStream_t>(stream), true, dtype, dy, gq, gs, M, N, wq, ws, K,
                 nullptr, dx);
}

int nrp_fp8_linear_weight_grad(nrp_context* ctx, void* stream, const void* dy, const uint8_t* xq,
                               const float* xs, int M, int N, int K, int dtype, void* dw,
                               void* dbias) {
  if (!ctx || (M && !dy) || !dw || M < 0 || K <= 0 || N <= 0)
    return failf(NRP_ERR_INVALID, "invalid fp8 weight gradient arguments");
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_sizes("fp8 weight gradient", {M, N, K})) return rc;
  if (int rc = check_codes("fp8 weight gradient: input", xq, xs, K, M == 0)) return rc;
  if (N % 8)
    return failf(NRP_ERR_UNSUPPORTED, "fp8 weight gradient: N = %d (needs a multiple of 8)", N);
  const int64_t es = elem(dtype), n = N, k = K;
  if (int rc = check_spans("fp8 weight gradient",
                           {{"dw", dw, n * k * es, es}, {"dbias", dbias, n * es, es}},
                           {{"dy", dy, M * n * 2, 16},
                            {"codes", xq, M * k, 16},
                            {"scales", xs, scale_bytes(M, k, 1), 4}}))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope ps(ctx, NRP_KERNEL_FP8_WGRAD, st);
  return status(nrp::launch_fp8_weight_grad(dtype == NRP_DTYPE_BF16, dy, xq, xs, M, N, K, dw,
                                            dbias, ctx->num_sms, ctx->d_err, st),
                "fp8 weight gradient");
}

int nrp_layer_norm(nrp_context* ctx, void* stream, int dtype, const void* x, int64_t rows,
                   int cols, const float* gamma, const float* beta, float eps, void* y,
                   float* mean, float* rstd) {
  if (!ctx || !gamma || !beta || (rows && (!x || !y)) || rows < 0 || cols <= 0)
    return failf(NRP_ERR_INVALID, "invalid layer norm arguments");
  if (int rc = check_sizes("layer norm", {cols})) return rc;
  if (rows && !mean != !rstd)
    return failf(NRP_ERR_INVALID, "layer norm: mean and rstd go together");
  if (!(eps >= 0.f)) return failf(NRP_ERR_INVALID, "layer norm: eps must not be negative");
  if (int rc = check_dtype(dtype)) return rc;
  const int64_t es = elem(dtype), bytes = rows * cols * es, vec = 4 * static_cast<int64_t>(cols);
  if (int rc = check_spans("layer norm",
                           {{"the output", y, bytes, es}, {"mean", mean, rows * 4, 4},
                            {"rstd", rstd, rows * 4, 4}},
                           {{"the input", x == y ? nullptr : x, bytes, es},
                            {"gamma", gamma, vec, 4}, {"beta", beta, vec, 4}}))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope ps(ctx, NRP_KERNEL_LAYERNORM, st);
  return status(nrp::launch_norm_fwd(dtype == NRP_DTYPE_BF16, x, rows, cols, gamma, beta, eps, y,
                                     mean, rstd, ctx->num_sms, st),
                "layer norm");
}

int nrp_layer_norm_backward_workspace(int64_t rows, int cols, int64_t* bytes) {
  if (!bytes || rows < 0 || cols <= 0) return failf(NRP_ERR_INVALID, "invalid layer norm size");
  if (int rc = check_sizes("layer norm backward", {cols})) return rc;
  *bytes = 4 * nrp::norm_bwd_partials(rows, cols);
  return NRP_OK;
}

int nrp_layer_norm_backward(nrp_context* ctx, void* stream, int dtype, const void* x,
                            const float* x_scales, const void* dy, const float* mean,
                            const float* rstd, const float* gamma, int64_t rows, int cols,
                            void* dx, float* dgamma, float* dbeta, void* workspace,
                            int64_t workspace_bytes) {
  if (!ctx || !gamma || (rows && (!x || !dy || !mean || !rstd || !dx)) || rows < 0 || cols <= 0)
    return failf(NRP_ERR_INVALID, "invalid layer norm backward arguments");
  if (int rc = check_sizes("layer norm backward", {cols})) return rc;
  if (!dgamma != !dbeta) return failf(NRP_ERR_INVALID, "layer norm: dgamma and dbeta go together");
  if (int rc = check_dtype(dtype)) return rc;
  if (x_scales)
    if (int rc = check_codes("layer norm backward: input", x, x_scales, cols, rows == 0)) return rc;
  const int64_t need = dgamma ? 4 * nrp::norm_bwd_partials(rows, cols) : 0;
  if (need) {
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
      return failf(NRP_ERR_INVALID,
                   "layer norm backward: workspace of %lld bytes (16-byte aligned) needed, got %lld",
                   static_cast<long long>(need), static_cast<long long>(workspace_bytes));
  }
  const int64_t es = elem(dtype), n = rows * cols, vec = 4 * static_cast<int64_t>(cols);
  if (int rc = check_spans(
          "layer norm backward",
          {{"dx", dx, n * es, es}, {"dgamma", dgamma, vec, 4}, {"dbeta", dbeta, vec, 4},
           {"workspace", dgamma ? workspace : nullptr, need, 4}},
          {{"the input", x, x_scales ? n : n * es, x_scales ? 16 : es},
           {"scales", x_scales, x_scales ? scale_bytes(rows, cols, 1) : 0, 4},
           {"dy", dy, n * es, es}, {"mean", mean, rows * 4, 4}, {"rstd", rstd, rows * 4, 4},
           {"gamma", gamma, vec, 4}}))
    return rc;
  if (nrp::select_device(ctx)) return NRP_ERR_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ProfScope ps(ctx, NRP_KERNEL_LAYERNORM_BWD, st);
  return status(nrp::launch_norm_bwd(dtype == NRP_DTYPE_BF16, x, x_scales, dy, mean, rstd, gamma,
                                     rows, cols, dx, dgamma, dbeta,
                                     static_cast<float*>(workspace), ctx->num_sms, st),
                "layer norm backward");
}

}  // extern "C"
