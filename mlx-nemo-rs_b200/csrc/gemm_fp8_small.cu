// gemm_fp8_small.cu -- the 8-bit linear's forward product for a streaming
// chunk's few rows (M <= 32): one launch that quantises x and multiplies.
//
// The work is reading the weight's codes once (4 MB at 4096 x 1024: 0.6 us of
// HBM), so what costs is latency: launches, dependent loads, reductions.  A CTA
// owns 16 or 32 weight rows and all of K, or a cluster of up to eight share K
// where that gives more SMs work; its eight warps take every eighth 128-block.
// A warp asks for its first block's codes, then the CTA quantises its part of x
// (as every other CTA of that part: 14 x 1024 values, from L2) into shared
// memory while they come, four blocks' loads in flight per lane.  mma.sync
// m16n8k32 takes the weight rows as the 16-row operand and up to 8 tokens as the
// other (a tcgen05 tile has 128 rows, of which 14 would be used); 64 consecutive
// codes of a row are four lanes' 16-byte loads, the same permutation of k on both
// sides.  A block's sum is scaled by its two scales and added in f32; the warps'
// partial results meet in shared memory, the CTAs' in the cluster's.
//
// Measured: 14 rows, 1024 to 4096, bf16 with bias 4.9 us (an empty kernel takes
// 2.2), 0.8 TB/s of weight.
#include <algorithm>

#include "fp8.h"
#include "fp8_quant.cuh"
#include "fp8_scales.cuh"

namespace nrp {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr size_t kMaxSmem = 200 * 1024;

// Bytes from one token's codes to the next: 64 mod 128, so that two tokens'
// 64-byte pieces fall on all banks.
__host__ __device__ inline int code_pitch(int K) { return (K + 127) / 128 * 128 + 64; }
inline int token_tiles(int M) { return M <= 8 ? 1 : M <= 16 ? 2 : 4; }
// K: the columns of one CTA
inline size_t smem_bytes(int M, int K, int rows) {
  const int tokens = 8 * token_tiles(M);
  return static_cast<size_t>(tokens) * (code_pitch(K) + 4 * qblocks(K)) +
         static_cast<size_t>(kWarps) * rows * tokens * 4;
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Args {
  const void* x;  // null: xq, xs are inputs
  uint8_t* xq;
  float* xs;
  const uint8_t* wq;
  const float* ws;
  const void* bias;
  void* y;
  int M, K, N, kb;
  int split;  // CTAs of a cluster, which share the kb blocks
};

// kRT: 16-row weight tiles per CTA; kNT: 8-token tiles.
template <typename T, int kRT, int kNT>
__global__ void __launch_bounds__(kThreads) fp8_small_kernel(const Args a) {
  constexpr int kRows = 16 * kRT, kTok = 8 * kNT;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tile = static_cast<int>(blockIdx.x) / a.split;
  const int rank = static_cast<int>(blockIdx.x) % a.split;
  const int tiles = static_cast<int>(gridDim.x) / a.split;
  const int b0 = a.kb * rank / a.split, nb = a.kb * (rank + 1) / a.split - b0;
  const int most = (a.kb + a.split - 1) / a.split;  // blocks of any rank at most
  const int pitch = code_pitch(most * kQBlock);
  uint8_t* sx = smem;                                         // [kTok][pitch]
  float* ss = reinterpret_cast<float*>(smem + kTok * pitch);  // [most][kTok] scales
  float* red = ss + kTok * most;                              // [warp][kTok][kRows]
  const int warp = warp_id(), lane = lane_id();
  const int g = lane >> 2, t = lane & 3;
  const int n0 = tile * kRows;
  pdl_launch_dependents();
  pdl_wait();

  // block b0 + b of the weight rows: 16 bytes per lane and 64 columns (zeros
  // off the end)
  auto load_w = [&](uint4 (&w)[2][2 * kRT], int b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = (b0 + b) * kQBlock + h * 64 + t * 16;
#pragma unroll
      for (int r = 0; r < 2 * kRT; ++r) {
        const int n = n0 + 8 * r + g;
        w[h][r] = n < a.N && k < a.K
                      ? __ldg(reinterpret_cast<const uint4*>(
                            a.wq + static_cast<int64_t>(n) * a.K + k))
                      : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  uint4 w[2][2 * kRT];
  if (warp < nb) load_w(w, warp);

  // x's codes and scales: eight lanes of 16 columns to a block, columns past K
  // as zeros (the last block's 64-byte pieces are read whole).  The codes of tokens
  // past M stay undefined, as their results are not stored; their scales are 1.
  // The 32 lane groups of a pass tile (token, block) by powers of two.
  constexpr int kFly = sizeof(T) == 4 ? 2 : 4;
  const int sub = threadIdx.x & 7;
  const int lb = nb >= 32 ? 5 : 32 - __clz(nb - 1);  // log2 of the blocks side by side
  const int gb = (threadIdx.x >> 3) & ((1 << lb) - 1), gm = threadIdx.x >> (3 + lb);
  for (int bb = 0; bb < nb; bb += 32)
    for (int mm = 0; mm < a.M; mm += kFly << (5 - lb)) {
      const int b = bb + gb, col = (b0 + b) * kQBlock + sub * 16;
      uint4 raw[kFly][kRawWords<T>];  // 16 elements; codes: [0]
      float sc[kFly];
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int m = mm + gm + (i << (5 - lb));
        const int64_t at = static_cast<int64_t>(m) * a.K + col;
        const bool in = m < a.M && b < nb && col < a.K;
        sc[i] = 0.f;
#pragma unroll
        for (int q = 0; q < kRawWords<T>; ++q)
          raw[i][q] = in && a.x ? __ldg(reinterpret_cast<const uint4*>(
                                            static_cast<const T*>(a.x) + at) + q)
                                : make_uint4(0u, 0u, 0u, 0u);
        if (in && !a.x) {
          raw[i][0] = __ldg(reinterpret_cast<const uint4*>(a.xq + at));
          sc[i] = a.xs[static_cast<int64_t>(m) * a.kb + b0 + b];
        }
      }
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int m = mm + gm + (i << (5 - lb));
        if (mm + (i << (5 - lb)) >= a.M) break;  // (the whole CTA)
        uint4 q = raw[i][0];
        float scale = sc[i];
        if (a.x) {
          q = quantize_block<T>(raw[i], scale);
          // (one of the part's CTAs hands the token's codes out)
          if (m < a.M && b < nb && col < a.K && m % tiles == tile) {
            *reinterpret_cast<uint4*>(a.xq + static_cast<int64_t>(m) * a.K + col) = q;
            if (sub == 0) a.xs[static_cast<int64_t>(m) * a.kb + b0 + b] = scale;
          }
        }
        if (m < a.M && b < nb) {
          *reinterpret_cast<uint4*>(sx + m * pitch + b * kQBlock + sub * 16) = q;
          if (sub == 0) ss[b * kTok + m] = scale;
        }
      }
    }
  for (int u = threadIdx.x; u < nb * kTok; u += kThreads)
    if (u % kTok >= a.M) ss[u] = 1.f;
  __syncthreads();

  float acc[kRT][kNT][4];
#pragma unroll
  for (int i = 0; i < kRT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
  const float* wsr = a.ws + static_cast<int64_t>(n0 / kQBlock) * a.kb + b0;  // (kRows divides 128)
  for (int b = warp; b < nb; b += kWarps) {
    const float wscale = wsr[b];
    float c[kRT][kNT][4];
#pragma unroll
    for (int i = 0; i < kRT; ++i)
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[i][j][e] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 xb[kNT];
#pragma unroll
      for (int j = 0; j < kNT; ++j)
        xb[j] = *reinterpret_cast<const uint4*>(sx + (8 * j + g) * pitch + b * kQBlock + h * 64 +
                                                t * 16);
#pragma unroll
      for (int i = 0; i < kRT; ++i) {
        const uint4 lo = w[h][2 * i], hi = w[h][2 * i + 1];  // rows g, g + 8
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          mma_e4m3(c[i][j], lo.x, hi.x, lo.y, hi.y, xb[j].x, xb[j].y);
          mma_e4m3(c[i][j], lo.z, hi.z, lo.w, hi.w, xb[j].z, xb[j].w);
        }
      }
    }
    if (b + kWarps < nb) load_w(w, b + kWarps);
    float s[kNT][2];
    bool in_range = true;
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      const float2 xsc = *reinterpret_cast<const float2*>(ss + b * kTok + 8 * j + 2 * t);
      s[j][0] = wscale * xsc.x;
      s[j][1] = wscale * xsc.y;
      in_range &= scale_in_range(s[j][0]) & scale_in_range(s[j][1]);
    }
    if (!in_range) {
#pragma unroll
      for (int j = 0; j < kNT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p;
          scale_factors(ss[b * kTok + 8 * j + 2 * t + h], wscale, p, s[j][h]);
#pragma unroll
          for (int i = 0; i < kRT; ++i) {
            c[i][j][h] *= p;
            c[i][j][2 + h] *= p;
          }
        }
    }
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int i = 0; i < kRT; ++i) {
        acc[i][j][0] = fmaf(c[i][j][0], s[j][0], acc[i][j][0]);
        acc[i][j][1] = fmaf(c[i][j][1], s[j][1], acc[i][j][1]);
        acc[i][j][2] = fmaf(c[i][j][2], s[j][0], acc[i][j][2]);
        acc[i][j][3] = fmaf(c[i][j][3], s[j][1], acc[i][j][3]);
      }
  }
  // the warps' partial sums, [token][row], in warp order
#pragma unroll
  for (int i = 0; i < kRT; ++i)
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        red[(warp * kTok + 8 * j + 2 * t + (e & 1)) * kRows + 16 * i + g + 8 * (e >> 1)] =
            acc[i][j][e];
  __syncthreads();
  auto store = [&](int u, float v) {
    const int m = u / kRows, n = n0 + u % kRows;
    if (m >= a.M || n >= a.N) return;
    T* o = static_cast<T*>(a.y) + static_cast<int64_t>(m) * a.N + n;
    if constexpr (sizeof(T) == 4) {
      if (a.bias) v += static_cast<const float*>(a.bias)[n];
      *o = v;
    } else {
      if (a.bias) v += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
      *o = __float2bfloat16_rn(v);
    }
  };
  for (int u = threadIdx.x; u < kTok * kRows; u += kThreads) {
    float v = red[u];
#pragma unroll
    for (int q = 1; q < kWarps; ++q) v += red[q * kTok * kRows + u];
    if (a.split == 1) store(u, v);
    else red[u] = v;  // (read by this thread alone so far)
  }
  if (a.split == 1) return;
  cluster_sync();
  const int share = kTok * kRows / a.split;
  for (int u = rank * share + threadIdx.x; u < (rank + 1) * share; u += kThreads)
    store(u, cluster_sum1(smem_u32(red + u), a.split));
  cluster_sync();  // no CTA leaves while another reads its sums
}

template <typename T, int kRT, int kNT>
cudaError_t launch(const Args& a, cudaStream_t stream) {
  static std::atomic<uint64_t> attr{0};
  auto* kernel = fp8_small_kernel<T, kRT, kNT>;
  if (cudaError_t e = smem_attr_once(kernel, static_cast<int>(kMaxSmem), attr)) return e;
  const int most = (a.kb + a.split - 1) / a.split;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((a.N + 16 * kRT - 1) / (16 * kRT) * a.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes(a.M, most * kQBlock, 16 * kRT);
  cfg.stream = stream;
  cudaLaunchAttribute la[2];
  la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[0].val.programmaticStreamSerializationAllowed = 1;
  la[1].id = cudaLaunchAttributeClusterDimension;
  la[1].val.clusterDim.x = static_cast<unsigned>(a.split);
  la[1].val.clusterDim.y = 1;
  la[1].val.clusterDim.z = 1;
  cfg.attrs = la;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T>
cudaError_t pick(Args a, int num_sms, cudaStream_t stream) {
  // 32 rows per CTA (x quantised half as often) where that still gives most
  // SMs a CTA; K split while that leaves two CTAs to an SM and a CTA eight
  // blocks (a cluster takes 1.7 us longer to start and join)
  const bool wide = 3 * ((a.N + 31) / 32) >= 2 * num_sms;
  const int tiles = wide ? (a.N + 31) / 32 : (a.N + 15) / 16;
  a.split = 1;
  while (a.split < 8 && tiles * a.split * 2 <= 2 * num_sms && a.kb / (a.split * 2) >= 8)
    a.split *= 2;
  switch (token_tiles(a.M)) {
    case 1: return wide ? launch<T, 2, 1>(a, stream) : launch<T, 1, 1>(a, stream);
    case 2: return wide ? launch<T, 2, 2>(a, stream) : launch<T, 1, 2>(a, stream);
    default: return wide ? launch<T, 2, 4>(a, stream) : launch<T, 1, 4>(a, stream);
  }
}

}  // namespace

// Every CTA quantises its part of x again: at 14 rows (4096 x 1024) 5.1 us in
// one launch against 4.8 us in two, of which the second costs the host 2.4 us;
// at 32 rows 8.3 us against 6.7 us.
bool fp8_small_quantizes(int M) { return M <= 16; }

bool fp8_small_supported(int M, int K) {
  return M <= kFp8SmallMaxM && smem_bytes(M, K, 32) <= kMaxSmem;
}

cudaError_t launch_fp8_small(bool bf16, const void* x, uint8_t* xq, float* xs, int M, int K,
                             const uint8_t* wq, const float* ws, int N, const void* bias, void* y,
                             int num_sms, cudaStream_t stream) {
  if (M <= 0) return cudaSuccess;
  const Args a{x, xq, xs, wq, ws, bias, y, M, K, N, static_cast<int>(qblocks(K)), 1};
  return bf16 ? pick<__nv_bfloat16>(a, num_sms, stream) : pick<float>(a, num_sms, stream);
}

}  // namespace nrp
