// gemm_fp8_wgrad.cu -- the weight's and bias' gradient of an 8-bit linear
// from the 8-bit checkpoint of its input:
//
//   dw[n, k] = sum_m dy[m, n] * x~[m, k],   db[n] = sum_m dy[m, n]
//
// x~ = code * scale of block (m, k / 128).  The scale changes along the
// reduction (tokens), so it cannot leave the sum as in the forward product:
// the codes are scaled on the way into the tensor cores.  Dequantising warps
// turn a [64 tokens][128 k] tile of codes into bf16 (exact for the
// quantiser's power-of-two scales) in swizzled shared memory, and the MMA
// takes it and the [64 tokens][256 n] tile of dy (TMA) both with the
// reduction along rows (MN-major), so neither is ever transposed in memory.
// The accumulator holds dw transposed (lanes k, columns n): a warp's store of
// one column n is 32 consecutive k.
//
// The bf16 checkpoint never exists in HBM, and the codes are half its bytes.
// The kernel is bound by the bf16 tensor rate.
//
// One tile per CTA.  Where the tiles do not fill the SMs, a cluster of 2, 4 or
// 8 CTAs splits the tokens of one tile; the partial tiles are summed in rank
// order through distributed shared memory, so the result does not depend on
// timing and needs no workspace.
//
// Warp roles (16 warps): 0 TMA producer, 1 TMEM allocator and MMA issuer,
// 4..7 the bias sums (in the tiles with k0 = 0, from the dy tiles in shared
// memory), 8..15 dequantisation; all store the result.
#include <algorithm>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.h"
#include "sm100.cuh"

namespace nrp {
namespace {

constexpr int kTK = 128;   // k columns of a tile: MMA M, one scale block
constexpr int kTN = 256;   // n columns of a tile: MMA N
constexpr int kTok = 64;   // tokens per stage
constexpr int kStages = 4;
constexpr int kRaw = 4;    // stages of the code ring
constexpr uint32_t kABytes = kTok * kTK * 2;   // two 64-column blocks of 8 KB
constexpr uint32_t kBBytes = kTok * kTN * 2;   // four of 8 KB
constexpr uint32_t kBlk = kTok * 128;          // bytes of a 64-column bf16 block
constexpr uint32_t kRawBytes = kTok * kTK;
constexpr int kThreads = 512;
constexpr size_t kSmem = 1024 + kStages * (kABytes + kBBytes) + kRaw * kRawBytes + 512;
static_assert(kSmem <= 232448, "shared memory budget");
static_assert(kTN * kTK * 4 + kTN * 4 <= kStages * (kABytes + kBBytes), "partial tile fits the stages");

struct Bars {
  uint64_t full[kStages];   // dy by TMA
  uint64_t deq[kStages];    // codes dequantised
  uint64_t empty[kStages];
  uint64_t rfull[kRaw];
  uint64_t rempty[kRaw];
  uint64_t done;
  uint32_t tmem_base;
  int abort;
};

struct Args {
  const float* xs;  // [M, kb]
  void* dw;
  void* db;  // null: none
  int M, N, K, kb, split;
  int* err;
};

template <typename TO>
__device__ __forceinline__ void store_one(TO* p, float v) {
  if constexpr (sizeof(TO) == 4) *p = v;
  else *p = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [ra];\n\t}\n"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

template <typename TO>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_wgrad_kernel(const __grid_constant__ CUtensorMap map_dy,  // bf16 [M, N], box (64, 64)
                     const __grid_constant__ CUtensorMap map_xq,  // u8 [M, K], box (128, 64)
                     const Args a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sA = base;
  uint8_t* sB = sA + kStages * kABytes;
  uint8_t* sR = sB + kStages * kBBytes;
  Bars* ss = reinterpret_cast<Bars*>(sR + kRaw * kRawBytes);
  const int warp = warp_id(), lane = lane_id();
  const int tiles_k = (a.K + kTK - 1) / kTK;
  const int tile = blockIdx.x / a.split, rank = blockIdx.x % a.split;
  const int kt = tile % tiles_k;
  const int k0 = kt * kTK, n0 = tile / tiles_k * kTN;
  const bool bias = a.db != nullptr && kt == 0;
  const int all = (a.M + kTok - 1) / kTok;
  const int st0 = static_cast<int>(static_cast<int64_t>(all) * rank / a.split);
  const int steps = static_cast<int>(static_cast<int64_t>(all) * (rank + 1) / a.split) - st0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ss->full[s], 1);
      mbar_init(&ss->deq[s], 8);
      mbar_init(&ss->empty[s], bias ? 5 : 1);  // the MMAs, and the bias warps
    }
    for (int s = 0; s < kRaw; ++s) {
      mbar_init(&ss->rfull[s], 1);
      mbar_init(&ss->rempty[s], 8);
    }
    mbar_init(&ss->done, 1);
    ss->abort = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_dy);
    prefetch_tensormap(&map_xq);
  }
  if (warp == 1) {
    tmem_alloc(&ss->tmem_base, kTN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ss->tmem_base;
  volatile int* abort_flag = &ss->abort;
  pdl_launch_dependents();
  pdl_wait();

  float bsum0 = 0.f, bsum1 = 0.f;  // bias warps: columns n0 + 2 * (thread - 128), + 1
  if (warp == 0) {
    // ---------------------------------------------------------- producer
    if (lane == 0) {
      int i = 0, r = 0;  // dy stages and code stages issued
      // the code ring runs ahead of the dy ring by up to its depth: each
      // round issues whatever has room, codes first
      for (; i < steps && !*abort_flag; ++i) {
        const int m0 = (st0 + i) * kTok;
        const int sr = r % kRaw;
        if (!mbar_wait(&ss->rempty[sr], ((r / kRaw) & 1) ^ 1, a.err, kDevTimeoutLoad)) {
          *abort_flag = 1;
          break;
        }
        mbar_arrive_expect_tx(&ss->rfull[sr], kRawBytes);
        tma_load_2d(sR + sr * kRawBytes, &map_xq, &ss->rfull[sr], k0, m0);
        ++r;
        const int s = i % kStages;
        if (!mbar_wait(&ss->empty[s], ((i / kStages) & 1) ^ 1, a.err, kDevTimeoutLoad)) {
          *abort_flag = 1;
          break;
        }
        mbar_arrive_expect_tx(&ss->full[s], kBBytes);
#pragma unroll
        for (int j = 0; j < kTN / 64; ++j)
          tma_load_2d(sB + s * kBBytes + j * kBlk, &map_dy, &ss->full[s], n0 + j * 64, m0);
      }
      if (*abort_flag) {  // the copies in flight land before the CTA goes
        for (int j = i > kStages ? i - kStages : 0; j < i; ++j)
          mbar_wait(&ss->full[j % kStages], (j / kStages) & 1, nullptr, 0);
        for (int j = r > kRaw ? r - kRaw : 0; j < r; ++j)
          mbar_wait(&ss->rfull[j % kRaw], (j / kRaw) & 1, nullptr, 0);
      }
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16_f32(kTK, kTN, 1, 1);
      for (int i = 0; i < steps; ++i) {
        const int s = i % kStages;
        if (*abort_flag || !mbar_wait(&ss->full[s], (i / kStages) & 1, a.err, kDevTimeoutLoad) ||
            !mbar_wait(&ss->deq[s], (i / kStages) & 1, a.err, kDevTimeoutLoad)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t a0 = smem_u32(sA + s * kABytes), b0 = smem_u32(sB + s * kBBytes);
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k)
          umma_ss(tmem, sdesc_sw128(a0 + k * 2048, kBlk, 1024),
                  sdesc_sw128(b0 + k * 2048, kBlk, 1024), idesc, (i | k) != 0);
        umma_commit(&ss->empty[s]);
      }
      umma_commit(&ss->done);
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------ dequantisation
    // thread: 16 codes (one 16-byte chunk c of the 128-byte row) of tokens
    // row and row + 32
    const int t = threadIdx.x - 256;
    const int row = t >> 3, c = t & 7;
    const int flip = c >> 2;
    const float* xs = a.xs + kt;
    float sc[2];
    auto scales = [&](int i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int m = (st0 + i) * kTok + row + 32 * h;
        sc[h] = i < steps && m < a.M ? xs[static_cast<int64_t>(m) * a.kb] : 0.f;
      }
    };
    scales(0);
    for (int i = 0; i < steps; ++i) {
      const int s = i % kStages, sr = i % kRaw;
      const float s0 = sc[0], s1 = sc[1];
      scales(i + 1);
      if (*abort_flag || !mbar_wait(&ss->rfull[sr], (i / kRaw) & 1, a.err, kDevTimeoutLoad)) {
        *abort_flag = 1;
        break;
      }
      uint4 q[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        q[h] = *reinterpret_cast<const uint4*>(sR + sr * kRawBytes + (row + 32 * h) * 128 + c * 16);
      __syncwarp();
      if (lane == 0) mbar_arrive(&ss->rempty[sr]);
      if (!mbar_wait(&ss->empty[s], ((i / kStages) & 1) ^ 1, a.err, kDevTimeoutLoad)) {
        *abort_flag = 1;
        break;
      }
      // chunk c: columns 16 c .. 16 c + 15 = 16-byte chunks 2 (c % 4), + 1 of
      // 64-column block c / 4
      uint8_t* dst = sA + s * kABytes + (c >> 2) * kBlk;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = h ? s1 : s0;
        const uint32_t w[4] = {q[h].x, q[h].y, q[h].z, q[h].w};
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(
              static_cast<__nv_fp8x2_storage_t>((w[e >> 1] >> (16 * (e & 1))) & 0xffffu),
              __NV_E4M3);
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hr));
          o[e] = pack_bf16x2(v.x * f, v.y * f);
        }
        // the two halves of a quarter warp's rows take the chunks in opposite
        // order, so their 16-byte stores fall on different banks
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int hi = p ^ flip;
          const uint4 v = hi ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(dst + sw128_offset(row + 32 * h, 2 * (c & 3) + hi)) = v;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ss->deq[s]);
    }
  } else if (warp >= 4 && bias) {
    // ----------------------------------------------------------- bias sums
    const int t = threadIdx.x - 128;  // columns 2t, 2t + 1
    const int chunk = (t & 31) >> 2, word = t & 3;
    for (int i = 0; i < steps; ++i) {
      const int s = i % kStages;
      if (*abort_flag || !mbar_wait(&ss->full[s], (i / kStages) & 1, a.err, kDevTimeoutLoad)) {
        *abort_flag = 1;
        break;
      }
      const uint8_t* b = sB + s * kBBytes + (t >> 5) * kBlk;
      float p0 = 0.f, p1 = 0.f;
#pragma unroll 16
      for (int m = 0; m < kTok; ++m) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(b + sw128_offset(m, chunk) + word * 4);
        p0 += __uint_as_float(u << 16);
        p1 += __uint_as_float(u & 0xffff0000u);
      }
      bsum0 += p0;
      bsum1 += p1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ss->empty[s]);
    }
  }

  // ------------------------------------------------------------- the result
  __syncwarp();
  const bool fine = mbar_wait(&ss->done, 0, a.err, kDevTimeoutMma);
  if (!fine) *abort_flag = 1;
  tc_fence_after();
  __syncthreads();
  const int quad = warp & 3, grp = warp >> 2;  // 64 columns of n each
  const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + grp * 64;
  TO* dw = static_cast<TO*>(a.dw);
  TO* db = static_cast<TO*>(a.db);
  if (a.split == 1) {
    if (!*abort_flag) {
      const int k = k0 + quad * 32 + lane;
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t r[32];
        tmem_ld32(taddr + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int n = n0 + grp * 64 + c + e;
          if (n < a.N && k < a.K)
            store_one(dw + static_cast<int64_t>(n) * a.K + k,
                      steps > 0 ? __uint_as_float(r[e]) : 0.f);
        }
      }
      if (bias && warp >= 4 && warp < 8) {
        const int n = n0 + 2 * (static_cast<int>(threadIdx.x) - 128);
        if (n < a.N) store_one(db + n, bsum0);
        if (n + 1 < a.N) store_one(db + n + 1, bsum1);
      }
    }
  } else {
    // partial tile [n][k] f32 and bias sums over the (drained) stages
    float* part = reinterpret_cast<float*>(base);
    float* bpart = part + kTN * kTK;
#pragma unroll
    for (int c = 0; c < 64; c += 32) {
      uint32_t r[32];
      tmem_ld32(taddr + c, r);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 32; ++e)
        part[(grp * 64 + c + e) * kTK + quad * 32 + lane] =
            steps > 0 ? __uint_as_float(r[e]) : 0.f;
    }
    if (bias && warp >= 4 && warp < 8) {
      bpart[2 * (threadIdx.x - 128)] = bsum0;
      bpart[2 * (threadIdx.x - 128) + 1] = bsum1;
    }
    cluster_sync();
    // this rank's columns, four k at a time, the ranks' tiles in order
    const int cols = kTN / a.split;
    for (int u = threadIdx.x; u < cols * (kTK / 4); u += kThreads) {
      const int nn = rank * cols + u / (kTK / 4), kk = (u % (kTK / 4)) * 4;
      const uint32_t at = smem_u32(part + nn * kTK + kk);
      float4 sum = ld_cluster_f4(at, 0);
      for (int q = 1; q < a.split; ++q) {
        const float4 v = ld_cluster_f4(at, q);
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      const int n = n0 + nn, k = k0 + kk;
      if (n < a.N && k < a.K) {  // K % 16 == 0: the four are inside together
        TO* o = dw + static_cast<int64_t>(n) * a.K + k;
        store_one(o, sum.x);
        store_one(o + 1, sum.y);
        store_one(o + 2, sum.z);
        store_one(o + 3, sum.w);
      }
    }
    if (bias)
      for (int u = threadIdx.x; u < cols / 4; u += kThreads) {
        const int nn = rank * cols + 4 * u;
        float4 sum = ld_cluster_f4(smem_u32(bpart + nn), 0);
        for (int q = 1; q < a.split; ++q) {
          const float4 v = ld_cluster_f4(smem_u32(bpart + nn), q);
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
        const float v[4] = {sum.x, sum.y, sum.z, sum.w};
        for (int e = 0; e < 4; ++e)
          if (n0 + nn + e < a.N) store_one(db + n0 + nn + e, v[e]);
      }
    cluster_sync();  // no CTA leaves while another reads its tile
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTN);
  }
}

template <typename TO>
cudaError_t launch(const void* dy, const uint8_t* xq, Args a, int num_sms, cudaStream_t stream) {
  static std::atomic<uint64_t> attr{0};
  auto* kernel = fp8_wgrad_kernel<TO>;
  if (cudaError_t e = smem_attr_once(kernel, static_cast<int>(kSmem), attr)) return e;
  CUtensorMap mdy, mxq;
  if (!make_tmap_2d(&mdy, dy, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.N, a.M,
                    static_cast<uint64_t>(a.N) * 2, 64, kTok, true) ||
      !make_tmap_2d(&mxq, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, a.K, kTK, kTok, false))
    return cudaErrorInvalidValue;
  const int64_t tiles = qblocks(a.K) * ((a.N + kTN - 1) / kTN);
  const int steps = (a.M + kTok - 1) / kTok;
  // the largest split whose clusters still fit the SMs at once, and that
  // leaves every CTA a step
  a.split = 1;
  while (a.split < 8 && tiles * a.split * 2 <= num_sms && a.split * 2 <= steps) a.split *= 2;
  if (tiles * a.split > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute la[2];
  la[0].id = cudaLaunchAttributeClusterDimension;
  la[0].val.clusterDim.x = static_cast<unsigned>(a.split);
  la[0].val.clusterDim.y = 1;
  la[0].val.clusterDim.z = 1;
  la[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = la;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, mdy, mxq, a);
}

}  // namespace

cudaError_t launch_fp8_weight_grad(bool bf16_out, const void* dy, const uint8_t* xq,
                                   const float* xs, int M, int N, int K, void* dw, void* db,
                                   int num_sms, int* err, cudaStream_t stream) {
  if (M <= 0) {  // no tokens: the sums are empty
    const size_t es = bf16_out ? 2 : 4;
    if (cudaError_t e = cudaMemsetAsync(dw, 0, static_cast<size_t>(N) * K * es, stream)) return e;
    return db ? cudaMemsetAsync(db, 0, N * es, stream) : cudaSuccess;
  }
  Args a{};
  a.xs = xs;
  a.dw = dw;
  a.db = db;
  a.M = M;
  a.N = N;
  a.K = K;
  a.kb = static_cast<int>(qblocks(K));
  a.err = err;
  return bf16_out ? launch<__nv_bfloat16>(dy, xq, a, num_sms, stream)
                  : launch<float>(dy, xq, a, num_sms, stream);
}

}  // namespace nrp
