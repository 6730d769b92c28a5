// gemm_fp8.cu -- products of block-scaled e4m3 matrices on tcgen05
// (kind::f8f6f4, f32 accumulation), the forward product and the input's
// gradient of an 8-bit linear:
//
//   y[m, n] = sum_b xs[m, b] * ws[b, n / 128] * sum_{r in block b} xq[m, r] * w(r, n)
//
// with r over the reduction in blocks of 128.  A block's scales are constant
// over its 128 products, so the tensor cores sum one block (four K = 32 steps)
// into a TMEM accumulator, and the epilogue warps read it, multiply by the two
// scales' product (one number per row and 128 columns) and add to f32
// registers; TMEM holds two to four accumulators, so the next blocks run
// meanwhile.  The scales may be any f32 values: where their product leaves f32's
// range, a sum is multiplied by one after the other.
//
// The weight is stored once, [out, in].  The forward product reads it with
// the reduction contiguous (K-major B operand); the input's gradient reduces
// over the output features, so its B tile comes from the same bytes with the
// reduction along rows (MN-major descriptor), with no transposed copy.
//
// Warp roles (10 warps): 0 TMA producer, 1 TMEM allocator and MMA issuer,
// 2..9 epilogue (two groups of four, each half of the tile's columns).  The
// grid is persistent, one CTA per SM; where the tiles are few and the
// reduction is long, a cluster shares a tile's reduction (launch).  An epilogue
// thread keeps 128 sums and two 16-column reads of TMEM in its 168 registers.
//
// Bound by getting the operands to the tensor cores: a 256-wide block is 48 KB
// into shared memory and 48 KB out of it, 768 cycles at 128 bytes each, for 512
// cycles of MMA (128 x 256 x 128 products at 16384 FLOP a cycle), and takes about
// 940 (the tensor pipe is active for 55% of them).  A tile's store is not hidden:
// the warps that add up the next tile's blocks make it, and TMEM holds two blocks.
// Measured from codes to bf16: 16000 x 4096 to 1024 70 us (1.91 PFLOP/s; 3.4
// waves of tiles take four), 16000 x 1024 to 4096 with bias 81 us, of whose 14 tiles
// to an SM 8 blocks each account for 55, 896 x 1024 to 1024 6.3 us.  Tried and slower:
// CTA pairs (256 x 256 tiles, 76 us against 71: the hand-off over the cluster),
// sixteen epilogue warps (80 against 71), the last wave's tiles in halves (68.3
// against 68.2).
#include <algorithm>

#include "fp8.h"
#include "fp8_scales.cuh"
#include "sm100.cuh"

namespace nrp {
namespace {

constexpr int kBM = 128;
constexpr int kBR = 128;  // reduction per stage: one scale block, one swizzle row
constexpr uint32_t kABytes = kBM * kBR;
constexpr int kThreads = 320;
constexpr int kEpiWarp0 = 2;
constexpr int kMaxStages = 6, kMaxBufs = 4;
constexpr uint32_t kSlabBytes = 32 * 128;  // per epilogue warp: 32 rows x 128 B

// An epilogue warp's scales, kChunk blocks ahead: two buffers of 32 rows (an
// odd pitch, for the banks) and the weight's.
constexpr int kChunk = 8, kScalePitch = kChunk + 1;
constexpr int kScaleBuf = 32 * kScalePitch + kChunk;
constexpr int kScaleFloats = 2 * kScaleBuf;

// ... and its part of the bias, for the tile at hand and the next.
constexpr uint32_t kBiasBytes = 128 * 4;

// A split tile's partial sums: four more floats to a row, for the banks.
constexpr int kPartPitch = 128 + 4;

template <int kBN>
struct Cfg {
  static constexpr int kStages = kBN == 256 ? 3 : 5;
  static constexpr int kBufs = 512 / kBN;  // accumulators in TMEM
  static constexpr uint32_t kBBytes = kBN * kBR;
  static constexpr size_t kSmem =
      1024 + kStages * (kABytes + kBBytes) +
      8 * (kSlabBytes + 4 * kScaleFloats + 2 * kBiasBytes) + 256;
};
static_assert(Cfg<256>::kSmem <= 232448 && Cfg<128>::kSmem <= 232448,
              "shared memory budget");
static_assert(kBM * kPartPitch * 4 <= Cfg<128>::kStages * (kABytes + Cfg<128>::kBBytes),
              "a split tile's sums fit the ring");

struct Bars {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tfull[kMaxBufs];
  uint64_t tempty[kMaxBufs];
  uint64_t drain;
  uint32_t tmem_base;
  int abort;
};

__device__ __forceinline__ void umma_f8_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                           uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// kind::f8f6f4 instruction descriptor: f32 accumulator (bit 4), A and B e4m3
// (format 0), A K-major, B major at bit 16, N >> 3 at 17, M >> 4 at 24.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N, int b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void copy4_async(float* dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src)
               : "memory");
}

struct Args {
  const float* xs;   // [M, rb]
  const float* ws;   // forward [ceil(NO/128), rb], trans [rb, ceil(NO/128)]
  const void* bias;  // [NO] in the output's type, or null
  void* y;           // [M, NO]
  int M, NO, rb;     // rb: reduction blocks
  int tma_out;       // y's rows are 16-byte multiples: stored through map_y
  int split;         // CTAs to a tile (a cluster), each with blocks of the reduction
  int* err;
};

template <typename TO>
__device__ __forceinline__ float to_f32(TO v) {
  if constexpr (sizeof(TO) == 4) return v;
  else return __bfloat162float(v);
}

// A slab's rows where they are no 16-byte multiples in y: each row's columns by
// neighbouring lanes (10877 x 112 to 114, bf16: 5.8 us, 23.5 with each lane storing
// its own row).  Out of line: it would cost the ordinary path registers.
template <typename TO>
__device__ __noinline__ void store_rows(const uint8_t* slab, TO* o, int ldo, int rows, int cols) {
  constexpr int kWords = 128 / static_cast<int>(sizeof(TO)) / 32;  // a lane's columns
  const int lane = lane_id();
  for (int r0 = 0; r0 < rows; r0 += 8) {
    TO v[8][kWords];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const int at = (lane + 32 * w) * static_cast<int>(sizeof(TO));
        v[i][w] = *reinterpret_cast<const TO*>(slab + sw128_offset(r0 + i, at >> 4) + (at & 15));
      }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        if (r0 + i < rows && lane + 32 * w < cols)
          o[static_cast<int64_t>(r0 + i) * ldo + lane + 32 * w] = v[i][w];
  }
}

// kSplit: a cluster of a.split CTAs shares one tile's reduction.
template <int kBN, bool kTrans, typename TO, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_x,
                    const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ CUtensorMap map_y, const Args a) {
  constexpr int kStages = Cfg<kBN>::kStages;
  constexpr uint32_t kBBytes = Cfg<kBN>::kBBytes;
  constexpr int kBufs = Cfg<kBN>::kBufs;
  constexpr int kHalfN = kBN / 2;  // columns of one epilogue group
  constexpr int kSlabCols = 128 / static_cast<int>(sizeof(TO));
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sA = base;
  uint8_t* sB = sA + kStages * kABytes;
  uint8_t* sE = sB + kStages * kBBytes;
  float* sS = reinterpret_cast<float*>(sE + 8 * kSlabBytes);
  [[maybe_unused]] float* part = reinterpret_cast<float*>(sA);  // kSplit: [128][kPartPitch]
  uint8_t* sBias = reinterpret_cast<uint8_t*>(sS + 8 * kScaleFloats);
  Bars* ss = reinterpret_cast<Bars*>(sBias + 8 * 2 * kBiasBytes);
  const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = lane_id();
  const int tiles_m = (a.M + kBM - 1) / kBM;
  const int tiles_n = (a.NO + kBN - 1) / kBN;
  const int num_tiles = tiles_m * tiles_n;
  // this CTA's tiles and blocks of the reduction
  const int first = kSplit ? blockIdx.x / a.split : blockIdx.x;
  const int step = kSplit ? num_tiles : gridDim.x;
  const int share = kSplit ? (a.rb + a.split - 1) / a.split : a.rb;
  const int lo = kSplit ? min(static_cast<int>(cluster_ctarank()) * share, a.rb) : 0;
  const int blocks = kSplit ? min(share, a.rb - lo) : a.rb;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ss->full[s], 1);
      mbar_init(&ss->empty[s], 1);
    }
    for (int b = 0; b < kBufs; ++b) {
      mbar_init(&ss->tfull[b], 1);
      mbar_init(&ss->tempty[b], 8);
    }
    mbar_init(&ss->drain, 1);
    ss->abort = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
  }
  if (warp == 1) {
    tmem_alloc(&ss->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(ss->tmem_base);
  volatile int* abort_flag = &ss->abort;
  // Whether a wait of this CTA has expired, alike in a warp's lanes: what follows
  // is for whole warps.
  auto aborted = [&] { return __any_sync(0xffffffffu, *abort_flag) != 0; };
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    // ---------------------------------------------------------- producer
    uint32_t it = 0;
    for (int t = first; t < num_tiles && !aborted(); t += step) {
      const int m0 = t / tiles_n * kBM, n0 = t % tiles_n * kBN;
      for (int b = 0; b < blocks; ++b, ++it) {
        const int s = it % kStages;
        if (!warp_mbar_wait(&ss->empty[s], ((it / kStages) & 1) ^ 1, a.err, kDevTimeoutLoad)) {
          *abort_flag = 1;
          break;
        }
        if (elect_one()) {
          uint8_t *A = sA + s * kABytes, *B = sB + s * kBBytes;
          mbar_arrive_expect_tx(&ss->full[s], kABytes + kBBytes);
          tma_load_2d(A, &map_x, &ss->full[s], (lo + b) * kBR, m0);
          if constexpr (!kTrans) {
            tma_load_2d(B, &map_w, &ss->full[s], (lo + b) * kBR, n0);  // [n][128 r]
          } else {
            // [r][128 n]: one box per 128 columns
#pragma unroll
            for (int j = 0; j < kBN; j += 128)
              tma_load_2d(B + j * kBR, &map_w, &ss->full[s], n0 + j, (lo + b) * kBR);
          }
        }
        __syncwarp();
      }
    }
    // after an abort: the copies in flight land before the CTA goes
    if (aborted() && lane == 0)
      for (uint32_t j = it > static_cast<uint32_t>(kStages) ? it - kStages : 0; j < it; ++j)
        mbar_wait(&ss->full[j % kStages], (j / kStages) & 1, nullptr, 0);
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = idesc_e4m3_f32(kBM, kBN, kTrans ? 1 : 0);
    uint32_t it = 0;
    for (int t = first; t < num_tiles && !aborted(); t += step) {
      for (int b = 0; b < blocks; ++b, ++it) {
        const int s = it % kStages, buf = it % kBufs;
        if (!warp_mbar_wait(&ss->tempty[buf], ((it / kBufs) & 1) ^ 1, a.err, kDevTimeoutEpi) ||
            !warp_mbar_wait(&ss->full[s], (it / kStages) & 1, a.err, kDevTimeoutLoad)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t a0 = smem_u32(sA + s * kABytes), b0 = smem_u32(sB + s * kBBytes);
#pragma unroll
          for (int k = 0; k < kBR / 32; ++k) {
            const uint64_t ad = sdesc_sw128(a0 + k * 32, 16, 1024);
            // MN-major: 32 reduction rows of 128 bytes per step, 128-column
            // blocks kBR * 128 bytes apart
            const uint64_t bd = kTrans ? sdesc_sw128(b0 + k * 32 * 128, kBR * 128, 1024)
                                       : sdesc_sw128(b0 + k * 32, 16, 1024);
            umma_f8_ss(tmem + buf * kBN, ad, bd, idesc, k != 0);
          }
          umma_commit(&ss->empty[s]);
          umma_commit(&ss->tfull[buf]);
        }
        __syncwarp();
      }
    }
    if (aborted()) {
      if (elect_one()) umma_commit(&ss->drain);
      __syncwarp();
      mbar_wait(&ss->drain, 0, nullptr, 0);
    }
  } else {
    // ---------------------------------------------------------- epilogue
    const int quad = warp & 3, group = (warp - kEpiWarp0) >> 2;
    uint8_t* slab = sE + (warp - kEpiWarp0) * kSlabBytes;
    const int ncb = (a.NO + 127) / 128;
    float* scales = sS + (warp - kEpiWarp0) * kScaleFloats;
    // Blocks 8 c .. 8 c + 7 of tile t's scales, asked for while the eight
    // before them are used.  (A load of each lane's own row per block, one block
    // ahead, touches 32 sectors an instruction: 16000 x 1024 x 4096 took 77 us
    // with it, 68 with these.)
    // With a tile's first scales comes its bias, in 4-byte words where it lies so
    // (loaded where it is added: 896 x 1024 to 4096 9.0 against 8.0 us, 16000 rows
    // 78.9 against 77.7).
    uint8_t* my_bias = sBias + (warp - kEpiWarp0) * 2 * kBiasBytes;
    constexpr int kWordCols = 4 / static_cast<int>(sizeof(TO));
    const bool bias_words = a.bias && reinterpret_cast<uintptr_t>(a.bias) % 4 == 0;
    auto prefetch = [&](int t, int c, int buf, int bias_buf) {
      const int nb = min((t % tiles_n * kBN + group * kHalfN) / 128, ncb - 1);
      if (!kSplit && c == 0 && bias_words) {
        const int n0 = t % tiles_n * kBN + group * kHalfN;
#pragma unroll
        for (int w = 0; w < kHalfN / kWordCols; w += 32) {
          const int n = n0 + (w + lane) * kWordCols;
          if (n + kWordCols <= a.NO)
            copy4_async(reinterpret_cast<float*>(my_bias + bias_buf * kBiasBytes) + w + lane,
                        reinterpret_cast<const float*>(static_cast<const TO*>(a.bias) + n));
        }
      }
      const int64_t b = lo + c * kChunk + (lane & 7);
      float* to = scales + buf * kScaleBuf;
      if (b < lo + blocks) {
        // a row's eight scales are one sector: four rows to an instruction
        const int row0 = t / tiles_n * kBM + quad * 32 + (lane >> 3);
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          copy4_async(to + (i + (lane >> 3)) * kScalePitch + (lane & 7),
                      a.xs + static_cast<int64_t>(min(row0 + i, a.M - 1)) * a.rb + b);
        if (lane < kChunk)
          copy4_async(to + 32 * kScalePitch + lane,
                      kTrans ? a.ws + b * ncb + nb : a.ws + static_cast<int64_t>(nb) * a.rb + b);
      }
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    const int chunks = (blocks + kChunk - 1) / kChunk;
    int sbuf = 0, tbuf = 0;  // the buffers of the scales and the tile's bias
    if (first < num_tiles) prefetch(first, 0, 0, 0);
    commit();
    uint32_t it = 0;
    for (int t = first; t < num_tiles && !aborted(); t += step) {
      const int m0 = t / tiles_n * kBM, n0 = t % tiles_n * kBN + group * kHalfN;
      float acc[kHalfN];
#pragma unroll
      for (int e = 0; e < kHalfN; ++e) acc[e] = 0.f;
      bool ok = true;
      for (int b = 0; b < blocks; ++b, ++it) {
        const int buf = it % kBufs;
        if (b % kChunk == 0) {
          const int c = b / kChunk;
          if (b) sbuf ^= 1;
          __syncwarp();  // the other buffer's readers are done
          if (c + 1 < chunks) prefetch(t, c + 1, sbuf ^ 1, 0);
          else if (t + step < num_tiles) prefetch(t + step, 0, sbuf ^ 1, tbuf ^ 1);
          commit();
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          __syncwarp();
        }
        const float* sc = scales + sbuf * kScaleBuf;
        const float s = sc[lane * kScalePitch + b % kChunk] * sc[32 * kScalePitch + b % kChunk];
        if (!warp_mbar_wait(&ss->tfull[buf], (it / kBufs) & 1, a.err, kDevTimeoutMma)) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr =
            tmem + (static_cast<uint32_t>(quad * 32) << 16) + buf * kBN + group * kHalfN;
        uint32_t r[2][16];
        tmem_ld16(taddr, r[0]);
        if (__any_sync(0xffffffffu, !scale_in_range(s))) {
          // (a loop of its own: a branch in the one below makes it spill)
          float p, q;
          scale_factors(sc[lane * kScalePitch + b % kChunk], sc[32 * kScalePitch + b % kChunk], p,
                        q);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < kHalfN; c += 16) {
            tmem_ld16(taddr + c, r[1]);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              acc[c + e] = fmaf(__uint_as_float(r[1][e]) * p, q, acc[c + e]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ss->tempty[buf]);
          continue;
        }
        // 16 columns are added up while the next 16 come from TMEM
#pragma unroll
        for (int c = 0; c < kHalfN; c += 16) {
          uint32_t(&cur)[16] = r[(c / 16) & 1];
          tmem_ld_wait();
          if (c + 16 < kHalfN) {
            tmem_ld16(taddr + c + 16, r[(c / 16 + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ss->tempty[buf]);
          }
#pragma unroll
          for (int e = 0; e < 16; e += 2)
            fma_f32x2v(acc[c + e], acc[c + e + 1], __uint_as_float(cur[e]),
                       __uint_as_float(cur[e + 1]), s, acc[c + e], acc[c + e + 1]);
        }
      }
      if (!ok) break;
      if constexpr (kSplit) {
        // the ring's loads and MMAs are done: this CTA's sums take its place
        float* to = part + (quad * 32 + lane) * kPartPitch + group * kHalfN;
#pragma unroll
        for (int e = 0; e < kHalfN; e += 4)
          *reinterpret_cast<float4*>(to + e) =
              make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
        break;
      }
      sbuf ^= 1;  // the next tile's first scales
      const TO* bias = static_cast<const TO*>(a.bias);
      const uint8_t* tile_bias = my_bias + tbuf * kBiasBytes;
      tbuf ^= 1;
      TO* y = static_cast<TO*>(a.y);
#pragma unroll
      for (int c = 0; c < kHalfN; c += kSlabCols) {
        if (n0 + c >= a.NO) break;  // warp-uniform
        if (bias) {
          if (bias_words && n0 + c + kSlabCols <= a.NO) {
#pragma unroll
            for (int e = 0; e < kSlabCols; e += 16 / static_cast<int>(sizeof(TO))) {
              const uint4 q =
                  *reinterpret_cast<const uint4*>(tile_bias + (c + e) * sizeof(TO));
              const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(TO) == 4) {
                  acc[c + e + i] += __uint_as_float(w[i]);
                } else {
                  acc[c + e + 2 * i] += __uint_as_float(w[i] << 16);
                  acc[c + e + 2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
                }
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < kSlabCols; ++e)
              if (n0 + c + e < a.NO) acc[c + e] += to_f32(bias[n0 + c + e]);
          }
        }
        if (lane == 0) bulk_wait_read<0>();  // the store before has read the slab
        __syncwarp();
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          uint4 q;
          if constexpr (sizeof(TO) == 4)
            q = make_uint4(__float_as_uint(acc[c + 4 * ch]), __float_as_uint(acc[c + 4 * ch + 1]),
                           __float_as_uint(acc[c + 4 * ch + 2]),
                           __float_as_uint(acc[c + 4 * ch + 3]));
          else
            q = make_uint4(pack_bf16x2(acc[c + 8 * ch], acc[c + 8 * ch + 1]),
                           pack_bf16x2(acc[c + 8 * ch + 2], acc[c + 8 * ch + 3]),
                           pack_bf16x2(acc[c + 8 * ch + 4], acc[c + 8 * ch + 5]),
                           pack_bf16x2(acc[c + 8 * ch + 6], acc[c + 8 * ch + 7]));
          *reinterpret_cast<uint4*>(slab + sw128_offset(lane, ch)) = q;
        }
        if (a.tma_out) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_y, slab, n0 + c, m0 + quad * 32);
            bulk_commit();
          }
        } else {
          __syncwarp();
          store_rows(slab, y + static_cast<int64_t>(m0 + quad * 32) * a.NO + n0 + c, a.NO,
                     min(32, a.M - (m0 + quad * 32)), a.NO - n0 - c);
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  if constexpr (kSplit) {
    // Each CTA adds up and stores every split-th row, the cluster's sums in
    // the order of their ranks.
    __syncwarp();
    cluster_sync();
    const int m0 = first / tiles_n * kBM, n0 = first % tiles_n * kBN;
    const int rows = min(kBM, a.M - m0), cols = min(kBN, a.NO - n0);
    const TO* bias = static_cast<const TO*>(a.bias);
    TO* y = static_cast<TO*>(a.y);
    for (int i = warp * a.split + static_cast<int>(cluster_ctarank()); i < rows;
         i += kThreads / 32 * a.split) {
      const int c = lane * 4;
      if (c >= cols) continue;
      const float4 q = cluster_sum4(smem_u32(part + i * kPartPitch + c), a.split);
      float v[4] = {q.x, q.y, q.z, q.w};
      TO* o = y + static_cast<int64_t>(m0 + i) * a.NO + n0 + c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (bias && c + e < cols) v[e] += to_f32(bias[n0 + c + e]);
      if (a.tma_out) {  // whole groups of four, 16 (8) byte aligned
        if constexpr (sizeof(TO) == 4)
          *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        else
          *reinterpret_cast<uint2*>(o) =
              make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < cols) {
            if constexpr (sizeof(TO) == 4) o[e] = v[e];
            else o[e] = __float2bfloat16_rn(v[e]);
          }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int kBN, bool kTrans, typename TO, bool kSplit>
cudaError_t launch(const uint8_t* xq, int R, const uint8_t* wq, Args a, int num_sms,
                   cudaStream_t stream) {
  static std::atomic<uint64_t> attr{0};
  constexpr int kSmem = static_cast<int>(Cfg<kBN>::kSmem);
  auto* kernel = gemm_fp8_kernel<kBN, kTrans, TO, kSplit>;
  if (cudaError_t e = smem_attr_once(kernel, kSmem, attr)) return e;
  constexpr int es = sizeof(TO);
  CUtensorMap mx, mw, my;
  bool ok = make_tmap_2d(&mx, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, R, a.M, R, kBR, kBM, true);
  ok = ok && (kTrans ? make_tmap_2d(&mw, wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.NO, R, a.NO, 128,
                                    kBR, true)
                     : make_tmap_2d(&mw, wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, R, a.NO, R, kBR,
                                    kBN, true));
  a.tma_out = (static_cast<int64_t>(a.NO) * es) % 16 == 0 &&
              reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
  my = mx;
  if (ok && a.tma_out)
    ok = make_tmap_2d(&my, a.y,
                      es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                      es, a.NO, a.M, static_cast<uint64_t>(a.NO) * es, 128 / es, 32, true);
  if (!ok) return cudaErrorInvalidValue;
  const int64_t tiles =
      ((a.M + kBM - 1) / kBM) * static_cast<int64_t>((a.NO + kBN - 1) / kBN);
  if (tiles > 0x7fffffff) return cudaErrorInvalidValue;
  if constexpr (kSplit) {
    // The split with the least estimate, in us: 0.33 a block of the reduction, 1.1
    // for a cluster and 0.2 for each of its CTAs; all clusters have to run at once
    // (on a B200 33 of four CTAs, 15 of eight).  Split against one CTA to a tile,
    // bf16 output: 64 rows, 1024 to 1024 5.1 against 5.9 us, 4096 to 1024 6.4 against
    // 13.8; 600 rows, 4096 to 1024 9.8 (three CTAs; two 11.8) against 15.0; 896 rows
    // 12.2 against 15.1; and two CTAs where none are taken, 896 rows, 1024 to 1024
    // 7.8 against 6.5.
    static std::atomic<int> fit[64][9];
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return e;
    a.split = 1;
    float best = 0.33f * static_cast<float>(a.rb);
    for (int s = 2; s <= 8 && a.rb / s >= 2 && tiles * s <= num_sms; ++s) {
      const float us = 1.1f + 0.2f * static_cast<float>(s) +
                       0.33f * static_cast<float>((a.rb + s - 1) / s);
      if (us >= best) continue;
      int f = fit[dev & 63][s].load(std::memory_order_relaxed);
      if (f == 0) {
        f = max_clusters(kernel, s, kThreads, kSmem);
        fit[dev & 63][s].store(f > 0 ? f : -1, std::memory_order_relaxed);
      }
      if (tiles <= f) {
        a.split = s;
        best = us;
      }
    }
    if (a.split == 1) return launch<kBN, kTrans, TO, false>(xq, R, wq, a, num_sms, stream);
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
    return cudaLaunchKernelEx(&cfg, kernel, mx, mw, my, a);
  }
  const int grid = static_cast<int>(std::min<int64_t>(tiles, num_sms));
  return launch_pdl(kernel, dim3(grid), dim3(kThreads), static_cast<size_t>(kSmem), stream, mx, mw,
                    my, a);
}

template <bool kTrans, typename TO>
cudaError_t pick(const uint8_t* xq, int R, const uint8_t* wq, const Args& a, int num_sms,
                 cudaStream_t stream) {
  // Tiles of 128 columns when each SM gets one at most, else of 256, which
  // load 3/4 of the bytes per product.  128 against 256, reduction 1024, bf16
  // output: 896 x 1024 (56 tiles) 6.4 against 7.9 us, 2000 x 1024 (128) 6.6
  // against 8.0; 2432 x 1024 (152) 9.5 against 8.2, 896 x 4096 (224) 10.4
  // against 8.4, 16000 x 4096 88 against 80.
  const int64_t narrow = static_cast<int64_t>((a.M + kBM - 1) / kBM) * ((a.NO + 127) / 128);
  if (narrow > num_sms) return launch<256, kTrans, TO, false>(xq, R, wq, a, num_sms, stream);
  if (a.rb >= 8 && 2 * narrow <= num_sms)  // (fewer blocks: no split pays)
    return launch<128, kTrans, TO, true>(xq, R, wq, a, num_sms, stream);
  return launch<128, kTrans, TO, false>(xq, R, wq, a, num_sms, stream);
}

}  // namespace

cudaError_t launch_gemm_fp8(bool bf16_out, bool trans, const uint8_t* xq, const float* xs, int M,
                            int R, const uint8_t* wq, const float* ws, int NO, const void* bias,
                            void* y, int num_sms, int* err, cudaStream_t stream) {
  if (M <= 0) return cudaSuccess;
  Args a{};
  a.xs = xs;
  a.ws = ws;
  a.bias = bias;
  a.y = y;
  a.M = M;
  a.NO = NO;
  a.rb = static_cast<int>(qblocks(R));
  a.err = err;
  if (trans)
    return bf16_out ? pick<true, __nv_bfloat16>(xq, R, wq, a, num_sms, stream)
                    : pick<true, float>(xq, R, wq, a, num_sms, stream);
  return bf16_out ? pick<false, __nv_bfloat16>(xq, R, wq, a, num_sms, stream)
                  : pick<false, float>(xq, R, wq, a, num_sms, stream);
}

}  // namespace nrp
