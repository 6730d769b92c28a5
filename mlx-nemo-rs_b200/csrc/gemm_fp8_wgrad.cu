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
//
// Tiles are 128 k x 256 n, one per CTA, or narrower for few tokens.  Where they
// do not fill the SMs, a cluster of 2 to 8 CTAs splits the tokens of one
// tile; the partial tiles are summed in rank order through distributed shared
// memory, so the result does not depend on timing and needs no workspace.  That
// sum costs about 4 us for four partial 256-wide tiles, which narrower ones save
// at the price of more conversion.  The bias' gradient is summed from the dy
// tiles in shared memory, which all of a column's tiles hold: each takes every
// tiles_k-th 8 columns, so that no CTA is the slowest.
//
// Bound by shared-memory traffic: per 64 tokens 48 KB of MMA operands, 40 KB of
// TMA writes and 24 KB of conversion, 896 cycles at 128 bytes each against the
// tensor cores' 512, which makes 121 us at 16000 x 4096 x 1024.  Measured there
// with bias: 142 us, 0.95 PFLOP/s; 749 x 1024 x 1024 10.2 us.  TMEM holds a
// segment's sums and the running ones (below), which leaves no room in it for
// the converted operand.  Tried and slower (then against 126 to 135): CTA pairs
// with 256 x 256 tiles (165, the hand-off of both CTAs' conversions to one
// issuer), 512-wide tiles (145), the k0 = 0 tiles summing all of the bias (170 to
// 195), CTAs of its own for the bias (133, but a second wave of clusters at 1024
// x 1024).
//
// Warp roles (23 warps): 0 TMA producer of dy, 1 TMEM allocator and MMA
// issuer, 2 TMA producer of the codes, 3..6 the bias, 7..22 dequantisation:
// four sets of four warps that take every fourth step, so that a set's waits
// hide under the other sets' work.  Warps 0..15 store the result.
#include <algorithm>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fp8.h"
#include "fp8_quant.cuh"
#include "sm100.cuh"

namespace nrp {
namespace {

constexpr int kTK = 128;    // k columns of a CTA: one scale block
constexpr int kTok = 64;    // tokens per stage
constexpr int kStages = 4;
constexpr int kSets = 4;    // dequantising sets of four warps
constexpr int kBiasWarp0 = 3, kBiasWarps = 4;
constexpr int kDeqWarp0 = kBiasWarp0 + kBiasWarps;
constexpr int kThreads = 32 * (kDeqWarp0 + 4 * kSets);
constexpr int kStoreThreads = 512;
// Steps between two additions of the accumulator to the running sum.  The
// tensor cores cut each addition to the accumulator off instead of rounding it,
// an error that grows with their number: 8e-6 of the result's norm after 1000 (16000
// tokens of 16000 x 4096 x 1024, an f32 product being off by 6e-7).  After 64
// additions the accumulator is added to a second one in f32, rounded to
// nearest, and starts again from zero: 3e-7, for 141 us against 131 (every 32
// steps 6e-7 and 137 us, every 64 1.4e-6 and 135 us).
constexpr int kSeg = 16;
static_assert(kSeg % kSets == 0 && kSeg > kSets, "every set starts every segment");
constexpr uint32_t kBlk = kTok * 128;         // bytes of a 64-column bf16 block
constexpr uint32_t kABytes = kTK / 64 * kBlk;
constexpr uint32_t kRawBytes = kTok * kTK;

// kTN: n columns of a tile (MMA N)
template <int kTN>
struct Cfg {
  static constexpr uint32_t kBBytes = kTN / 64 * kBlk;
  static constexpr size_t kSmem = 1024 + kStages * (kABytes + kBBytes + kRawBytes) + kTN * 4 + 256;
  static_assert(kSmem <= 232448, "shared memory budget");
  static_assert(kTN * kTK * 4 <= kStages * (kABytes + kBBytes), "a partial tile fits the stages");
};

struct Bars {
  uint64_t full[kStages];   // dy by TMA
  uint64_t deq[kStages];    // codes dequantised
  uint64_t empty[kStages];
  uint64_t rfull[kStages];   // codes by TMA
  uint64_t rempty[kStages];
  uint64_t seg_full, seg_empty;  // a segment's sums are complete; are taken
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

// Two bf16 (low half first) of two codes in bytes 0 and 1 (sel 0x1404 of the
// word) or 2 and 3 (0x3424), times f.  A code's seven exponent and mantissa
// bits, moved to bf16's places, read as value * 2^-120 (the biases are 7 and
// 127; subnormal codes come out as bf16 subnormals, which the multiply
// takes); f is the block's scale * 2^120.  The NaN code is not one here.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t w, uint32_t f) {
  const uint32_t t = __byte_perm(w, 0u, kSel);  // each code in the high byte of its half
  const uint32_t v = (t & 0x80008000u) | ((t >> 4) & 0x07F007F0u);
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(f));
  return d;
}
// Before a barrier arrival that hands shared memory back to TMA: the thread's
// reads of it are complete, and ordered before the copy that overwrites it.  The
// arrival alone is not enough (generic reads against writes of the async
// proxy): without this, stages that come round again were overwritten under
// their readers.
__device__ __forceinline__ void reads_done() { fence_proxy_async_smem(); }
// Whether a byte of w is the NaN code.
__device__ __forceinline__ bool has_nan_code(uint32_t w) {
  return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
}

// Four consecutive elements; wide: 16 (or 8) bytes at once.
template <typename TO>
__device__ __forceinline__ void store_four(TO* p, float4 v, bool wide) {
  if (!wide) {
    store_one(p, v.x);
    store_one(p + 1, v.y);
    store_one(p + 2, v.z);
    store_one(p + 3, v.w);
  } else if constexpr (sizeof(TO) == 4) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
}

// Adds a segment's sums to the running sums kTN columns further on (`more`: there
// are some) in a quarter of the tile's columns, once full completes the phase
// `parity`, and arrives on empty.  Out of line, as inlined it takes registers from the
// conversion, which at 80 a thread (23 warps) spills 100 to 190 bytes all the same:
// the addresses and counts around the loops.
template <int kTN>
__device__ __noinline__ bool add_segment(uint32_t at, bool more, uint64_t* full, uint64_t* empty,
                                         uint32_t parity, int* err) {
  if (!warp_mbar_wait_hot(full, parity, err, kDevTimeoutMma)) return false;
  tc_fence_after();
#pragma unroll 1
  for (int c = 0; c < kTN / kSets; c += 16) {
    uint32_t r[16], t[16];
    tmem_ld16(at + c, r);
    if (more) tmem_ld16(at + kTN + c, t);
    tmem_ld_wait();
    if (more) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(t[e]));
    }
    tmem_st16(at + kTN + c, r);
  }
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if (lane_id() == 0) mbar_arrive(empty);
  return true;
}

template <int kTN, typename TO>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_wgrad_kernel(const __grid_constant__ CUtensorMap map_dy,  // bf16 [M, N], box (64, 64)
                     const __grid_constant__ CUtensorMap map_xq,  // u8 [M, K], box (128, 64)
                     const Args a) {
  constexpr uint32_t kBBytes = Cfg<kTN>::kBBytes;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sA = base;
  uint8_t* sB = sA + kStages * kABytes;
  uint8_t* sR = sB + kStages * kBBytes;
  float* sBias = reinterpret_cast<float*>(sR + kStages * kRawBytes);  // [kTN]
  Bars* ss = reinterpret_cast<Bars*>(sBias + kTN);
  const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = lane_id();
  const int tiles_k = (a.K + kTK - 1) / kTK;
  const int tile = static_cast<int>(blockIdx.x) / a.split;
  const int rank = static_cast<int>(blockIdx.x) % a.split;
  const int kt = tile % tiles_k;
  const int k0 = kt * kTK, n0 = tile / tiles_k * kTN;
  const int all = (a.M + kTok - 1) / kTok;
  const int st0 = static_cast<int>(static_cast<int64_t>(all) * rank / a.split);
  const int steps = static_cast<int>(static_cast<int64_t>(all) * (rank + 1) / a.split) - st0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ss->full[s], 1);
      mbar_init(&ss->deq[s], 4);
      mbar_init(&ss->rfull[s], 1);
      mbar_init(&ss->rempty[s], 4);
      mbar_init(&ss->empty[s], a.db ? 1 + kBiasWarps : 1);  // the MMAs, the bias warps
    }
    mbar_init(&ss->seg_full, 1);
    mbar_init(&ss->seg_empty, 4 * kSets);
    mbar_init(&ss->done, 1);
    ss->abort = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_dy);
    prefetch_tensormap(&map_xq);
  }
  if (warp == 1) {
    tmem_alloc(&ss->tmem_base, 2 * kTN);  // a segment's sums, the sum of the segments
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
  // A lane's wait, given up at once when another of the CTA has expired; the lanes
  // agree on it by `agreed`, at the latest where the warp comes together anyway.
  auto lane_wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return !*abort_flag && mbar_wait_hot(bar, parity, a.err, code);
  };
  auto agreed = [&](bool fine) {
    if (!__all_sync(0xffffffffu, fine)) {
      *abort_flag = 1;
      return false;
    }
    __syncwarp();  // (a vote orders no memory, which the arrivals after it need)
    return true;
  };
  pdl_launch_dependents();
  pdl_wait();

  if (warp == 0) {
    // ---------------------------------------------------- producer of dy
    int i = 0;
    for (; i < steps && !aborted(); ++i) {
      const int s = i % kStages;
      if (!warp_mbar_wait_hot(&ss->empty[s], ((i / kStages) & 1) ^ 1, a.err, kDevTimeoutLoad)) {
        *abort_flag = 1;
        break;
      }
      if (elect_one()) {
        mbar_arrive_expect_tx(&ss->full[s], kBBytes);
#pragma unroll
        for (int j = 0; j < kTN / 64; ++j)
          tma_load_2d(sB + s * kBBytes + j * kBlk, &map_dy, &ss->full[s], n0 + j * 64,
                      (st0 + i) * kTok);
      }
      __syncwarp();
    }
    if (aborted() && lane == 0)  // the copies in flight land before the CTA goes
      for (int j = i > kStages ? i - kStages : 0; j < i; ++j)
        mbar_wait(&ss->full[j % kStages], (j / kStages) & 1, nullptr, 0);
  } else if (warp == 2) {
    // ------------------------------------------------- producer of the codes
    int i = 0;
    for (; i < steps && !aborted(); ++i) {
      const int s = i % kStages;
      if (!warp_mbar_wait_hot(&ss->rempty[s], ((i / kStages) & 1) ^ 1, a.err, kDevTimeoutLoad)) {
        *abort_flag = 1;
        break;
      }
      if (elect_one()) {
        mbar_arrive_expect_tx(&ss->rfull[s], kRawBytes);
        tma_load_2d(sR + s * kRawBytes, &map_xq, &ss->rfull[s], k0, (st0 + i) * kTok);
      }
      __syncwarp();
    }
    if (aborted() && lane == 0)
      for (int j = i > kStages ? i - kStages : 0; j < i; ++j)
        mbar_wait(&ss->rfull[j % kStages], (j / kStages) & 1, nullptr, 0);
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc = idesc_bf16_f32(kTK, kTN, 1, 1);
    for (int i = 0; i < steps; ++i) {
      const int s = i % kStages;
      const uint32_t parity = (i / kStages) & 1;
      if (aborted() || !warp_mbar_wait_hot(&ss->full[s], parity, a.err, kDevTimeoutLoad) ||
          !warp_mbar_wait_hot(&ss->deq[s], parity, a.err, kDevTimeoutLoad)) {
        *abort_flag = 1;
        break;
      }
      if (i > 0 && i % kSeg == 0 &&
          !warp_mbar_wait_hot(&ss->seg_empty, (i / kSeg - 1) & 1, a.err, kDevTimeoutEpi)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a0 = smem_u32(sA + s * kABytes), b0 = smem_u32(sB + s * kBBytes);
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k)
          umma_ss(tmem, sdesc_sw128(a0 + k * 2048, kBlk, 1024),
                  sdesc_sw128(b0 + k * 2048, kBlk, 1024), idesc, (i % kSeg | k) != 0);
        umma_commit(&ss->empty[s]);
        if ((i + 1) % kSeg == 0 && i + 1 < steps) umma_commit(&ss->seg_full);
      }
      __syncwarp();
    }
    if (elect_one()) umma_commit(&ss->done);
    __syncwarp();
    // (the other warps wait at the CTA's barrier: its end bounds no wait)
    if (!warp_mbar_wait(&ss->done, 0, a.err, kDevTimeoutMma)) *abort_flag = 1;
  } else if (warp >= kBiasWarp0 && warp < kDeqWarp0) {
    // ----------------------------------------------------------- bias sums
    // the tile's 8-column chunks kt, kt + tiles_k, ...: four to a round over
    // the warps, a lane tokens lane and lane + 32
    if (a.db) {
      constexpr int kOwn = kTN / 8 / kBiasWarps;  // chunks a warp has at most
      const int c0 = kt + (warp - kBiasWarp0) * tiles_k, cstep = kBiasWarps * tiles_k;
      float sum[kOwn][8];
#pragma unroll
      for (int j = 0; j < kOwn; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[j][e] = 0.f;
      for (int i = 0; i < steps; ++i) {
        const int s = i % kStages;
        const bool fine = lane_wait(&ss->full[s], (i / kStages) & 1, kDevTimeoutLoad);
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          const int c = c0 + j * cstep;
          if (c >= kTN / 8) break;
#pragma unroll
          for (int h = 0; h < kTok; h += 32) {
            const uint4 q = *reinterpret_cast<const uint4*>(
                sB + s * kBBytes + (c >> 3) * kBlk + sw128_offset(h + lane, c & 7));
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sum[j][2 * e] += __uint_as_float(w[e] << 16);
              sum[j][2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
            }
          }
        }
        reads_done();
        if (!agreed(fine)) break;
        if (lane == 0) mbar_arrive(&ss->empty[s]);
      }
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        const int c = c0 + j * cstep;
        if (c >= kTN / 8) break;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v = sum[j][e];
#pragma unroll
          for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          if (lane == 0) sBias[c * 8 + e] = v;
        }
      }
    }
  } else {
    // ------------------------------------------------------ dequantisation
    // set `set` of four warps takes steps set, set + kSets, ...; a thread 16
    // codes (one 16-byte chunk c of the 128-byte row) of tokens row, row + 16, ...
    constexpr int kRowsT = kTok / 16;
    const int set = (warp - kDeqWarp0) >> 2;
    const int t = threadIdx.x - 32 * (kDeqWarp0 + 4 * set);
    const int row = t >> 3, c = t & 7;
    // chunk c: columns 16 c .. 16 c + 15 = 16-byte chunks 2 (c % 4), + 1 of
    // 64-column block c / 4.  Chunks 4..7 store their second half first, so
    // that the 16-byte stores of a row's eight threads fall on different banks
    const int flip = c >> 2;
    const uint32_t at0 = (c >> 2) * kBlk + sw128_offset(row, 2 * (c & 3) + flip);
    const uint32_t at1 = (c >> 2) * kBlk + sw128_offset(row, 2 * (c & 3) + (flip ^ 1));
    const float* xs = a.xs + kt;
    float sc[kRowsT];
    auto scales = [&](int i) {
#pragma unroll
      for (int h = 0; h < kRowsT; ++h) {
        const int m = (st0 + i) * kTok + row + 16 * h;
        sc[h] = i < steps && m < a.M ? xs[static_cast<int64_t>(m) * a.kb] : 0.f;
      }
    };
    scales(set);
    const uint32_t quarter =
        tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + set * (kTN / kSets);
    // Behind its first step of a segment, which the MMAs then find ready, a set
    // takes its quarter of the segment before.
    auto take_segment = [&](int b) -> bool {
      if (!aborted() &&
          add_segment<kTN>(quarter, b > 1, &ss->seg_full, &ss->seg_empty, (b - 1) & 1, a.err))
        return true;
      *abort_flag = 1;
      return false;
    };
    int taken = 0;
    for (int i = set; i < steps; i += kSets) {
      const int s = i % kStages;
      const uint32_t round = i / kStages;
      float sn[kRowsT];
#pragma unroll
      for (int h = 0; h < kRowsT; ++h) sn[h] = sc[h];
      scales(i + kSets);
      bool fine = lane_wait(&ss->rfull[s], round & 1, kDevTimeoutLoad);
      uint4 q[kRowsT];
#pragma unroll
      for (int h = 0; h < kRowsT; ++h)
        q[h] = *reinterpret_cast<const uint4*>(sR + s * kRawBytes + (row + 16 * h) * 128 + c * 16);
      reads_done();
      if (!agreed(fine)) break;
      if (lane == 0) mbar_arrive(&ss->rempty[s]);
      uint32_t out[kRowsT][8];
#pragma unroll
      for (int h = 0; h < kRowsT; ++h) {
        const float f = sn[h];
        const uint32_t w[4] = {flip ? q[h].z : q[h].x, flip ? q[h].w : q[h].y,
                               flip ? q[h].x : q[h].z, flip ? q[h].y : q[h].w};
        uint32_t(&o)[8] = out[h];
        // a power of two in [2^-117, 2^7] and no NaN code: the product is
        // exact, by bits; anything else rounded once
        const uint32_t fb = __float_as_uint(f);
        const bool nan = has_nan_code(w[0]) | has_nan_code(w[1]) | has_nan_code(w[2]) |
                         has_nan_code(w[3]);
        if ((fb & 0x807fffffu) == 0 && fb - (10u << 23) <= (124u << 23) && !nan) {
          const uint32_t f2 = ((fb >> 16) + (120u << 7)) * 0x10001u;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[2 * e] = codes_to_bf16<0x1404>(w[e], f2);
            o[2 * e + 1] = codes_to_bf16<0x3424>(w[e], f2);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(
                static_cast<__nv_fp8x2_storage_t>((w[e >> 1] >> (16 * (e & 1))) & 0xffffu),
                __NV_E4M3);
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&hr));
            o[e] = pack_bf16x2(code_times(v.x, f), code_times(v.y, f));
          }
        }
      }
      // only the stores wait for the MMAs that still read the stage
      fine = lane_wait(&ss->empty[s], (round & 1) ^ 1, kDevTimeoutLoad);
      uint8_t* dst = sA + s * kABytes;
#pragma unroll
      for (int h = 0; h < kRowsT; ++h) {
        // (16 rows on: two 1024-byte atoms, the same place in them)
        *reinterpret_cast<uint4*>(dst + at0 + 2048 * h) =
            make_uint4(out[h][0], out[h][1], out[h][2], out[h][3]);
        *reinterpret_cast<uint4*>(dst + at1 + 2048 * h) =
            make_uint4(out[h][4], out[h][5], out[h][6], out[h][7]);
      }
      fence_proxy_async_smem();
      if (!agreed(fine)) break;
      if (lane == 0) mbar_arrive(&ss->deq[s]);
      if (i >= kSeg && i % kSeg < kSets) {
        if (!take_segment(i / kSeg)) break;
        ++taken;
      }
    }
    // a last segment too short for this set to have a step in it
    if (taken < (steps - 1) / kSeg && !aborted()) take_segment((steps - 1) / kSeg);
  }

  // ------------------------------------------------------------- the result
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // After an expired wait (the context's error word names it) this CTA's sums are
  // NaN, in its tile or its share of one.
  const bool lost = *abort_flag != 0;
  const int quad = warp & 3, grp = warp >> 2;  // 32 columns of n at a time
  const bool storer = threadIdx.x < kStoreThreads;
  const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  // 32 columns of the result: the last segment's, and the sum of those before
  auto sums = [&](int c, float (&v)[32]) {
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      uint32_t r[16], t[16];
      tmem_ld16(taddr + c + h, r);
      if (steps > kSeg) tmem_ld16(taddr + kTN + c + h, t);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e)
        v[h + e] = __uint_as_float(r[e]) + (steps > kSeg ? __uint_as_float(t[e]) : 0.f);
    }
    if (lost) {
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(0x7fc00000u);
    }
  };
  if (lost && threadIdx.x < kTN) sBias[threadIdx.x] = __uint_as_float(0x7fc00000u);
  TO* dw = static_cast<TO*>(a.dw);
  TO* db = static_cast<TO*>(a.db);
  // bias columns this CTA summed (this rank writes its share of them)
  auto bias_here = [&](int c) { return db && (c >> 3) % tiles_k == kt && n0 + c < a.N; };
  if (a.split == 1) {
    if (storer) {
      const int k = k0 + quad * 32 + lane;
#pragma unroll 1
      for (int c = grp * 32; c < kTN; c += 128) {
        float v[32];
        sums(c, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int n = n0 + c + e;
          if (n < a.N && k < a.K)
            store_one(dw + static_cast<int64_t>(n) * a.K + k, v[e]);
        }
      }
      if (threadIdx.x < kTN && bias_here(threadIdx.x))
        store_one(db + n0 + threadIdx.x, sBias[threadIdx.x]);
    }
  } else {
    // partial sums [kTN n][128 k] f32 over the (drained) stages
    float* part = reinterpret_cast<float*>(base);
    if (storer) {
#pragma unroll 1
      for (int c = grp * 32; c < kTN; c += 128) {
        float v[32];
        sums(c, v);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          part[(c + e) * kTK + quad * 32 + lane] = v[e];
      }
    }
    cluster_sync();
    // this rank's columns, four k at a time, the ranks' tiles in order
    const int c0 = kTN * rank / a.split, cols = kTN * (rank + 1) / a.split - c0;
    const bool wide = reinterpret_cast<uintptr_t>(dw) % 16 == 0;
    constexpr int kFly = 3;  // units whose loads are in flight together
    for (int u0 = threadIdx.x; u0 < cols * (kTK / 4); u0 += kFly * kThreads) {
      float4 sum[kFly];
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int u = min(u0 + i * kThreads, cols * (kTK / 4) - 1);
        const int nn = c0 + u / (kTK / 4), kk = (u % (kTK / 4)) * 4;
        sum[i] = cluster_sum4(smem_u32(part + nn * kTK + kk), a.split);
      }
#pragma unroll
      for (int i = 0; i < kFly; ++i) {
        const int u = u0 + i * kThreads;
        const int n = n0 + c0 + u / (kTK / 4), k = k0 + (u % (kTK / 4)) * 4;
        if (u < cols * (kTK / 4) && n < a.N && k < a.K)  // K % 16 == 0: all four are inside
          store_four(dw + static_cast<int64_t>(n) * a.K + k, sum[i], wide);
      }
    }
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const int nn = c0 + c;
      if (bias_here(nn)) store_one(db + n0 + nn, cluster_sum1(smem_u32(sBias + nn), a.split));
    }
    cluster_sync();  // no CTA leaves while another reads its tile
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 2 * kTN);
  }
}

// How a tile width would run: the CTAs that share a tile's tokens, and about how
// long it takes.
struct Plan {
  int split;
  float us;
};
// kStart: a launch whose tiles are not shared, with the result's store; kJoin: the
// partial tiles' sum over a cluster, and kRank for each of its CTAs; kStep: a
// step of 64 tokens.  From 1024 x 1024 (64 / 128 / 256 columns: 100 tokens 5.7 / 7.9 /
// 9.3 us, 749 tokens 10.1 / 10.1 / 12.6, 1500 tokens 15.2 / 12.8 / 14.2, 5000 tokens
// 38 / 25 / 21.7; these are tiles of 1, 2 and 4 CTAs).  With them 5000 x 560 x 120
// takes 64 columns and eight CTAs to a tile (11.6 us, 18.0 with 256), 12000 x 768 x
// 768 256 and seven (30.8, 38.7 with four).
template <int kTN>
constexpr float kStep = kTN == 256 ? 0.56f : kTN == 128 ? 0.41f : 0.36f;
template <int kTN>
constexpr float kJoin = kTN == 256 ? 4.2f : kTN == 128 ? 1.8f : 1.f;
constexpr float kStart = 5.f, kRank = 0.2f;

template <int kTN, typename TO>
cudaError_t allow_smem() {
  static std::atomic<uint64_t> attr{0};
  return smem_attr_once(fp8_wgrad_kernel<kTN, TO>, static_cast<int>(Cfg<kTN>::kSmem), attr);
}

// Puts width kTN in place of `best` if it runs faster.
template <int kTN, typename TO>
cudaError_t plan(const Args& a, int num_sms, int dev, Plan& best, int& width) {
  static std::atomic<int> fit[64][9];  // clusters that run at once, by size
  const int64_t tiles = qblocks(a.K) * ((a.N + kTN - 1) / kTN);
  const int steps = (a.M + kTok - 1) / kTok;
  auto better = [&](int split, float us) {
    if (width != 0 && us >= best.us) return;
    best = {split, us};
    width = kTN;
  };
  better(1, kStart + kStep<kTN> * static_cast<float>(steps) *
                         static_cast<float>((tiles + num_sms - 1) / num_sms));
  // all clusters have to run at once (on a B200 33 of four CTAs, 15 of eight)
  for (int s = 2; s <= 8 && s <= steps && tiles * s <= num_sms; ++s) {
    int f = fit[dev & 63][s].load(std::memory_order_relaxed);
    if (f == 0) {
      if (cudaError_t e = allow_smem<kTN, TO>()) return e;
      f = max_clusters(fp8_wgrad_kernel<kTN, TO>, s, kThreads, Cfg<kTN>::kSmem);
      fit[dev & 63][s].store(f > 0 ? f : -1, std::memory_order_relaxed);
    }
    if (tiles <= f)
      better(s, kStart + kJoin<kTN> + kRank * static_cast<float>(s) +
                    kStep<kTN> * static_cast<float>((steps + s - 1) / s));
  }
  return cudaSuccess;
}

template <int kTN, typename TO>
cudaError_t launch(const void* dy, const uint8_t* xq, const Args& a, cudaStream_t stream) {
  if (cudaError_t e = allow_smem<kTN, TO>()) return e;
  CUtensorMap mdy, mxq;
  if (!make_tmap_2d(&mdy, dy, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.N, a.M,
                    static_cast<uint64_t>(a.N) * 2, 64, kTok, true) ||
      !make_tmap_2d(&mxq, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.K, a.M, a.K, kTK, kTok, false))
    return cudaErrorInvalidValue;
  const int64_t tiles = qblocks(a.K) * ((a.N + kTN - 1) / kTN);
  if (tiles * a.split > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.split));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<kTN>::kSmem;
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
  return cudaLaunchKernelEx(&cfg, fp8_wgrad_kernel<kTN, TO>, mdy, mxq, a);
}

template <typename TO>
cudaError_t pick(const void* dy, const uint8_t* xq, Args a, int num_sms, cudaStream_t stream) {
  Plan best{};
  int width = 0, dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (cudaError_t e = plan<64, TO>(a, num_sms, dev, best, width)) return e;
  if (cudaError_t e = plan<128, TO>(a, num_sms, dev, best, width)) return e;
  if (cudaError_t e = plan<256, TO>(a, num_sms, dev, best, width)) return e;
  a.split = best.split;
  if (width == 64) return launch<64, TO>(dy, xq, a, stream);
  if (width == 128) return launch<128, TO>(dy, xq, a, stream);
  return launch<256, TO>(dy, xq, a, stream);
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
  return bf16_out ? pick<__nv_bfloat16>(dy, xq, a, num_sms, stream)
                  : pick<float>(dy, xq, a, num_sms, stream);
}

}  // namespace nrp
