// pw_linear.cu -- linear layer over a 16-bit weight on tcgen05 / TMEM:
//   y[t, r] = round(act(sum_c x[t, c] W[r, c] + bias[r]) + residual[t, r]).
//
// Weight rows are the TMEM lanes (A), tokens the columns (B), both K-major in
// shared memory (128B swizzle, written by TMA, zero past the matrices' ends, so
// no size is special).  With weight rows on the lanes a warp's store covers 32
// consecutive outputs of one token, whatever the output's stride or alignment,
// and the bias is one value per thread.  In both kernels a producer warp fills
// the TMA ring, an MMA warp issues tcgen05.mma.kind::f16 into TMEM accumulators,
// and eight epilogue warps empty them.
//
//  * k_linear_pair, for many tokens and 16-bit outputs: two CTAs on one 256 x 256
//    tile (cta_group::2): each holds its 128 weight rows and half of the tokens,
//    so the shared memory that a tensor core reads per product is half of what a
//    128 x 256 tile of one CTA needs.  Persistent pairs, two accumulators, all of
//    a tile's K in one accumulator.  Bound by the tensor pipe.
//  * k_linear_tile, for the widths between and for what a pair's accumulator would not
//    hold exactly enough (f32 outputs, long K): 128 x 32, 64 or 128 tiles of one CTA.
//    K runs in segments of 512 columns: each gets a fresh accumulator, and the epilogue
//    adds the segments in registers.  (The tensor pipe truncates when it adds to an
//    accumulator: over 4096 columns in one accumulator an f32 result was 4.4e-6 off,
//    with segments it is below 1e-6; a 16-bit result does not show it.)
//
// When the tiles are fewer than the SMs, the CTAs (pairs) of a cluster split K:
// HBM bounds these widths, and a stream over a third of the SMs does not reach
// it.  They exchange their sums through distributed shared memory, 16 bytes per
// store, and each finishes its share of the tokens, so the join is as parallel as
// the products (77 x 5000 x 1024: 12.7 us when each lane sent single values and
// joined token by token, 7.7 us so).
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "pw_cluster.cuh"
#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"
#include "pw_tc.cuh"

namespace pw {
namespace lin {

using namespace clu;
using tc::elect_one;
using tc::smem_desc_sw128;
using tc::tc_fence_after;
using tc::tc_fence_before;

constexpr int kProducerWarp = 0;
constexpr int kMmaWarp = 1;
constexpr int kEpiWarp0 = 2;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr uint32_t kBlockK = 64;        // columns of a k-block: one 128-byte line
constexpr uint32_t kSmemLimit = 227u * 1024u;
// A 64-column block takes about 512 cycles in either kernel (a pair's products; a
// tile's operands through L2).
constexpr TileCost kCost{512u, 4000u, 8000u};
constexpr uint32_t kTokenGroup = 8;     // token tiles that neighbouring CTAs share weights over

template <int BN>
struct TileCfg {
  static constexpr uint32_t KBS = 2;  // k-blocks per stage: 32 KB of weights per TMA box
  static constexpr uint32_t A_BYTES = KBS * kTileRows * 128u;
  static constexpr uint32_t B_BYTES = KBS * (uint32_t)BN * 128u;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr uint32_t NST = (kSmemLimit - 2048u) / STAGE < 6u ? (kSmemLimit - 2048u) / STAGE : 6u;
  static constexpr uint32_t NACC = 4;    // accumulators: segments in flight
  static constexpr uint32_t SEG = 4;     // stages per segment: 512 columns
  static constexpr uint32_t BARS = NST * STAGE;
  static constexpr uint32_t MISC = BARS + (2u * NST + 2u * NACC) * 8u;
  static constexpr uint32_t SMEM = MISC + 16u + 1024u;  // + alignment slack
  static constexpr uint32_t TMEM_COLS = NACC * (uint32_t)BN;
  static_assert(SMEM <= kSmemLimit, "shared memory");
  // the K splits' exchange reuses the ring: [split][token of the share][128 rows] f32
  static_assert(((uint32_t)BN + 8u * kMaxSplits) * kTileRows * 4u <= NST * STAGE, "exchange buffer");
};

struct PairCfg {
  static constexpr uint32_t BN = 256;               // tokens of the pair's tile, half of them per CTA
  static constexpr uint32_t A_BYTES = kTileRows * 128u;
  static constexpr uint32_t B_BYTES = BN / 2u * 128u;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;  // one k-block
  static constexpr uint32_t NST = 7;
  static constexpr uint32_t BARS = NST * STAGE;
  static constexpr uint32_t MISC = BARS + (2u * NST + 4u) * 8u;
  static constexpr uint32_t SMEM = MISC + 16u + 1024u;
  static constexpr uint32_t TMEM_COLS = 2u * BN;
  static_assert(SMEM <= kSmemLimit, "shared memory");
  static_assert((BN + 8u * kMaxSplits) * kTileRows * 4u <= NST * STAGE, "exchange buffer");
};

struct Args {
  LinearArgs a;
  CUtensorMap wmap, xmap;
  uint32_t k3d;  // the maps have a k-block dimension (encode_rows16_map)
  uint32_t row_tiles, token_tiles, stages, splits;
};

// kind::f16 instruction descriptor: D f32, A and B both bf16 or both f16, K-major.
__device__ __forceinline__ uint32_t instr_desc16(uint32_t n, uint32_t m, bool bf16) {
  const uint32_t t = bf16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// One MMA (M, N, K = 16) issued by one lane of the converged warp.
__device__ __forceinline__ void mma_f16_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}

// The pair's MMA (M = 256 over both CTAs, N = 256), issued in the leading CTA.
__device__ __forceinline__ void mma_f16_pair_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}

struct Shared {
  uint8_t *ring;
  uint64_t *full, *empty, *tfull, *tempty;
  uint32_t *tmem_base;
  volatile int *abort;
};

// Tile u: neighbouring tiles share their token tiles within a group of
// kTokenGroup, so that the tiles in flight reuse both operands in L2.
__device__ __forceinline__ void tile_of(const Args &A, uint32_t u, uint32_t &row_tile, uint32_t &token_tile) {
  const uint32_t per = kTokenGroup * A.row_tiles, g = u / per, in = u % per;
  const uint32_t width = min(kTokenGroup, A.token_tiles - g * kTokenGroup);
  row_tile = in / width;
  token_tile = g * kTokenGroup + in % width;
}

// The residual of output column c, tokens t0 .. t0 + n - 1 (n >= 1): loads only,
// all N in flight, so they can be issued before what they are added to is ready.
// Past the last token they repeat it.
template <int N>
__device__ __forceinline__ void load_residual(const EpilogueArgs &e, uint64_t t0, uint32_t c, uint32_t n,
                                              uint32_t (&raw)[N]) {
  const uint64_t at = t0 * e.residual_stride + c;
  if (e.residual_dtype == PW_DTYPE_F32) {
    const uint32_t *p = static_cast<const uint32_t *>(e.residual) + at;
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) raw[j] = p[min(j, n - 1u) * e.residual_stride];
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(e.residual) + at;
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) raw[j] = p[min(j, n - 1u) * e.residual_stride];
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_rows(const float (&v)[N], T *p, uint64_t stride, uint32_t n) {
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
    if (j < n) p[j * stride] = from_f32<T>(v[j]);
}

// The epilogue of one thread: output column c of tokens t0 .. t0 + n - 1, raw its
// residual (load_residual).
template <int N>
__device__ __forceinline__ void finish(const EpilogueArgs &e, float (&v)[N], float bias, const uint32_t (&raw)[N],
                                       uint64_t t0, uint32_t c, uint32_t n, uint32_t *flags) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] += bias;
  activate_all(v, e.act);
  if (e.residual) {
    if (e.residual_dtype == PW_DTYPE_F32) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += __uint_as_float(raw[j]);
    } else if (e.residual_dtype == PW_DTYPE_BF16) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += __uint_as_float(raw[j] << 16);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += __half2float(__ushort_as_half((unsigned short)raw[j]));
    }
  }
  uint32_t top = 0u;
#pragma unroll
  for (uint32_t j = 0; j < N; ++j)
    if (j < n) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  if (top >= overflow_bits(e.y_dtype)) raise_flag(flags, PW_FLAG_NONFINITE_ROUND);
  const uint64_t at = t0 * e.y_stride + c;
  if (e.y_dtype == PW_DTYPE_F32) store_rows(v, static_cast<float *>(e.y) + at, e.y_stride, n);
  else if (e.y_dtype == PW_DTYPE_BF16) store_rows(v, static_cast<__nv_bfloat16 *>(e.y) + at, e.y_stride, n);
  else store_rows(v, static_cast<__half *>(e.y) + at, e.y_stride, n);
}

// The rest of a split tile's epilogue, from the CTA's own sums sent: joins and
// finishes this thread's row (output column c) for its half of the share, 8
// tokens at a time (each CTA runs this once: a short loop, because code that is
// fetched for the first time costs more than it computes).
__device__ __forceinline__ void finish_share(const Exchange &x, const LinearArgs &a, float bias, uint32_t tok0,
                                             uint32_t c, uint32_t row, uint32_t half) {
  const bool mine = c < a.rows;
  const uint32_t first = x.split * x.share, mid = x.share / 2u & ~7u;
  // tokens [begin, end) of the share
  const uint32_t in_tile = first < x.cols ? min(x.share, x.cols - first) : 0u;
  const uint32_t begin = half ? mid : 0u, end = half ? in_tile : min(mid, in_tile);
  uint32_t raw[8];
  const bool add = mine && a.ep.residual != nullptr;
  if (add && begin < end) load_residual(a.ep, tok0 + first + begin, c, min(8u, end - begin), raw);
  __syncwarp();
  cluster_sync_all();  // every CTA's sums have arrived
#pragma unroll 1
  for (uint32_t b = begin; b < end; b += 8u) {
    const uint32_t n = min(8u, end - b);
    uint32_t cur[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) cur[j] = raw[j];
    if (add && b + 8u < end) load_residual(a.ep, tok0 + first + b + 8u, c, min(8u, end - b - 8u), raw);
    float v[8];
    x.receive8(v, b, row);
    if (mine) finish(a.ep, v, bias, cur, tok0 + first + b, c, n, a.flags);
  }
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) k_linear_tile(const __grid_constant__ Args A) {
  using C = TileCfg<BN>;
  constexpr uint32_t NST = C::NST, NACC = C::NACC;
  const LinearArgs &a = A.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared sh;
  sh.ring = smem;
  sh.full = reinterpret_cast<uint64_t *>(smem + C::BARS);
  sh.empty = sh.full + NST;
  sh.tfull = sh.empty + NST;
  sh.tempty = sh.tfull + NACC;
  sh.tmem_base = reinterpret_cast<uint32_t *>(smem + C::MISC);
  sh.abort = reinterpret_cast<volatile int *>(smem + C::MISC + 4);

  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < NST; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);  // tcgen05.commit after the stage's MMAs
    }
    for (uint32_t i = 0; i < NACC; ++i) {
      mbar_init(&sh.tfull[i], 1);           // tcgen05.commit after the segment's MMAs
      mbar_init(&sh.tempty[i], kEpiWarps);  // one arrive per epilogue warp
    }
    *sh.abort = 0;
    mbar_fence_init();
  }
  if (warp == (uint32_t)kProducerWarp && elect_one()) {
    prefetch_map(&A.wmap);
    prefetch_map(&A.xmap);
  }
  if (warp == (uint32_t)kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(sh.tmem_base)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem = *sh.tmem_base;
  // A cluster takes a tile, its CTA `rank` the K stages [st0, st1).  With K
  // splits there is one tile per cluster (the exchange reuses the ring).
  const uint32_t total = A.row_tiles * A.token_tiles;
  const uint32_t splits = A.splits, rank = blockIdx.x % splits;
  const uint32_t u_begin = blockIdx.x / splits, u_step = gridDim.x / splits;
  const uint32_t st0 = A.stages * rank / splits, st1 = A.stages * (rank + 1u) / splits;

  if (warp == (uint32_t)kProducerWarp) {
    uint32_t slot = 0, phase = 0, issued = 0, parity = 0;
    for (uint32_t u = u_begin; u < total; u += u_step) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const int row0 = (int)(rt * kTileRows), tok0 = (int)(tt * BN);
      for (uint32_t st = st0; st < st1; ++st) {
        if (bounded_wait(sh.abort, &sh.empty[slot], phase ^ 1u, a.flags)) {
          uint8_t *dst = sh.ring + slot * C::STAGE;
          const int kb = (int)(st * C::KBS);
          if (elect_one()) {
            mbar_arrive_expect_tx(&sh.full[slot], C::STAGE);
            if (A.k3d) {
              tc::tma_load_3d(dst, &A.wmap, 0, row0, kb, &sh.full[slot]);
              tc::tma_load_3d(dst + C::A_BYTES, &A.xmap, 0, tok0, kb, &sh.full[slot]);
            } else {
#pragma unroll
              for (int j = 0; j < (int)C::KBS; ++j) {
                tc::tma_load_3d(dst + j * (kTileRows * 128u), &A.wmap, (kb + j) * (int)kBlockK, row0, 0,
                                &sh.full[slot]);
                tc::tma_load_3d(dst + C::A_BYTES + j * (BN * 128u), &A.xmap, (kb + j) * (int)kBlockK, tok0, 0,
                                &sh.full[slot]);
              }
            }
          }
          __syncwarp();
          issued |= 1u << slot;
          parity = (parity & ~(1u << slot)) | (phase << slot);
        }
        if (++slot == NST) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    // every copy in flight lands before the CTA can exit
    for (uint32_t i = 0; i < NST; ++i)
      if (issued & (1u << i))
        if (!mbar_wait(&sh.full[i], (parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
  } else if (warp == (uint32_t)kMmaWarp) {
    const uint32_t idesc = instr_desc16(BN, kTileRows, a.dtype == PW_DTYPE_BF16);
    const uint64_t ring_desc = smem_desc_sw128(smem_addr(sh.ring));
    uint32_t slot = 0, phase = 0, acc = 0, aphase = 0, pending = 0, pend_parity = 0;
    for (uint32_t u = u_begin; u < total; u += u_step) {
      bool ok_acc = true;
      for (uint32_t st = st0; st < st1; ++st) {
        const uint32_t in_seg = (st - st0) % C::SEG;
        if (in_seg == 0u) {
          ok_acc = bounded_wait(sh.abort, &sh.tempty[acc], aphase ^ 1u, a.flags);
          tc_fence_after();
        }
        const bool ok = bounded_wait(sh.abort, &sh.full[slot], phase, a.flags) && ok_acc;
        tc_fence_after();
        if (ok) {
          const uint32_t d = tmem + acc * (uint32_t)BN;
          const uint64_t ad = ring_desc + ((slot * C::STAGE) >> 4);
          const uint64_t bd = ad + (C::A_BYTES >> 4);
#pragma unroll
          for (uint32_t j = 0; j < C::KBS; ++j)
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s)
              mma_f16_elect(d, ad + ((j * kTileRows * 128u) >> 4) + 2u * s, bd + ((j * BN * 128u) >> 4) + 2u * s, idesc,
                            (in_seg | j | s) ? 1u : 0u);
        }
        tc::mma_commit_elect(&sh.empty[slot]);
        if (++slot == NST) {
          slot = 0;
          phase ^= 1u;
        }
        if (in_seg == C::SEG - 1u || st + 1u == st1) {
          tc::mma_commit_elect(&sh.tfull[acc]);
          pending |= 1u << acc;
          pend_parity = (pend_parity & ~(1u << acc)) | (aphase << acc);
          if (++acc == NACC) {
            acc = 0;
            aphase ^= 1u;
          }
        }
      }
    }
    // every MMA is complete before the columns are freed
    for (uint32_t i = 0; i < NACC; ++i)
      if (pending & (1u << i))
        if (!mbar_wait(&sh.tfull[i], (pend_parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
  } else {
    // two warps per TMEM lane quarter, each half of the token columns (all of
    // them for the first when there are only 32)
    const uint32_t quarter = warp % 4u, half = (warp - kEpiWarp0) / 4u;
    constexpr uint32_t COLS = BN >= 64 ? BN / 2 : 32, CH = COLS / 32u;
    const uint32_t col0 = half * COLS;
    const bool active = col0 < (uint32_t)BN;
    const uint32_t row = quarter * 32u + lane;  // of the tile
    uint32_t acc = 0, aphase = 0;
    for (uint32_t u = u_begin; u < total; u += u_step) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const uint32_t c = rt * kTileRows + row, tok0 = tt * BN;
      const bool mine = c < a.rows;
      const float bias = mine && a.ep.bias ? load_elem(a.ep.bias, c, a.ep.bias_dtype) : 0.0f;
      float sum[CH][32];
#pragma unroll
      for (uint32_t q = 0; q < CH; ++q)
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[q][j] = 0.0f;
      for (uint32_t st = st0; st < st1; st += C::SEG) {
        const bool ok = __all_sync(0xffffffffu, bounded_wait(sh.abort, &sh.tfull[acc], aphase, a.flags));
        tc_fence_after();
        if (ok && active) {
          const uint32_t src = tmem + ((quarter * 32u) << 16) + acc * (uint32_t)BN + col0;
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q) {
            float v[32];
            tc::tmem_ld32(src + 32u * q, v);
            tc::tmem_wait_ld(v);
#pragma unroll
            for (int j = 0; j < 32; ++j) sum[q][j] += v[j];
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_relaxed(&sh.tempty[acc]);
        if (++acc == NACC) {
          acc = 0;
          aphase ^= 1u;
        }
      }
      if (splits == 1u) {
        if (active && mine)
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q) {
            const uint32_t t0 = tok0 + col0 + 32u * q;
            if (t0 < a.width) {
              const uint32_t n = min(32u, a.width - t0);
              uint32_t raw[32];
              if (a.ep.residual) load_residual(a.ep, t0, c, n, raw);
              finish(a.ep, sum[q], bias, raw, t0, c, n, a.flags);
            }
          }
      } else {
        const Exchange x(sh.ring, splits, rank, 1u, 0u, min((uint32_t)BN, a.width - tok0));
        __syncwarp();
        cluster_sync_all();  // every CTA's MMAs have read their last stage
        if (active)
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q) x.send32(sum[q], col0 + 32u * q, row);
        finish_share(x, a, bias, tok0, c, row, half);
      }
    }
  }
  if (splits > 1u && warp < (uint32_t)kEpiWarp0) {
    // the epilogue's two cluster barriers count every thread
    __syncwarp();
    cluster_sync_all();
    cluster_sync_all();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == (uint32_t)kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
}

__global__ void __launch_bounds__(kThreads, 1) k_linear_pair(const __grid_constant__ Args A) {
  using C = PairCfg;
  constexpr uint32_t NST = C::NST, BN = C::BN;
  const LinearArgs &a = A.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared sh;
  sh.ring = smem;
  sh.full = reinterpret_cast<uint64_t *>(smem + C::BARS);
  sh.empty = sh.full + NST;
  sh.tfull = sh.empty + NST;
  sh.tempty = sh.tfull + 2;
  sh.tmem_base = reinterpret_cast<uint32_t *>(smem + C::MISC);
  sh.abort = reinterpret_cast<volatile int *>(smem + C::MISC + 4);

  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
  // cluster CTAs 2 k and 2 k + 1 are the pair of K split k
  const uint32_t cta = cluster_rank(), rank = cta & 1u, lead = cta & ~1u;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < NST; ++i) {
      mbar_init(&sh.full[i], 1);   // the leading CTA's: both CTAs' loads complete on it
      mbar_init(&sh.empty[i], 1);  // each CTA's: the pair's commit after the stage's MMAs
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&sh.tfull[i], 1);                // each CTA's: the pair's commit after the tile's MMAs
      mbar_init(&sh.tempty[i], 2u * kEpiWarps);  // the leading CTA's: both CTAs' epilogue warps
    }
    *sh.abort = 0;
    mbar_fence_init();
  }
  if (warp == (uint32_t)kProducerWarp && elect_one()) {
    prefetch_map(&A.wmap);
    prefetch_map(&A.xmap);
  }
  if (warp == (uint32_t)kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(sh.tmem_base)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();  // both CTAs' barriers are initialised
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem = *sh.tmem_base;
  // a cluster takes a tile; with K splits only one (the exchange reuses the ring)
  const uint32_t splits = A.splits, split = cta / 2u;
  const uint32_t total = A.row_tiles * A.token_tiles;
  const uint32_t u_begin = blockIdx.x / (2u * splits), u_step = gridDim.x / (2u * splits);
  const uint32_t kb0 = A.stages * split / splits, kb1 = A.stages * (split + 1u) / splits;

  if (warp == (uint32_t)kProducerWarp) {
    // this CTA's 128 weight rows and its half of the tokens
    uint32_t slot = 0, phase = 0, issued = 0, parity = 0;
    for (uint32_t u = u_begin; u < total; u += u_step) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const int row0 = (int)(rt * 2u * kTileRows + rank * kTileRows), tok0 = (int)(tt * BN + rank * (BN / 2u));
      for (uint32_t kb = kb0; kb < kb1; ++kb) {
        if (bounded_wait(sh.abort, &sh.empty[slot], phase ^ 1u, a.flags)) {
          uint8_t *dst = sh.ring + slot * C::STAGE;
          if (elect_one()) {
            const uint32_t bar = map_rank(smem_addr(&sh.full[slot]), lead);
            if (rank == 0u) mbar_arrive_expect_tx(&sh.full[slot], 2u * C::STAGE);
            if (A.k3d) {
              tma_load_pair(dst, &A.wmap, 0, row0, (int)kb, bar);
              tma_load_pair(dst + C::A_BYTES, &A.xmap, 0, tok0, (int)kb, bar);
            } else {
              tma_load_pair(dst, &A.wmap, (int)(kb * kBlockK), row0, 0, bar);
              tma_load_pair(dst + C::A_BYTES, &A.xmap, (int)(kb * kBlockK), tok0, 0, bar);
            }
          }
          __syncwarp();
          issued |= 1u << slot;
          parity = (parity & ~(1u << slot)) | (phase << slot);
        }
        if (++slot == NST) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
    // every copy in flight lands before either CTA can exit
    if (rank == 0u)
      for (uint32_t i = 0; i < NST; ++i)
        if (issued & (1u << i))
          if (!mbar_wait(&sh.full[i], (parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
  } else if (warp == (uint32_t)kMmaWarp) {
    if (rank == 0u) {
      const uint32_t idesc = instr_desc16(BN, 2u * kTileRows, a.dtype == PW_DTYPE_BF16);
      const uint64_t ring_desc = smem_desc_sw128(smem_addr(sh.ring));
      uint32_t slot = 0, phase = 0, acc = 0, aphase = 0, pending = 0, pend_parity = 0;
      for (uint32_t u = u_begin; u < total; u += u_step) {
        const bool ok_acc = bounded_wait<true>(sh.abort, &sh.tempty[acc], aphase ^ 1u, a.flags);
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (uint32_t kb = kb0; kb < kb1; ++kb) {
          const bool ok = bounded_wait(sh.abort, &sh.full[slot], phase, a.flags) && ok_acc;
          tc_fence_after();
          if (ok) {
            const uint64_t ad = ring_desc + ((slot * C::STAGE) >> 4);
            const uint64_t bd = ad + (C::A_BYTES >> 4);
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s)
              mma_f16_pair_elect(d, ad + 2u * s, bd + 2u * s, idesc, (kb != kb0 || s) ? 1u : 0u);
          }
          mma_commit_pair_elect(&sh.empty[slot], 3u << lead);
          if (++slot == NST) {
            slot = 0;
            phase ^= 1u;
          }
        }
        mma_commit_pair_elect(&sh.tfull[acc], 3u << lead);
        pending |= 1u << acc;
        pend_parity = (pend_parity & ~(1u << acc)) | (aphase << acc);
        if (++acc == 2u) {
          acc = 0;
          aphase ^= 1u;
        }
      }
      // every MMA is complete before either CTA's columns are freed
      for (uint32_t i = 0; i < 2; ++i)
        if (pending & (1u << i))
          if (!mbar_wait(&sh.tfull[i], (pend_parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
    }
  } else {
    // this CTA's 128 rows: two warps per TMEM lane quarter, half of the tokens each
    const uint32_t quarter = warp % 4u, half = (warp - kEpiWarp0) / 4u, col0 = half * (BN / 2u);
    uint32_t acc = 0, aphase = 0;
    for (uint32_t u = u_begin; u < total; u += u_step) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const uint32_t row = quarter * 32u + lane, c = rt * 2u * kTileRows + rank * kTileRows + row;
      const bool mine = c < a.rows;
      const float bias = mine && a.ep.bias ? load_elem(a.ep.bias, c, a.ep.bias_dtype) : 0.0f;
      // 32 tokens at a time, their residual loaded one step ahead (the first
      // while the tile's products still run)
      const uint32_t t_begin = tt * BN + col0;
      const bool add = mine && a.ep.residual != nullptr && splits == 1u;
      uint32_t raw[32];
      if (add && t_begin < a.width) load_residual(a.ep, t_begin, c, min(32u, a.width - t_begin), raw);
      const bool ok = __all_sync(0xffffffffu, bounded_wait(sh.abort, &sh.tfull[acc], aphase, a.flags));
      tc_fence_after();
      const uint32_t src = tmem + ((quarter * 32u) << 16) + acc * BN + col0;
      if (splits > 1u) {
        const Exchange x(sh.ring, splits, split, 2u, rank, min(BN, a.width - tt * BN));
        __syncwarp();
        cluster_sync_all();  // every pair's MMAs have read their last stage
        if (ok) {
#pragma unroll 1
          for (uint32_t q = 0; q < BN / 2u; q += 32u) {
            float v[32];
            tc::tmem_ld32(src + q, v);
            tc::tmem_wait_ld(v);
            x.send32(v, col0 + q, row);
          }
        }
        finish_share(x, a, bias, tt * BN, c, row, half);
      } else if (ok) {
#pragma unroll 1
        for (uint32_t q = 0; q < BN / 2u; q += 32u) {
          float v[32];
          tc::tmem_ld32(src + q, v);
          tc::tmem_wait_ld(v);
          const uint32_t t0 = t_begin + q, t1 = t0 + 32u;
          uint32_t cur[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) cur[j] = raw[j];
          if (add && q + 32u < BN / 2u && t1 < a.width) load_residual(a.ep, t1, c, min(32u, a.width - t1), raw);
          if (mine && t0 < a.width) finish(a.ep, v, bias, cur, t0, c, min(32u, a.width - t0), a.flags);
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_relaxed_remote(map_rank(smem_addr(&sh.tempty[acc]), lead));
      if (++acc == 2u) {
        acc = 0;
        aphase ^= 1u;
      }
    }
  }

  if (A.splits > 1u && warp < (uint32_t)kEpiWarp0) {
    // the epilogue's two cluster barriers count every thread
    __syncwarp();
    cluster_sync_all();
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  cluster_sync_all();  // neither CTA's shared memory or columns go before both are done
  tc_fence_after();
  if (warp == (uint32_t)kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
}

// The kernel's arguments over tiles of `rows` x `tokens`, boxes of `box_tokens`
// tokens and `kbs` k-blocks per stage; false when a map cannot be made.
bool make_args(const LinearArgs &a, uint32_t rows, uint32_t tokens, uint32_t box_tokens, uint32_t kbs, Args &A) {
  A.a = a;
  A.k3d = a.cols % kBlockK == 0u;
  const uint32_t kb = A.k3d ? kbs : 0u;
  if (!encode_rows16_map(&A.wmap, a.w, a.rows, a.cols, a.w_stride, a.dtype, kTileRows, kb) ||
      !encode_rows16_map(&A.xmap, a.x, a.width, a.cols, a.x_stride, a.dtype, box_tokens, kb))
    return false;
  A.row_tiles = (a.rows + rows - 1u) / rows;
  A.token_tiles = (a.width + tokens - 1u) / tokens;
  A.stages = (a.cols + kbs * kBlockK - 1u) / (kbs * kBlockK);
  A.splits = 1u;
  return (uint64_t)A.row_tiles * A.token_tiles <= 0x7fffffffull / kMaxSplits;
}

template <int BN>
cudaError_t launch_tile(const LinearArgs &a, int num_sms, cudaStream_t stream) {
  using C = TileCfg<BN>;
  Args A{};
  if (!make_args(a, kTileRows, BN, BN, C::KBS, A)) return cudaErrorInvalidValue;
  cudaError_t e = allow_smem<k_linear_tile<BN>>(C::SMEM);
  if (e != cudaSuccess) return e;
  const uint32_t tiles = A.row_tiles * A.token_tiles, sms = (uint32_t)num_sms;
  A.splits =
      best_splits<k_linear_tile<BN>>(kCost, tiles, A.stages * C::KBS, kMaxSplits, 1u, kThreads, C::SMEM, num_sms).n;
  Launch l(A.splits > 1u ? tiles * A.splits : tiles < sms ? tiles : sms, kThreads, A.splits, C::SMEM, stream);
  e = cudaLaunchKernelEx(&l.cfg, k_linear_tile<BN>, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_pair(const LinearArgs &a, int num_sms, cudaStream_t stream) {
  using C = PairCfg;
  Args A{};
  if (!make_args(a, 2u * kTileRows, C::BN, C::BN / 2u, 1u, A)) return cudaErrorInvalidValue;
  cudaError_t e = allow_smem<k_linear_pair>(C::SMEM);
  if (e != cudaSuccess) return e;
  const uint32_t tiles = A.row_tiles * A.token_tiles, pairs = (uint32_t)num_sms / 2u;
  A.splits = best_splits<k_linear_pair>(kCost, tiles, A.stages, kMaxSplits / 2u, 2u, kThreads, C::SMEM, num_sms).n;
  Launch l(2u * (A.splits > 1u ? tiles * A.splits : tiles < pairs ? tiles : pairs), kThreads, 2u * A.splits, C::SMEM,
           stream);
  e = cudaLaunchKernelEx(&l.cfg, k_linear_pair, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

// ------------------------------------------------------------- row conversion
// x rows in another type, or not 16-byte aligned: one pass into aligned rows.
template <typename T>
__global__ void k_convert_rows(const void *__restrict__ x, uint64_t x_stride, uint32_t x_dtype, uint32_t rows,
                               uint32_t cols, T *__restrict__ out, uint64_t out_stride) {
  pdl_wait();
  pdl_launch_dependents();
  for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y)
    for (uint32_t c = blockIdx.x * blockDim.x + threadIdx.x; c < cols; c += gridDim.x * blockDim.x)
      out[(uint64_t)r * out_stride + c] = from_f32<T>(load_elem(x, (uint64_t)r * x_stride + c, x_dtype));
}

}  // namespace lin

cudaError_t launch_convert_rows(const void *x, uint64_t x_stride, uint32_t x_dtype, uint32_t rows, uint32_t cols,
                                void *out, uint64_t out_stride, uint32_t dtype, cudaStream_t stream) {
  const dim3 grid((cols + 255u) / 256u < 64u ? (cols + 255u) / 256u : 64u, rows < 4096u ? rows : 4096u);
  if (dtype == PW_DTYPE_BF16)
    return launch_kernel(lin::k_convert_rows<__nv_bfloat16>, grid, dim3(256), 0, stream, x, x_stride, x_dtype, rows,
                         cols, static_cast<__nv_bfloat16 *>(out), out_stride);
  return launch_kernel(lin::k_convert_rows<__half>, grid, dim3(256), 0, stream, x, x_stride, x_dtype, rows, cols,
                       static_cast<__half *>(out), out_stride);
}

cudaError_t launch_linear(const LinearArgs &a, int num_sms, cudaStream_t stream) {
  if (a.rows == 0 || a.cols == 0 || (a.dtype != PW_DTYPE_BF16 && a.dtype != PW_DTYPE_F16)) return cudaErrorInvalidValue;
  if (a.width == 0) return cudaSuccess;
  // One token tile of the narrow kernel streams at HBM rate; its second tile
  // costs registers, and with rows enough for every SM the tile kernel's ring is
  // faster (16 tokens, 4096 columns: 512 rows 3.9 against 5.9 us, 4096 rows 8.8 against 8.6 us,
  // 16384 rows 30.0 against 25.1 us).
  if (a.width <= 8u || (a.width <= 16u && a.rows <= 16u * (uint32_t)num_sms))
    return launch_linear_narrow(a, num_sms, stream);
  // A pair's accumulator takes all of K, in K / 16 additions that truncate by up to 2^-23:
  // within a quarter of the output's half step (bf16 2^-8, f16 2^-11) for these K.  The
  // tile's segments cost time (2048 x 4096 x 16384: pairs 201 us, tiles 300 us).
  const uint32_t pair_cols = a.ep.y_dtype == PW_DTYPE_BF16 ? 131072u : a.ep.y_dtype == PW_DTYPE_F16 ? 16384u : 0u;
  if (a.cols <= pair_cols && a.width > 128u) return lin::launch_pair(a, num_sms, stream);
  // Below and above, the token count chooses: a wide tile reads the weights for fewer
  // column tiles, a narrow one pads less.  us at 32 / 64 / 128 / pair, bf16:
  //    32 tokens  [4096, 4096]  9.3 /  9.4 / 10.6 / 13.7   [16384, 4096] 26.2 / 26.7 / 28.4 / 28.9
  //    64         [4096, 8192] 17.5 / 16.0 / 17.4 / 20.7   [16384, 4096] 29.8 / 27.2 / 29.8 / 30.2
  //   128         [4096, 8192] 26.2 / 19.5 / 19.2 / 22.6   [16384, 4096] 48.0 / 32.7 / 30.7 / 32.7
  //   200         [4096, 8192] 47.0 / 28.5 / 24.9 / 24.7
  //   256         [4096, 4096] 26.5 / 16.8 / 16.6 / 19.6   [16384, 4096] 79.8 / 53.3 / 42.0 / 34.4
  //   512         [4096, 8192] 89.4 / 51.3 / 38.8 / 32.9
  // Where the tiles are few it is not always the best: 256 tokens of [4096, 4096] above, and
  // 100 of them 15.6 / 12.7 / 13.6 / 15.6.
  if (a.width <= 32u) return lin::launch_tile<32>(a, num_sms, stream);
  if (a.width <= 64u) return lin::launch_tile<64>(a, num_sms, stream);
  return lin::launch_tile<128>(a, num_sms, stream);
}

}  // namespace pw
