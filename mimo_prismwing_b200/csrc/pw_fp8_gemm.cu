// pw_fp8_gemm.cu -- block-scaled FP8 linear layer on codes, for more tokens than
// pw_fp8_narrow.cu takes (the equation stands there).
//
// Tokens are the TMEM lanes (A), weight rows the columns (B): a thread then has
// one token, whose scale of a column block is one value, and the weight scale is
// one value for the 64 or 128 columns that a warp reads, so promoting a block is
// acc += d * (S xs) with packed FMAs.  Every 128-column block gets a fresh
// accumulator (the checkpoint's f32 scales are not powers of two, which the
// hardware block scaling would need), so the epilogue warps read 128 x columns of
// TMEM per block while the MMA warp fills the next accumulator.
//
//  * PAIR, for more than 128 tokens: two CTAs on a 256-token x 256-row tile
//    (cta_group::2), 128 tokens of each CTA's own and half of the weight rows
//    each.  A 128 x 128 tile of one CTA needs 8 KB of operands from shared memory
//    per 64 cycles of products, all that shared memory gives, before TMA has
//    written any; a pair's needs half of that.  Eight epilogue warps hold 128
//    sums per thread: setmaxnreg moves the registers of the other four to them.
//    One token takes 128 sums x 32 blocks of promotion, so the pipe that bounds
//    this kernel is the epilogue's FMAs and TMEM reads together with the MMAs.
//  * one CTA, up to 128 tokens: 128 x 128 tiles, bound by the weight stream.  When
//    the tiles are fewer than the SMs a cluster's CTAs split K and exchange their
//    sums (pw_cluster.cuh).
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "pw_cluster.cuh"
#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"
#include "pw_tc.cuh"

namespace pw {
namespace fp8g {

using namespace clu;
using tc::elect_one;
using tc::smem_desc_sw128;
using tc::tc_fence_after;
using tc::tc_fence_before;

constexpr int kProducerWarp = 0;
constexpr int kMmaWarp = 1;
constexpr int kEpiWarp0 = 4;  // warps 2 and 3 fill the first warpgroup (setmaxnreg works on whole ones)
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr uint32_t kSmemLimit = 227u * 1024u;
constexpr uint32_t kMaxBlocks = 32;   // K <= 4096
constexpr uint32_t kTokenGroup = 8;   // token tiles that neighbouring pairs share weights over
// Register split of PAIR: 256 x 224 + 128 x 40 of the 384 x 168 at launch.
constexpr int kRegsLaunch = 168, kRegsEpi = 224, kRegsOther = 40;
static_assert(kEpiWarps * 32 * kRegsEpi + kEpiWarp0 * 32 * kRegsOther <= kThreads * kRegsLaunch, "register split");

template <bool PAIR>
struct Cfg {
  static constexpr uint32_t BN = PAIR ? 256u : 128u;    // weight rows of a tile
  static constexpr uint32_t KBS = PAIR ? 1u : 2u;       // column blocks per stage
  static constexpr uint32_t A_BYTES = KBS * kTileRows * 128u;
  static constexpr uint32_t B_BYTES = KBS * 128u * 128u;  // this CTA's 128 weight rows
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr uint32_t NST = PAIR ? 6u : 3u;
  static constexpr uint32_t NACC = PAIR ? 2u : 4u;
  static constexpr uint32_t COLS = BN / 2u;  // a thread's columns: two warps per lane quarter
  static constexpr uint32_t XS = NST * STAGE;  // token scales [2 tiles][4 quarters][32 blocks][32 tokens] f32
  static constexpr uint32_t BARS = XS + 2u * 4u * kMaxBlocks * 32u * 4u;
  static constexpr uint32_t MISC = BARS + (2u * NST + 2u * NACC) * 8u;
  static constexpr uint32_t SMEM = MISC + 16u + 1024u;  // + alignment slack
  static constexpr uint32_t TMEM_COLS = NACC * BN;
  static_assert(SMEM <= kSmemLimit, "shared memory");
  static_assert((BN + 8u * kMaxSplits) * kTileRows * 4u <= NST * STAGE, "exchange buffer");
};

struct Args {
  Fp8CodesArgs a;
  CUtensorMap wmap, xmap;
  uint32_t row_tiles, token_tiles, stages, splits;
  uint32_t box_tokens;  // token rows that a stage loads
};

struct Shared {
  uint8_t *ring;
  float *xs;
  uint64_t *full, *empty, *tfull, *tempty;
  uint32_t *tmem_base;
  volatile int *abort;
};

__device__ __forceinline__ void mma_f8_pair_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}

__device__ __forceinline__ void tile_of(const Args &A, uint32_t u, uint32_t &row_tile, uint32_t &token_tile) {
  const uint32_t per = kTokenGroup * A.row_tiles, g = u / per, in = u % per;
  const uint32_t width = min(kTokenGroup, A.token_tiles - g * kTokenGroup);
  row_tile = in / width;
  token_tile = g * kTokenGroup + in % width;
}

template <bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) k_fp8_gemm(const __grid_constant__ Args A) {
  using C = Cfg<PAIR>;
  constexpr uint32_t NST = C::NST, NACC = C::NACC, BN = C::BN, CH = C::COLS / 32u;
  const Fp8CodesArgs &a = A.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Shared sh;
  sh.ring = smem;
  sh.xs = reinterpret_cast<float *>(smem + C::XS);
  sh.full = reinterpret_cast<uint64_t *>(smem + C::BARS);
  sh.empty = sh.full + NST;
  sh.tfull = sh.empty + NST;
  sh.tempty = sh.tfull + NACC;
  sh.tmem_base = reinterpret_cast<uint32_t *>(smem + C::MISC);
  sh.abort = reinterpret_cast<volatile int *>(smem + C::MISC + 4);

  const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
  // PAIR: cluster CTAs 2 k and 2 k + 1 are the pair of K split k; else CTA k is split k
  const uint32_t splits = A.splits, cta = PAIR || splits > 1u ? cluster_rank() : 0u;
  const uint32_t rank = PAIR ? cta & 1u : 0u, lead = PAIR ? cta & ~1u : cta, split = PAIR ? cta / 2u : cta;
  constexpr uint32_t CTAS = PAIR ? 2u : 1u;
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < NST; ++i) {
      mbar_init(&sh.full[i], 1);   // PAIR: the leading CTA's, both CTAs' loads complete on it
      mbar_init(&sh.empty[i], 1);  // commit after the stage's MMAs (PAIR: in both CTAs)
    }
    for (uint32_t i = 0; i < NACC; ++i) {
      mbar_init(&sh.tfull[i], 1);                  // commit after a block's MMAs
      mbar_init(&sh.tempty[i], CTAS * kEpiWarps);  // PAIR: the leading CTA's, both CTAs' warps
    }
    *sh.abort = 0;
    mbar_fence_init();
  }
  if (warp == (uint32_t)kProducerWarp && elect_one()) {
    prefetch_map(&A.wmap);
    prefetch_map(&A.xmap);
  }
  if (warp == (uint32_t)kMmaWarp) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(sh.tmem_base)),
                   "r"(C::TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(sh.tmem_base)),
                   "r"(C::TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) {
    __syncwarp();
    cluster_sync_all();  // both CTAs' barriers are initialised
  }
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t tmem = *sh.tmem_base;
  const uint32_t kblocks = a.K / 128u;
  // a cluster takes a tile; with K splits only one (the exchange reuses the ring)
  const uint32_t total = A.row_tiles * A.token_tiles;
  const uint32_t u_begin = blockIdx.x / (CTAS * splits), u_step = gridDim.x / (CTAS * splits);
  const uint32_t st0 = A.stages * split / splits, st1 = A.stages * (split + 1u) / splits;
  const uint32_t kb0 = st0 * C::KBS, kb1 = min(st1 * C::KBS, kblocks);  // its column blocks
  const bool qkv = a.layout != PW_LAYOUT_PLAIN;

  if (warp < (uint32_t)kEpiWarp0) {
    if (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == (uint32_t)kProducerWarp) {
      uint32_t slot = 0, phase = 0, issued = 0, parity = 0;
      const uint32_t bytes = C::B_BYTES + C::KBS * A.box_tokens * 128u;
      for (uint32_t u = u_begin; u < total; u += u_step) {
        uint32_t rt, tt;
        tile_of(A, u, rt, tt);
        const uint32_t row0 = rt * BN + rank * 128u;
        const int tok0 = (int)((tt * CTAS + rank) * kTileRows);
        // QKV: the CTA's two 64-row halves are each one run of checkpoint rows
        uint32_t src0 = row0, src1 = 0, unused;
        if (qkv) {
          map_row(a.layout, row0, src0, unused);
          map_row(a.layout, row0 + 64u, src1, unused);
        }
        for (uint32_t st = st0; st < st1; ++st) {
          if (bounded_wait(sh.abort, &sh.empty[slot], phase ^ 1u, a.flags)) {
            uint8_t *dst = sh.ring + slot * C::STAGE;
            const int kb = (int)(st * C::KBS);
            if (elect_one()) {
              if (PAIR) {
                const uint32_t bar = map_rank(smem_addr(&sh.full[slot]), lead);
                if (rank == 0u) mbar_arrive_expect_tx(&sh.full[slot], 2u * bytes);
                tma_load_pair(dst, &A.xmap, 0, tok0, kb, bar);
                if (!qkv) {
                  tma_load_pair(dst + C::A_BYTES, &A.wmap, 0, (int)src0, kb, bar);
                } else {
                  tma_load_pair(dst + C::A_BYTES, &A.wmap, 0, (int)src0, kb, bar);
                  tma_load_pair(dst + C::A_BYTES + 64u * 128u, &A.wmap, 0, (int)src1, kb, bar);
                }
              } else {
                mbar_arrive_expect_tx(&sh.full[slot], bytes);
                tc::tma_load_3d(dst, &A.xmap, 0, tok0, kb, &sh.full[slot]);
                if (!qkv) {
                  tc::tma_load_3d(dst + C::A_BYTES, &A.wmap, 0, (int)src0, kb, &sh.full[slot]);
                } else {
#pragma unroll
                  for (int j = 0; j < (int)C::KBS; ++j) {
                    uint8_t *d = dst + C::A_BYTES + j * (128u * 128u);
                    tc::tma_load_3d(d, &A.wmap, 0, (int)src0, kb + j, &sh.full[slot]);
                    tc::tma_load_3d(d + 64u * 128u, &A.wmap, 0, (int)src1, kb + j, &sh.full[slot]);
                  }
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
      // every copy in flight lands before the CTA (either CTA of the pair) can exit
      if (rank == 0u)
        for (uint32_t i = 0; i < NST; ++i)
          if (issued & (1u << i))
            if (!mbar_wait(&sh.full[i], (parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
    } else if (warp == (uint32_t)kMmaWarp && rank == 0u) {
      const uint32_t idesc = tc::instr_desc(BN, CTAS * kTileRows);
      const uint64_t ring_desc = smem_desc_sw128(smem_addr(sh.ring));
      uint32_t slot = 0, phase = 0, acc = 0, aphase = 0, pending = 0, pend_parity = 0;
      for (uint32_t u = u_begin; u < total; u += u_step) {
        for (uint32_t st = st0; st < st1; ++st) {
          const bool ok_full = bounded_wait(sh.abort, &sh.full[slot], phase, a.flags);
          tc_fence_after();
#pragma unroll
          for (uint32_t j = 0; j < C::KBS; ++j) {
            if (st * C::KBS + j >= kblocks) break;
            const bool ok = bounded_wait<PAIR>(sh.abort, &sh.tempty[acc], aphase ^ 1u, a.flags) && ok_full;
            tc_fence_after();
            if (ok) {
              const uint32_t d = tmem + acc * BN;
              // codes: a block's box_tokens rows follow one another; weights: 128 rows
              const uint64_t ad = ring_desc + ((slot * C::STAGE + j * A.box_tokens * 128u) >> 4);
              const uint64_t bd = ring_desc + ((slot * C::STAGE + C::A_BYTES + j * 128u * 128u) >> 4);
#pragma unroll
              for (uint32_t s = 0; s < 4; ++s) {
                if (PAIR)
                  mma_f8_pair_elect(d, ad + 2u * s, bd + 2u * s, idesc, s ? 1u : 0u);
                else
                  tc::mma_f8_elect(d, ad + 2u * s, bd + 2u * s, idesc, s ? 1u : 0u);
              }
            }
            if (PAIR)
              mma_commit_pair_elect(&sh.tfull[acc], 3u << lead);
            else
              tc::mma_commit_elect(&sh.tfull[acc]);
            pending |= 1u << acc;
            pend_parity = (pend_parity & ~(1u << acc)) | (aphase << acc);
            if (++acc == NACC) {
              acc = 0;
              aphase ^= 1u;
            }
          }
          if (PAIR)
            mma_commit_pair_elect(&sh.empty[slot], 3u << lead);
          else
            tc::mma_commit_elect(&sh.empty[slot]);
          if (++slot == NST) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      // every MMA is complete before the columns are freed
      for (uint32_t i = 0; i < NACC; ++i)
        if (pending & (1u << i))
          if (!mbar_wait(&sh.tfull[i], (pend_parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
    }
    if (splits > 1u) {
      // the epilogue's two cluster barriers count every thread
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    if (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // two warps per TMEM lane quarter: 32 tokens, half of the tile's columns each
    const uint32_t quarter = warp % 4u, half = (warp - kEpiWarp0) / 4u, col0 = half * C::COLS;
    const uint32_t row = quarter * 32u + lane;  // this thread's token of the CTA
    const uint32_t cols = tmem + ((quarter * 32u) << 16) + col0;
    // Token scales: the quarter's two warps copy its 32 tokens' ([block][token]:
    // read by lane without conflicts) for the next tile while this one runs.
    auto xs_fetch = [&](uint32_t u, uint32_t buf) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const uint32_t tok0 = (tt * CTAS + rank) * kTileRows + quarter * 32u;
      float *dst = sh.xs + (buf * 4u + quarter) * (kMaxBlocks * 32u);
      for (uint32_t e = half * 32u + lane; e < 32u * kblocks; e += 64u) {
        const uint32_t kb = e / 32u, t = e % 32u;
        if (tok0 + t < a.width) tc::cp_async4(dst + kb * 32u + t, a.scales + (uint64_t)(tok0 + t) * kblocks + kb);
      }
      tc::cp_async_commit();
    };
    // Weight scales: lane l holds block l of the scale rows of the warp's columns
    // (64 or 128 rows of one 128-row block, or of two 64-row QKV runs).
    auto ws_load = [&](uint32_t u, float &w0, float &w1) {
      uint32_t rt, tt, unused, s0, s1;
      tile_of(A, u, rt, tt);
      const uint32_t r = rt * BN + col0;
      w0 = w1 = 0.0f;
      if (r >= a.rows || lane >= kblocks) return;
      map_row(a.layout, r, unused, s0);
      w0 = w1 = __ldg(a.ws + (uint64_t)s0 * kblocks + lane);
      if (C::COLS > 64u && qkv) {
        map_row(a.layout, r + 64u, unused, s1);
        w1 = __ldg(a.ws + (uint64_t)s1 * kblocks + lane);
      }
    };
    uint32_t acc_slot = 0, aphase = 0, ti = 0;
    float wn0 = 0.0f, wn1 = 0.0f;
    if (u_begin < total) {
      ws_load(u_begin, wn0, wn1);
      xs_fetch(u_begin, 0u);
    }
    for (uint32_t u = u_begin; u < total; u += u_step, ++ti) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const uint32_t tok_q = (tt * CTAS + rank) * kTileRows + quarter * 32u;  // the warp's first token
      const uint32_t rows_here = tok_q < a.width ? min(32u, a.width - tok_q) : 0u;
      const uint32_t c_base = rt * BN + col0;  // the warp's first output column
      const bool active = rows_here != 0u && c_base < a.rows;
      tc::cp_async_wait_all();
      named_bar_sync(2u + quarter, 64u);  // this tile's scales are here, the other buffer is free
      float *xsb = sh.xs + ((ti & 1u) * 4u + quarter) * (kMaxBlocks * 32u);
      if (u + u_step < total) xs_fetch(u + u_step, (ti & 1u) ^ 1u);
      const float wc0 = wn0, wc1 = wn1;
      if (u + u_step < total) ws_load(u + u_step, wn0, wn1);

      float2 acc[CH][16];
#pragma unroll
      for (uint32_t q = 0; q < CH; ++q)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[q][i] = make_float2(0.0f, 0.0f);
      if (active) {
        // A chunk of 32 columns loads while the previous one is promoted, across
        // blocks too; the accumulator goes back to the MMA once its last chunk is
        // in registers.
        float v[2][32];
        bool ok = __all_sync(0xffffffffu, bounded_wait(sh.abort, &sh.tfull[acc_slot], aphase, a.flags));
        tc_fence_after();
        tc::tmem_ld32(cols + acc_slot * BN, v[0]);
        tc::tmem_wait_ld(v[0]);
#pragma unroll 1
        for (uint32_t kb = kb0; kb < kb1; ++kb) {
          const float x = xsb[kb * 32u + lane];
          const float s0 = ok ? __fmul_rn(__shfl_sync(0xffffffffu, wc0, kb), x) : 0.0f;
          const float s1 = C::COLS > 64u ? (ok ? __fmul_rn(__shfl_sync(0xffffffffu, wc1, kb), x) : 0.0f) : s0;
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q) {
            const float s = q < 2u ? s0 : s1;
            const float2 s2 = make_float2(s, s);
            float(&now)[32] = v[q & 1u];
            float(&next)[32] = v[(q & 1u) ^ 1u];
            bool load = true;
            if (q + 1u < CH) {
              tc::tmem_ld32(cols + acc_slot * BN + 32u * (q + 1u), next);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                if (PAIR)
                  arrive_remote(map_rank(smem_addr(&sh.tempty[acc_slot]), lead));
                else
                  mbar_arrive(&sh.tempty[acc_slot]);
              }
              if (++acc_slot == NACC) {
                acc_slot = 0;
                aphase ^= 1u;
              }
              load = kb + 1u < kb1;
              if (load) {
                ok = __all_sync(0xffffffffu, bounded_wait(sh.abort, &sh.tfull[acc_slot], aphase, a.flags));
                tc_fence_after();
                tc::tmem_ld32(cols + acc_slot * BN, next);
              }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
              acc[q][i] = __ffma2_rn(make_float2(now[2 * i], now[2 * i + 1]), s2, acc[q][i]);
            if (load) tc::tmem_wait_ld(next);
          }
        }
      } else {
        // no tokens or no rows here: keep the accumulators' handshake
        for (uint32_t kb = kb0; kb < kb1; ++kb) {
          bounded_wait(sh.abort, &sh.tfull[acc_slot], aphase, a.flags);
          tc_fence_after();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR)
              arrive_remote(map_rank(smem_addr(&sh.tempty[acc_slot]), lead));
            else
              mbar_arrive(&sh.tempty[acc_slot]);
          }
          if (++acc_slot == NACC) {
            acc_slot = 0;
            aphase ^= 1u;
          }
        }
      }

      if (splits > 1u) {
        const Exchange x(sh.ring, splits, split, CTAS, rank, min(BN, a.rows - rt * BN));
        __syncwarp();
        cluster_sync_all();  // every CTA's MMAs have read their last stage
        if (active) {
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q)
            x.send32(reinterpret_cast<const float(&)[32]>(acc[q]), col0 + 32u * q, row);
        }
        __syncwarp();
        cluster_sync_all();  // every CTA's sums have arrived
        const uint32_t first = x.split * x.share, mid = x.share / 2u & ~7u;
        const uint32_t in_tile = first < x.cols ? min(x.share, x.cols - first) : 0u;
        const uint32_t begin = half ? mid : 0u, end = half ? in_tile : min(mid, in_tile);
        bool ok = true;
        if (tok_q + lane < a.width)
#pragma unroll 1
          for (uint32_t b = begin; b < end; b += 8u) {  // rows are a multiple of 64: whole eights
            float v[8];
            x.receive8(v, b, row);
            const uint32_t c = rt * BN + first + b;
            ok = finish4(a.ep, make_float4(v[0], v[1], v[2], v[3]), bias4(a.ep, c), tok_q + lane, c) && ok;
            ok = finish4(a.ep, make_float4(v[4], v[5], v[6], v[7]), bias4(a.ep, c + 4u), tok_q + lane, c + 4u) && ok;
          }
        if (!ok) raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
      } else {
        // Outputs through staging rows in this tile's scale buffer, which the
        // quarter no longer needs once both of its warps are past the last block:
        // 16 columns at a time, a 64-byte row per token (16-byte chunk i at
        // position i ^ ((token >> 1) & 3), so that neither side conflicts), then
        // four columns per thread, coalesced.
        named_bar_sync(2u + quarter, 64u);
        if (active) {
          uint8_t *stg = reinterpret_cast<uint8_t *>(xsb) + half * 2048u;
          bool ok = true;
#pragma unroll
          for (uint32_t h = 0; h < C::COLS / 16u; ++h) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
              const float2 lo = acc[h / 2u][8u * (h % 2u) + 2u * i], hi = acc[h / 2u][8u * (h % 2u) + 2u * i + 1u];
              *reinterpret_cast<float4 *>(stg + lane * 64u + ((i ^ ((lane >> 1) & 3u)) << 4)) =
                  make_float4(lo.x, lo.y, hi.x, hi.y);
            }
            __syncwarp();
            const uint32_t c = lane % 4u, col = c_base + h * 16u + c * 4u;
            const float4 bias = bias4(a.ep, col);
#pragma unroll 1
            for (uint32_t r = lane / 4u; r < rows_here; r += 8u) {
              const float4 q = *reinterpret_cast<const float4 *>(stg + r * 64u + ((c ^ ((r >> 1) & 3u)) << 4));
              ok = finish4(a.ep, q, bias, tok_q + r, col) && ok;
            }
            __syncwarp();
          }
          if (!ok) raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (PAIR) {
    __syncwarp();
    cluster_sync_all();  // neither CTA's shared memory or columns go before both are done
  }
  tc_fence_after();
  if (warp == (uint32_t)kMmaWarp) {
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
  }
}

template <bool PAIR>
cudaError_t launch_one(const Fp8CodesArgs &a, int num_sms, cudaStream_t stream) {
  using C = Cfg<PAIR>;
  constexpr auto kernel = k_fp8_gemm<PAIR>;
  cudaError_t e = allow_smem<k_fp8_gemm<PAIR>>(C::SMEM);
  if (e != cudaSuccess) return e;
  if (PAIR) {
    // the register split must fit what the launch allocates, or setmaxnreg would wait for good
    static std::atomic<int> regs{0};
    if (regs.load(std::memory_order_relaxed) == 0) {
      cudaFuncAttributes at;
      if ((e = cudaFuncGetAttributes(&at, kernel)) != cudaSuccess) return e;
      regs.store(at.numRegs, std::memory_order_relaxed);
    }
    if (regs.load(std::memory_order_relaxed) < kRegsLaunch) return cudaErrorInvalidConfiguration;
  }
  Args A{};
  A.a = a;
  const bool qkv = a.layout != PW_LAYOUT_PLAIN;
  // up to 128 tokens a stage loads whole 32-token chunks of them
  A.box_tokens = PAIR ? 128u : (a.width + 31u) / 32u * 32u;
  if (!encode_weight_map(&A.wmap, a.w, a.rows, a.K, qkv ? 64u : 128u, qkv ? 1u : C::KBS) ||
      !encode_weight_map(&A.xmap, a.codes, a.width, a.K, A.box_tokens, C::KBS))
    return cudaErrorInvalidValue;
  constexpr uint32_t kTokens = PAIR ? 256u : 128u;
  A.row_tiles = (a.rows + C::BN - 1u) / C::BN;
  A.token_tiles = (a.width + kTokens - 1u) / kTokens;
  A.stages = (a.K / 128u + C::KBS - 1u) / C::KBS;
  const uint64_t tiles = (uint64_t)A.row_tiles * A.token_tiles;
  if (tiles > 0x7fffffffull / kMaxSplits) return cudaErrorInvalidValue;
  constexpr uint32_t CTAS = PAIR ? 2u : 1u;
  A.splits = best_splits<k_fp8_gemm<PAIR>>(tiles, A.stages * C::KBS, kMaxSplits / CTAS, CTAS, kThreads, C::SMEM, num_sms);
  const uint64_t at_once = (uint64_t)num_sms / CTAS;
  const uint32_t clusters = (uint32_t)(A.splits > 1u ? tiles * A.splits : tiles < at_once ? tiles : at_once);
  Launch l(CTAS * clusters, kThreads, CTAS * A.splits, C::SMEM, stream);
  e = cudaLaunchKernelEx(&l.cfg, kernel, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace fp8g

cudaError_t launch_fp8_gemm(const Fp8CodesArgs &a, int num_sms, cudaStream_t stream) {
  if (a.width == 0 || a.rows % 64u || a.K == 0 || a.K % 128u || a.K > 128u * fp8g::kMaxBlocks) return cudaErrorInvalidValue;
  return a.width <= 128u ? fp8g::launch_one<false>(a, num_sms, stream) : fp8g::launch_one<true>(a, num_sms, stream);
}

}  // namespace pw
