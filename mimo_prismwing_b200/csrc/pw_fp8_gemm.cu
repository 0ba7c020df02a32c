// pw_fp8_gemm.cu -- block-scaled FP8 linear layer on codes, for more tokens than
// pw_fp8_narrow.cu takes (the equation stands there).
//
// Tokens are the TMEM lanes (A), weight rows the columns (B): a thread then has
// one token, whose scale of a column block is one value, and the weight scale is
// one value for the 64 or 128 columns that a warp reads, so promoting a block is
// acc += d * (S xs).  (Packed FMAs, two values per instruction, were slower: 45 cycles
// for a warp's 32 values against 36.)  Every 128-column block gets a fresh
// accumulator (the checkpoint's f32 scales are not powers of two, which the
// hardware block scaling would need), so the epilogue warps read 128 x columns of
// TMEM per block while the MMA warp fills the next accumulator.
//
//  * PAIR, for many tokens: two CTAs on a 256-token x 256-row tile
//    (cta_group::2), 128 tokens of each CTA's own and half of the weight rows
//    each.  A 128 x 128 tile of one CTA needs 8 KB of operands from shared memory
//    per 64 cycles of products, all that shared memory gives, before TMA has
//    written any; a pair's needs half of that.  Eight epilogue warps hold 128
//    sums per thread: setmaxnreg moves the registers of the other four to them.
//    What bounds it is the promotion: a block's takes 950 cycles against 512 of
//    products (when 2048 x 16384 x 4096 took 164 us: 126 with an eighth of the FMAs, 152
//    with a quarter of the MMAs, 99 with both, 165 without the weights' loads).  Sixteen
//    warps with 64 sums each, with the registers that leaves, were slower, and so were
//    128-column accumulators, handed back by halves.
//  * one CTA, for the widths between: 128 x 128 tiles, 640 cycles per column block, of
//    which shared memory takes 512 (32 KB written by TMA, 32 KB read by the MMAs); with
//    few tokens the weight stream bounds it.  When the tiles are fewer than the SMs a
//    cluster's CTAs split K and exchange their sums (pw_cluster.cuh).
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
// Measured cycles (B200 at 1.9 GHz): the one-CTA tile 640 per block and 5500 per wave,
// 13500 where K splits are joined; a pair's, of four times the products, 950 and 11000.
// (Pairs do not split K: joining took them 28000, and wherever that beat an unsplit pair,
// split one-CTA tiles beat both.)  In us, one CTA / pair: 512 x 4096 x 4096 15.0 / 22.9, 768 x
// 4096 x 4096 27.9 / 23.9, 384 x 13568 x 4096 41.0 / 43.8, 1024 x 13568 x 4096 83.6 / 65.4;
// unsplit / split one-CTA tiles: 203 x 4096 x 2048 9.6 / 10.8, 64 x 4096 x 4096 14.4 / 9.9.
constexpr TileCost kCostOne{640u, 5500u, 13500u};
constexpr uint64_t kPairBlock = 950u, kPairWave = 11000u;
constexpr uint32_t kTokenGroup = 8;   // token tiles that neighbouring pairs share weights over
// Register split: 256 x 240 + 128 x 24, all of the 384 x 168 at launch.
constexpr int kRegsLaunch = 168, kRegsEpi = 240, kRegsOther = 24;
static_assert(kEpiWarps * 32 * kRegsEpi + kEpiWarp0 * 32 * kRegsOther <= kThreads * kRegsLaunch, "register split");

// RES: the residual comes into the output boxes by TMA (2048 x 16384 x 4096 bf16: 219 us
// with it read and added on the way out, 184 so).  That takes four boxes per warp to
// hide, and the ring gives way to them; without a residual four stages cost 6%.
template <bool PAIR, bool RES>
struct Cfg {
  static constexpr uint32_t BN = PAIR ? 256u : 128u;    // weight rows of a tile
  static constexpr uint32_t A_BYTES = kTileRows * 128u;  // a stage is one column block
  static constexpr uint32_t B_BYTES = 128u * 128u;       // this CTA's 128 weight rows
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr uint32_t NST = RES ? 4u : 5u;
  static constexpr uint32_t NACC = PAIR ? 2u : 4u;
  static constexpr uint32_t G = PAIR ? 2u : 4u;  // blocks whose scales are fetched together, as registers allow
  static constexpr uint32_t COLS = BN / 2u;  // a thread's columns: two warps per lane quarter
  static constexpr uint32_t BOXES = RES ? 4u : 2u;  // 2 KB output boxes per epilogue warp
  static constexpr uint32_t STG = NST * STAGE;
  static constexpr uint32_t XS = STG + kEpiWarps * BOXES * 2048u;  // token scales [2 tiles][4 quarters][32 tokens][32 blocks] f32
  static constexpr uint32_t WS = XS + 2u * 4u * 32u * kMaxBlocks * 4u;  // weight scales [2 tiles][BN / 64 runs of rows][32 blocks]
  static constexpr uint32_t BARS = WS + 2u * (BN / 64u) * kMaxBlocks * 4u;
  static constexpr uint32_t RBARS = BARS + (2u * NST + 2u * NACC) * 8u;  // residual boxes
  static constexpr uint32_t MISC = RBARS + kEpiWarps * BOXES * 8u;
  static constexpr uint32_t SMEM = MISC + 16u + 1024u;  // + alignment slack
  static constexpr uint32_t TMEM_COLS = NACC * BN;
  static_assert(SMEM <= kSmemLimit, "shared memory");
  // the ring and, behind it, the boxes, which K splits do not use
  static_assert(PAIR || (BN + 8u * kMaxSplits) * kTileRows * 4u <= XS, "exchange buffer");
};

struct Args {
  Fp8CodesArgs a;
  CUtensorMap wmap, xmap, ymap, rmap;
  bool tma_y;  // outputs by way of ymap: rows at 16-byte boundaries, no residual or RES
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

// For the thread that issues them all.
template <bool PAIR>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
}

__device__ __forceinline__ void lds(float (&v)[4], uint32_t at) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(at));
}
__device__ __forceinline__ void lds(float (&v)[2], uint32_t at) {
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(at));
}

__device__ __forceinline__ void tile_of(const Args &A, uint32_t u, uint32_t &row_tile, uint32_t &token_tile) {
  const uint32_t per = kTokenGroup * A.row_tiles, g = u / per, in = u % per;
  const uint32_t width = min(kTokenGroup, A.token_tiles - g * kTokenGroup);
  row_tile = in / width;
  token_tile = g * kTokenGroup + in % width;
}

template <bool PAIR, bool RES>
__global__ void __launch_bounds__(kThreads, 1) k_fp8_gemm(const __grid_constant__ Args A) {
  using C = Cfg<PAIR, RES>;
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
  // a cluster is a pair, or the CTAs that split a tile's K
  const uint32_t splits = PAIR || RES ? 1u : A.splits, cta = PAIR || splits > 1u ? cluster_rank() : 0u;
  const uint32_t rank = PAIR ? cta : 0u, lead = PAIR ? 0u : cta, split = PAIR ? 0u : cta;
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
    for (uint32_t i = 0; i < kEpiWarps * C::BOXES; ++i) mbar_init(reinterpret_cast<uint64_t *>(smem + C::RBARS) + i, 1);
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
  const bool qkv = a.layout != PW_LAYOUT_PLAIN;

  if (warp < (uint32_t)kEpiWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == (uint32_t)kProducerWarp) {
      uint32_t slot = 0, phase = 0, issued = 0, parity = 0;
      const uint32_t bytes = C::B_BYTES + A.box_tokens * 128u;
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
            const int kb = (int)st;
            if (elect_one()) {
              if (PAIR) {
                const uint32_t bar = map_rank(smem_addr(&sh.full[slot]), lead);
                if (rank == 0u) mbar_arrive_expect_tx(&sh.full[slot], 2u * bytes);
                tma_load_pair(dst, &A.xmap, 0, tok0, kb, bar);
                tma_load_pair(dst + C::A_BYTES, &A.wmap, 0, (int)src0, kb, bar);
                if (qkv) tma_load_pair(dst + C::A_BYTES + 64u * 128u, &A.wmap, 0, (int)src1, kb, bar);
              } else {
                mbar_arrive_expect_tx(&sh.full[slot], bytes);
                tc::tma_load_3d(dst, &A.xmap, 0, tok0, kb, &sh.full[slot]);
                tc::tma_load_3d(dst + C::A_BYTES, &A.wmap, 0, (int)src0, kb, &sh.full[slot]);
                if (qkv) tc::tma_load_3d(dst + C::A_BYTES + 64u * 128u, &A.wmap, 0, (int)src1, kb, &sh.full[slot]);
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
    } else if (warp == (uint32_t)kMmaWarp && rank == 0u && elect_one()) {
      // one thread: an election per instruction costs as much as an MMA takes
      const uint32_t idesc = tc::instr_desc(BN, CTAS * kTileRows);
      const uint64_t ring_desc = smem_desc_sw128(smem_addr(sh.ring));
      uint32_t slot = 0, phase = 0, acc = 0, aphase = 0, pending = 0, pend_parity = 0;
      for (uint32_t u = u_begin; u < total; u += u_step) {
        for (uint32_t st = st0; st < st1; ++st) {
          const bool ok_full = bounded_wait(sh.abort, &sh.full[slot], phase, a.flags);
          tc_fence_after();
          const bool ok = bounded_wait<PAIR>(sh.abort, &sh.tempty[acc], aphase ^ 1u, a.flags) && ok_full;
          tc_fence_after();
          if (ok) {
            const uint32_t d = tmem + acc * BN;
            const uint64_t ad = ring_desc + ((slot * C::STAGE) >> 4);
            const uint64_t bd = ad + (C::A_BYTES >> 4);
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s) mma_f8<PAIR>(d, ad + 2u * s, bd + 2u * s, idesc, s ? 1u : 0u);
          }
          mma_commit<PAIR>(&sh.tfull[acc], 3u);
          mma_commit<PAIR>(&sh.empty[slot], 3u);
          pending |= 1u << acc;
          pend_parity = (pend_parity & ~(1u << acc)) | (aphase << acc);
          if (++acc == NACC) {
            acc = 0;
            aphase ^= 1u;
          }
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
    __syncwarp();
    if (splits > 1u) {
      // the epilogue's two cluster barriers count every thread
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // two warps per TMEM lane quarter: 32 tokens, half of the tile's columns each
    const uint32_t quarter = warp % 4u, half = (warp - kEpiWarp0) / 4u, col0 = half * C::COLS;
    const uint32_t row = quarter * 32u + lane;  // this thread's token of the CTA
    const uint32_t cols = tmem + ((quarter * 32u) << 16) + col0;
    // The next tile's scales are copied while this one runs: token scales by the
    // quarter's two warps, a row of 32 blocks per token (G blocks i at position i ^
    // token: a lane's G blocks are one load without conflicts); weight scales, per 64
    // rows, by all warps.
    const uint32_t shift = 32u - __clz(kblocks - 1u);  // 2^shift >= kblocks (__clz(0) is 32)
    const auto fetch_scales = [&](uint32_t u, uint32_t buf) {
      uint32_t rt, tt, unused, row;
      tile_of(A, u, rt, tt);
      const uint32_t tok0 = (tt * CTAS + rank) * kTileRows + quarter * 32u;
      float *dst = sh.xs + (buf * 4u + quarter) * (kMaxBlocks * 32u);
      // 2^shift lanes per token
      const uint32_t kb = lane & ((1u << shift) - 1u), step = 64u >> shift;
      if (kb < kblocks)
        for (uint32_t t = (half * 32u + lane) >> shift; t < 32u && tok0 + t < a.width; t += step)
          tc::cp_async4(dst + t * 32u + ((kb / C::G) ^ (t % (32u / C::G))) * C::G + kb % C::G,
                        a.scales + (uint64_t)(tok0 + t) * kblocks + kb);
      const uint32_t run = warp - kEpiWarp0, r = rt * BN + run * 64u;
      if (run < BN / 64u && r < a.rows && lane < kblocks) {
        map_row(a.layout, r, unused, row);
        tc::cp_async4(reinterpret_cast<float *>(smem + C::WS) + (buf * (BN / 64u) + run) * 32u + lane,
                      a.ws + (uint64_t)row * kblocks + lane);
      }
      tc::cp_async_commit();
    };
    const uint32_t tempty_lead = map_rank(smem_addr(sh.tempty), lead);
    const bool quad_r = quad_access(a.ep.residual, a.ep.residual_stride, a.ep.residual_dtype);
    const bool quad_y = quad_access(a.ep.y, a.ep.y_stride, a.ep.y_dtype);
    // this warp's output boxes: 32 tokens x 64 bytes, `box` counts them over all tiles
    const uint32_t box_cols = a.ep.y_dtype == PW_DTYPE_F32 ? 16u : 32u, per_tile = C::COLS / box_cols;
    uint32_t box = 0;
    const auto box_at = [&](uint32_t b) {
      return smem_addr(smem + C::STG) + ((warp - kEpiWarp0) * C::BOXES + b % C::BOXES) * 2048u;
    };
    const auto box_bar = [&](uint32_t b) {
      return reinterpret_cast<uint64_t *>(smem + C::RBARS) + (warp - kEpiWarp0) * C::BOXES + b % C::BOXES;
    };
    const auto fetch_box = [&](uint32_t b, uint32_t col, uint32_t tok) {  // its residual
      mbar_arrive_expect_tx(box_bar(b), 2048u);
      tma_load_2d(box_at(b), &A.rmap, (int)col, (int)tok, box_bar(b));
    };
    uint32_t acc_slot = 0, aphase = 0, ti = 0;
    if (u_begin < total) fetch_scales(u_begin, 0u);
    for (uint32_t u = u_begin; u < total; u += u_step, ++ti) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const uint32_t tok_q = (tt * CTAS + rank) * kTileRows + quarter * 32u;  // the warp's first token
      const uint32_t rows_here = tok_q < a.width ? min(32u, a.width - tok_q) : 0u;
      const uint32_t c_base = rt * BN + col0;  // the warp's first output column
      const bool active = rows_here != 0u && c_base < a.rows;
      tc::cp_async_wait_all();
      named_bar_sync(2u, kEpiWarps * 32u);  // this tile's scales are here, the other buffer is free
      float *xsb = sh.xs + ((ti & 1u) * 4u + quarter) * (kMaxBlocks * 32u);
      if (u + u_step < total) fetch_scales(u + u_step, (ti & 1u) ^ 1u);

      if (RES && active && lane == 0) {
        tma_store_wait_read<0>();  // the last tile's outputs have left the boxes
        for (uint32_t i = 0; i < C::BOXES && i < per_tile; ++i) fetch_box(box + i, c_base + i * box_cols, tok_q);
      }
      float acc[C::COLS];
#pragma unroll
      for (uint32_t i = 0; i < C::COLS; ++i) acc[i] = 0.0f;
      if (active) {
        // A chunk of 32 columns loads while the previous one is promoted; the
        // accumulator goes back to the MMA once its last chunk is in registers.  A warp
        // issues in order, so what takes long to come back is asked for early: the next
        // accumulator's barrier half a chunk before it is needed, scales G blocks at
        // a time before the last chunk of the G (a load and two shuffles per block cost a
        // tenth of the loop).
        float v[2][32];
        float xg[C::G], wg[C::COLS / 64u][C::G], sg[C::COLS / 64u][C::G];
        const uint32_t xs_at = smem_addr(xsb) + lane * 128u;
        const uint32_t ws_at = smem_addr(smem + C::WS) + (((ti & 1u) * (BN / 64u) + half * (C::COLS / 64u)) * 128u);
        const auto ask = [&](uint32_t kb) {  // for the G blocks around kb
          lds(xg, xs_at + ((kb / C::G) ^ (lane % (32u / C::G))) * (4u * C::G));
#pragma unroll
          for (uint32_t h = 0; h < C::COLS / 64u; ++h) lds(wg[h], ws_at + h * 128u + (kb / C::G) * (4u * C::G));
        };
        const auto answer = [&]() {
#pragma unroll
          for (uint32_t h = 0; h < C::COLS / 64u; ++h)
#pragma unroll
            for (uint32_t i = 0; i < C::G; ++i) sg[h][i] = __fmul_rn(wg[h][i], xg[i]);
        };
        const auto next_scale = [&]() {
#pragma unroll
          for (uint32_t h = 0; h < C::COLS / 64u; ++h)
#pragma unroll
            for (uint32_t i = 0; i + 1u < C::G; ++i) sg[h][i] = sg[h][i + 1u];
        };
        ask(st0);
        answer();
        for (uint32_t i = 0; i < st0 % C::G; ++i) next_scale();
        bounded_wait(sh.abort, &sh.tfull[acc_slot], aphase, a.flags);
        __syncwarp();
        tc_fence_after();
        tc::tmem_ld32(cols + acc_slot * BN, v[0]);
        tc::tmem_wait_ld(v[0]);
#pragma unroll 1
        for (uint32_t kb = st0; kb < st1; ++kb) {
          const bool more = kb + 1u < st1;
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q) {
            const float s = sg[q / 2u][0];
            float(&now)[32] = v[q & 1u];
            float(&next)[32] = v[(q & 1u) ^ 1u];
            const bool last = q + 1u == CH;
            bool ready = true;
            if (!last) {
              tc::tmem_ld32(cols + acc_slot * BN + 32u * (q + 1u), next);
            } else {
              if (kb % C::G == C::G - 1u && more) ask(kb + 1u);
              tc_fence_before();
              __syncwarp();
              if (lane == 0) arrive_relaxed_remote(tempty_lead + acc_slot * 8u);
              if (++acc_slot == NACC) {
                acc_slot = 0;
                aphase ^= 1u;
              }
              if (more) ready = look<false, false>(&sh.tfull[acc_slot], aphase);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[32u * q + i] = __fmaf_rn(now[i], s, acc[32u * q + i]);
            if (last && more) {
              if (!ready) bounded_wait(sh.abort, &sh.tfull[acc_slot], aphase, a.flags);
              __syncwarp();
              tc_fence_after();
              tc::tmem_ld32(cols + acc_slot * BN, next);
            }
#pragma unroll
            for (int i = 16; i < 32; ++i) acc[32u * q + i] = __fmaf_rn(now[i], s, acc[32u * q + i]);
            if (!last || more) tc::tmem_wait_ld(next);
          }
          if (kb % C::G == C::G - 1u) answer();
          else next_scale();
        }
      } else {
        // no tokens or no rows here: keep the accumulators' handshake
        for (uint32_t kb = st0; kb < st1; ++kb) {
          bounded_wait(sh.abort, &sh.tfull[acc_slot], aphase, a.flags);
          tc_fence_after();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_relaxed_remote(tempty_lead + acc_slot * 8u);
          if (++acc_slot == NACC) {
            acc_slot = 0;
            aphase ^= 1u;
          }
        }
      }

      if (!PAIR && !RES && splits > 1u) {
        const Exchange x(sh.ring, splits, split, 1u, 0u, min(BN, a.rows - rt * BN));
        __syncwarp();
        cluster_sync_all();  // every CTA's MMAs have read their last stage
        if (active) {
#pragma unroll
          for (uint32_t q = 0; q < CH; ++q) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = acc[32u * q + i];
            x.send32(v, col0 + 32u * q, row);
          }
        }
        const uint32_t first = x.split * x.share, mid = x.share / 2u & ~7u;
        const uint32_t in_tile = first < x.cols ? min(x.share, x.cols - first) : 0u;
        // this thread's token, columns [begin, end) of the share, eight at a time
        // (rows are a multiple of 128), their residual and bias one step ahead
        const uint32_t begin = half ? mid : 0u, end = half ? in_tile : min(mid, in_tile);
        const bool mine = tok_q + lane < a.width;
        Quads<2, false> g{tok_q + lane, rt * BN + first + begin, 0u};
        uint32_t raw[2][4];
        float4 bias[2];
        auto fetch = [&]() {
          bias[0] = bias4(a.ep, g.c);
          bias[1] = bias4(a.ep, g.c + 4u);
          if (a.ep.residual) load_quads(a.ep, g, quad_r, raw);
        };
        if (mine && begin < end) fetch();
        __syncwarp();
        cluster_sync_all();  // every CTA's sums have arrived
        bool ok = true;
        if (mine)
#pragma unroll 1
          for (uint32_t b = begin; b < end; b += 8u) {
            const Quads<2, false> now = g;
            uint32_t cur[2][4];
            float4 cur_bias[2] = {bias[0], bias[1]};
#pragma unroll
            for (int i = 0; i < 8; ++i) cur[i / 4][i % 4] = raw[i / 4][i % 4];
            g.c += 8u;
            if (b + 8u < end) fetch();
            float v[8];
            x.receive8(v, b, row);
            ok = finish_quads(a.ep, now, v, cur_bias, cur, quad_r, quad_y) && ok;
          }
        if (!ok) raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
      } else if (RES || A.tma_y) {
        // Each thread packs its token's next columns into a 64-byte row of a box (16-byte
        // chunk i at position i ^ ((token >> 1) & 3)), which leaves by TMA while the next is
        // made; the residual came into the same place by TMA while the products ran.  The
        // loop is rolled (the sums move down 32 registers per turn): unrolled, its code left
        // the instruction cache and a tile's epilogue took as long as its products.
        // lane l loads the bias of the warp's columns 4 l .. 4 l + 3
        float4 biasc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (active && 4u * lane < C::COLS) biasc = bias4(a.ep, c_base + 4u * lane);
        if (active) {
          float most = 0.0f;
          if (!RES) box = 0;  // a tile's boxes are a multiple of BOXES
          const uint32_t box_end = box + per_tile;
#pragma unroll 1
          for (uint32_t h = 0; h < C::COLS / 32u; ++h) {
            float v[32];
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) v[i] = acc[i];
            if (a.ep.bias) {
#pragma unroll
              for (uint32_t j = 0; j < 8; ++j) {
                v[4u * j] += __shfl_sync(0xffffffffu, biasc.x, h * 8u + j);
                v[4u * j + 1u] += __shfl_sync(0xffffffffu, biasc.y, h * 8u + j);
                v[4u * j + 2u] += __shfl_sync(0xffffffffu, biasc.z, h * 8u + j);
                v[4u * j + 3u] += __shfl_sync(0xffffffffu, biasc.w, h * 8u + j);
              }
            }
            activate_all(v, a.ep.act);
            // a box: 16 columns of f32 from v[16 part], else all 32
            auto put = [&](uint32_t part, bool wide) {
              const uint32_t to = box_at(box);
              if (RES) {
                // waits on its own limit: the copy lands before the CTA can exit
                if (!mbar_wait(box_bar(box), (box / C::BOXES) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
              } else if (lane == 0) {
                tma_store_wait_read<C::BOXES - 1u>();
              }
              __syncwarp();
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t at = to + lane * 64u + ((i ^ ((lane >> 1) & 3u)) << 4);
                float *x = wide ? v + 16u * part + 4u * i : v + 8u * i;
                uint4 q;
                if (RES) {
                  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                               : "r"(at));
                  if (wide)
                    x[0] += __uint_as_float(q.x), x[1] += __uint_as_float(q.y), x[2] += __uint_as_float(q.z),
                        x[3] += __uint_as_float(q.w);
                  else
                    add8(x, q, a.ep.residual_dtype);
                }
                most = max_abs(max_abs(most, x[0], x[1]), x[2], x[3]);
                if (wide) {
                  q = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                } else {
                  most = max_abs(max_abs(most, x[4], x[5]), x[6], x[7]);
                  q = pack8(x, a.ep.y_dtype);
                }
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w)
                             : "memory");
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
              if (lane == 0) {
                tma_store(&A.ymap, (int)(c_base + 32u * h + 16u * part), (int)tok_q, to);
                // the box before it has left, if only just: the residual of the one that follows there
                if (RES && box + C::BOXES - 1u < box_end && box + per_tile > box_end) {
                  tma_store_wait_read<1>();
                  fetch_box(box + C::BOXES - 1u, c_base + (box + C::BOXES - 1u + per_tile - box_end) * box_cols, tok_q);
                }
              }
              ++box;
            };
            if (a.ep.y_dtype == PW_DTYPE_F32) {
              put(0u, true);
              put(1u, true);
            } else {
              put(0u, false);
            }
#pragma unroll
            for (uint32_t i = 0; i + 32u < C::COLS; ++i) acc[i] = acc[i + 32u];
          }
          // a token past the end (its sums are of no value) is not stored
          if (tok_q + lane < a.width && __float_as_uint(most) >= overflow_bits(a.ep.y_dtype))
            raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
        }
      } else {
        // Outputs through staging rows in this tile's scale buffer, which the
        // quarter no longer needs once both of its warps are past the last block:
        // 16 columns at a time, a 64-byte row per token (16-byte chunk i at
        // position i ^ ((token >> 1) & 3), so that neither side conflicts), then
        // four columns of a few tokens per thread, coalesced.  The loop is rolled
        // (the sums move down 16 registers per turn): unrolled, its code left the
        // instruction cache and a tile's epilogue took as long as its products.
        // lane l loads the bias of the warp's columns 4 l .. 4 l + 3
        float4 biasc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (active && 4u * lane < C::COLS) biasc = bias4(a.ep, c_base + 4u * lane);
        named_bar_sync(3u + quarter, 64u);
        if (active) {
          uint8_t *stg = reinterpret_cast<uint8_t *>(xsb) + half * 2048u;
          const uint32_t c4 = lane % 4u, r0 = lane / 4u;
          bool ok = true;
#pragma unroll 1
          for (uint32_t h = 0; h < C::COLS / 16u; ++h) {
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
              *reinterpret_cast<float4 *>(stg + lane * 64u + ((i ^ ((lane >> 1) & 3u)) << 4)) =
                  make_float4(acc[4u * i], acc[4u * i + 1u], acc[4u * i + 2u], acc[4u * i + 3u]);
            __syncwarp();
            const uint32_t col = c_base + h * 16u + c4 * 4u;
            const uint32_t from = h * 4u + c4;
            const float4 bias[1] = {
                make_float4(__shfl_sync(0xffffffffu, biasc.x, from), __shfl_sync(0xffffffffu, biasc.y, from),
                            __shfl_sync(0xffffffffu, biasc.z, from), __shfl_sync(0xffffffffu, biasc.w, from))};
            // a pair's thread has registers for its four tokens at once
            constexpr uint32_t R = PAIR ? 4u : 2u;
#pragma unroll 1
            for (uint32_t r = r0; r < rows_here; r += 8u * R) {
              const Quads<R, true> g{tok_q + r, col, rows_here - r};
              uint32_t raw[R][4];
              if (a.ep.residual) load_quads(a.ep, g, quad_r, raw);
              float q[4u * R];
#pragma unroll
              for (uint32_t j = 0; j < R; ++j) {
                const uint32_t rj = r + 8u * j;
                const float4 f = *reinterpret_cast<const float4 *>(stg + rj * 64u + ((c4 ^ ((rj >> 1) & 3u)) << 4));
                q[4u * j] = f.x, q[4u * j + 1u] = f.y, q[4u * j + 2u] = f.z, q[4u * j + 3u] = f.w;
              }
              ok = finish_quads(a.ep, g, q, bias, raw, quad_r, quad_y) && ok;
            }
            __syncwarp();
#pragma unroll
            for (uint32_t i = 0; i + 16u < C::COLS; ++i) acc[i] = acc[i + 16u];
            __syncwarp();
          }
          if (!ok) raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
        }
      }
    }
  }

  // the outputs are written before the grid can be complete for the kernel behind it
  if (warp >= (uint32_t)kEpiWarp0 && lane == 0) tma_store_wait();
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

// Tiles, column blocks, and the best K split of one-CTA tiles on these sizes.
template <bool PAIR>
Splits plan(const Fp8CodesArgs &a, int num_sms, uint32_t &row_tiles, uint32_t &token_tiles, uint32_t &stages) {
  using C = Cfg<PAIR, false>;
  constexpr uint32_t kTokens = (PAIR ? 2u : 1u) * kTileRows;
  row_tiles = (a.rows + C::BN - 1u) / C::BN;
  token_tiles = (a.width + kTokens - 1u) / kTokens;
  stages = a.K / 128u;
  const uint64_t tiles = (uint64_t)row_tiles * token_tiles;
  if constexpr (PAIR) {
    const uint64_t pairs = (uint64_t)num_sms / 2u;
    return {1u, (tiles + pairs - 1u) / pairs * (stages * kPairBlock + kPairWave)};
  } else {
    return best_splits<k_fp8_gemm<false, false>>(kCostOne, tiles, stages, kMaxSplits, 1u, kThreads, C::SMEM, num_sms);
  }
}

// Raises the kernel's shared-memory limit, without which its occupancy is none.
template <bool PAIR, bool RES>
cudaError_t prepare() {
  cudaError_t e = allow_smem<k_fp8_gemm<PAIR, RES>>(Cfg<PAIR, RES>::SMEM);
  if (e != cudaSuccess) return e;
  // the register split must fit what the launch allocates, or setmaxnreg would wait for good
  static std::atomic<int> regs{0};
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes at;
    if ((e = cudaFuncGetAttributes(&at, k_fp8_gemm<PAIR, RES>)) != cudaSuccess) return e;
    regs.store(at.numRegs, std::memory_order_relaxed);
  }
  return regs.load(std::memory_order_relaxed) < kRegsLaunch ? cudaErrorInvalidConfiguration : cudaSuccess;
}

template <bool PAIR, bool RES>
cudaError_t launch_as(const Args &A, uint32_t clusters, cudaStream_t stream) {
  constexpr uint32_t CTAS = PAIR ? 2u : 1u;
  cudaError_t e = prepare<PAIR, RES>();
  if (e != cudaSuccess) return e;
  Launch l(CTAS * clusters, kThreads, CTAS * A.splits, Cfg<PAIR, RES>::SMEM, stream);
  e = cudaLaunchKernelEx(&l.cfg, k_fp8_gemm<PAIR, RES>, A);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <bool PAIR>
cudaError_t launch_one(const Fp8CodesArgs &a, int num_sms, cudaStream_t stream) {
  constexpr uint32_t CTAS = PAIR ? 2u : 1u;
  Args A{};
  A.a = a;
  A.splits = plan<PAIR>(a, num_sms, A.row_tiles, A.token_tiles, A.stages).n;
  const bool qkv = a.layout != PW_LAYOUT_PLAIN;
  // up to 128 tokens a stage loads whole 32-token chunks of them
  A.box_tokens = a.width > 96u ? 128u : (a.width + 31u) / 32u * 32u;
  if (!encode_weight_map(&A.wmap, a.w, a.rows, a.K, qkv ? 64u : 128u, 1u) ||
      !encode_weight_map(&A.xmap, a.codes, a.width, a.K, A.box_tokens, 1u))
    return cudaErrorInvalidValue;
  const uint64_t tiles = (uint64_t)A.row_tiles * A.token_tiles, at_once = (uint64_t)num_sms / CTAS;
  if (tiles > 0x7fffffffull / kMaxSplits) return cudaErrorInvalidValue;
  const uint32_t clusters = (uint32_t)(A.splits > 1u ? tiles * A.splits : tiles < at_once ? tiles : at_once);
  bool res = false;
  if (A.splits == 1u) {
    const auto fits = [&](CUtensorMap *map, const void *at, uint64_t stride, uint32_t dtype) {
      return reinterpret_cast<uintptr_t>(at) % 16u == 0u && encode_out_map(map, at, a.width, a.rows, stride, dtype, 32u);
    };
    const bool y = fits(&A.ymap, a.ep.y, a.ep.y_stride, a.ep.y_dtype);
    // the sums join the residual in its place: elements of one size
    res = y && a.ep.residual && (a.ep.residual_dtype == PW_DTYPE_F32) == (a.ep.y_dtype == PW_DTYPE_F32) &&
          fits(&A.rmap, a.ep.residual, a.ep.residual_stride, a.ep.residual_dtype);
    A.tma_y = y && (res || !a.ep.residual);
  }
  return res ? launch_as<PAIR, true>(A, clusters, stream) : launch_as<PAIR, false>(A, clusters, stream);
}

}  // namespace fp8g

cudaError_t launch_fp8_gemm(const Fp8CodesArgs &a, int num_sms, cudaStream_t stream) {
  using namespace fp8g;
  // a warp of the pair's epilogue takes 128 output columns whole
  if (a.width == 0 || a.rows == 0 || a.rows % 128u || a.K == 0 || a.K % 128u || a.K > 128u * kMaxBlocks)
    return cudaErrorInvalidValue;
  const cudaError_t e = prepare<false, false>();
  if (e != cudaSuccess) return e;
  uint32_t r, t, s;
  if (a.width <= 128u || plan<false>(a, num_sms, r, t, s).cost <= plan<true>(a, num_sms, r, t, s).cost)
    return launch_one<false>(a, num_sms, stream);
  return launch_one<true>(a, num_sms, stream);
}

}  // namespace pw
