// pw_cluster.cuh -- what the clustered tensor kernels share: CTA pairs (the
// cta_group::2 forms of loads and commits), distributed shared memory, bounded
// waits that sleep, the exchange that joins K splits, and cluster launches.
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "pw_device.cuh"
#include "pw_internal.h"

namespace pw {
namespace clu {

constexpr uint32_t kMaxSplits = 8;   // CTAs of a portable cluster
constexpr uint32_t kTileRows = 128;  // rows of a CTA's tile: TMEM lanes

// Arrives on the barrier at this offset in both CTAs once the MMAs so far are complete.
__device__ __forceinline__ void mma_commit_pair_elect(uint64_t *bar, uint32_t pair_mask) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)pair_mask)
      : "memory");
}
// The same for a kernel whose MMAs one thread issues; without PAIR on this CTA's barrier.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint64_t *bar, uint32_t pair_mask) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)pair_mask)
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}
// A tile load into this CTA's shared memory that completes on the pair's
// leading CTA's barrier (a shared::cluster address).
__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
      "%4}], [%5];" ::"r"(smem_addr(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of this CTA's shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Arrivals that hand a TMEM accumulator back to the MMA: what they order is the
// tcgen05.ld before them (tcgen05.wait::ld and the before_thread_sync fence), no
// memory, so they are relaxed.  (As releases they waited for the warp's stores
// and copies each time.)
__device__ __forceinline__ void arrive_relaxed_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_relaxed(uint64_t *bar) {
  asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void store_remote4(uint32_t addr, float x, float y, float z, float w) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                   dst),
               "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
               : "memory");
}
// A box from shared memory to global memory, and the end of its reading for all but
// the last N boxes that this thread sent.
__device__ __forceinline__ void tma_store(const CUtensorMap *map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
               "r"(src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// The end of their writing.
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// One look at a barrier's phase; SLEEP: waits in hardware for up to 100 us, woken
// by the phase's completion.  PAIR: the pair's other CTA arrives on the barrier too.
template <bool PAIR, bool SLEEP>
__device__ __forceinline__ bool look(uint64_t *bar, uint32_t parity) {
  constexpr uint32_t kSleepNs = 100000;
  uint32_t done;
  if (SLEEP && PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity), "r"(kSleepNs)
        : "memory");
  else if (SLEEP)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity), "r"(kSleepNs)
        : "memory");
  else if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
  return done != 0u;
}

// Bounded wait (1 s) that sleeps between looks: ten warps polling in a loop took a
// fifth of the ALU's issue slots.  The first look does not sleep (FP8 pairs at 2048 x
// 16384 x 4096: 221 us, 224 when it did).  `abort` (shared memory) makes a CTA's other
// waits give up once one has.
template <bool PAIR = false>
__device__ __forceinline__ bool bounded_wait(volatile int *abort, uint64_t *bar, uint32_t parity, uint32_t *flags) {
  if (look<PAIR, false>(bar, parity)) return true;
  const uint64_t start = global_timer_ns();
  do {
    if (*abort) return false;
    if (look<PAIR, true>(bar, parity)) return true;
  } while (global_timer_ns() - start <= kWaitLimitNs);
  *abort = 1;
  raise_flag(flags, PW_FLAG_WAIT_TIMEOUT);
  return false;
}

// Joining K splits of a tile of 128 rows (TMEM lanes) x `cols` accumulator
// columns.  Split k finishes columns [k share, (k + 1) share); share is a multiple
// of 8, so that a quad of columns has one owner and each half of the epilogue warps
// whole quads.  The sums travel as [source split][quad of the share][128 rows][4
// columns] f32 into the owners' rings, (cols + 8 splits) * 512 bytes at most.
struct Exchange {
  uint32_t ring;    // this CTA's ring
  uint32_t splits, split, step, base;  // split k is the cluster's CTA base + step k
  uint32_t cols, share;
  __device__ __forceinline__ Exchange(uint8_t *r, uint32_t n_splits, uint32_t k, uint32_t cta_step, uint32_t cta_base,
                                      uint32_t n_cols)
      : ring(smem_addr(r)), splits(n_splits), split(k), step(cta_step), base(cta_base), cols(n_cols) {
    share = ((n_cols + n_splits - 1u) / n_splits + 7u) & ~7u;
  }
  __device__ __forceinline__ uint32_t slot(uint32_t from, uint32_t col_of_share, uint32_t row) const {
    return ((from * (share / 4u) + col_of_share / 4u) * kTileRows + row) * 16u;
  }
  // this row's sums of columns c0 .. c0 + 31 (c0 % 32 == 0) to their owners
  __device__ __forceinline__ void send32(const float (&v)[32], uint32_t c0, uint32_t row) const {
    uint32_t to = c0 / share, at = c0 % share;
    uint32_t dst = to < splits ? map_rank(ring + slot(split, 0u, row), base + step * to) : 0u;
#pragma unroll
    for (uint32_t q = 0; q < 8; ++q) {
      if (c0 + 4u * q < cols) store_remote4(dst + slot(0u, at, 0u), v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      at += 4u;
      if (at == share && to + 1u < splits) {
        at = 0u;
        ++to;
        dst = map_rank(ring + slot(split, 0u, row), base + step * to);
      }
    }
  }
  // this row's joined sums of columns b .. b + 7 of this CTA's share
  __device__ __forceinline__ void receive8(float (&v)[8], uint32_t b, uint32_t row) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    for (uint32_t s = 0; s < splits; ++s)
#pragma unroll
      for (uint32_t q = 0; q < 2; ++q) {
        float x, y, z, w;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(x), "=f"(y), "=f"(z), "=f"(w)
                     : "r"(ring + slot(s, b + 4u * q, row)));
        v[4 * q] += x;
        v[4 * q + 1] += y;
        v[4 * q + 2] += z;
        v[4 * q + 3] += w;
      }
  }
};

// A launch of `cluster` CTAs per cluster (1: none).
struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  Launch(uint32_t grid, uint32_t threads, uint32_t cluster, uint32_t smem, cudaStream_t stream) {
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1u ? 2 : 1;
  }
};

// Clusters of each size that run at once.  An SM holds one CTA, and a cluster
// stays within a GPC, so sizes that do not divide the GPCs leave SMs idle (of a
// B200's 148: 132 CTAs in clusters of 4 or 6, 120 in clusters of 8).
template <auto Kernel>
uint32_t clusters_at_once(uint32_t cluster, uint32_t threads, uint32_t smem, int num_sms) {
  static std::atomic<int> known[kMaxSplits + 1];
  if (cluster == 1u) return (uint32_t)num_sms;
  int n = known[cluster].load(std::memory_order_relaxed);
  if (n == 0) {
    Launch l(cluster, threads, cluster, smem, nullptr);
    if (cudaOccupancyMaxActiveClusters(&n, Kernel, &l.cfg) != cudaSuccess || n < 1) n = num_sms / (int)kMaxSplits;
    known[cluster].store(n, std::memory_order_relaxed);
  }
  return (uint32_t)n;
}

// A tile kernel's time in cycles: per column block, and per wave of tiles
// without and with the exchange of K splits.
struct TileCost {
  uint32_t block, wave, wave_split;
};
struct Splits {
  uint32_t n;
  uint64_t cost;
};

// K splits of `tiles` tiles: the count with the least time over the waves of
// clusters.  Every split keeps four column blocks.
template <auto Kernel>
Splits best_splits(const TileCost &t, uint64_t tiles, uint32_t k_blocks, uint32_t most, uint32_t cta_per_split,
                   uint32_t threads, uint32_t smem, int num_sms) {
  Splits best{1u, ~(uint64_t)0};
  for (uint32_t s = 1u; s <= most && (s == 1u || s * 4u <= k_blocks); ++s) {
    const uint64_t n = clusters_at_once<Kernel>(s * cta_per_split, threads, smem, num_sms);
    const uint64_t cost = (tiles + n - 1u) / n * ((uint64_t)k_blocks * t.block / s + (s > 1u ? t.wave_split : t.wave));
    if (cost < best.cost) best = {s, cost};
  }
  return best;
}

}  // namespace clu
}  // namespace pw
