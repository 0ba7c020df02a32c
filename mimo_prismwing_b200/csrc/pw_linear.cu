// pw_linear.cu -- linear layer over a 16-bit weight on tcgen05 / TMEM:
//   y[t, r] = round(act(sum_c x[t, c] W[r, c] + bias[r]) + residual[t, r]).
//
// A tile is 128 weight rows (TMEM lanes) x BN tokens (TMEM columns): A = W,
// B = x, both K-major in shared memory (128B swizzle, written by TMA, zero
// past the matrices' ends, so no size is special).  With weight rows on the
// lanes a warp's store covers 32 consecutive outputs of one token, whatever
// the output's stride or alignment, and the bias is one value per thread.
// Persistent CTAs, one per SM: a producer warp fills the TMA ring, an MMA warp
// issues tcgen05.mma.kind::f16 into one of two TMEM accumulators, eight
// epilogue warps empty the other.  Sums are f32 over the whole K.
#include <cstdint>
#include <cstdlib>
#include <cuda.h>
#include <cuda_runtime.h>

#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"
#include "pw_tc.cuh"

namespace pw {
namespace lin {

using tc::elect_one;
using tc::smem_desc_sw128;
using tc::tc_fence_after;
using tc::tc_fence_before;

constexpr int kProducerWarp = 0;
constexpr int kMmaWarp = 1;
constexpr int kEpiWarp0 = 2;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr uint32_t kTileRows = 128;
constexpr uint32_t kBlockK = 64;        // columns of a k-block: one 128-byte line
constexpr uint32_t kSmemLimit = 227u * 1024u;
constexpr uint32_t kTokenGroup = 8;     // token tiles that neighbouring CTAs share weights over

template <int BN>
struct Cfg {
  static constexpr uint32_t KBS = BN == 256 ? 1u : 2u;  // k-blocks per stage
  static constexpr uint32_t A_BYTES = KBS * kTileRows * 128u;
  static constexpr uint32_t B_BYTES = KBS * (uint32_t)BN * 128u;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr uint32_t NST = (kSmemLimit - 2048u) / STAGE < 6u ? (kSmemLimit - 2048u) / STAGE : 6u;
  static constexpr uint32_t BARS = NST * STAGE;
  static constexpr uint32_t MISC = BARS + (2u * NST + 4u) * 8u;
  static constexpr uint32_t SMEM = MISC + 16u + 1024u;  // + alignment slack
  static constexpr uint32_t TMEM_COLS = 2u * (uint32_t)BN;
  static_assert(SMEM <= kSmemLimit, "shared memory");
};

struct Args {
  LinearArgs a;
  CUtensorMap wmap, xmap;
  uint32_t w3d, x3d;  // the maps have a k-block dimension (encode_rows16_map)
  uint32_t row_tiles, token_tiles, stages;
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

struct Shared {
  uint8_t *ring;
  uint64_t *full, *empty, *tfull, *tempty;
  uint32_t *tmem_base;
  volatile int *abort;
};

__device__ __forceinline__ bool lwait(const Shared &sh, uint64_t *bar, uint32_t parity, uint32_t *flags) {
  if (*sh.abort) return false;
  if (mbar_wait(bar, parity)) return true;
  *sh.abort = 1;
  raise_flag(flags, PW_FLAG_WAIT_TIMEOUT);
  return false;
}

// Tile u: neighbouring tiles share their token tiles within a group of
// kTokenGroup, so that the tiles in flight reuse both operands in L2.
__device__ __forceinline__ void tile_of(const Args &A, uint32_t u, uint32_t &row_tile, uint32_t &token_tile) {
  const uint32_t per = kTokenGroup * A.row_tiles, g = u / per, in = u % per;
  const uint32_t width = min(kTokenGroup, A.token_tiles - g * kTokenGroup);
  row_tile = in / width;
  token_tile = g * kTokenGroup + in % width;
}

template <typename T>
__device__ __forceinline__ void add_rows(float (&v)[32], const T *p, uint64_t stride, uint32_t n) {
  float r[32];
#pragma unroll
  for (uint32_t j = 0; j < 32; ++j) r[j] = j < n ? to_f32(p[j * stride]) : 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < 32; ++j) v[j] += r[j];
}

template <typename T>
__device__ __forceinline__ void store_rows(const float (&v)[32], T *p, uint64_t stride, uint32_t n) {
#pragma unroll
  for (uint32_t j = 0; j < 32; ++j)
    if (j < n) p[j * stride] = from_f32<T>(v[j]);
}

// The epilogue of one thread: output column c of tokens t0 .. t0 + n - 1.
__device__ __forceinline__ void finish32(const EpilogueArgs &e, float (&v)[32], float bias, uint64_t t0, uint32_t c,
                                         uint32_t n, uint32_t *flags) {
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] += bias;
  activate_all(v, e.act);
  if (e.residual) {
    const uint64_t at = t0 * e.residual_stride + c;
    if (e.residual_dtype == PW_DTYPE_F32) add_rows(v, static_cast<const float *>(e.residual) + at, e.residual_stride, n);
    else if (e.residual_dtype == PW_DTYPE_BF16)
      add_rows(v, static_cast<const __nv_bfloat16 *>(e.residual) + at, e.residual_stride, n);
    else add_rows(v, static_cast<const __half *>(e.residual) + at, e.residual_stride, n);
  }
  uint32_t top = 0u;
#pragma unroll
  for (uint32_t j = 0; j < 32; ++j)
    if (j < n) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  if (top >= overflow_bits(e.y_dtype)) raise_flag(flags, PW_FLAG_NONFINITE_ROUND);
  const uint64_t at = t0 * e.y_stride + c;
  if (e.y_dtype == PW_DTYPE_F32) store_rows(v, static_cast<float *>(e.y) + at, e.y_stride, n);
  else if (e.y_dtype == PW_DTYPE_BF16) store_rows(v, static_cast<__nv_bfloat16 *>(e.y) + at, e.y_stride, n);
  else store_rows(v, static_cast<__half *>(e.y) + at, e.y_stride, n);
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) k_linear_tc(const __grid_constant__ Args A) {
  using C = Cfg<BN>;
  constexpr uint32_t NST = C::NST;
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
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < NST; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);  // tcgen05.commit after the stage's MMAs
    }
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(&sh.tfull[i], 1);           // tcgen05.commit after the tile's MMAs
      mbar_init(&sh.tempty[i], kEpiWarps);  // one arrive per epilogue warp
    }
    *sh.abort = 0;
    mbar_fence_init();
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
  const uint32_t total = A.row_tiles * A.token_tiles;

  if (warp == (uint32_t)kProducerWarp) {
    uint32_t slot = 0, phase = 0, issued = 0, parity = 0;
    for (uint32_t u = blockIdx.x; u < total; u += gridDim.x) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const int row0 = (int)(rt * kTileRows), tok0 = (int)(tt * BN);
      for (uint32_t st = 0; st < A.stages; ++st) {
        if (lwait(sh, &sh.empty[slot], phase ^ 1u, a.flags)) {
          uint8_t *dst = sh.ring + slot * C::STAGE;
          const int kb = (int)(st * C::KBS);
          if (elect_one()) {
            mbar_arrive_expect_tx(&sh.full[slot], C::STAGE);
            if (A.w3d) {
              tc::tma_load_3d(dst, &A.wmap, 0, row0, kb, &sh.full[slot]);
            } else {
#pragma unroll
              for (int j = 0; j < (int)C::KBS; ++j)
                tc::tma_load_3d(dst + j * (kTileRows * 128u), &A.wmap, (kb + j) * (int)kBlockK, row0, 0, &sh.full[slot]);
            }
            if (A.x3d) {
              tc::tma_load_3d(dst + C::A_BYTES, &A.xmap, 0, tok0, kb, &sh.full[slot]);
            } else {
#pragma unroll
              for (int j = 0; j < (int)C::KBS; ++j)
                tc::tma_load_3d(dst + C::A_BYTES + j * (BN * 128u), &A.xmap, (kb + j) * (int)kBlockK, tok0, 0,
                                &sh.full[slot]);
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
    for (uint32_t u = blockIdx.x; u < total; u += gridDim.x) {
      const bool ok_acc = lwait(sh, &sh.tempty[acc], aphase ^ 1u, a.flags);
      tc_fence_after();
      const uint32_t d = tmem + acc * (uint32_t)BN;
      for (uint32_t st = 0; st < A.stages; ++st) {
        const bool ok = lwait(sh, &sh.full[slot], phase, a.flags) && ok_acc;
        tc_fence_after();
        if (ok) {
          const uint64_t ad = ring_desc + ((slot * C::STAGE) >> 4);
          const uint64_t bd = ad + (C::A_BYTES >> 4);
#pragma unroll
          for (uint32_t j = 0; j < C::KBS; ++j)
#pragma unroll
            for (uint32_t s = 0; s < 4; ++s)
              mma_f16_elect(d, ad + ((j * kTileRows * 128u) >> 4) + 2u * s, bd + ((j * BN * 128u) >> 4) + 2u * s, idesc,
                            (st | j | s) ? 1u : 0u);
        }
        tc::mma_commit_elect(&sh.empty[slot]);
        if (++slot == NST) {
          slot = 0;
          phase ^= 1u;
        }
      }
      tc::mma_commit_elect(&sh.tfull[acc]);
      pending |= 1u << acc;
      pend_parity = (pend_parity & ~(1u << acc)) | (aphase << acc);
      if (++acc == 2u) {
        acc = 0;
        aphase ^= 1u;
      }
    }
    // every MMA is complete before the columns are freed
    for (uint32_t i = 0; i < 2; ++i)
      if (pending & (1u << i))
        if (!mbar_wait(&sh.tfull[i], (pend_parity >> i) & 1u)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
  } else {
    // two warps per TMEM lane quarter, each half of the token columns (all of
    // them for the first when there are only 32)
    const uint32_t quarter = warp % 4u, half = (warp - kEpiWarp0) / 4u;
    constexpr uint32_t COLS = BN >= 64 ? BN / 2 : 32;
    const uint32_t col0 = half * COLS;
    uint32_t acc = 0, aphase = 0;
    for (uint32_t u = blockIdx.x; u < total; u += gridDim.x) {
      uint32_t rt, tt;
      tile_of(A, u, rt, tt);
      const uint32_t c = rt * kTileRows + quarter * 32u + lane;
      const bool mine = c < a.rows;
      const float bias = mine && a.ep.bias ? load_elem(a.ep.bias, c, a.ep.bias_dtype) : 0.0f;
      const bool ok = lwait(sh, &sh.tfull[acc], aphase, a.flags);
      tc_fence_after();
      const uint32_t src = tmem + ((quarter * 32u) << 16) + acc * (uint32_t)BN + col0;
      if (ok && col0 < (uint32_t)BN) {
        for (uint32_t q = 0; q < COLS; q += 32u) {
          float v[32];
          tc::tmem_ld32(src + q, v);
          tc::tmem_wait_ld(v);
          const uint32_t t0 = tt * BN + col0 + q;
          if (mine && t0 < a.width) finish32(a.ep, v, bias, t0, c, min(32u, a.width - t0), a.flags);
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.tempty[acc]);
      if (++acc == 2u) {
        acc = 0;
        aphase ^= 1u;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == (uint32_t)kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
}

template <int BN>
cudaError_t launch_tc(const LinearArgs &a, int num_sms, cudaStream_t stream) {
  using C = Cfg<BN>;
  Args A{};
  A.a = a;
  A.w3d = a.cols % kBlockK == 0u;
  A.x3d = A.w3d;
  const uint32_t kb = A.w3d ? C::KBS : 0u;
  if (!encode_rows16_map(&A.wmap, a.w, a.rows, a.cols, a.w_stride, a.dtype, kTileRows, kb) ||
      !encode_rows16_map(&A.xmap, a.x, a.width, a.cols, a.x_stride, a.dtype, BN, kb))
    return cudaErrorInvalidValue;
  A.row_tiles = (a.rows + kTileRows - 1u) / kTileRows;
  A.token_tiles = (a.width + (uint32_t)BN - 1u) / (uint32_t)BN;
  A.stages = (a.cols + C::KBS * kBlockK - 1u) / (C::KBS * kBlockK);
  cudaError_t e = allow_smem<k_linear_tc<BN>>(C::SMEM);
  if (e != cudaSuccess) return e;
  const uint64_t tiles = (uint64_t)A.row_tiles * A.token_tiles;
  if (tiles > 0x7fffffffull) return cudaErrorInvalidValue;
  const uint32_t grid = tiles < (uint64_t)num_sms ? (uint32_t)tiles : (uint32_t)num_sms;
  return launch_kernel(k_linear_tc<BN>, dim3(grid), dim3(kThreads), C::SMEM, stream, A);
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
  if (a.width <= 16u && !getenv("PW_NONARROW")) return launch_linear_narrow(a, num_sms, stream);
  if (a.width <= 32u) return lin::launch_tc<32>(a, num_sms, stream);
  if (a.width <= 64u) return lin::launch_tc<64>(a, num_sms, stream);
  if (a.width <= 128u) return lin::launch_tc<128>(a, num_sms, stream);
  return lin::launch_tc<256>(a, num_sms, stream);
}

}  // namespace pw
