// pw_linear_narrow.cu -- the linear layer for a few tokens (pw_linear.cu has the
// equation): every weight byte is used at most 16 times, so the kernel is a
// weight stream and HBM bounds it.
//
// What it takes is enough loads in flight on every SM from the first
// microsecond, for weights of any shape.  A warp owns 16 weight rows and a
// share of K and loads its weights straight into registers, 16 bytes per lane
// and sixteen loads deep (eight with two token tiles); no shared memory, no
// barrier in the loop.  The lanes' 8 consecutive columns are fed to mma.m16n8k16 in place: the MMA sums over k in
// any order as long as both operands agree, so lane t of a quad supplies its
// columns 0..3 and 4..7 as the k positions that the fragment layout gives it,
// and x, loaded the same way, does too.  (Warp MMAs are far from the tensor
// roof, and 16 tokens are far below it.)  K is split over the eight warps of a
// CTA and, for weights of few rows, over the CTAs of a cluster; the sums join in
// a fixed order through (distributed) shared memory, without atomics or a
// workspace.
//
// Measured, us of one token x [rows, cols] bf16 (a tensor-core tile kernel with a
// TMA ring, one 128-row tile per CTA, took 21.6, 12.6, 20.6, 38.5 for the first
// four and 186.7 for the last, at eight tokens):
//                            4096x8192 4096x4096 1024x8192 256x16384 152576x4096
//   8 loads deep,  8 warps      15.3      8.8       9.2      12.5      203.6
//   8 loads deep, 16 warps      13.7      7.3       6.4       8.6      190.7
//   16 loads deep, 8 warps      13.2      7.0       6.9       9.2      183.2
//   8 deep, 8 warps x 4 CTAs    15.9     10.2       5.3       5.8      307.0
#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_runtime.h>

#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"

namespace pw {
namespace narrow {

constexpr uint32_t kMaxWarps = 8;
constexpr uint32_t kRows = 16;   // weight rows of a CTA
constexpr uint32_t kChunk = 32;  // columns of a load: 4 lanes x 8
template <int NT>
struct Depth {
  // chunks in flight, two weight loads per lane each: two token tiles need the registers
  static constexpr uint32_t value = NT == 1 ? 8u : 4u;
};

__device__ __forceinline__ uint4 ldg_stream(const void *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// x is the previous kernel's output, which it may still write while this kernel is
// resident: an ordinary load, not one of read-only data.
__device__ __forceinline__ uint4 load_x(const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); }

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <bool BF16>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 columns from `c` of a 16-bit row that has `cols`, zero past its end.
__device__ __forceinline__ uint4 load_tail(const uint16_t *row, uint32_t c, uint32_t cols) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i)
    if (c + i < cols) w[i / 2u] |= (uint32_t)row[c + i] << (16u * (i % 2u));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// NT: token tiles of 8.  The cluster's CTAs share 16 weight rows.
template <bool BF16, int NT>
__global__ void __launch_bounds__(kMaxWarps * 32, 2)
    k_linear_narrow(const LinearArgs a, const uint32_t splits, const uint32_t ahead) {
  namespace cg = cooperative_groups;
  constexpr uint32_t kDeep = Depth<NT>::value;
  __shared__ float part[kMaxWarps][8 * NT][kRows + 1];
  __shared__ float total[8 * NT][kRows];
  const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, g = lane / 4u, t = lane % 4u;
  const uint32_t warps = blockDim.x / 32u;
  const uint32_t split = blockIdx.x % splits, row0 = blockIdx.x / splits * kRows;

  const uint16_t *w = static_cast<const uint16_t *>(a.w), *x = static_cast<const uint16_t *>(a.x);
  // rows past the end read the last one; their sums are not stored
  const uint16_t *w0 = w + (uint64_t)min(row0 + g, a.rows - 1u) * a.w_stride;
  const uint16_t *w1 = w + (uint64_t)min(row0 + g + 8u, a.rows - 1u) * a.w_stride;
  const uint16_t *xr[NT];
  bool token[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    token[n] = g + 8u * n < a.width;
    xr[n] = x + (uint64_t)(token[n] ? g + 8u * n : 0u) * a.x_stride;
  }
  // Under programmatic dependent launch the CTAs that run first start while the
  // previous kernel drains: they ask L2 for their first weights, which needs no
  // order with what that kernel writes (a prefetch moves a line to where every
  // write goes).
  if (blockIdx.x < ahead) {
    const uint32_t q = split * warps + warp;
    if ((q + 1u) * kChunk * kDeep <= a.cols && t % 2u == 0u) {
#pragma unroll
      for (uint32_t j = 0; j < kDeep; ++j) {
        prefetch_l2(w0 + q * kChunk * kDeep + t * 8u + j * kChunk);
        prefetch_l2(w1 + q * kChunk * kDeep + t * 8u + j * kChunk);
      }
    }
  }
  pdl_wait();
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;

  // this warp's chunks: every (splits * warps)-th group of kDeep
  const uint32_t whole = a.cols / 8u;  // columns in whole vectors
  const uint32_t groups = (a.cols + kChunk * kDeep - 1u) / (kChunk * kDeep);
  for (uint32_t q = split * warps + warp; q < groups; q += splits * warps) {
    const uint32_t c0 = q * kChunk * kDeep + t * 8u;
    uint4 wa[kDeep], wb[kDeep], xv[kDeep][NT];
    if ((q + 1u) * kChunk * kDeep <= a.cols) {
#pragma unroll
      for (uint32_t j = 0; j < kDeep; ++j) {
        wa[j] = ldg_stream(w0 + c0 + j * kChunk);
        wb[j] = ldg_stream(w1 + c0 + j * kChunk);
      }
#pragma unroll
      for (uint32_t j = 0; j < kDeep; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          xv[j][n] = token[n] ? load_x(xr[n] + c0 + j * kChunk) : make_uint4(0u, 0u, 0u, 0u);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < kDeep; ++j) {
        const uint32_t c = c0 + j * kChunk;
        const bool in = c / 8u < whole;
        wa[j] = in ? ldg_stream(w0 + c) : load_tail(w0, c, a.cols);
        wb[j] = in ? ldg_stream(w1 + c) : load_tail(w1, c, a.cols);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          xv[j][n] = !token[n] ? make_uint4(0u, 0u, 0u, 0u)
                     : in      ? load_x(xr[n] + c)
                               : load_tail(xr[n], c, a.cols);
      }
    }
    // Each group's products get accumulators of their own, added in f32: the MMA truncates
    // when it adds to one (2400 rows x 65536 columns of one sign: 3.1e-5 off in one per
    // warp).
    float d[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[n][i] = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < kDeep; ++j)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma16<BF16>(d[n], wa[j].x, wb[j].x, wa[j].y, wb[j].y, xv[j][n].x, xv[j][n].y);
        mma16<BF16>(d[n], wa[j].z, wb[j].z, wa[j].w, wb[j].w, xv[j][n].z, xv[j][n].w);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] += d[n][i];
  }
  pdl_launch_dependents();

  // lane holds rows g, g + 8 x tokens 2 t, 2 t + 1 of each tile
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][8 * n + 2 * t + (i & 1)][g + (i >= 2 ? 8u : 0u)] = acc[n][i];
  __syncthreads();
  constexpr uint32_t kOut = 8u * NT * kRows;  // 128 or 256 outputs
  for (uint32_t i = threadIdx.x; i < kOut; i += blockDim.x) {
    const uint32_t n = i / kRows, r = i % kRows;
    float sum = part[0][n][r];
    for (uint32_t k = 1; k < warps; ++k) sum += part[k][n][r];
    total[n][r] = sum;
  }
  if (splits > 1u) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (split == 0u)
      for (uint32_t i = threadIdx.x; i < kOut; i += blockDim.x) {
        float sum = (&total[0][0])[i];
        for (uint32_t s = 1; s < splits; ++s) sum += cluster.map_shared_rank(&total[0][0], s)[i];
        (&total[0][0])[i] = sum;  // read back by this thread only
      }
    cluster.sync();  // the other CTAs' sums stay until they are read
    if (split != 0u) return;
  }
  for (uint32_t i = threadIdx.x; i < kOut; i += blockDim.x) {
    const uint32_t n = i / kRows, c = row0 + i % kRows;
    if (n < a.width && c < a.rows &&
        !store_elem(a.ep.y, (uint64_t)n * a.ep.y_stride + c, a.ep.y_dtype,
                    epilogue_value(a.ep, (&total[0][0])[i], n, c)))
      raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
  }
}

template <bool BF16, int NT>
cudaError_t launch_one(const LinearArgs &a, int num_sms, cudaStream_t stream) {
  // A warp per group of loads, up to eight; then 2 to 8 CTAs of a cluster while
  // two CTAs per SM still hold them all and every warp keeps a group.
  constexpr uint32_t kGroup = kChunk * Depth<NT>::value;
  const uint32_t units = (a.rows + kRows - 1u) / kRows, groups = (a.cols + kGroup - 1u) / kGroup;
  const uint32_t warps = groups < kMaxWarps ? groups : kMaxWarps;
  uint32_t splits = 1u;
  while (splits < 8u && units * splits <= (uint32_t)num_sms && splits * 2u * warps <= groups) splits *= 2u;
  const uint64_t grid = (uint64_t)units * splits;
  if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(warps * 32u);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1u ? 2 : 1;
  // The first wave, in whole-K launches of one token tile (one token of 8192 x 4096
  // in a row of calls: 13.1 us without, 11.0 us with; with two tiles or splits, and
  // in later waves, it gains nothing).
  const uint32_t ahead = pdl_enabled() && NT == 1 && splits == 1u ? 2u * (uint32_t)num_sms : 0u;
  cudaError_t e = cudaLaunchKernelEx(&cfg, k_linear_narrow<BF16, NT>, a, splits, ahead);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace narrow

cudaError_t launch_linear_narrow(const LinearArgs &a, int num_sms, cudaStream_t stream) {
  using namespace narrow;
  if (a.width == 0 || a.width > 16u) return cudaErrorInvalidValue;
  const bool bf16 = a.dtype == PW_DTYPE_BF16;
  if (a.width <= 8u) return bf16 ? launch_one<true, 1>(a, num_sms, stream) : launch_one<false, 1>(a, num_sms, stream);
  return bf16 ? launch_one<true, 2>(a, num_sms, stream) : launch_one<false, 2>(a, num_sms, stream);
}

}  // namespace pw
