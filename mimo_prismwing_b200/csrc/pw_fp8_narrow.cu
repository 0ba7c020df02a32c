// pw_fp8_narrow.cu -- block-scaled FP8 linear layer on codes, for a few tokens:
//   y[t, r] = round(act(sum_kb dot_kb S[r / 128, kb] xs[t, kb] + bias[r]) + residual[t, r]),
//   dot_kb = sum over the 128 columns of block kb of dec(W[r, c]) dec(code[t, c]).
//
// A weight stream, bound by HBM, built like pw_linear_narrow.cu: a warp owns 16
// (or 32) weight rows and a share of the column blocks and loads its e4m3 bytes straight
// into registers, 16 per lane and load, all of its first blocks in flight at
// once; a quad's lanes feed their 16 consecutive columns to two mma.m16n8k32 in
// place (the sum over k does not care which column sits at which k position as
// long as weights and codes agree).  A block's MMAs start from zero and
// their sum is promoted by its two scales with one FMA, as the checkpoint's f32
// block scales require.  The CTA's eight warps join in a fixed tree.
//
// Measured at 8 tokens, us, for [13568, 4096] / [16384, 4096] / [4096, 2048] (the
// ring kernels of pw_fp8_linear, one CTA per SM: 19.1 for the first):
//   2 blocks in flight, 8 warps, 3 CTAs per SM   11.4 / 14.7 / 3.3
//   2 blocks,           8 warps, 2 CTAs          12.8 / 15.8 / 3.4
//   4 blocks,           8 warps, 2 CTAs          13.4 / 16.8 / 3.4
//   2 blocks,           4 warps, 6 CTAs          11.1 / 18.2 / 4.0
//   4 blocks,           2 warps, 8 CTAs          12.9 / 15.6 / 5.6
// From 9 tokens on a CTA with weights of many rows takes 32 of them, so that the codes,
// twice as many, are read half as often (16 tokens, 16 / 32 rows per CTA: [8192, 4096]
// 11.2 / 9.4, [4096, 4096] 5.3 / 6.8, where too few CTAs are left).
#include <cstdint>
#include <cuda_runtime.h>

#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"

namespace pw {
namespace fp8n {

constexpr uint32_t kWarps = 8;

__device__ __forceinline__ uint4 ldg_stream(const void *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: token tiles of 8.  RT: row tiles of 16 of a CTA.  4 KB of weights per warp are in
// flight: two column blocks of 16 rows or one of 32.
template <int NT, int RT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) k_fp8_narrow(const Fp8CodesArgs a) {
  constexpr uint32_t kRows = 16u * RT, DEEP = 2u / RT;
  __shared__ float part[kWarps][8 * NT][kRows + 1];
  const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, g = lane / 4u, t = lane % 4u;
  const uint32_t row0 = blockIdx.x * kRows, kblocks = a.K / 128u, warps = blockDim.x / 32u;
  // 64 rows of a layout are consecutive checkpoint rows with one scale row
  uint32_t src, srow;
  map_row(a.layout, row0, src, srow);
  const uint8_t *w0 = a.w + (uint64_t)(src + g) * a.K + t * 16u;
  const float *ws_row = a.ws + (uint64_t)srow * kblocks;
  pdl_wait();
  float acc[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;

  for (uint32_t k0 = warp * DEEP; k0 < kblocks; k0 += warps * DEEP) {
    uint4 wv[DEEP][RT][2][2], xv[DEEP][NT][2];  // weights: [block][row tile][rows g, g + 8][half]
    float ws[DEEP], xs[DEEP][NT][2];
#pragma unroll
    for (uint32_t j = 0; j < DEEP; ++j) {
      const bool in = k0 + j < kblocks;
#pragma unroll
      for (uint32_t r = 0; r < 2u * RT; ++r)
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
          wv[j][r / 2u][r % 2u][h] = in ? ldg_stream(w0 + (uint64_t)(8u * r) * a.K + (k0 + j) * 128u + 64u * h)
                                        : make_uint4(0u, 0u, 0u, 0u);
    }
    // codes and scales are the previous kernel's output, which it may still write while
    // this kernel is resident: ordinary loads, not ones of read-only data
#pragma unroll
    for (uint32_t j = 0; j < DEEP; ++j) {
      const bool in = k0 + j < kblocks;
      ws[j] = in ? __ldg(ws_row + k0 + j) : 0.0f;
#pragma unroll
      for (uint32_t n = 0; n < NT; ++n) {
        const uint32_t tok = g + 8u * n;
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
          xv[j][n][h] = in && tok < a.width ? *reinterpret_cast<const uint4 *>(
                                                  a.codes + (uint64_t)tok * a.K + (k0 + j) * 128u + 64u * h + t * 16u)
                                            : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
          const uint32_t ot = 8u * n + 2u * t + i;
          xs[j][n][i] = in && ot < a.width ? a.scales[(uint64_t)ot * kblocks + k0 + j] : 0.0f;
        }
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < DEEP; ++j)
#pragma unroll
      for (uint32_t n = 0; n < NT; ++n) {
        const float c0 = __fmul_rn(ws[j], xs[j][n][0]), c1 = __fmul_rn(ws[j], xs[j][n][1]);
#pragma unroll
        for (uint32_t r = 0; r < RT; ++r) {
          float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            const uint4 wa = wv[j][r][0][h], wb = wv[j][r][1][h];
            mma_e4m3(d, wa.x, wb.x, wa.y, wb.y, xv[j][n][h].x, xv[j][n][h].y);
            mma_e4m3(d, wa.z, wb.z, wa.w, wb.w, xv[j][n][h].z, xv[j][n][h].w);
          }
          acc[r][n][0] = __fmaf_rn(d[0], c0, acc[r][n][0]);
          acc[r][n][1] = __fmaf_rn(d[1], c1, acc[r][n][1]);
          acc[r][n][2] = __fmaf_rn(d[2], c0, acc[r][n][2]);
          acc[r][n][3] = __fmaf_rn(d[3], c1, acc[r][n][3]);
        }
      }
  }
  pdl_launch_dependents();

  // lane holds rows g, g + 8 x tokens 2 t, 2 t + 1 of each tile
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][8 * n + 2 * t + (i & 1)][16 * r + g + (i >= 2 ? 8u : 0u)] = acc[r][n][i];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 8u * NT * kRows; i += blockDim.x) {
    const uint32_t n = i / kRows, r = i % kRows, c = row0 + r;
    if (n >= a.width) continue;
    float p[kWarps];
#pragma unroll
    for (uint32_t k = 0; k < kWarps; ++k) p[k] = k < warps ? part[k][n][r] : 0.0f;
    const float sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    if (!store_elem(a.ep.y, (uint64_t)n * a.ep.y_stride + c, a.ep.y_dtype, epilogue_value(a.ep, sum, n, c)))
      raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
  }
}

template <int NT, int RT>
cudaError_t launch_one(const Fp8CodesArgs &a, cudaStream_t stream) {
  constexpr uint32_t kRows = 16u * RT, DEEP = 2u / RT;
  const uint32_t groups = (a.K / 128u + DEEP - 1u) / DEEP, warps = groups < kWarps ? groups : kWarps;
  return launch_kernel(k_fp8_narrow<NT, RT>, dim3(a.rows / kRows), dim3(warps * 32u), 0, stream, a);
}

}  // namespace fp8n

cudaError_t launch_fp8_narrow(const Fp8CodesArgs &a, int num_sms, cudaStream_t stream) {
  if (a.width == 0 || a.width > 16u || a.rows % 64u || a.K % 128u) return cudaErrorInvalidValue;
  if (a.width <= 8u) return fp8n::launch_one<1, 1>(a, stream);
  return a.rows >= 32u * (uint32_t)num_sms ? fp8n::launch_one<2, 2>(a, stream) : fp8n::launch_one<2, 1>(a, stream);
}

}  // namespace pw
