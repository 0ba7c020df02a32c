// pw_add_norm.cu -- the residual's addition, RMSNorm and its FP8 output in one
// pass over the rows:
//   s = round(x + residual), v = s / sqrt(mean(s^2) + eps) * w,
//   y = round(v), scale_g = max(absmax_g v, 1e-10) / 448, code = e4m3(v / scale_g).
//
// About 10 operations per element against 5-9 bytes: bound by HBM, and for a
// few rows by one chain of load, reduction, store.  A CTA holds a whole row in
// registers (8 elements per thread and step), so x and residual are read once
// and every output is written once; the weight's 8 values per step stay in
// registers over the rows of a persistent CTA.  The sum of squares is f32:
// per-thread chains of at most 32 squares, then a fixed tree.
#include <cstdint>
#include <cuda_runtime.h>

#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"

namespace pw {
namespace addnorm {

constexpr uint32_t kMaxThreads = 512;
constexpr uint32_t kMaxHidden = 16384;

// Column of element k (0..7) of a thread's step.  A warp's step covers 256
// columns.  With vectors a lane holds 8 consecutive columns, a 128-column
// group is half a warp; without, a lane holds every 32nd column, so that
// single-element accesses are coalesced, and a group is four elements of every lane.
template <bool VEC>
__device__ __forceinline__ uint32_t column(uint32_t step_base, uint32_t lane, uint32_t k) {
  return VEC ? step_base + lane * 8u + k : step_base + k * 32u + lane;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void load8<__half>(const __half *p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  if (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    T h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(v[i]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(h);
  }
}

// Row values of one step: loads (zero past the row's end).
template <typename T, bool VEC>
__device__ __forceinline__ void load_step(const T *row, uint32_t base, uint32_t lane, uint32_t hidden, float (&v)[8]) {
  if (VEC) {
    if (base + lane * 8u < hidden) {
      load8<T>(row + base + lane * 8u, v);
      return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t c = column<false>(base, lane, k);
      v[k] = c < hidden ? to_f32(row[c]) : 0.0f;
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_step(T *row, uint32_t base, uint32_t lane, uint32_t hidden, const float (&v)[8]) {
  if (VEC) {
    if (base + lane * 8u < hidden) store8<T>(row + base + lane * 8u, v);
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t c = column<false>(base, lane, k);
      if (c < hidden) row[c] = from_f32<T>(v[k]);
    }
  }
}

// Sum over the CTA, the same value in every thread.  `part` alternates between
// two rows of kMaxThreads / 32 floats, so one barrier per sum is enough.
__device__ __forceinline__ float cta_sum(float v, float *part) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const uint32_t warps = blockDim.x / 32u;
  if (warps == 1u) return v;
  if (threadIdx.x % 32u == 0u) part[threadIdx.x / 32u] = v;
  __syncthreads();
  float s = 0.0f;
  for (uint32_t w = 0; w < warps; ++w) s += part[w];
  return s;
}

// STEPS: steps of 8 columns per thread (hidden <= 8 * STEPS * blockDim.x).
template <typename T, bool VEC, int STEPS>
__global__ void __launch_bounds__(kMaxThreads) k_add_norm(const AddNormArgs a) {
  __shared__ float part[2][kMaxThreads / 32];
  const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
  const uint32_t hidden = a.hidden, groups = (hidden + 127u) / 128u;
  pdl_wait();
  pdl_launch_dependents();

  uint32_t base[STEPS];
  float w[STEPS][8];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    base[i] = ((uint32_t)i * (blockDim.x / 32u) + warp) * 256u;
    switch (a.w_dtype) {
      case PW_NORM_F32:
        load_step<float, VEC>(static_cast<const float *>(a.weight), base[i], lane, hidden, w[i]);
        break;
      case PW_NORM_BF16:
        load_step<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16 *>(a.weight), base[i], lane, hidden, w[i]);
        break;
      default: load_step<__half, VEC>(static_cast<const __half *>(a.weight), base[i], lane, hidden, w[i]);
    }
  }

  uint32_t turn = 0;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + (uint64_t)row * a.x_stride;
    float s[STEPS][8];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) load_step<T, VEC>(x, base[i], lane, hidden, s[i]);
    if (a.residual) {
      const T *r = static_cast<const T *>(a.residual) + (uint64_t)row * a.residual_stride;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        float v[8];
        load_step<T, VEC>(r, base[i], lane, hidden, v);
        // the stream is kept, and normalized, as its type holds it
#pragma unroll
        for (int k = 0; k < 8; ++k) s[i][k] = to_f32(from_f32<T>(s[i][k] + v[k]));
      }
    }
    if (a.sum) {
      T *o = static_cast<T *>(a.sum) + (uint64_t)row * a.sum_stride;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) store_step<T, VEC>(o, base[i], lane, hidden, s[i]);
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) sq = fmaf(s[i][k], s[i][k], sq);
    sq = cta_sum(sq, part[turn]);
    turn ^= 1u;
    float pre = 1.0f;
    if (!finite(sq)) {  // uniform: a non-finite value, or squares beyond f32
      bool ok = true;
      pre = 8.271806125530277e-25f;  // 2^-80: the squares of scaled values cannot overflow
      sq = 0.0f;
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          ok = ok && finite(s[i][k]);
          const float v = s[i][k] * pre;
          sq = fmaf(v, v, sq);
        }
      if (!ok) raise_flag(a.flags, PW_FLAG_NONFINITE_INPUT);
      sq = cta_sum(sq, part[turn]);
      turn ^= 1u;
    }
    // next to scaled squares eps (at most f32's range) vanishes unless it is as large as they are
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sq, (float)hidden) + a.eps * pre * pre));
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[i][k] = s[i][k] * pre * inv * w[i][k];

    uint32_t top = 0u;  // largest |v| by its bits (a NaN's are above infinity's)
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(s[i][k]) & 0x7fffffffu);
    if (top >= overflow_bits(a.y ? a.y_dtype : PW_DTYPE_F32)) raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
    if (a.y) {
      if (a.y_dtype == a.dtype) {
        T *o = static_cast<T *>(a.y) + (uint64_t)row * a.y_stride;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) store_step<T, VEC>(o, base[i], lane, hidden, s[i]);
      } else {
        float *o = static_cast<float *>(a.y) + (uint64_t)row * a.y_stride;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) store_step<float, VEC>(o, base[i], lane, hidden, s[i]);
      }
    }
    if (a.codes) {
      uint8_t *codes = a.codes + (uint64_t)row * hidden;
      float *scales = a.scales + (uint64_t)row * groups;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (VEC) {
          float m = 0.0f;
#pragma unroll
          for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(s[i][k]));
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
          const Fp8GroupScale g = Fp8GroupScale::of(m);
          const uint32_t c = base[i] + lane * 8u;
          if (c < hidden) {
            uint2 q;
            q.x = encode2(g.quotient(s[i][0]), g.quotient(s[i][1])) |
                  encode2(g.quotient(s[i][2]), g.quotient(s[i][3])) << 16;
            q.y = encode2(g.quotient(s[i][4]), g.quotient(s[i][5])) |
                  encode2(g.quotient(s[i][6]), g.quotient(s[i][7])) << 16;
            *reinterpret_cast<uint2 *>(codes + c) = q;
            if (lane % 16u == 0u) scales[c / 128u] = g.scale;
          }
        } else {
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {  // the step's two groups
            float m = 0.0f;
#pragma unroll
            for (uint32_t k = 4 * h; k < 4 * h + 4; ++k) m = fmaxf(m, fabsf(s[i][k]));
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const Fp8GroupScale g = Fp8GroupScale::of(m);
#pragma unroll
            for (uint32_t k = 4 * h; k < 4 * h + 4; ++k) {
              const uint32_t c = column<false>(base[i], lane, k);
              if (c < hidden) codes[c] = (uint8_t)(encode2(g.quotient(s[i][k]), 0.0f) & 0xffu);
            }
            if (lane == 0u && base[i] + 128u * h < hidden) scales[base[i] / 128u + h] = g.scale;
          }
        }
      }
    }
  }
}

template <typename T, bool VEC, int STEPS>
cudaError_t launch_one(const AddNormArgs &a, uint32_t threads, int num_sms, cudaStream_t stream) {
  const uint32_t per_sm = 2048u / threads < 8u ? 2048u / threads : 8u;
  const uint32_t grid = a.rows < (uint32_t)num_sms * per_sm ? a.rows : (uint32_t)num_sms * per_sm;
  return launch_kernel(k_add_norm<T, VEC, STEPS>, dim3(grid), dim3(threads), 0, stream, a);
}

template <typename T, bool VEC>
cudaError_t launch_steps(const AddNormArgs &a, int num_sms, cudaStream_t stream) {
  const uint32_t warp_steps = (a.hidden + 255u) / 256u;  // 1..64
  const uint32_t steps = warp_steps <= 8u ? 1u : warp_steps <= 32u ? 2u : 4u;
  const uint32_t threads = (warp_steps + steps - 1u) / steps * 32u;
  if (steps == 1u) return launch_one<T, VEC, 1>(a, threads, num_sms, stream);
  if (steps == 2u) return launch_one<T, VEC, 2>(a, threads, num_sms, stream);
  return launch_one<T, VEC, 4>(a, threads, num_sms, stream);
}

inline bool aligned(const void *p, uint64_t stride, size_t elem) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u && stride * elem % 16u == 0u;
}

template <typename T>
cudaError_t launch_type(const AddNormArgs &a, int num_sms, cudaStream_t stream) {
  const size_t yz = a.y_dtype == PW_DTYPE_F32 ? 4u : sizeof(T);
  const bool vec = a.hidden % 8u == 0u && aligned(a.weight, 0, 1) && aligned(a.x, a.x_stride, sizeof(T)) &&
                   (!a.residual || aligned(a.residual, a.residual_stride, sizeof(T))) &&
                   (!a.sum || aligned(a.sum, a.sum_stride, sizeof(T))) && (!a.y || aligned(a.y, a.y_stride, yz)) &&
                   (!a.codes || (reinterpret_cast<uintptr_t>(a.codes) & 7u) == 0u);
  return vec ? launch_steps<T, true>(a, num_sms, stream) : launch_steps<T, false>(a, num_sms, stream);
}

}  // namespace addnorm

cudaError_t launch_add_norm(const AddNormArgs &a, int num_sms, cudaStream_t stream) {
  if (a.hidden == 0 || a.hidden > addnorm::kMaxHidden) return cudaErrorInvalidValue;
  if (a.rows == 0) return cudaSuccess;
  switch (a.dtype) {
    case PW_DTYPE_F32: return addnorm::launch_type<float>(a, num_sms, stream);
    case PW_DTYPE_BF16: return addnorm::launch_type<__nv_bfloat16>(a, num_sms, stream);
    case PW_DTYPE_F16: return addnorm::launch_type<__half>(a, num_sms, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace pw
