// pw_epilogue.cuh -- element types and the linear layers' epilogue:
// y = round(activation(sum + bias) + residual), everything before the one
// rounding in f32.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "pw_device.cuh"
#include "pw_internal.h"

namespace pw {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Smallest |f32| bit pattern that rounding to the dtype turns into an infinity
// (f16: 65520, halfway above the largest finite value, where ties go up).
__device__ __forceinline__ uint32_t overflow_bits(uint32_t dtype) {
  return dtype == PW_DTYPE_F32 ? 0x7f800000u : dtype == PW_DTYPE_BF16 ? kBf16OverflowBits : 0x477ff000u;
}

// One element of a PW_DTYPE_* array (the dtype is uniform over the grid).
__device__ __forceinline__ float load_elem(const void *p, uint64_t i, uint32_t dtype) {
  if (dtype == PW_DTYPE_F32) return static_cast<const float *>(p)[i];
  if (dtype == PW_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return __half2float(static_cast<const __half *>(p)[i]);
}

// Stores v rounded to the dtype; false when the stored value is not finite.
__device__ __forceinline__ bool store_elem(void *p, uint64_t i, uint32_t dtype, float v) {
  if (dtype == PW_DTYPE_F32) {
    static_cast<float *>(p)[i] = v;
    return finite(v);
  }
  if (dtype == PW_DTYPE_BF16) {
    const __nv_bfloat16 r = __float2bfloat16_rn(v);
    static_cast<__nv_bfloat16 *>(p)[i] = r;
    return finite(__bfloat162float(r));
  }
  const __half r = __float2half_rn(v);
  static_cast<__half *>(p)[i] = r;
  return finite(__half2float(r));
}

// The activations from their formulas, to a few ulps of f32 (__fdividef: 2),
// without branches, so that the compiler interleaves several values.
// exp(-v) overflows to infinity for v < -88 and the quotient is then -0, the limit.
//
// GELU: v (1 + erf(v / sqrt 2)) / 2 cancels below v ~ -4, so with z = |v| / sqrt 2
// it is h = v erfc(z) / 2 for v < 0 and v - h for v > 0.  erfc(z) = exp(-z^2) t Q(t),
// t = 1 / (1 + 0.4 z): Q is a degree-8 polynomial fitted here to exp(z^2) erfc(z) / t
// over z in [0, 10.5] by iteratively reweighted least squares in relative error
// (largest 6.6e-8; with f32 arithmetic 5.5e-7 for |v| < 3, growing with v^2 2^-24
// in the tail).  CUDA's erfcf has branches that kept the values of a thread from
// overlapping: a 8192 x 16384 x 4096 layer took 877 us with it, 709 us without
// an activation.
__device__ __forceinline__ float gelu(float v) {
  const float t = __fdividef(1.0f, fmaf(0.4f * 0.70710678f, fabsf(v), 1.0f));
  float q = 0.04211849719f;
  q = fmaf(q, t, -0.1445513666f);
  q = fmaf(q, t, 0.09278277308f);
  q = fmaf(q, t, 0.07784505188f);
  q = fmaf(q, t, 0.08678550273f);
  q = fmaf(q, t, 0.190383628f);
  q = fmaf(q, t, 0.202661037f);
  q = fmaf(q, t, 0.2263343185f);
  q = fmaf(q, t, 0.2256406248f);
  const float h = 0.5f * v * (exp2f(-0.72134752f * v * v) * (t * q));
  return v < 0.0f ? h : v - h;
}
__device__ __forceinline__ float activate(float v, uint32_t act) {
  switch (act) {
    case PW_ACT_RELU: return v < 0.0f ? 0.0f : v;  // a NaN stays a NaN
    case PW_ACT_GELU: return gelu(v);
    case PW_ACT_GELU_TANH: {
      // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
      const float u = 1.5957691216057308f * fmaf(0.044715f * v * v, v, v);
      return __fdividef(v, 1.0f + expf(-u));
    }
    case PW_ACT_SILU: return __fdividef(v, 1.0f + expf(-v));
    default: return v;
  }
}

// One output: `sum` for token t, output column c.
__device__ __forceinline__ float epilogue_value(const EpilogueArgs &e, float sum, uint64_t t, uint32_t c) {
  if (e.bias) sum += load_elem(e.bias, c, e.bias_dtype);
  sum = activate(sum, e.act);
  if (e.residual) sum += load_elem(e.residual, t * e.residual_stride + c, e.residual_dtype);
  return sum;
}

__device__ __forceinline__ float4 bias4(const EpilogueArgs &e, uint32_t c) {
  if (!e.bias) return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  return make_float4(load_elem(e.bias, c, e.bias_dtype), load_elem(e.bias, c + 1u, e.bias_dtype),
                     load_elem(e.bias, c + 2u, e.bias_dtype), load_elem(e.bias, c + 3u, e.bias_dtype));
}

// v[i] = activation(v[i]): one branch for all of them.
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], uint32_t act) {
  switch (act) {
    case PW_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], PW_ACT_RELU);
      break;
    case PW_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], PW_ACT_GELU);
      break;
    case PW_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], PW_ACT_GELU_TANH);
      break;
    case PW_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate(v[i], PW_ACT_SILU);
      break;
    default: break;
  }
}

// The epilogue of four consecutive columns c .. c + 3 (c % 4 == 0) of token t,
// with one access per array where its rows allow.  False when a stored value
// is not finite.
__device__ __forceinline__ bool finish4(const EpilogueArgs &e, float4 q, float4 bias, uint64_t t, uint32_t c) {
  float v[4] = {q.x + bias.x, q.y + bias.y, q.z + bias.z, q.w + bias.w};
  activate_all(v, e.act);
  const uint32_t rz = e.residual_dtype == PW_DTYPE_F32 ? 4u : 2u, yz = e.y_dtype == PW_DTYPE_F32 ? 4u : 2u;
  if (e.residual) {
    const uint8_t *p = static_cast<const uint8_t *>(e.residual) + (t * e.residual_stride + c) * rz;
    if ((reinterpret_cast<uintptr_t>(p) & (4u * rz - 1u)) == 0u) {
      if (rz == 4u) {
        const float4 r = *reinterpret_cast<const float4 *>(p);
        v[0] += r.x, v[1] += r.y, v[2] += r.z, v[3] += r.w;
      } else {
        const uint2 r = *reinterpret_cast<const uint2 *>(p);
        if (e.residual_dtype == PW_DTYPE_BF16) {
          v[0] += __uint_as_float(r.x << 16), v[1] += __uint_as_float(r.x & 0xffff0000u);
          v[2] += __uint_as_float(r.y << 16), v[3] += __uint_as_float(r.y & 0xffff0000u);
        } else {
          const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&r.x));
          const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&r.y));
          v[0] += a.x, v[1] += a.y, v[2] += b.x, v[3] += b.y;
        }
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) v[i] += load_elem(e.residual, t * e.residual_stride + c + i, e.residual_dtype);
    }
  }
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  uint8_t *p = static_cast<uint8_t *>(e.y) + (t * e.y_stride + c) * yz;
  if ((reinterpret_cast<uintptr_t>(p) & (4u * yz - 1u)) == 0u) {
    if (yz == 4u) {
      *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (e.y_dtype == PW_DTYPE_BF16) {
      *reinterpret_cast<uint2 *>(p) = make_uint2(pack_bf16x2_rn(v[0], v[1]), pack_bf16x2_rn(v[2], v[3]));
    } else {
      const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
      *reinterpret_cast<uint2 *>(p) =
          make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) store_elem(e.y, t * e.y_stride + c + i, e.y_dtype, v[i]);
  }
  return top < overflow_bits(e.y_dtype);
}

}  // namespace pw
