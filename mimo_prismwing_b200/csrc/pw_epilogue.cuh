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
// The logistic function by exp of the negative magnitude, so that neither it nor the
// divisor (1 to 2) leaves f32's range and the tail keeps its digits:
// v / (1 + exp(-u)) = v exp(u) / (1 + exp(u)), the latter for u < 0.
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
  // far right of zero the tail is 0 times a bounded factor, not times an infinite v
  const float h = 0.5f * fminf(v, 64.0f) * (exp2f(-0.72134752f * v * v) * (t * q));
  return v < 0.0f ? h : v - h;
}
// v / (1 + exp(-u)) for a u of v's sign.
__device__ __forceinline__ float gated(float v, float u) {
  const float e = expf(-fabsf(u));
  return __fdividef(u < 0.0f ? v * e : v, 1.0f + e);
}
__device__ __forceinline__ float activate(float v, uint32_t act) {
  switch (act) {
    case PW_ACT_RELU: return v < 0.0f ? 0.0f : v;  // a NaN stays a NaN
    case PW_ACT_GELU: return gelu(v);
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u))
    case PW_ACT_GELU_TANH: return gated(v, 1.5957691216057308f * fmaf(0.044715f * v * v, v, v));
    case PW_ACT_SILU: return gated(v, v);
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

// max(|a|, |b|, |c|), a NaN if any is one.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
}

// 8 values in a 16-byte word of a 16-bit type.
__device__ __forceinline__ uint4 pack8(const float *v, uint32_t dtype) {
  if (dtype == PW_DTYPE_BF16)
    return make_uint4(pack_bf16x2_rn(v[0], v[1]), pack_bf16x2_rn(v[2], v[3]), pack_bf16x2_rn(v[4], v[5]),
                      pack_bf16x2_rn(v[6], v[7]));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// v[i] += 8 values of a 16-bit type.
__device__ __forceinline__ void add8(float *v, uint4 q, uint32_t dtype) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = dtype == PW_DTYPE_BF16 ? make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u))
                                            : __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] += f.x;
    v[2 * i + 1] += f.y;
  }
}

// Whether four consecutive elements from any column c, c % 4 == 0, of these rows can
// be accessed at once.
__device__ __forceinline__ bool quad_access(const void *p, uint64_t stride, uint32_t dtype) {
  const uint32_t z = dtype == PW_DTYPE_F32 ? 4u : 2u;
  return reinterpret_cast<uintptr_t>(p) % (4u * z) == 0u && stride % 4u == 0u;
}

// R quads of four columns (column % 4 == 0) of a thread: DOWN: columns c .. c + 3 of
// the tokens t0 + 8 j with 8 j < n; else columns c + 4 j .. of token t0, n ignored.
template <int R, bool DOWN>
struct Quads {
  uint64_t t0;
  uint32_t c, n;
  __device__ __forceinline__ bool in(uint32_t j) const { return !DOWN || 8u * j < n; }
  __device__ __forceinline__ uint64_t at(uint32_t j, uint64_t stride) const {
    return DOWN ? (t0 + 8u * j) * stride + c : t0 * stride + c + 4u * j;
  }
};

// Their residual: loads only, all in flight, so they can be issued before what
// they are added to is ready (past the end: the first quad again).
template <int R, bool DOWN>
__device__ __forceinline__ void load_quads(const EpilogueArgs &e, const Quads<R, DOWN> &g, bool quad_residual,
                                           uint32_t (&raw)[R][4]) {
  if (!quad_residual) {
#pragma unroll
    for (uint32_t j = 0; j < R; ++j)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        raw[j][i] =
            __float_as_uint(load_elem(e.residual, g.at(g.in(j) ? j : 0u, e.residual_stride) + i, e.residual_dtype));
  } else if (e.residual_dtype == PW_DTYPE_F32) {
#pragma unroll
    for (uint32_t j = 0; j < R; ++j) {
      const uint4 q = *reinterpret_cast<const uint4 *>(static_cast<const uint32_t *>(e.residual) +
                                                       g.at(g.in(j) ? j : 0u, e.residual_stride));
      raw[j][0] = q.x, raw[j][1] = q.y, raw[j][2] = q.z, raw[j][3] = q.w;
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < R; ++j) {
      const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(e.residual) +
                                                       g.at(g.in(j) ? j : 0u, e.residual_stride));
      raw[j][0] = q.x, raw[j][1] = q.y, raw[j][2] = raw[j][3] = 0u;
    }
  }
}

// Their epilogue.  False when a stored value is not finite.
template <int R, bool DOWN>
__device__ __forceinline__ bool finish_quads(const EpilogueArgs &e, const Quads<R, DOWN> &g, float (&v)[4 * R],
                                             const float4 (&bias)[DOWN ? 1 : R], const uint32_t (&raw)[R][4],
                                             bool quad_residual, bool quad_y) {
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const float4 b = bias[DOWN ? 0 : j];
    v[4 * j] += b.x, v[4 * j + 1] += b.y, v[4 * j + 2] += b.z, v[4 * j + 3] += b.w;
  }
  activate_all(v, e.act);
  if (e.residual) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float r[4];
      if (!quad_residual || e.residual_dtype == PW_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __uint_as_float(raw[j][i]);
      } else if (e.residual_dtype == PW_DTYPE_BF16) {
        r[0] = __uint_as_float(raw[j][0] << 16), r[1] = __uint_as_float(raw[j][0] & 0xffff0000u);
        r[2] = __uint_as_float(raw[j][1] << 16), r[3] = __uint_as_float(raw[j][1] & 0xffff0000u);
      } else {
        const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&raw[j][0]));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&raw[j][1]));
        r[0] = lo.x, r[1] = lo.y, r[2] = hi.x, r[3] = hi.y;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * j + i] += r[i];
    }
  }
  uint32_t top = 0u;
#pragma unroll
  for (uint32_t j = 0; j < R; ++j) {
    if (!g.in(j)) continue;
    const float *q = v + 4 * j;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(q[i]) & 0x7fffffffu);
    const uint64_t at = g.at(j, e.y_stride);
    if (!quad_y) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) store_elem(e.y, at + i, e.y_dtype, q[i]);
    } else if (e.y_dtype == PW_DTYPE_F32) {
      *reinterpret_cast<float4 *>(static_cast<float *>(e.y) + at) = make_float4(q[0], q[1], q[2], q[3]);
    } else if (e.y_dtype == PW_DTYPE_BF16) {
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(e.y) + at) =
          make_uint2(pack_bf16x2_rn(q[0], q[1]), pack_bf16x2_rn(q[2], q[3]));
    } else {
      const __half2 lo = __floats2half2_rn(q[0], q[1]), hi = __floats2half2_rn(q[2], q[3]);
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(e.y) + at) =
          make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
    }
  }
  return top < overflow_bits(e.y_dtype);
}

}  // namespace pw
