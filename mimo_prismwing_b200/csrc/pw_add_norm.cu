// pw_add_norm.cu -- the residual's addition, RMSNorm and its FP8 output in one
// pass over the rows:
//   s = round(x + residual), v = s / sqrt(mean(s^2) + eps) * w,
//   y = round(v), scale_g = max(absmax_g v, 1e-10) / 448, code = e4m3(v / scale_g).
//
// About 10 operations per element against 5-9 bytes: bound by HBM, and for a
// few rows by one chain of load, reduction, store.  A CTA holds a whole row in
// registers (8 elements per thread and step), so x and residual are read once
// and every output is written once; the weight comes from L1.  The sum of
// squares is f32: per-thread chains of at most 32 squares, then a fixed tree.
// With several rows per CTA the next rows of x and residual are on their way
// into a shared-memory ring (cp.async.bulk, one thread) while a row is reduced
// and stored; otherwise a CTA's loads would wait for its barrier and stores.
#include <cstdint>
#include <cuda_runtime.h>

#include <type_traits>

#include "pw_device.cuh"
#include "pw_epilogue.cuh"
#include "pw_internal.h"

namespace pw {
namespace addnorm {

constexpr uint32_t kMaxThreads = 512;
constexpr uint32_t kSlimThreads = 128;
constexpr uint32_t kMaxHidden = 16384;

// How a thread's step of 8 columns is accessed: element by element, as 16-byte
// vectors, or as vectors in a row that the CTA's steps cover exactly.
enum Access { kElements, kVectors, kFull };

// Column of element k (0..7) of a thread's step.  A warp's step covers 256
// columns.  With vectors a lane holds 8 consecutive columns, a 128-column
// group is half a warp; without, a lane holds every 32nd column, so that
// single-element accesses are coalesced, and a group is four elements of every lane.
template <Access VEC>
__device__ __forceinline__ uint32_t column(uint32_t step_base, uint32_t lane, uint32_t k) {
  return VEC != kElements ? step_base + lane * 8u + k : step_base + k * 32u + lane;
}

// 8 values of a 16-bit type in a 16-byte word, rounded with one conversion per pair.
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]);
template <>
__device__ __forceinline__ uint4 pack8<__nv_bfloat16>(const float (&v)[8]) {
  return make_uint4(pack_bf16x2_rn(v[0], v[1]), pack_bf16x2_rn(v[2], v[3]), pack_bf16x2_rn(v[4], v[5]),
                    pack_bf16x2_rn(v[6], v[7]));
}
template <>
__device__ __forceinline__ uint4 pack8<__half>(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void unpack8(uint4 q, float (&v)[8]);
template <>
__device__ __forceinline__ void unpack8<__nv_bfloat16>(uint4 q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void unpack8<__half>(uint4 q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    unpack8<T>(*reinterpret_cast<const uint4 *>(p), v);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4 *>(p) = pack8<T>(v);
  }
}

// a + b as T holds it.  For the 16-bit types one packed addition per pair gives
// what an f32 addition and a rounding give: the f32 sum is exact when the
// exponents are less than 17 (bf16; f16: 14) apart, and beyond that the smaller
// value is too small to move the larger one's rounding either way.
template <typename T>
__device__ __forceinline__ void add_words(uint4 &a, uint4 b) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  T2 *p = reinterpret_cast<T2 *>(&a);
  const T2 *q = reinterpret_cast<const T2 *>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __hadd2(p[i], q[i]);
}

// The group's quotient as Fp8GroupScale::quotient; the conversion to e4m3 saturates.
__device__ __forceinline__ float code_quotient(const Fp8GroupScale &g, float v) {
  const float q0 = __fmul_rn(v, g.rcp);
  const float q1 = __fmaf_rn(__fmaf_rn(-q0, g.scale, v), g.rcp, q0);
  return copysignf(__fmaf_rn(__fmaf_rn(-q1, g.scale, v), g.rcp, q1), v);
}

// Row values of one step: loads (zero past the row's end).
template <typename T, Access VEC>
__device__ __forceinline__ void load_step(const T *row, uint32_t base, uint32_t lane, uint32_t hidden, float (&v)[8]) {
  if (VEC == kFull) {
    load8<T>(row + base + lane * 8u, v);
  } else if (VEC == kVectors) {
    if (base + lane * 8u < hidden) {
      load8<T>(row + base + lane * 8u, v);
      return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.0f;
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t c = column<kElements>(base, lane, k);
      v[k] = c < hidden ? to_f32(row[c]) : 0.0f;
    }
  }
}

template <typename T, Access VEC>
__device__ __forceinline__ void store_step(T *row, uint32_t base, uint32_t lane, uint32_t hidden, const float (&v)[8]) {
  if (VEC != kElements) {
    if (VEC == kFull || base + lane * 8u < hidden) store8<T>(row + base + lane * 8u, v);
  } else {
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
      const uint32_t c = column<kElements>(base, lane, k);
      if (c < hidden) row[c] = from_f32<T>(v[k]);
    }
  }
}

// Sum over the CTA, the same value in every thread: within the warps, then over
// the at most 16 warps' sums.  `part` alternates between two rows, so one
// barrier per sum is enough.
__device__ __forceinline__ float cta_sum(float v, float *part) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const uint32_t warps = blockDim.x / 32u, lane = threadIdx.x % 32u;
  if (warps == 1u) return v;
  if (lane == 0u) part[threadIdx.x / 32u] = v;
  __syncthreads();
  v = lane % 16u < warps ? part[lane % 16u] : 0.0f;
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr uint32_t kMaxStages = 4;
constexpr uint32_t kRingBytes = 192u * 1024u;  // rings of an SM's CTAs together; the rest stays L1

// One row of x and residual into ring slot `slot`.
template <typename T>
__device__ __forceinline__ void fetch_row(const AddNormArgs &a, uint8_t *ring, uint64_t *full, uint32_t slot,
                                          uint32_t row) {
  const uint32_t bytes = a.hidden * (uint32_t)sizeof(T), per = a.residual ? 2u * bytes : bytes;
  uint8_t *dst = ring + slot * per;
  mbar_arrive_expect_tx(&full[slot], per);
  bulk_g2s(dst, static_cast<const T *>(a.x) + (uint64_t)row * a.x_stride, bytes, &full[slot]);
  if (a.residual)
    bulk_g2s(dst + bytes, static_cast<const T *>(a.residual) + (uint64_t)row * a.residual_stride, bytes, &full[slot]);
}

// STEPS: steps of 8 columns per thread (hidden <= 8 * STEPS * blockDim.x).
// stages: ring slots, or 0 to load rows straight into registers.
// SLIM: registers for a fifth CTA of four warps per SM.
template <typename T, Access VEC, int STEPS, bool SLIM>
__global__ void __launch_bounds__(SLIM ? kSlimThreads : kMaxThreads, SLIM ? 5 : STEPS == 1 ? 3 : STEPS == 2 ? 2 : 1)
    k_add_norm(const AddNormArgs a, const uint32_t stages) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float part[2][kMaxThreads / 32];
  __shared__ uint64_t full[kMaxStages];
  const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
  const uint32_t hidden = a.hidden, groups = (hidden + 127u) / 128u;
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t slot_bytes = hidden * (uint32_t)sizeof(T) * (a.residual ? 2u : 1u);
  if (VEC != kElements && stages) {
    if (threadIdx.x == 0) {
      for (uint32_t i = 0; i < stages; ++i) mbar_init(&full[i], 1);
      mbar_fence_init();
    }
    __syncthreads();
  }
  if (VEC != kElements && stages && threadIdx.x == 0)
    for (uint32_t i = 0; i < stages && blockIdx.x + i * gridDim.x < a.rows; ++i)
      fetch_row<T>(a, ring, full, i, blockIdx.x + i * gridDim.x);

  auto base_of = [&](int i) { return ((uint32_t)i * (blockDim.x / 32u) + warp) * 256u; };
  uint32_t turn = 0, slot = 0, phase = 0;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + (uint64_t)row * a.x_stride;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + (uint64_t)row * a.residual_stride : nullptr;
    if (VEC != kElements && stages) {
      x = reinterpret_cast<const T *>(ring + slot * slot_bytes);
      if (a.residual) r = x + hidden;
      if (!mbar_wait(&full[slot], phase)) raise_flag(a.flags, PW_FLAG_WAIT_TIMEOUT);
    }
    // the stream is kept, and normalized, as its type holds it
    float s[STEPS][8];
    T *o_sum = a.sum ? static_cast<T *>(a.sum) + (uint64_t)row * a.sum_stride : nullptr;
    if constexpr (VEC != kElements && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const uint32_t c = base_of(i) + lane * 8u;
        const bool in = VEC == kFull || c < hidden;
        uint4 q = make_uint4(0u, 0u, 0u, 0u);
        if (in) {
          q = *reinterpret_cast<const uint4 *>(x + c);
          if (r) add_words<T>(q, *reinterpret_cast<const uint4 *>(r + c));
          if (o_sum) *reinterpret_cast<uint4 *>(o_sum + c) = q;
        }
        unpack8<T>(q, s[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) load_step<T, VEC>(x, base_of(i), lane, hidden, s[i]);
      if (r) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          float v[8];
          load_step<T, VEC>(r, base_of(i), lane, hidden, v);
#pragma unroll
          for (int k = 0; k < 8; ++k) s[i][k] = to_f32(from_f32<T>(s[i][k] + v[k]));
        }
      }
      if (o_sum) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) store_step<T, VEC>(o_sum, base_of(i), lane, hidden, s[i]);
      }
    }
    // 16-bit weights are on their way before the reduction's barrier
    uint4 wq[STEPS];
    if (VEC != kElements && a.w_dtype != PW_NORM_F32) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const uint32_t c = base_of(i) + lane * 8u;
        wq[i] = VEC == kFull || c < hidden
                    ? __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.weight) + c))
                    : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) sq = fmaf(s[i][k], s[i][k], sq);
    sq = cta_sum(sq, part[turn]);
    turn ^= 1u;
    if (VEC != kElements && stages) {
      // past that barrier every thread has its part of the row: refill the slot
      const uint32_t next = row + stages * gridDim.x;
      if (threadIdx.x == 0 && next < a.rows) fetch_row<T>(a, ring, full, slot, next);
      if (++slot == stages) {
        slot = 0;
        phase ^= 1u;
      }
    }
    float eps = a.eps;
    if (!finite(sq)) {  // uniform: a non-finite value, or squares beyond f32
      bool ok = true;
      constexpr float kDown = 8.271806125530277e-25f;  // 2^-80: squares of scaled values cannot overflow
      eps = eps * kDown * kDown;  // vanishes unless it is as large as they are
      sq = 0.0f;
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          ok = ok && finite(s[i][k]);
          s[i][k] *= kDown;
          sq = fmaf(s[i][k], s[i][k], sq);
        }
      if (!ok) raise_flag(a.flags, PW_FLAG_NONFINITE_INPUT);
      sq = cta_sum(sq, part[turn]);
      turn ^= 1u;
    }
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(sq, (float)hidden) + eps));
    float top[STEPS][2];  // largest |v| of the step's elements 0..3 and 4..7
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      float w[8];
      if (VEC != kElements && a.w_dtype == PW_NORM_BF16)
        unpack8<__nv_bfloat16>(wq[i], w);
      else if (VEC != kElements && a.w_dtype == PW_NORM_F16)
        unpack8<__half>(wq[i], w);
      else if (a.w_dtype == PW_NORM_F32)
        load_step<float, VEC>(static_cast<const float *>(a.weight), base_of(i), lane, hidden, w);
      else if (a.w_dtype == PW_NORM_BF16)
        load_step<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16 *>(a.weight), base_of(i), lane, hidden, w);
      else
        load_step<__half, VEC>(static_cast<const __half *>(a.weight), base_of(i), lane, hidden, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[i][k] = s[i][k] * inv * w[k];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        top[i][h] = max_abs(max_abs(s[i][4 * h], s[i][4 * h + 1], s[i][4 * h + 2]), s[i][4 * h + 3], 0.0f);
    }

    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) most = max_abs(most, top[i][0], top[i][1]);
    if (__float_as_uint(most) >= overflow_bits(a.y ? a.y_dtype : PW_DTYPE_F32))  // a NaN too
      raise_flag(a.flags, PW_FLAG_NONFINITE_ROUND);
    if (a.y) {
      if (a.y_dtype == a.dtype) {
        T *o = static_cast<T *>(a.y) + (uint64_t)row * a.y_stride;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) store_step<T, VEC>(o, base_of(i), lane, hidden, s[i]);
      } else {
        float *o = static_cast<float *>(a.y) + (uint64_t)row * a.y_stride;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) store_step<float, VEC>(o, base_of(i), lane, hidden, s[i]);
      }
    }
    if (a.codes) {
      uint8_t *codes = a.codes + (uint64_t)row * hidden;
      float *scales = a.scales + (uint64_t)row * groups;
      // A warp's steps hold 2 * STEPS groups.  Their maxima first, then every
      // lane computes one group's scale and reciprocal (two IEEE divisions:
      // one evaluation instead of one per step) and the others read it.
      constexpr uint32_t N = 2u * STEPS;
      float m[N];  // vectors: both halves of m[2 i] are in their own lanes
      if (VEC != kElements) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          m[i] = fmaxf(top[i][0], top[i][1]);
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
        }
      } else {
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            m[2 * i + h] = top[i][h];
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1)
              m[2 * i + h] = fmaxf(m[2 * i + h], __shfl_xor_sync(0xffffffffu, m[2 * i + h], o));
          }
      }
      float mine = m[0];
      const uint32_t turns = VEC != kElements ? (uint32_t)STEPS : N;
#pragma unroll
      for (uint32_t i = 1; i < turns; ++i)
        if (lane % 16u == i) mine = m[i];
      const Fp8GroupScale own = Fp8GroupScale::of(mine);
      if (VEC != kElements) {
        // lane 16 h + i holds the group of step i's half h
        const uint32_t g = base_of((int)(lane % 16u)) / 128u + lane / 16u;
        if (lane % 16u < (uint32_t)STEPS && g < groups) scales[g] = own.scale;
      } else {
        const uint32_t g = base_of((int)(lane / 2u)) / 128u + lane % 2u;
        if (lane < N && g < groups) scales[g] = own.scale;
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (VEC != kElements) {
          Fp8GroupScale g;
          g.scale = __shfl_sync(0xffffffffu, own.scale, (lane & 16u) + (uint32_t)i);
          g.rcp = __shfl_sync(0xffffffffu, own.rcp, (lane & 16u) + (uint32_t)i);
          const uint32_t c = base_of(i) + lane * 8u;
          if (VEC == kFull || c < hidden) {
            uint2 q;
            q.x = encode2(code_quotient(g, s[i][0]), code_quotient(g, s[i][1])) |
                  encode2(code_quotient(g, s[i][2]), code_quotient(g, s[i][3])) << 16;
            q.y = encode2(code_quotient(g, s[i][4]), code_quotient(g, s[i][5])) |
                  encode2(code_quotient(g, s[i][6]), code_quotient(g, s[i][7])) << 16;
            *reinterpret_cast<uint2 *>(codes + c) = q;
          }
        } else {
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            Fp8GroupScale g;
            g.scale = __shfl_sync(0xffffffffu, own.scale, 2u * (uint32_t)i + h);
            g.rcp = __shfl_sync(0xffffffffu, own.rcp, 2u * (uint32_t)i + h);
#pragma unroll
            for (uint32_t k = 4 * h; k < 4 * h + 4; ++k) {
              const uint32_t c = column<kElements>(base_of(i), lane, k);
              if (c < hidden) codes[c] = (uint8_t)(encode2(code_quotient(g, s[i][k]), 0.0f) & 0xffu);
            }
          }
        }
      }
    }
  }
}

// CTAs of `threads` that fit an SM together by their registers.
template <auto Kernel>
uint32_t resident(uint32_t threads) {
  static std::atomic<int> known[kMaxThreads / 32 + 1];
  int n = known[threads / 32u].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, Kernel, (int)threads, 0) != cudaSuccess || n < 1) n = 1;
    known[threads / 32u].store(n, std::memory_order_relaxed);
  }
  return (uint32_t)n;
}

template <typename T, Access VEC, int STEPS, bool SLIM>
cudaError_t launch_one(const AddNormArgs &a, uint32_t threads, int num_sms, cudaStream_t stream) {
  const uint32_t per_sm = resident<k_add_norm<T, VEC, STEPS, SLIM>>(threads);
  uint32_t stages = 0;
  // The ring pays when CTAs run several rows (without it the first and last case
  // below took 21.5 and 204 us).  Slots share what the resident CTAs have of shared memory.
  const uint32_t row_bytes = a.hidden * (uint32_t)sizeof(T) * (a.residual ? 2u : 1u);
  if (VEC != kElements && a.rows > (uint32_t)num_sms * per_sm) {
    stages = kRingBytes / per_sm / row_bytes;
    stages = stages > kMaxStages ? kMaxStages : stages < 2u ? 0u : stages;
  }
  const uint32_t most = (uint32_t)num_sms * per_sm;
  const uint32_t grid = a.rows < most ? a.rows : most;
  if (stages) {
    cudaError_t e = allow_smem<k_add_norm<T, VEC, STEPS, SLIM>>(kRingBytes);
    if (e != cudaSuccess) return e;
  }
  return launch_kernel(k_add_norm<T, VEC, STEPS, SLIM>, dim3(grid), dim3(threads), stages * row_bytes, stream, a, stages);
}

template <typename T, Access VEC>
cudaError_t launch_shape(const AddNormArgs &a, uint32_t steps, uint32_t threads, int num_sms, cudaStream_t stream) {
  if (steps == 1u) return launch_one<T, VEC, 1, false>(a, threads, num_sms, stream);
  if (steps == 2u) return launch_one<T, VEC, 2, false>(a, threads, num_sms, stream);
  // Fewer registers make more CTAs resident, and a turn of each slower: worth it when
  // the rows then take fewer turns (bf16 with residual and codes, usual / slim: 2048 x
  // 4096, 4 / 3 turns, 14.7 / 13.8 us; 16384 x 1024, 7 / 6 turns, 23.9 / 22.5 us; 2048 x
  // 2048, 2 turns both, 7.3 / 8.0 us; f32 rows leave slim CTAs no ring: 2048 x 4096 20.4 /
  // 22.9 us).
  if constexpr (VEC != kElements && sizeof(T) == 2) {
    if (threads <= kSlimThreads) {
      const uint32_t usual = resident<k_add_norm<T, VEC, 4, false>>(threads) * (uint32_t)num_sms;
      const uint32_t slim = resident<k_add_norm<T, VEC, 4, true>>(threads) * (uint32_t)num_sms;
      if ((a.rows + slim - 1u) / slim < (a.rows + usual - 1u) / usual)
        return launch_one<T, VEC, 4, true>(a, threads, num_sms, stream);
    }
  }
  return launch_one<T, VEC, 4, false>(a, threads, num_sms, stream);
}

template <typename T, Access VEC>
cudaError_t launch_steps(const AddNormArgs &a, int num_sms, cudaStream_t stream) {
  // With few rows, all the threads that a row can use.  With many, four steps per
  // thread, so that fewer threads repeat a row's reductions and scales (measured
  // at 2 / 4 steps: 2048 x 4096 bf16 with residual and codes 16.6 / 15.8 us, 8192
  // rows 46.7 / 41.9 us, 16384 x 8192 f16 to f16 108.7 / 94.2 us).  Element access
  // needs twice the registers, so two steps unless the row needs four (777 x 5003
  // f32: 16.8 us at two, 18.9 us at four).
  const uint32_t warp_steps = (a.hidden + 255u) / 256u;  // 1..64
  const uint32_t least = warp_steps <= 16u ? 1u : warp_steps <= 32u ? 2u : 4u;
  const uint32_t best = warp_steps >= 4u && VEC != kElements ? 4u : warp_steps >= 2u ? 2u : 1u;
  const uint32_t steps = a.rows <= 2u * (uint32_t)num_sms || best < least ? least : best;
  const uint32_t threads = (warp_steps + steps - 1u) / steps * 32u;
  if (VEC == kVectors && a.hidden == threads * 8u * steps)
    return launch_shape<T, kFull>(a, steps, threads, num_sms, stream);
  return launch_shape<T, VEC>(a, steps, threads, num_sms, stream);
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
  return vec ? launch_steps<T, kVectors>(a, num_sms, stream) : launch_steps<T, kElements>(a, num_sms, stream);
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
