// policy_common.h -- element types, matrix instructions and activations of the policy network's kernels (gfx950).
#pragma once
#include <hip/hip_runtime.h>

#include "../../../include/mjlab_policy.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// VEC: elements of a 16-byte chunk.
template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int DTYPE = MJLAB_DTYPE_F32, VEC = 4; };
template <> struct Elem<_Float16> { static constexpr int DTYPE = MJLAB_DTYPE_F16, VEC = 8; };
template <> struct Elem<__bf16> { static constexpr int DTYPE = MJLAB_DTYPE_BF16, VEC = 8; };

template <typename T> struct alignas(16) Chunk {
  T e[Elem<T>::VEC];
};

// 16 bytes from / to any element address: global memory takes unaligned 16-byte accesses here, so rows of odd length keep the wide path.
template <typename T> __device__ __forceinline__ Chunk<T> load_chunk(const T* p) {
  Chunk<T> c;
  __builtin_memcpy(&c, p, 16);
  return c;
}
template <typename T> __device__ __forceinline__ void store_chunk(T* p, const Chunk<T>& c) { __builtin_memcpy(p, &c, 16); }

// the first `n` elements of a chunk (n <= 0: none), the rest zero
template <typename T> __device__ __forceinline__ Chunk<T> load_part(const T* p, long long n) {
  constexpr int V = Elem<T>::VEC;
  if (n >= V) return load_chunk(p);
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < V; ++i) c.e[i] = i < n ? p[i] : (T)0.f;
  return c;
}
template <typename T> __device__ __forceinline__ void store_part(T* p, const Chunk<T>& c, long long n) {
  constexpr int V = Elem<T>::VEC;
  if (n >= V) { store_chunk(p, c); return; }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = c.e[i];
}

// ---- activations, in float.  NaN goes through every one of them.  The device library's erff, expm1f and tanhf cost a hundred instructions each, and a layer's
// epilogue runs one per output: a gated layer of 24576 x 512 x 1365 (bf16, silu) with its backward pass took 260 us more with them than with the forms below
// (and wider stores).
__device__ __forceinline__ float rcp_f(float x) { return __builtin_amdgcn_rcpf(x); }  // 1 ulp
__device__ __forceinline__ float sigmoid_f(float z) { return rcp_f(1.f + __expf(-z)); }

// exp(z) - 1 for z <= 0: the series to z^7 above -1/4 (next term: 2^-14 / 40320 of z, 2^-29), the difference below
__device__ __forceinline__ float expm1_neg(float z) {
  const float s = z * (1.f + z * (1.f / 2 + z * (1.f / 6 + z * (1.f / 24 + z * (1.f / 120 + z * (1.f / 720 + z * (1.f / 5040)))))));
  const float d = __expf(z) - 1.f;
  return z > -0.25f ? s : d;
}

// The odd series to z^9 below 1/4 (next term: 2^-20 * 0.0089 of z), 1 - 2 / (1 + exp 2z) above
__device__ __forceinline__ float tanh_f(float z) {
  const float q = z * z;
  const float s = z * (1.f + q * (-1.f / 3 + q * (2.f / 15 + q * (-17.f / 315 + q * (62.f / 2835)))));
  const float d = 1.f - 2.f * rcp_f(1.f + __expf(2.f * z));
  return q < 0.0625f ? s : d;
}

// (1 + erf(z / sqrt 2)) / 2 with e = exp(-z^2 / 2).  Abramowitz and Stegun 7.1.26, off by 0.75e-7 at most: enough for 16 bits.  FINE, for float outputs: the
// Chebyshev fit of erfc whose relative error is 1.2e-7 everywhere (Press et al., Numerical Recipes, 6.2), since small values show theirs; e adds the rounding of its
// argument, z^2 / 2 times 2^-24 of itself.
// (24576 x 512 x 512 float, us: the first form 90, the second 93, erfcf 117.)
template <bool FINE> __device__ __forceinline__ float normal_cdf(float z, float e) {
  if constexpr (FINE) {
    const float x = 0.70710678f * __builtin_fabsf(z), t = rcp_f(1.f + 0.5f * x);
    const float q = 1.48851587f + t * (-0.82215223f + t * 0.17087277f);
    const float r = 0.37409196f + t * (0.09678418f + t * (-0.18628806f + t * (0.27886807f + t * (-1.13520398f + t * q))));
    const float tail = 0.5f * t * e * __expf(-1.26551223f + t * (1.00002368f + t * r));
    return z < 0.f ? tail : 1.f - tail;
  }
  const float t = rcp_f(1.f + 0.3275911f * 0.70710678f * __builtin_fabsf(z));
  const float tail = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return z < 0.f ? tail : 1.f - tail;
}

// FINE: for float outputs
template <int ACT, bool FINE> __device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == MJLAB_ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == MJLAB_ACT_ELU) return z > 0.f ? z : expm1_neg(z);
  if constexpr (ACT == MJLAB_ACT_TANH) return tanh_f(z);
  if constexpr (ACT == MJLAB_ACT_SIGMOID) return sigmoid_f(z);
  if constexpr (ACT == MJLAB_ACT_SILU) return z * sigmoid_f(z);
  if constexpr (ACT == MJLAB_ACT_GELU) return z * normal_cdf<FINE>(z, __expf(-0.5f * z * z));
  return z;
}

// Derivative at z.  Beyond |z| = 100 the derivative of each is its limit to all 24 bits: z is cut there, so that a z that 16 bits hold
// as infinite gives the limit and not infinity times zero.
template <int ACT, bool FINE> __device__ __forceinline__ float act_slope(float z) {
  z = z > 100.f ? 100.f : (z < -100.f ? -100.f : z);
  if constexpr (ACT == MJLAB_ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if constexpr (ACT == MJLAB_ACT_ELU) return z > 0.f ? 1.f : __expf(z);
  if constexpr (ACT == MJLAB_ACT_TANH) { const float e = __expf(-2.f * __builtin_fabsf(z)), r = rcp_f(1.f + e); return 4.f * e * r * r; }
  if constexpr (ACT == MJLAB_ACT_SIGMOID) { const float e = __expf(-__builtin_fabsf(z)), r = rcp_f(1.f + e); return e * r * r; }
  if constexpr (ACT == MJLAB_ACT_SILU) { const float s = sigmoid_f(z); return s * (1.f + z * (1.f - s)); }
  if constexpr (ACT == MJLAB_ACT_GELU) { const float e = __expf(-0.5f * z * z); return normal_cdf<FINE>(z, e) + z * 0.39894228f * e; }
  return 1.f;
}

// The derivative from the output y of a layer without residual, where y determines it (off by 2^-24 of 1 where y is float)
__host__ __device__ constexpr bool slope_from_output(int act) { return act == MJLAB_ACT_RELU || act == MJLAB_ACT_ELU || act == MJLAB_ACT_TANH || act == MJLAB_ACT_SIGMOID; }
template <int ACT> __device__ __forceinline__ float act_slope_out(float y) {
  if constexpr (ACT == MJLAB_ACT_RELU) return y > 0.f ? 1.f : (y <= 0.f ? 0.f : y);
  if constexpr (ACT == MJLAB_ACT_ELU) return y > 0.f ? 1.f : 1.f + y;
  if constexpr (ACT == MJLAB_ACT_TANH) return 1.f - y * y;
  return y * (1.f - y);  // (sigmoid)
}

// One uniform branch for a whole block of elements: f(Act<..>) with the activation as a type
template <int A> struct Act {
  static constexpr int value = A;
};
template <typename F> __device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case MJLAB_ACT_RELU: f(Act<MJLAB_ACT_RELU>()); break;
    case MJLAB_ACT_ELU: f(Act<MJLAB_ACT_ELU>()); break;
    case MJLAB_ACT_TANH: f(Act<MJLAB_ACT_TANH>()); break;
    case MJLAB_ACT_SIGMOID: f(Act<MJLAB_ACT_SIGMOID>()); break;
    case MJLAB_ACT_SILU: f(Act<MJLAB_ACT_SILU>()); break;
    case MJLAB_ACT_GELU: f(Act<MJLAB_ACT_GELU>()); break;
    default: f(Act<MJLAB_ACT_NONE>());
  }
}

// Workgroup b of n: consecutive workgroups go to the eight XCDs in turn, each with an L2 of its own, so the index is dealt out such that
// one XCD works on neighbouring tiles (which share operand rows).
__device__ __forceinline__ long long xcd_tile(long long b, long long n) {
  const long long per = n / 8, rest = n % 8, x = b % 8, i = b / 8;
  return x * per + (x < rest ? x : rest) + i;
}
