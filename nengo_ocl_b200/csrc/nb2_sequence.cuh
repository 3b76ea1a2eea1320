// Shared by the sequence operators (causal convolution, selective scan, residual norm):
// element types, vector loads and the layout of their tables.
//
// A sequence array holds one (rows x channels) block per sequence, rows `stride` elements
// apart, channels next to each other.  The table of a launch is an int64 matrix
// [fields][n_seq]: field 0 the number of rows, then (start, stride) of each array in
// elements, so that offsets past 2^31 need no care in the kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "nb2_common.cuh"
#include "../../include/nengo_b200.h"

__device__ __forceinline__ float nb2_to_float(float v) { return v; }
__device__ __forceinline__ float nb2_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float nb2_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T nb2_from_float(float v);
template <>
__device__ __forceinline__ float nb2_from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half nb2_from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 nb2_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
struct IsHalf {
  static constexpr bool value = false;
};
template <>
struct IsHalf<__half> {
  static constexpr bool value = true;
};

// V elements next to each other: one 16-byte access when V * sizeof(T) == 16 (the caller has
// checked the alignment), single elements otherwise.
template <typename T, int V>
struct SeqVecA {
  alignas(V * sizeof(T) >= 16 ? 16 : V * sizeof(T)) T e[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V * sizeof(T) == 16)
      *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (V * sizeof(T) == 8)
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    else if constexpr (V > 1 && V * sizeof(T) == 4)
      *reinterpret_cast<uint32_t*>(e) = *reinterpret_cast<const uint32_t*>(p);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = p[i];
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V * sizeof(T) == 16)
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
    else if constexpr (V * sizeof(T) == 8)
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    else if constexpr (V > 1 && V * sizeof(T) == 4)
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(e);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = e[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = nb2_from_float<T>(0.0f);
  }
  // (a pair of bfloat16 is two shifts of its word)
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (V > 1 && sizeof(T) == 2 && !IsHalf<T>::value) {
      const uint32_t w = reinterpret_cast<const uint32_t*>(e)[i >> 1];
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    } else {
      return nb2_to_float(e[i]);
    }
  }
  // rounds v, two to a conversion where the type has one
  __device__ __forceinline__ void put(const float (&v)[V]) {
    if constexpr (V > 1 && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        if constexpr (IsHalf<T>::value)
          reinterpret_cast<__half2*>(e)[i >> 1] = __floats2half2_rn(v[i], v[i + 1]);
        else
          reinterpret_cast<__nv_bfloat162*>(e)[i >> 1] = __floats2bfloat162_rn(v[i], v[i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = nb2_from_float<T>(v[i]);
    }
  }
};
// The gates' sigmoid, for every type: the fast exponential is off by (2 + 1.2 |v|) * 2^-23 of its value and the fast
// division by 2 * 2^-23, which where the sigmoid is not small is less than a sum of a few products; at v = -20
// (the sigmoid is 2e-9) it is 3e-6 of it.  With expf no output of the float32 workloads comes closer to the formulas than
// by a thirtieth, and the calls take longer: convolution 8192 x 4096 bfloat16 40.0 -> 45.4 us, training 4096 x 2048
// float32 53.4 -> 54.8, scan training 4096 x 2048 x 16 float32 423 -> 427, norm 8192 x 4096 bfloat16 69.4 -> 74.3.
__device__ __forceinline__ float nb2_sigmoid(float v) { return __fdividef(1.0f, 1.0f + __expf(-v)); }
// d/dv [v sigmoid(v)]
__device__ __forceinline__ float nb2_silu_slope(float v) {
  const float s = nb2_sigmoid(v);
  return s * (1.0f + v * (1.0f - s));
}

// A column's share of the sum over units that warp w of 8 adds: every eighth unit in order, 16 of them apart
// and then these (shorter chains of additions; loads of 16 in flight).  The same result every time.
__device__ __forceinline__ float nb2_sum_units(const float* column, int64_t pitch, int n_units, int w) {
  float sum = 0.0f;
  const float* at = column + w * pitch;
  int left = (n_units - w + 7) / 8;  // of this warp
  for (; left >= 16; left -= 16) {
    float v[16], part = 0.0f;
#pragma unroll
    for (int q = 0; q < 16; ++q, at += 8 * pitch) v[q] = *at;
#pragma unroll
    for (int q = 0; q < 16; ++q) part += v[q];
    sum += part;
  }
  float part = 0.0f;
#pragma unroll 8
  for (int q = 0; q < left; ++q, at += 8 * pitch) part += *at;
  return sum + part;
}

// The launch's device must be the calling thread's current one: the pointers belong to it.
#define NB2_REQUIRE_DEVICE(ordinal)                                                     \
  do {                                                                                  \
    int dev__ = -1;                                                                     \
    NB2_CUDA(cudaGetDevice(&dev__));                                                    \
    NB2_REQUIRE(dev__ == (ordinal), "the plan's device is not the current CUDA device"); \
  } while (0)

#define NB2_SEQ_DTYPE(dtype, ...)                       \
  do {                                                  \
    if ((dtype) == NB2_F32) {                           \
      using T = float;                                  \
      __VA_ARGS__;                                      \
    } else if ((dtype) == NB2_F16) {                    \
      using T = __half;                                 \
      __VA_ARGS__;                                      \
    } else {                                            \
      using T = __nv_bfloat16;                          \
      __VA_ARGS__;                                      \
    }                                                   \
  } while (0)
