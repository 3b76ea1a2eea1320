// The norms around a block with its gate and residual scale, row by row:
//   u = x silu(gate);  v = u rsqrt(mean over the group of u^2 + eps) weight;  y = residual + scale v;
//   h = y rsqrt(mean(y^2) + eps) norm_weight
// (the gate before or after the first norm, every part optional), and the backward pass.  Bound by memory: a
// block holds a whole row in registers, NV vectors of V channels to a thread, so each array is read or
// written once, and all of a row's loads are in flight before its first sum is needed.  Measured (B200, bfloat16): 8192 rows
// x 4096, all parts, 70 us = 4.8 TB/s, 0.73 of the copy rate (without the copies ahead 110); backward 87 us for 4096
// rows, 3.0 TB/s: its sums hold a block of 512 threads a multiprocessor, whose four phases a row do not overlap.
#pragma once
#include "nb2_sequence.cuh"

struct NormPlace {
  int64_t start, stride;
};
__device__ __forceinline__ NormPlace norm_place(const int64_t* table, int n_seq, int array, int k) {
  return {table[(size_t)(1 + 2 * array) * n_seq + k], table[(size_t)(2 + 2 * array) * n_seq + k]};
}

// ---- sums over the row, or over groups of its channels -------------------------------------------------
// Vector v of a row (V neighbouring channels) sits with thread v % blockDim, so a warp holds 32 neighbours.
enum NormSums {
  kNormWarps,   // whole row, or groups of whole warps' vectors: a shuffle sum per warp, then the group's warps
  kNormLanes,   // groups of 1, 2, .. 16 vectors: shuffles alone
  kNormShares,  // anything else: every vector's share through shared memory
};
static int norm_sums(int vecs, int groups) {
  const int per = vecs / groups;
  if (groups == 1 || per % 32 == 0) return kNormWarps;
  return 32 % per == 0 ? kNormLanes : kNormShares;
}
// floats of one buffer
__host__ __device__ inline int norm_buffer(int kind, int vecs, int groups) {
  return kind == kNormWarps ? (vecs + 31) / 32 : kind == kNormLanes ? 0 : vecs + groups;
}

// floats of the backward pass's two, an even number
__host__ __device__ inline int norm_buffers(int kind, int vecs, int groups) {
  const int one = norm_buffer(kind, vecs, groups);
  return kind == kNormShares ? (one + 1) / 2 * 2 : 2 * one;
}

// part[i] becomes the sum over the group of vector threadIdx.x + i blockDim.x.  One barrier (kNormShares: three):
// the caller alternates buffers so that a buffer is not written again before the next barrier.
template <int NV>
__device__ __forceinline__ void norm_reduce(float (&part)[NV], int kind, int vecs, int groups, float* buf) {
  const int lane = threadIdx.x & 31;
  if (kind == kNormLanes) {
    const int per = vecs / groups;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      for (int w = 1; w < per; w *= 2) part[i] += __shfl_xor_sync(0xffffffffu, part[i], w);
    return;
  }
  if (groups == 1) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += part[i];
#pragma unroll
    for (int w = 16; w >= 1; w /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    if (lane == 0) buf[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = lane < (int)blockDim.x / 32 ? buf[lane] : 0.0f;
#pragma unroll
    for (int w = 16; w >= 1; w /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
#pragma unroll
    for (int i = 0; i < NV; ++i) part[i] = sum;
    return;
  }
  if (kind == kNormWarps) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int w = 16; w >= 1; w /= 2) part[i] += __shfl_xor_sync(0xffffffffu, part[i], w);
      const int v = threadIdx.x + i * blockDim.x;
      if (lane == 0 && v < vecs) buf[v >> 5] = part[i];
    }
    __syncthreads();
    const int per = vecs / groups / 32;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = min(threadIdx.x + i * (int)blockDim.x, vecs - 1), first = v / (per * 32) * per;
      part[i] = 0.0f;
      for (int q = 0; q < per; ++q) part[i] += buf[first + q];
    }
    return;
  }
  const int per = vecs / groups;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < vecs) buf[v] = part[i];
  }
  __syncthreads();
  for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
    float s = 0.0f;
    for (int i = lane; i < per; i += 32) s += buf[g * per + i];
#pragma unroll
    for (int w = 16; w >= 1; w /= 2) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (lane == 0) buf[vecs + g] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    part[i] = v < vecs ? buf[vecs + v / per] : 0.0f;
  }
}

// V parameters from channel c on; ones (or another value) without an array
template <int V>
__device__ __forceinline__ void norm_params(const float* p, int c, int vec, float otherwise, float (&out)[V]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = otherwise;
  } else if (V % 4 == 0 && vec) {
#pragma unroll
    for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(out + e) = __ldg(reinterpret_cast<const float4*>(p + c + e));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = __ldg(p + c + e);
  }
}

// Parameters of the thread's channels (the product of two, if there are two): in registers for all rows of a unit
// where they fit, else loaded (from L1) with every use.
template <int V, int NV>
struct NormParams {
  static constexpr bool kHeld = NV * V <= 8;
  float held[kHeld ? NV : 1][V];
  const float *p, *q;
  int vec, last;
  float otherwise;  // in q's place
  __device__ __forceinline__ NormParams(const float* p, const float* q, float otherwise, int vec, int vecs)
      : p(p), q(q), vec(vec), last(vecs - 1), otherwise(otherwise) {
    if constexpr (kHeld)
#pragma unroll
      for (int i = 0; i < NV; ++i) load(i, held[i]);
  }
  __device__ __forceinline__ void load(int i, float (&out)[V]) const {
    const int c = min(threadIdx.x + i * (int)blockDim.x, last) * V;
    float more[V];
    norm_params<V>(p, c, vec, 1.0f, out);
    norm_params<V>(q, c, vec, otherwise, more);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] *= more[e];
  }
  __device__ __forceinline__ void get(int i, float (&out)[V]) const {
    if constexpr (kHeld) {
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = held[i][e];
    } else {
      load(i, out);
    }
  }
};

template <int NV>
struct NormThreads {
  static constexpr int kMost = NV <= 2 ? 512 : 1024;
};

// The rows of N arrays on their way to a block.  Rows of 16-byte vectors that fit (kAsync) are copied to shared
// memory kDepth - 1 rows ahead; a thread copies and reads its own vectors only, so no barrier is needed, and
// nothing is held in registers meanwhile.  Others are loaded where they are used.
template <typename T, int V, int NV, int N>
struct NormRows {
  static constexpr bool kAsync = V * sizeof(T) == 16 && NV <= 2;
  static constexpr int kDepth = N == 5 && NV == 2 ? 2 : 3;  // (N x 16 KB a row at most)
  const T* from[N];
  int64_t stride[N];
  int vecs;
  char* smem;
  __host__ __device__ static int bytes(int vecs) { return kAsync ? kDepth * N * vecs * 16 : 0; }
  __device__ __forceinline__ void ahead(int t, int rows) const {
    if constexpr (kAsync) {
      if (t < rows)
#pragma unroll
        for (int q = 0; q < N; ++q)
          if (from[q])
#pragma unroll
            for (int i = 0; i < NV; ++i) {
              const int v = threadIdx.x + i * blockDim.x;
              if (v < vecs) {
                const unsigned to = (unsigned)__cvta_generic_to_shared(smem + ((t % kDepth * N + q) * vecs + v) * 16);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from[q] + t * stride[q] + v * V) : "memory");
              }
            }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  }
  __device__ __forceinline__ void begin(int rows) const {
#pragma unroll
    for (int t = 0; t < kDepth - 1; ++t) ahead(t, rows);
  }
  // row t is there (after the call that asks for row t + kDepth - 1)
  __device__ __forceinline__ void wait() const {
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
  }
  __device__ __forceinline__ void get(int q, int i, int t, SeqVecA<T, V>& out) const {
    const int v = threadIdx.x + i * blockDim.x;
    if (!from[q] || v >= vecs)
      out.zero();
    else if constexpr (kAsync)
      out.load(reinterpret_cast<const T*>(smem + ((t % kDepth * N + q) * vecs + v) * 16));
    else
      out.load(from[q] + t * stride[q] + v * V);
  }
};

enum NormGate { kNoGate, kGateFirst, kGateLast };

// One or two vectors to a thread up to 512 threads, then as many as 1024 threads need.
static int norm_vectors(int vecs) {
  if (vecs <= 1024) return vecs <= 512 ? 1 : 2;
  int nv = 4;
  while (nv * 1024 < vecs) nv *= 2;
  return nv;
}

template <typename A>
static int norm_check(const A& a) {
  NB2_REQUIRE(a.table && a.units && a.x, "null pointer");
  NB2_REQUIRE(a.dtype >= NB2_F32 && a.dtype <= NB2_BF16, "dtype");
  NB2_REQUIRE(a.n_seq >= 1 && a.n_units >= 1 && a.unit_rows >= 1, "shape");
  NB2_REQUIRE(a.channels >= 1 && a.channels <= NB2_NORM_MAX_CHANNELS && a.groups >= 1 && a.channels % a.groups == 0,
              "channels / groups");
  const int V = a.dtype == NB2_F32 ? 4 : 8;
  NB2_REQUIRE(!a.vec || (a.channels / a.groups) % V == 0, "vec");
  NB2_REQUIRE_DEVICE(a.device);
  return NB2_OK;
}

template <typename K, typename A>
static cudaError_t norm_launch(K kernel, cudaStream_t s, const A& a, int vecs, int nv, int buffers, int ahead) {
  const int kind = norm_sums(vecs, a.groups), threads = ((vecs + nv - 1) / nv + 31) / 32 * 32;
  // `buffers` of the groups' sums and two of the row's, two values from each of up to 32 warps
  const int group = buffers == 2 ? norm_buffers(kind, vecs, a.groups) : norm_buffer(kind, vecs, a.groups);
  const size_t smem = (size_t)(group + 128) * sizeof(float) + ahead;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return nb2_launch(kernel, dim3(a.n_units), dim3(threads), smem, s, a, kind);
}

#define NORM_CASE(kernel, n) \
  return norm_launch(kernel<T, V, n, GATE>, s, a, vecs, n, buffers, NormRows<T, V, n, arrays>::bytes(vecs))
// (V == 1, rows that do not allow 16-byte accesses: fewer variants)
#define NORM_BY_VECTORS(kernel)                             \
  const int vecs = a.channels / V, nv = norm_vectors(vecs); \
  if constexpr (V == 1) {                                   \
    if (nv > 4) NORM_CASE(kernel, 32);                      \
  }                                                         \
  if constexpr (V == 4) {                                   \
    if (nv > 4) NORM_CASE(kernel, 8);                       \
  }                                                         \
  if (nv > 2) NORM_CASE(kernel, 4);                         \
  if constexpr (V > 1) {                                    \
    if (nv > 1) NORM_CASE(kernel, 2);                       \
  } else {                                                  \
    if (nv > 1) NORM_CASE(kernel, 4);                       \
  }                                                         \
  NORM_CASE(kernel, 1)
