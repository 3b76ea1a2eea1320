// The norms around a block with its gate and residual scale, row by row:
//   u = x silu(gate);  v = u rsqrt(mean over the group of u^2 + eps) weight;  y = residual + scale v;
//   h = y rsqrt(mean(y^2) + eps) norm_weight
// (the gate before or after the first norm, every part optional), and the backward pass.  Bound by memory: a
// block holds a whole row in registers, NV vectors of V channels to a thread, so each array is read or
// written once, and all of a row's loads are in flight before its first sum is needed.
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

template <typename T, int V, int NV, int GATE>
__global__ void __launch_bounds__(NormThreads<NV>::kMost, NV == 1 ? 2 : 1) nb2_residual_norm_kernel(const nb2_residual_norm_args a, int kind) {
  extern __shared__ __align__(16) float shared[];
  float* sums = shared;
  nb2_pdl_wait();
  const int k = a.units[2 * blockIdx.x];
  const int64_t t0 = a.units[2 * blockIdx.x + 1];
  const int rows = (int)(min(t0 + a.unit_rows, a.table[k]) - t0);
  const int vecs = a.channels / V, tid = threadIdx.x, step = blockDim.x;
  const float inv_group = (float)a.groups / (float)a.channels, inv_row = 1.0f / (float)a.channels;
  NormRows<T, V, NV, 3> in;  // x, gate, residual
  in.vecs = vecs;
  in.smem = reinterpret_cast<char*>(sums);
  {
    const void* const base[3] = {a.x, GATE != kNoGate ? a.gate : nullptr, a.residual};
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const NormPlace p = norm_place(a.table, a.n_seq, q == 0 ? 0 : q + 2, k);
      in.from[q] = base[q] ? (const T*)base[q] + p.start + t0 * p.stride : nullptr;
      in.stride[q] = p.stride;
    }
  }
  in.begin(rows);
  sums += in.bytes(vecs) / sizeof(float);
  const NormPlace py = norm_place(a.table, a.n_seq, 1, k), ph = norm_place(a.table, a.n_seq, 2, k);
  T* y = a.y ? (T*)a.y + py.start + t0 * py.stride + tid * V : nullptr;
  T* h = a.h ? (T*)a.h + ph.start + t0 * ph.stride + tid * V : nullptr;
  const NormParams<V, NV> scaled(a.weight, a.scale, a.scale_value, a.param_vec, vecs),
      norm_weight(a.norm_weight, nullptr, 1.0f, a.param_vec, vecs);
  const bool normed = a.weight != nullptr;
  float* row_sums = sums + norm_buffer(kind, vecs, a.groups);
  for (int t = 0; t < rows; ++t) {
    in.ahead(t + in.kDepth - 1, rows);
    in.wait();
    float u[NV][V], part[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      SeqVecA<T, V> xv, gv;
      in.get(0, i, t, xv);
      if constexpr (GATE == kGateFirst) in.get(1, i, t, gv);
      part[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[i][e] = xv[e];
        if constexpr (GATE == kGateFirst) u[i][e] *= gv[e] * nb2_sigmoid(gv[e]);
        part[i] = fmaf(u[i][e], u[i][e], part[i]);
      }
    }
    if (normed) norm_reduce<NV>(part, kind, vecs, a.groups, sums);
    float ss[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float inv = normed ? rsqrtf(fmaf(part[i], inv_group, a.eps)) : 1.0f;
      float w[V];
      scaled.get(i, w);
      SeqVecA<T, V> rv, gv, o;
      in.get(2, i, t, rv);
      if constexpr (GATE == kGateLast) in.get(1, i, t, gv);
      ss[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = u[i][e] * inv;
        if constexpr (GATE == kGateLast) v *= gv[e] * nb2_sigmoid(gv[e]);
        u[i][e] = fmaf(w[e], v, rv[e]);  // (zeros past the row's end)
        o.e[e] = nb2_from_float<T>(u[i][e]);
        ss[i] = fmaf(u[i][e], u[i][e], ss[i]);
      }
      if (y && tid + i * step < vecs) o.store(y + i * step * V);
    }
    if (h) {
      norm_reduce<NV>(ss, kNormWarps, vecs, 1, row_sums + (t & 1) * 32);
      const float inv = rsqrtf(fmaf(ss[0], inv_row, a.eps));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float w[V];
        norm_weight.get(i, w);
        SeqVecA<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.e[e] = nb2_from_float<T>(u[i][e] * inv * w[e]);
        if (tid + i * step < vecs) o.store(h + i * step * V);
      }
      h += ph.stride;
    } else if (normed) {
      __syncthreads();  // (the buffer's next use)
    }
    if (y) y += py.stride;
  }
}

// Backward, with ^ marking normed values, r the row's y, q = dr scale weight:
//   dr = dy + inv_r (dh w_n - r^ mean(dh w_n r^)),  du = inv_u (q - u^ mean over the group(q u^))
// with q times silu(gate) when the gate comes after, and the gate's product rule around it.  The gradients of
// weight and scale are one sum S = sum over rows of dr u^ (silu(gate)) times scale and weight.  S and the
// gradient of norm_weight are summed over the unit's rows, in registers while they fit (kInRegisters), else in
// the unit's own rows of `part` in memory.
template <typename T, int V, int NV, int GATE>
__global__ void __launch_bounds__(NormThreads<NV>::kMost, 1) nb2_residual_norm_grad_kernel(const nb2_residual_norm_grad_args a, int kind) {
  constexpr bool kInRegisters = NV * V <= 16;
  extern __shared__ __align__(16) float shared[];
  float* sums = shared;
  nb2_pdl_wait();
  const int k = a.units[2 * blockIdx.x];
  const int64_t t0 = a.units[2 * blockIdx.x + 1];
  const int rows = (int)(min(t0 + a.unit_rows, a.table[k]) - t0);
  const int vecs = a.channels / V, tid = threadIdx.x, step = blockDim.x;
  const float inv_group = (float)a.groups / (float)a.channels, inv_row = 1.0f / (float)a.channels;
  NormRows<T, V, NV, 5> in;  // x, gate, residual, dy, dh
  in.vecs = vecs;
  in.smem = reinterpret_cast<char*>(sums);
  {
    const void* const base[5] = {a.x, GATE != kNoGate ? a.gate : nullptr, a.dh ? a.residual : nullptr, a.dy, a.dh};
#pragma unroll
    for (int q = 0; q < 5; ++q) {
      const NormPlace p = norm_place(a.table, a.n_seq, q, k);
      in.from[q] = base[q] ? (const T*)base[q] + p.start + t0 * p.stride : nullptr;
      in.stride[q] = p.stride;
    }
  }
  in.begin(rows);
  sums += in.bytes(vecs) / sizeof(float);
  const NormPlace pdx = norm_place(a.table, a.n_seq, 5, k), pdg = norm_place(a.table, a.n_seq, 6, k),
                  pdr = norm_place(a.table, a.n_seq, 7, k);
  T* dx = (T*)a.dx + pdx.start + t0 * pdx.stride + tid * V;
  T* dgate = GATE != kNoGate && a.dgate ? (T*)a.dgate + pdg.start + t0 * pdg.stride + tid * V : nullptr;
  T* dresidual = a.dresidual ? (T*)a.dresidual + pdr.start + t0 * pdr.stride + tid * V : nullptr;
  // of q u^ (the shares' sum begins with a barrier: one buffer does), then of r^2 and dh w_n r
  float* group_sums = kind == kNormShares ? sums : sums + norm_buffer(kind, vecs, a.groups);
  float* row_sums = sums + norm_buffers(kind, vecs, a.groups);
  const NormParams<V, NV> scaled(a.weight, a.scale, a.scale_value, a.param_vec, vecs),
      norm_weight(a.norm_weight, nullptr, 1.0f, a.param_vec, vecs);
  const bool normed = a.weight != nullptr, heads = a.dh != nullptr;
  float* part_of = a.part + (size_t)blockIdx.x * 2 * a.channels;
  float acc[2][kInRegisters ? NV : 1][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (kInRegisters) {
        acc[0][i][e] = acc[1][i][e] = 0.0f;
      } else {
        const int c = (tid + i * step) * V + e;
        if (c < a.channels) part_of[c] = part_of[a.channels + c] = 0.0f;
      }
    }
  auto add = [&](int which, int i, int e, float value) {
    if constexpr (kInRegisters)
      acc[which][i][e] += value;
    else if (tid + i * step < vecs)
      part_of[(size_t)which * a.channels + (tid + i * step) * V + e] += value;
  };
  for (int t = 0; t < rows; ++t) {
    in.ahead(t + in.kDepth - 1, rows);
    in.wait();
    float part[NV], u[NV][V], r[NV][V], s[NV][V], inv[NV];  // s: sigmoid(gate)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      SeqVecA<T, V> xv, gv;
      in.get(0, i, t, xv);
      if constexpr (GATE != kNoGate) in.get(1, i, t, gv);
      part[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[i][e] = xv[e];
        if constexpr (GATE != kNoGate) s[i][e] = nb2_sigmoid(gv[e]);
        if constexpr (GATE == kGateFirst) u[i][e] *= gv[e] * s[i][e];
        part[i] = fmaf(u[i][e], u[i][e], part[i]);
      }
    }
    if (normed) norm_reduce<NV>(part, kind, vecs, a.groups, sums);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      inv[i] = normed ? rsqrtf(fmaf(part[i], inv_group, a.eps)) : 1.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) u[i][e] *= inv[i];  // u^ from here on
    }
    float rinv = 0.0f, proj = 0.0f;
    if (heads) {
      float ss[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        float w[V], wn[V];
        scaled.get(i, w);
        norm_weight.get(i, wn);
        SeqVecA<T, V> gv, rv, dh;
        if constexpr (GATE == kGateLast) in.get(1, i, t, gv);
        in.get(2, i, t, rv);
        in.get(4, i, t, dh);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float v = u[i][e];
          if constexpr (GATE == kGateLast) v *= gv[e] * s[i][e];
          r[i][e] = fmaf(w[e], v, rv[e]);  // (zeros past the row's end)
          ss[0] = fmaf(r[i][e], r[i][e], ss[0]);
          ss[1] = fmaf(dh[e] * wn[e], r[i][e], ss[1]);
        }
      }
      // both sums with one barrier
#pragma unroll
      for (int w = 16; w >= 1; w /= 2) {
        ss[0] += __shfl_xor_sync(0xffffffffu, ss[0], w);
        ss[1] += __shfl_xor_sync(0xffffffffu, ss[1], w);
      }
      float2* buf = reinterpret_cast<float2*>(row_sums) + (t & 1) * 32;
      const int lane = tid & 31;
      if (lane == 0) buf[tid >> 5] = make_float2(ss[0], ss[1]);
      __syncthreads();
      const float2 of = lane < step / 32 ? buf[lane] : make_float2(0.0f, 0.0f);
      ss[0] = of.x, ss[1] = of.y;
#pragma unroll
      for (int w = 16; w >= 1; w /= 2) {
        ss[0] += __shfl_xor_sync(0xffffffffu, ss[0], w);
        ss[1] += __shfl_xor_sync(0xffffffffu, ss[1], w);
      }
      rinv = rsqrtf(fmaf(ss[0], inv_row, a.eps));
      proj = ss[1] * rinv * inv_row;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float w[V], wn[V];
      scaled.get(i, w);
      SeqVecA<T, V> gv, dy, dh, o;
      if constexpr (GATE == kGateLast) in.get(1, i, t, gv);
      in.get(3, i, t, dy);
      float dr[V];
#pragma unroll
      for (int e = 0; e < V; ++e) dr[e] = dy[e];
      if (heads) {
        norm_weight.get(i, wn);
        in.get(4, i, t, dh);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float hat = r[i][e] * rinv;
          add(1, i, e, dh[e] * hat);
          dr[e] = fmaf(rinv, fmaf(dh[e], wn[e], -hat * proj), dr[e]);
        }
      }
      part[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        o.e[e] = nb2_from_float<T>(dr[e]);
        float hat = u[i][e];
        if constexpr (GATE == kGateLast) hat *= gv[e] * s[i][e];
        add(0, i, e, dr[e] * hat);
        r[i][e] = dr[e] * w[e];  // q (without the late gate) from here on
        part[i] = fmaf(r[i][e], hat, part[i]);
      }
      if (dresidual && tid + i * step < vecs) o.store(dresidual + i * step * V);
    }
    if (normed) norm_reduce<NV>(part, kind, vecs, a.groups, group_sums);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float mean = part[i] * inv_group;
      SeqVecA<T, V> xv, gv, ox, og;
      if constexpr (GATE == kGateFirst) in.get(0, i, t, xv);
      if constexpr (GATE != kNoGate) in.get(1, i, t, gv);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float sg = 1.0f, slope = 0.0f, du = r[i][e];
        if constexpr (GATE != kNoGate) {
          sg = gv[e] * s[i][e];
          slope = fmaf(sg, 1.0f - s[i][e], s[i][e]);  // of g sigmoid(g)
        }
        if constexpr (GATE == kGateLast) {
          og.e[e] = nb2_from_float<T>(du * u[i][e] * slope);
          du *= sg;
        }
        if (normed) du = inv[i] * fmaf(-u[i][e], mean, du);
        if constexpr (GATE == kGateFirst) {
          og.e[e] = nb2_from_float<T>(du * xv[e] * slope);
          du *= sg;
        }
        ox.e[e] = nb2_from_float<T>(du);
      }
      if (tid + i * step >= vecs) continue;
      ox.store(dx + i * step * V);
      if constexpr (GATE != kNoGate)
        if (dgate) og.store(dgate + i * step * V);
    }
    if (normed && !heads) __syncthreads();  // (the buffers' next use)
    dx += pdx.stride;
    if (dgate) dgate += pdg.stride;
    if (dresidual) dresidual += pdr.stride;
  }
  if constexpr (kInRegisters)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (tid + i * step >= vecs) continue;
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < V; ++e) part_of[(size_t)q * a.channels + (tid + i * step) * V + e] = acc[q][i][e];
    }
}

// Parameter gradients from the units' partial sums, units in order within eight interleaved runs (as the
// convolution's): the same result every time.  A block owns 32 columns of [2][channels].
__global__ void __launch_bounds__(256) nb2_norm_grad_sum_kernel(const nb2_residual_norm_grad_args a) {
  nb2_pdl_enter();
  __shared__ float run[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = 2ll * a.channels, i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (i < n)
    for (int u = w; u < a.n_units; u += 8) s += a.part[(int64_t)u * n + i];
  run[w][lane] = s;
  __syncthreads();
  if (w == 0 && i < n) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; ++r) sum += run[r][lane];
    if (i < a.channels) {
      if (a.dweight) a.dweight[i] = sum * (a.scale ? a.scale[i] : a.scale_value);
      if (a.dscale) a.dscale[i] = sum * (a.weight ? a.weight[i] : 1.0f);
    } else if (a.dnorm_weight) {
      a.dnorm_weight[i - a.channels] = sum;
    }
  }
}

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

template <typename T, int V, int GATE>
static cudaError_t norm_dispatch(cudaStream_t s, const nb2_residual_norm_args& a) {
  constexpr int buffers = 1, arrays = 3;
  NORM_BY_VECTORS(nb2_residual_norm_kernel);
}
template <typename T, int V, int GATE>
static cudaError_t norm_dispatch(cudaStream_t s, const nb2_residual_norm_grad_args& a) {
  constexpr int buffers = 2, arrays = 5;
  NORM_BY_VECTORS(nb2_residual_norm_grad_kernel);
}
template <typename T, int V, typename A>
static cudaError_t norm_by_gate(cudaStream_t s, const A& a) {
  if (!a.gate) return norm_dispatch<T, V, kNoGate>(s, a);
  return a.gate_first ? norm_dispatch<T, V, kGateFirst>(s, a) : norm_dispatch<T, V, kGateLast>(s, a);
}

extern "C" int nb2_residual_norm(void* stream, const nb2_residual_norm_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_residual_norm_args& a = *args;
  if (int e = norm_check(a)) return e;
  NB2_REQUIRE(a.y || a.h, "no output");
  NB2_SEQ_DTYPE(a.dtype, if (a.vec) NB2_CUDA((norm_by_gate<T, 16 / sizeof(T)>(nb2_stream(stream), a)));
                else NB2_CUDA((norm_by_gate<T, 1>(nb2_stream(stream), a))));
  return NB2_OK;
}

extern "C" int nb2_residual_norm_grad(void* stream, const nb2_residual_norm_grad_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_residual_norm_grad_args& a = *args;
  if (int e = norm_check(a)) return e;
  NB2_REQUIRE(a.dx && a.part && (a.dy || a.dh), "null pointer");
  NB2_REQUIRE((!a.dgate || a.gate) && (!a.dweight || a.weight) && (!a.dscale || a.scale) && (!a.dnorm_weight || a.dh),
              "gradients");
  NB2_SEQ_DTYPE(a.dtype, if (a.vec) NB2_CUDA((norm_by_gate<T, 16 / sizeof(T)>(nb2_stream(stream), a)));
                else NB2_CUDA((norm_by_gate<T, 1>(nb2_stream(stream), a))));
  if (a.dweight || a.dscale || a.dnorm_weight)
    NB2_CUDA(nb2_launch(nb2_norm_grad_sum_kernel, dim3((unsigned)((2ll * a.channels + 31) / 32)), dim3(256), 0,
                        nb2_stream(stream), a));
  return NB2_OK;
}
