// Forward pass of the residual norm.
#include "nb2_seq_norm.cuh"

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
        u[i][e] = fmaf(w[e], v, rv[e]);
        ss[i] = fmaf(u[i][e], u[i][e], ss[i]);
      }
      // (past the row's end: 0 times an infinite 1 / sqrt(0 + eps), weight or scale, left out of the sum)
      if (tid + i * step >= vecs) ss[i] = 0.0f;
      if (y && tid + i * step < vecs) {
        o.put(u[i]);
        o.store(y + i * step * V);
      }
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
        for (int e = 0; e < V; ++e) w[e] *= u[i][e] * inv;
        o.put(w);
        if (tid + i * step < vecs) o.store(h + i * step * V);
      }
      h += ph.stride;
    } else if (normed) {
      __syncthreads();  // (the buffer's next use)
    }
    if (y) y += py.stride;
  }
}

template <typename T, int V, int GATE>
static cudaError_t norm_dispatch(cudaStream_t s, const nb2_residual_norm_args& a) {
  constexpr int buffers = 1, arrays = 3;
  NORM_BY_VECTORS(nb2_residual_norm_kernel);
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
