// Backward pass of the residual norm.
#include "nb2_seq_norm.cuh"

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
        float mine[2] = {ss[0], ss[1]};
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float v = u[i][e];
          if constexpr (GATE == kGateLast) v *= gv[e] * s[i][e];
          r[i][e] = fmaf(w[e], v, rv[e]);
          mine[0] = fmaf(r[i][e], r[i][e], mine[0]);
          mine[1] = fmaf(dh[e] * wn[e], r[i][e], mine[1]);
        }
        // (past the row's end: 0 times an infinite 1 / sqrt(0 + eps), weight or scale, left out of the sums)
        if (tid + i * step < vecs) ss[0] = mine[0], ss[1] = mine[1];
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
        float hat = u[i][e];
        if constexpr (GATE == kGateLast) hat *= gv[e] * s[i][e];
        add(0, i, e, dr[e] * hat);
        r[i][e] = dr[e] * w[e];  // q (without the late gate) from here on
        part[i] = fmaf(r[i][e], hat, part[i]);
      }
      if (tid + i * step >= vecs) part[i] = 0.0f;
      if (dresidual && tid + i * step < vecs) {
        o.put(dr);
        o.store(dresidual + i * step * V);
      }
    }
    if (normed) norm_reduce<NV>(part, kind, vecs, a.groups, group_sums);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float mean = part[i] * inv_group;
      SeqVecA<T, V> xv, gv, o;
      float ox[V], og[V];
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
          og[e] = du * u[i][e] * slope;
          du *= sg;
        }
        if (normed) du = inv[i] * fmaf(-u[i][e], mean, du);
        if constexpr (GATE == kGateFirst) {
          og[e] = du * xv[e] * slope;
          du *= sg;
        }
        ox[e] = du;
      }
      if (tid + i * step >= vecs) continue;
      o.put(ox);
      o.store(dx + i * step * V);
      if constexpr (GATE != kNoGate)
        if (dgate) {
          o.put(og);
          o.store(dgate + i * step * V);
        }
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
  run[w][lane] = i < n ? nb2_sum_units(a.part + i, n, a.n_units, w) : 0.0f;
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
