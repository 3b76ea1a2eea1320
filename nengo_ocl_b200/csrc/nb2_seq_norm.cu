// The norms around a block with its gate and residual scale, row by row:
//   u = x silu(gate);  v = u rsqrt(mean over the group of u^2 + eps) weight;  y = residual + scale v;
//   h = y rsqrt(mean(y^2) + eps) norm_weight
// (the gate before or after the first norm, every part optional), and the backward pass.  A block holds
// a whole row in registers, NV vectors of V channels to a thread, so each array is read or written once.
#include "nb2_sequence.cuh"

struct NormPlace {
  int64_t start, stride;
};
__device__ __forceinline__ NormPlace norm_place(const int64_t* table, int n_seq, int array, int k) {
  return {table[(size_t)(1 + 2 * array) * n_seq + k], table[(size_t)(2 + 2 * array) * n_seq + k]};
}

// Sum over the block, the same on every thread.  scratch: 33 floats, free again after the next barrier.
__device__ __forceinline__ float norm_block_sum(float v, float* scratch) {
#pragma unroll
  for (int w = 16; w >= 1; w /= 2) v += __shfl_xor_sync(0xffffffffu, v, w);
  if (blockDim.x == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = (threadIdx.x & 31) < blockDim.x / 32 ? scratch[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int w = 16; w >= 1; w /= 2) s += __shfl_xor_sync(0xffffffffu, s, w);
  return s;
}

// Per vector i of the thread: the sum of part[i] over the vectors of its group.  groups == 1: one block
// sum.  Else every vector's share goes to shared memory and a warp adds up each group in order.
template <int NV>
__device__ __forceinline__ void norm_group_sums(float (&part)[NV], int vecs, int groups, float* scratch, float* shares) {
  if (groups == 1) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += part[i];
    s = norm_block_sum(s, scratch);
#pragma unroll
    for (int i = 0; i < NV; ++i) part[i] = s;
    return;
  }
  const int per = vecs / groups;
  float* sums = shares + vecs;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < vecs) shares[v] = part[i];
  }
  __syncthreads();
  for (int g = threadIdx.x >> 5; g < groups; g += blockDim.x >> 5) {
    float s = 0.0f;
    for (int i = threadIdx.x & 31; i < per; i += 32) s += shares[g * per + i];
#pragma unroll
    for (int w = 16; w >= 1; w /= 2) s += __shfl_xor_sync(0xffffffffu, s, w);
    if ((threadIdx.x & 31) == 0) sums[g] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    part[i] = v < vecs ? sums[v / per] : 0.0f;
  }
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(1024) nb2_residual_norm_kernel(const nb2_residual_norm_args a) {
  extern __shared__ float shares[];
  __shared__ float scratch[32];
  nb2_pdl_enter();
  const int k = a.units[2 * blockIdx.x];
  const int64_t t0 = a.units[2 * blockIdx.x + 1], t1 = min(t0 + a.unit_rows, a.table[k]);
  const int vecs = a.channels / V;
  const float inv_group = (float)a.groups / (float)a.channels, inv_row = 1.0f / (float)a.channels;
  const NormPlace px = norm_place(a.table, a.n_seq, 0, k), py = norm_place(a.table, a.n_seq, 1, k),
                  ph = norm_place(a.table, a.n_seq, 2, k), pg = norm_place(a.table, a.n_seq, 3, k),
                  pr = norm_place(a.table, a.n_seq, 4, k);
  for (int64_t t = t0; t < t1; ++t) {
    const T* x = (const T*)a.x + px.start + t * px.stride;
    const T* gate = (const T*)a.gate + pg.start + t * pg.stride;
    const T* residual = (const T*)a.residual + pr.start + t * pr.stride;
    SeqVecA<T, V> gv[NV];
    float u[NV][V], part[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      SeqVecA<T, V> r;
      r.zero();
      gv[i].zero();
      if (v < vecs) {
        r.load(x + v * V);
        if (a.gate) gv[i].load(gate + v * V);
      }
      part[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u[i][e] = r[e];
        if (a.gate && a.gate_first) u[i][e] *= gv[i][e] * nb2_sigmoid(gv[i][e]);
        part[i] = fmaf(u[i][e], u[i][e], part[i]);
      }
    }
    if (a.weight) norm_group_sums<NV>(part, vecs, a.groups, scratch, shares);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= vecs) continue;
      const float inv = rsqrtf(fmaf(part[i], inv_group, a.eps));
      SeqVecA<T, V> r;
      r.zero();
      if (a.residual) r.load(residual + v * V);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float o = u[i][e];
        if (a.weight) o *= inv * a.weight[v * V + e];
        if (a.gate && !a.gate_first) o *= gv[i][e] * nb2_sigmoid(gv[i][e]);
        u[i][e] = fmaf(a.scale ? a.scale[v * V + e] : a.scale_value, o, r[e]);
        ss = fmaf(u[i][e], u[i][e], ss);
      }
      if (a.y) {
        SeqVecA<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.e[e] = nb2_from_float<T>(u[i][e]);
        o.store((T*)a.y + py.start + t * py.stride + v * V);
      }
    }
    if (a.h) {
      const float inv = rsqrtf(fmaf(norm_block_sum(ss, scratch), inv_row, a.eps));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= vecs) continue;
        SeqVecA<T, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e)
          o.e[e] = nb2_from_float<T>(u[i][e] * inv * (a.norm_weight ? a.norm_weight[v * V + e] : 1.0f));
        o.store((T*)a.h + ph.start + t * ph.stride + v * V);
      }
    }
  }
}

// Backward, with ^ marking normed values, r the row's y, o the block's output before the residual:
//   dr = dy + inv_r (dh w_n - r^ mean(dh w_n r^)),  do = scale dr,  du = inv_u (dv w - u^ mean over the group(dv w u^))
// where dv = do (times silu(gate) when the gate comes after), and the gate's product rule around it.
// Parameter gradients are summed over the unit's rows in registers and left per unit in `part`.
template <typename T, int V, int NV>
__global__ void __launch_bounds__(V == 1 || NV > 2 ? 1024 : 512) nb2_residual_norm_grad_kernel(const nb2_residual_norm_grad_args a) {
  extern __shared__ float shares[];
  __shared__ float scratch[32];
  nb2_pdl_enter();
  const int k = a.units[2 * blockIdx.x];
  const int64_t t0 = a.units[2 * blockIdx.x + 1], t1 = min(t0 + a.unit_rows, a.table[k]);
  const int vecs = a.channels / V;
  const float inv_group = (float)a.groups / (float)a.channels, inv_row = 1.0f / (float)a.channels;
  const NormPlace px = norm_place(a.table, a.n_seq, 0, k), pg = norm_place(a.table, a.n_seq, 1, k),
                  pr = norm_place(a.table, a.n_seq, 2, k), pdy = norm_place(a.table, a.n_seq, 3, k),
                  pdh = norm_place(a.table, a.n_seq, 4, k), pdx = norm_place(a.table, a.n_seq, 5, k),
                  pdg = norm_place(a.table, a.n_seq, 6, k), pdr = norm_place(a.table, a.n_seq, 7, k);
  float dw[NV][V], dsc[NV][V], dn[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = dsc[i][e] = dn[i][e] = 0.0f;
  for (int64_t t = t0; t < t1; ++t) {
    const T* x = (const T*)a.x + px.start + t * px.stride;
    const T* gate = (const T*)a.gate + pg.start + t * pg.stride;
    SeqVecA<T, V> xv[NV], gv[NV];
    float part[NV], r[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      xv[i].zero();
      gv[i].zero();
      if (v < vecs) {
        xv[i].load(x + v * V);
        if (a.gate) gv[i].load(gate + v * V);
      }
      part[i] = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float u = xv[i][e];
        if (a.gate && a.gate_first) u *= gv[i][e] * nb2_sigmoid(gv[i][e]);
        part[i] = fmaf(u, u, part[i]);
      }
    }
    if (a.weight) norm_group_sums<NV>(part, vecs, a.groups, scratch, shares);
    float inv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) inv[i] = a.weight ? rsqrtf(fmaf(part[i], inv_group, a.eps)) : 1.0f;
    // r: first the row's y, from here on dr
    float rinv = 0.0f, proj = 0.0f;
    if (a.dh) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= vecs) continue;
        SeqVecA<T, V> res;
        res.zero();
        if (a.residual) res.load((const T*)a.residual + pr.start + t * pr.stride + v * V);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float o = xv[i][e];
          if (a.gate && a.gate_first) o *= gv[i][e] * nb2_sigmoid(gv[i][e]);
          if (a.weight) o *= inv[i] * a.weight[v * V + e];
          if (a.gate && !a.gate_first) o *= gv[i][e] * nb2_sigmoid(gv[i][e]);
          r[i][e] = fmaf(a.scale ? a.scale[v * V + e] : a.scale_value, o, res[e]);
          ss = fmaf(r[i][e], r[i][e], ss);
        }
      }
      rinv = rsqrtf(fmaf(norm_block_sum(ss, scratch), inv_row, a.eps));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v >= vecs) continue;
        SeqVecA<T, V> dh;
        dh.load((const T*)a.dh + pdh.start + t * pdh.stride + v * V);
#pragma unroll
        for (int e = 0; e < V; ++e)
          proj = fmaf(dh[e] * (a.norm_weight ? a.norm_weight[v * V + e] : 1.0f), r[i][e] * rinv, proj);
      }
      proj = norm_block_sum(proj, scratch) * inv_row;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      part[i] = 0.0f;
      if (v >= vecs) continue;
      SeqVecA<T, V> dy, dh, o;
      dy.zero();
      dh.zero();
      if (a.dy) dy.load((const T*)a.dy + pdy.start + t * pdy.stride + v * V);
      if (a.dh) dh.load((const T*)a.dh + pdh.start + t * pdh.stride + v * V);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float dr = dy[e];
        if (a.dh) {
          const float hat = r[i][e] * rinv;
          dn[i][e] = fmaf(dh[e], hat, dn[i][e]);
          dr = fmaf(rinv, fmaf(dh[e], a.norm_weight ? a.norm_weight[v * V + e] : 1.0f, -hat * proj), dr);
        }
        r[i][e] = dr;
        o.e[e] = nb2_from_float<T>(dr);
        const float sg = a.gate ? gv[i][e] * nb2_sigmoid(gv[i][e]) : 1.0f;
        const float u = xv[i][e] * (a.gate_first ? sg : 1.0f), hat = u * inv[i];
        const float w = a.weight ? a.weight[v * V + e] : 1.0f, late = a.gate_first ? 1.0f : sg;
        dsc[i][e] = fmaf(dr, hat * w * late, dsc[i][e]);
        const float dv = dr * (a.scale ? a.scale[v * V + e] : a.scale_value) * late;
        dw[i][e] = fmaf(dv, hat, dw[i][e]);
        part[i] = fmaf(dv * w, hat, part[i]);
      }
      if (a.dresidual) o.store((T*)a.dresidual + pdr.start + t * pdr.stride + v * V);
    }
    if (a.weight) norm_group_sums<NV>(part, vecs, a.groups, scratch, shares);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v >= vecs) continue;
      SeqVecA<T, V> ox, og;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = gv[i][e], sg = a.gate ? g * nb2_sigmoid(g) : 1.0f;
        const float u = xv[i][e] * (a.gate_first ? sg : 1.0f);
        const float w = a.weight ? a.weight[v * V + e] : 1.0f, late = a.gate_first ? 1.0f : sg;
        const float dlast = r[i][e] * (a.scale ? a.scale[v * V + e] : a.scale_value), dv = dlast * late;
        float du = dv;
        if (a.weight) du = inv[i] * fmaf(dv, w, -u * inv[i] * part[i] * inv_group);
        ox.e[e] = nb2_from_float<T>(du * (a.gate_first ? sg : 1.0f));
        og.e[e] = nb2_from_float<T>(a.gate ? (a.gate_first ? du * xv[i][e] : dlast * u * inv[i] * w) * nb2_silu_slope(g) : 0.0f);
      }
      ox.store((T*)a.dx + pdx.start + t * pdx.stride + v * V);
      if (a.dgate) og.store((T*)a.dgate + pdg.start + t * pdg.stride + v * V);
    }
  }
  float* out = a.part + (size_t)blockIdx.x * 3 * a.channels;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v >= vecs) continue;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      out[v * V + e] = dw[i][e];
      out[a.channels + v * V + e] = dsc[i][e];
      out[2 * a.channels + v * V + e] = dn[i][e];
    }
  }
}

// Sums of the units' partial parameter gradients in order, eight interleaved runs (as the convolution's).
__global__ void __launch_bounds__(256) nb2_norm_grad_sum_kernel(const float* part, int n_units, int channels, float* dw,
                                                                float* dscale, float* dnorm) {
  nb2_pdl_enter();
  __shared__ float run[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = 3ll * channels, i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (i < n)
    for (int u = w; u < n_units; u += 8) s += part[(int64_t)u * n + i];
  run[w][lane] = s;
  __syncthreads();
  if (w == 0 && i < n) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; ++r) sum += run[r][lane];
    const int which = (int)(i / channels), c = (int)(i - (int64_t)which * channels);
    float* out = which == 0 ? dw : which == 1 ? dscale : dnorm;
    if (out) out[c] = sum;
  }
}

// Threads and vectors a thread that hold a row of `vecs` vectors: two vectors to a thread while the
// block has room.
struct NormShape {
  int threads, nv;
};
static NormShape norm_shape(int vecs, int max_threads) {
  int threads = 32;
  while (threads < max_threads && threads * 2 < vecs) threads *= 2;
  int nv = 1;
  while (nv * threads < vecs) nv *= 2;
  return {threads, nv};
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
static cudaError_t norm_launch(K kernel, cudaStream_t s, const A& a, int threads, int vecs) {
  const size_t smem = a.groups > 1 ? (size_t)(vecs + a.groups) * sizeof(float) : 0;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return nb2_launch(kernel, dim3(a.n_units), dim3(threads), smem, s, a);
}

template <typename T, int V>
static cudaError_t norm_dispatch(cudaStream_t s, const nb2_residual_norm_args& a) {
  const int vecs = a.channels / V;
  const NormShape n = norm_shape(vecs, 1024);
  if constexpr (V == 1) {
    if (n.nv > 8) return norm_launch(nb2_residual_norm_kernel<T, V, 32>, s, a, n.threads, vecs);
  }
  if (n.nv > 4) return norm_launch(nb2_residual_norm_kernel<T, V, 8>, s, a, n.threads, vecs);
  if (n.nv > 2) return norm_launch(nb2_residual_norm_kernel<T, V, 4>, s, a, n.threads, vecs);
  return norm_launch(nb2_residual_norm_kernel<T, V, 2>, s, a, n.threads, vecs);
}

template <typename T, int V>
static cudaError_t norm_dispatch(cudaStream_t s, const nb2_residual_norm_grad_args& a) {
  const int vecs = a.channels / V;
  NormShape n = norm_shape(vecs, 512);
  if (n.nv > 2) n = norm_shape(vecs, 1024);
  if constexpr (V == 1) {
    if (n.nv > 8) return norm_launch(nb2_residual_norm_grad_kernel<T, V, 32>, s, a, n.threads, vecs);
  }
  if (n.nv > 4) return norm_launch(nb2_residual_norm_grad_kernel<T, V, 8>, s, a, n.threads, vecs);
  if (n.nv > 2) return norm_launch(nb2_residual_norm_grad_kernel<T, V, 4>, s, a, n.threads, vecs);
  return norm_launch(nb2_residual_norm_grad_kernel<T, V, 2>, s, a, n.threads, vecs);
}

extern "C" int nb2_residual_norm(void* stream, const nb2_residual_norm_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_residual_norm_args& a = *args;
  if (int e = norm_check(a)) return e;
  NB2_REQUIRE(a.y || a.h, "no output");
  NB2_SEQ_DTYPE(a.dtype, if (a.vec) NB2_CUDA((norm_dispatch<T, 16 / sizeof(T)>(nb2_stream(stream), a)));
                else NB2_CUDA((norm_dispatch<T, 1>(nb2_stream(stream), a))));
  return NB2_OK;
}

extern "C" int nb2_residual_norm_grad(void* stream, const nb2_residual_norm_grad_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_residual_norm_grad_args& a = *args;
  if (int e = norm_check(a)) return e;
  NB2_REQUIRE(a.dx && a.part && (a.dy || a.dh), "null pointer");
  NB2_REQUIRE((!a.dgate || a.gate) && (!a.dweight || a.weight) && (!a.dscale || a.scale) && (!a.dnorm_weight || a.dh),
              "gradients");
  NB2_SEQ_DTYPE(a.dtype, if (a.vec) NB2_CUDA((norm_dispatch<T, 16 / sizeof(T)>(nb2_stream(stream), a)));
                else NB2_CUDA((norm_dispatch<T, 1>(nb2_stream(stream), a))));
  if (a.dweight || a.dscale || a.dnorm_weight)
    NB2_CUDA(nb2_launch(nb2_norm_grad_sum_kernel, dim3((unsigned)((3ll * a.channels + 31) / 32)), dim3(256), 0,
                        nb2_stream(stream), a.part, a.n_units, a.channels, a.dweight, a.dscale, a.dnorm_weight));
  return NB2_OK;
}
