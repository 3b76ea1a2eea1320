// Short causal convolution along the rows of sequences, one filter per channel (depthwise), and its
// backward pass:
//   pre[t] = bias + sum_j w[j] x[t - W + 1 + j],   y = pre or pre sigmoid(pre)
//   dpre = dy * act'(pre),  dx[p] = sum_j w[j] dpre[p + W - 1 - j],  dw[j] = sum_t dpre[t] x[t - W + 1 + j]
// Rows before the first one come from the state, which is also a sequence's last W - 1 rows.
#include "nb2_sequence.cuh"

#define CONV_THREADS 128

struct ConvPlace {
  int64_t start, stride;
};
__device__ __forceinline__ ConvPlace conv_place(const int64_t* table, int n_seq, int array, int k) {
  return {table[(size_t)(1 + 2 * array) * n_seq + k], table[(size_t)(2 + 2 * array) * n_seq + k]};
}

template <int V, int W>
__device__ __forceinline__ void conv_weights(const float* w, const float* bias, int c, float (&wr)[W][V], float (&b)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < W; ++j) wr[j][v] = w[(size_t)(c + v) * W + j];
    b[v] = bias ? bias[c + v] : 0.0f;
  }
}

// The thread's V channels of row p of a sequence: the state's rows stand before row 0 (zeros without one).
template <typename T, int V, int W>
__device__ __forceinline__ void conv_row(SeqVecA<T, V>& r, const T* x, int64_t xs, const T* state, int64_t ss, int64_t p) {
  if (p >= 0)
    r.load(x + p * xs);
  else if (state)
    r.load(state + (p + W - 1) * ss);
  else
    r.zero();
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(CONV_THREADS) nb2_causal_conv_kernel(const nb2_causal_conv_args a, int tiles) {
  nb2_pdl_enter();
  const int unit = blockIdx.x / tiles;
  const int c = ((blockIdx.x - unit * tiles) * CONV_THREADS + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int k = a.units[2 * unit];
  const int64_t t0 = a.units[2 * unit + 1], len = a.table[k];
  const int64_t t1 = min(t0 + a.unit_rows, len);
  const ConvPlace px = conv_place(a.table, a.n_seq, 0, k), py = conv_place(a.table, a.n_seq, 1, k);
  const T* x = (const T*)a.x + px.start + c;
  T* y = (T*)a.y + py.start + c;
  const T* state = nullptr;
  int64_t ss = 0;
  if (a.state) {
    const ConvPlace p = conv_place(a.table, a.n_seq, 2, k);
    state = (const T*)a.state + p.start + c;
    ss = p.stride;
  }
  float w[W][V], b[V];
  conv_weights<V, W>(a.w, a.bias, c, w, b);
  float win[W][V];  // rows t - W + 1 .. t
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    SeqVecA<T, V> r;
    conv_row<T, V, W>(r, x, px.stride, state, ss, t0 - (W - 1) + j);
#pragma unroll
    for (int v = 0; v < V; ++v) win[j + 1][v] = r[v];
  }
  for (int64_t t = t0; t < t1; ++t) {
    SeqVecA<T, V> r, o;
    r.load(x + t * px.stride);
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) win[j][v] = win[j + 1][v];
      win[W - 1][v] = r[v];
      float s = b[v];
#pragma unroll
      for (int j = 0; j < W; ++j) s = fmaf(w[j][v], win[j][v], s);
      o.e[v] = nb2_from_float<T>(a.silu ? s * nb2_sigmoid(s) : s);
    }
    o.store(y + t * py.stride);
  }
  // The unit that read the old state writes the new one (so that the two may be the same rows): its
  // threads have read what they overwrite, and later rows of the old state are read before they are.
  if (a.new_state && t0 == 0) {
    const ConvPlace p = conv_place(a.table, a.n_seq, 3, k);
    T* out = (T*)a.new_state + p.start + c;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      SeqVecA<T, V> r;
      conv_row<T, V, W>(r, x, px.stride, state, ss, len - (W - 1) + j);
      r.store(out + j * p.stride);
    }
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(CONV_THREADS) nb2_causal_conv_grad_kernel(const nb2_causal_conv_grad_args a, int tiles) {
  nb2_pdl_enter();
  const int unit = blockIdx.x / tiles;
  const int c = ((blockIdx.x - unit * tiles) * CONV_THREADS + threadIdx.x) * V;
  if (c >= a.channels) return;
  const int k = a.units[2 * unit];
  const int64_t t0 = a.units[2 * unit + 1], len = a.table[k];
  const int64_t t1 = min(t0 + a.unit_rows, len);
  const ConvPlace px = conv_place(a.table, a.n_seq, 0, k), pdy = conv_place(a.table, a.n_seq, 1, k),
                  pdx = conv_place(a.table, a.n_seq, 2, k);
  const T* x = (const T*)a.x + px.start + c;
  const T* dy = (const T*)a.dy + pdy.start + c;
  T* dx = (T*)a.dx + pdx.start + c;
  const T *state = nullptr, *dnew = nullptr;
  T* dstate = nullptr;
  int64_t ss = 0, ds = 0, ns = 0;
  if (a.state) {
    const ConvPlace p = conv_place(a.table, a.n_seq, 3, k);
    state = (const T*)a.state + p.start + c, ss = p.stride;
  }
  if (a.dstate) {
    const ConvPlace p = conv_place(a.table, a.n_seq, 4, k);
    dstate = (T*)a.dstate + p.start + c, ds = p.stride;
  }
  if (a.dnew_state) {
    const ConvPlace p = conv_place(a.table, a.n_seq, 5, k);
    dnew = (const T*)a.dnew_state + p.start + c, ns = p.stride;
  }
  float w[W][V], b[V], dw[W][V], db[V];
  conv_weights<V, W>(a.w, a.bias, c, w, b);
  float xw[W][V], gw[W][V];  // x and dpre of rows t - W + 1 .. t
#pragma unroll
  for (int j = 0; j < W; ++j) {
    SeqVecA<T, V> r;
    r.zero();
    if (j < W - 1) conv_row<T, V, W>(r, x, px.stride, state, ss, t0 - (W - 1) + j);
#pragma unroll
    for (int v = 0; v < V; ++v) dw[j][v] = 0.0f, gw[j][v] = 0.0f, xw[(j + 1) % W][v] = r[v];
  }
#pragma unroll
  for (int v = 0; v < V; ++v) db[v] = 0.0f;
  // The gradient of row p needs dpre of rows p .. p + W - 1, so the walk goes W - 1 rows past the unit;
  // the first unit also emits the W - 1 rows before the sequence, the state's gradient.
  for (int64_t t = t0; t < t1 + W - 1; ++t) {
    SeqVecA<T, V> rx, rg;
    rx.zero();
    rg.zero();
    const bool in = t < len;
    if (in) {
      rx.load(x + t * px.stride);
      rg.load(dy + t * pdy.stride);
    }
    const bool own = t < t1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) xw[j][v] = xw[j + 1][v], gw[j][v] = gw[j + 1][v];
      xw[W - 1][v] = rx[v];
      float g = 0.0f;
      if (in) {
        g = rg[v];
        if (a.silu) {
          float s = b[v];
#pragma unroll
          for (int j = 0; j < W; ++j) s = fmaf(w[j][v], xw[j][v], s);
          g *= nb2_silu_slope(s);
        }
        if (own) {
          db[v] += g;
#pragma unroll
          for (int j = 0; j < W; ++j) dw[j][v] = fmaf(g, xw[j][v], dw[j][v]);
        }
      }
      gw[W - 1][v] = g;
    }
    const int64_t p = t - (W - 1);
    if (p < t0 && !(t0 == 0 && dstate)) continue;
    SeqVecA<T, V> add, o;
    add.zero();
    if (dnew && p >= len - (W - 1)) add.load(dnew + (p - len + (W - 1)) * ns);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = add[v];
#pragma unroll
      for (int j = 0; j < W; ++j) s = fmaf(w[W - 1 - j][v], gw[j][v], s);
      o.e[v] = nb2_from_float<T>(s);
    }
    if (p >= 0)
      o.store(dx + p * pdx.stride);
    else
      o.store(dstate + (p + W - 1) * ds);
  }
  float* part = a.part + (size_t)unit * (W + 1) * a.channels + c;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int j = 0; j < W; ++j) part[(size_t)j * a.channels + v] = dw[j][v];
    part[(size_t)W * a.channels + v] = db[v];
  }
}

// Sums of the units' partial parameter gradients, units in order within eight interleaved runs:
// the same result every time.  A block owns 32 columns of [taps + 1][channels].
__global__ void __launch_bounds__(256) nb2_conv_grad_sum_kernel(const float* part, int n_units, int taps, int channels,
                                                                float* dw, float* dbias) {
  nb2_pdl_enter();
  __shared__ float run[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t n = (int64_t)(taps + 1) * channels, i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (i < n)
    for (int u = w; u < n_units; u += 8) s += part[(int64_t)u * n + i];
  run[w][lane] = s;
  __syncthreads();
  if (w == 0 && i < n) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; ++r) sum += run[r][lane];
    const int j = (int)(i / channels), c = (int)(i - (int64_t)j * channels);
    if (j < taps)
      dw[(size_t)c * taps + j] = sum;
    else if (dbias)
      dbias[c] = sum;
  }
}

// Every block of a grid-stride loop owns 32 columns: eight interleaved runs over the parts, then their sum.
__global__ void __launch_bounds__(256) nb2_seq_sum_parts_kernel(const float* part, int64_t n_parts, int64_t n, float* out) {
  nb2_pdl_enter();
  __shared__ float run[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int64_t b = blockIdx.x; b * 32 < n; b += gridDim.x) {
    const int64_t i = b * 32 + lane;
    float s = 0.0f;
    if (i < n)
      for (int64_t u = w; u < n_parts; u += 8) s += part[u * n + i];
    run[w][lane] = s;
    __syncthreads();
    if (w == 0 && i < n) {
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 8; ++r) sum += run[r][lane];
      out[i] = sum;
    }
    __syncthreads();
  }
}

cudaError_t nb2_seq_sum_parts(cudaStream_t s, const float* part, int64_t n_parts, int64_t n, float* out) {
  const int64_t blocks = (n + 31) / 32;
  return nb2_launch(nb2_seq_sum_parts_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, part,
                    n_parts, n, out);
}

template <typename T, int V>
static cudaError_t conv_launch(cudaStream_t s, const nb2_causal_conv_args& a) {
  const int tiles = (a.channels + V * CONV_THREADS - 1) / (V * CONV_THREADS);
  const dim3 grid((unsigned)a.n_units * tiles), block(CONV_THREADS);
#define NB2_CASE(W) \
  case W: return nb2_launch(nb2_causal_conv_kernel<T, V, W>, grid, block, 0, s, a, tiles)
  switch (a.taps) {
    NB2_CASE(1); NB2_CASE(2); NB2_CASE(3); NB2_CASE(4); NB2_CASE(5); NB2_CASE(6); NB2_CASE(7);
    default: return nb2_launch(nb2_causal_conv_kernel<T, V, 8>, grid, block, 0, s, a, tiles);
  }
#undef NB2_CASE
}

template <typename T, int V>
static cudaError_t conv_grad_launch(cudaStream_t s, const nb2_causal_conv_grad_args& a) {
  const int tiles = (a.channels + V * CONV_THREADS - 1) / (V * CONV_THREADS);
  const dim3 grid((unsigned)a.n_units * tiles), block(CONV_THREADS);
#define NB2_CASE(W) \
  case W: return nb2_launch(nb2_causal_conv_grad_kernel<T, V, W>, grid, block, 0, s, a, tiles)
  switch (a.taps) {
    NB2_CASE(1); NB2_CASE(2); NB2_CASE(3); NB2_CASE(4); NB2_CASE(5); NB2_CASE(6); NB2_CASE(7);
    default: return nb2_launch(nb2_causal_conv_grad_kernel<T, V, 8>, grid, block, 0, s, a, tiles);
  }
#undef NB2_CASE
}

template <typename A>
static int conv_check(const A& a) {
  NB2_REQUIRE(a.table && a.units && a.x && a.w, "null pointer");
  NB2_REQUIRE(a.dtype >= NB2_F32 && a.dtype <= NB2_BF16, "dtype");
  NB2_REQUIRE(a.n_seq >= 1 && a.n_units >= a.n_seq && a.channels >= 1, "shape");
  NB2_REQUIRE(a.taps >= 1 && a.taps <= NB2_CONV_MAX_TAPS && a.unit_rows >= 1 && a.unit_rows >= a.taps - 1, "taps");
  NB2_REQUIRE((int64_t)a.n_units * ((a.channels + CONV_THREADS - 1) / CONV_THREADS) < (1ll << 31), "too many units");
  NB2_REQUIRE_DEVICE(a.device);
  return NB2_OK;
}

extern "C" int nb2_causal_conv(void* stream, const nb2_causal_conv_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_causal_conv_args& a = *args;
  if (int e = conv_check(a)) return e;
  NB2_REQUIRE(a.y, "null pointer");
  NB2_SEQ_DTYPE(a.dtype, if (a.vec) NB2_CUDA((conv_launch<T, 16 / sizeof(T)>(nb2_stream(stream), a)));
                else NB2_CUDA((conv_launch<T, 1>(nb2_stream(stream), a))));
  return NB2_OK;
}

extern "C" int nb2_causal_conv_grad(void* stream, const nb2_causal_conv_grad_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_causal_conv_grad_args& a = *args;
  if (int e = conv_check(a)) return e;
  NB2_REQUIRE(a.dy && a.dx && a.dw && a.part, "null pointer");
  NB2_SEQ_DTYPE(a.dtype, if (a.vec) NB2_CUDA((conv_grad_launch<T, 16 / sizeof(T)>(nb2_stream(stream), a)));
                else NB2_CUDA((conv_grad_launch<T, 1>(nb2_stream(stream), a))));
  const int64_t n = (int64_t)(a.taps + 1) * a.channels;
  NB2_CUDA(nb2_launch(nb2_conv_grad_sum_kernel, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, nb2_stream(stream), a.part,
                      a.n_units, a.taps, a.channels, a.dw, a.dbias));
  return NB2_OK;
}
