// Short causal convolution along the rows of sequences, one filter per channel (depthwise), and its
// backward pass:
//   pre[t] = bias + sum_j w[j] x[t - W + 1 + j],   y = pre or pre sigmoid(pre)
//   dpre = dy * act'(pre),  dx[p] = sum_j w[j] dpre[p + W - 1 - j],  dw[j] = sum_t dpre[t] x[t - W + 1 + j]
// Rows before the first one come from the state, which is also a sequence's last W - 1 rows.
//
// Memory would allow 20 us for 8192 rows x 4096 channels in bfloat16; the kernel takes 40: with 4 taps and the silu a value
// is 30 instructions (counted; 0.72 of the issue slots), and the window and weights of four channels leave 24 warps to a multiprocessor (float32: 20).  Eight
// channels to a thread 47 us, weights read from memory by each thread 54, one row at a time 81.
#include "nb2_sequence.cuh"

#define CONV_THREADS 128

struct ConvPlace {
  int64_t start, stride;
};
__device__ __forceinline__ ConvPlace conv_place(const int64_t* table, int n_seq, int array, int k) {
  return {table[(size_t)(1 + 2 * array) * n_seq + k], table[(size_t)(2 + 2 * array) * n_seq + k]};
}

// The weights of a block's channels lie together in memory, V W of them to a thread: read in a row by all
// threads and handed out through shared memory (an odd pitch keeps a warp's reads in different banks).
template <int V, int W>
struct ConvWeights {
  static constexpr int kEach = V * W, kPitch = kEach | 1, kFloats = CONV_THREADS * kPitch;
  static __device__ __forceinline__ void stage(float* smem, const float* w, int c0, int channels) {
    const int n = min(CONV_THREADS * V, channels - c0) * W;
    const float* from = w + (size_t)c0 * W;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += CONV_THREADS) smem[i / kEach * kPitch + i % kEach] = from[i];
  }
  static __device__ __forceinline__ void get(const float* smem, const float* bias, int c, float (&wr)[W][V], float (&b)[V]) {
    const float* mine = smem + threadIdx.x * kPitch;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int j = 0; j < W; ++j) wr[j][v] = mine[v * W + j];
      b[v] = bias ? bias[c + v] : 0.0f;
    }
  }
};

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

// The thread's V channels of the rows to come, kRows at a time: copied to shared memory while the ones
// before them are worked on (a thread copies and reads its own channels only: no barrier).  Single elements, and a
// unit of one group, are loaded straight into registers.
template <typename T, int V, int kRows, int N>
struct ConvRows {
  static constexpr int kBytes = V * (int)sizeof(T), kAhead = 2;
  static constexpr bool kAsync = kBytes == 16 || kBytes == 8;
  const T* from[N];
  int64_t stride[N];
  int64_t end;  // rows from here on are zeros
  bool async;
  char* smem;
  __host__ __device__ static constexpr int bytes() { return kAsync ? kAhead * kRows * N * CONV_THREADS * kBytes : 0; }
  __device__ __forceinline__ char* slot(int group, int i, int q) const {
    return smem + (((group % kAhead * kRows + i) * N + q) * CONV_THREADS + threadIdx.x) * kBytes;
  }
  __device__ __forceinline__ void ahead(int64_t t, int64_t stop, int group) const {
    if constexpr (kAsync)
      if (async) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (t + i < stop)
#pragma unroll
            for (int q = 0; q < N; ++q) {
              const unsigned to = (unsigned)__cvta_generic_to_shared(slot(group, i, q));
              const T* row = from[q] + (t + i) * stride[q];
              if constexpr (kBytes == 16)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(row) : "memory");
              else
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(row) : "memory");
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
  }
  __device__ __forceinline__ void begin(int64_t t, int64_t stop) {
    end = stop;
    async = kAsync && stop - t > kRows;
#pragma unroll
    for (int g = 0; g < kAhead - 1; ++g) ahead(t + g * kRows, stop, g);
  }
  // group of rows t .. t + kRows - 1
  __device__ __forceinline__ void get(int64_t t, int group, SeqVecA<T, V> (&r)[N][kRows]) const {
    ahead(t + (kAhead - 1) * kRows, end, group + kAhead - 1);
    if constexpr (kAsync)
      if (async) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int q = 0; q < N; ++q) {
        if (t + i >= end)
          r[q][i].zero();
        else if (kAsync && async)
          r[q][i].load(reinterpret_cast<const T*>(slot(group, i, q)));
        else
          r[q][i].load(from[q] + (t + i) * stride[q]);
      }
  }
};

template <typename T, int V, int W, bool SILU>
__global__ void __launch_bounds__(CONV_THREADS) nb2_causal_conv_kernel(const nb2_causal_conv_args a, int tiles) {
  nb2_pdl_enter();
  extern __shared__ __align__(16) char smem[];
  const int unit = blockIdx.x / tiles;
  const int c0 = (blockIdx.x - unit * tiles) * CONV_THREADS * V, c = c0 + threadIdx.x * V;
  float* weights = reinterpret_cast<float*>(smem + ConvRows<T, V, 8, 1>::bytes());
  ConvWeights<V, W>::stage(weights, a.w, c0, a.channels);
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
  constexpr int kRows = 8;
  ConvRows<T, V, kRows, 1> in;
  in.smem = smem;
  in.from[0] = x;
  in.stride[0] = px.stride;
  if (c < a.channels) in.begin(t0, t1);
  __syncthreads();
  if (c >= a.channels) return;
  float w[W][V], b[V];
  ConvWeights<V, W>::get(weights, a.bias, c, w, b);
  float win[W][V];  // rows t - W + 1 .. t
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    SeqVecA<T, V> r;
    conv_row<T, V, W>(r, x, px.stride, state, ss, t0 - (W - 1) + j);
#pragma unroll
    for (int v = 0; v < V; ++v) win[j + 1][v] = r[v];
  }
  int group = 0;
  for (int64_t tb = t0; tb < t1; tb += kRows, ++group) {
    const int rows = (int)min((int64_t)kRows, t1 - tb);
    SeqVecA<T, V> r[1][kRows];
    in.get(tb, group, r);
    // (no way out of this loop: the window then moves by renaming registers)
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float out[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) win[j][v] = win[j + 1][v];
        win[W - 1][v] = r[0][i][v];
        float s = b[v];
#pragma unroll
        for (int j = 0; j < W; ++j) s = fmaf(w[j][v], win[j][v], s);
        out[v] = s;
      }
      if (SILU)
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] *= nb2_sigmoid(out[v]);
      SeqVecA<T, V> o;
      o.put(out);
      if (i < rows) o.store(y + (tb + i) * py.stride);
    }
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

template <typename T, int V, int W, bool SILU>
__global__ void __launch_bounds__(CONV_THREADS) nb2_causal_conv_grad_kernel(const nb2_causal_conv_grad_args a, int tiles) {
  nb2_pdl_enter();
  extern __shared__ __align__(16) char smem[];
  const int unit = blockIdx.x / tiles;
  const int c0 = (blockIdx.x - unit * tiles) * CONV_THREADS * V, c = c0 + threadIdx.x * V;
  float* weights = reinterpret_cast<float*>(smem + ConvRows<T, V, 4, 2>::bytes());
  ConvWeights<V, W>::stage(weights, a.w, c0, a.channels);
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
  constexpr int kRows = 4;
  ConvRows<T, V, kRows, 2> in;
  in.smem = smem;
  in.from[0] = x, in.from[1] = dy;
  in.stride[0] = px.stride, in.stride[1] = pdy.stride;
  if (c < a.channels) in.begin(t0, min(t1 + W - 1, len));
  __syncthreads();
  if (c >= a.channels) return;
  float w[W][V], b[V], dw[W][V], db[V];
  ConvWeights<V, W>::get(weights, a.bias, c, w, b);
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
  int group = 0;
  for (int64_t tb = t0; tb < t1 + W - 1; tb += kRows, ++group) {
    SeqVecA<T, V> r[2][kRows];
    in.get(tb, group, r);
    float group_w[W][V], group_b[V];  // (the group's rows apart, then the groups: shorter chains of additions)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      group_b[v] = 0.0f;
#pragma unroll
      for (int j = 0; j < W; ++j) group_w[j][v] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t t = tb + i, p = t - (W - 1);
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) xw[j][v] = xw[j + 1][v], gw[j][v] = gw[j + 1][v];
        xw[W - 1][v] = r[0][i][v];
        float g = r[1][i][v];
        if (SILU) {
          float s = b[v];
#pragma unroll
          for (int j = 0; j < W; ++j) s = fmaf(w[j][v], xw[j][v], s);
          g *= nb2_silu_slope(s);
        }
        gw[W - 1][v] = t < len ? g : 0.0f;
      }
      if (t < t1)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          group_b[v] += gw[W - 1][v];
#pragma unroll
          for (int j = 0; j < W; ++j) group_w[j][v] = fmaf(gw[W - 1][v], xw[j][v], group_w[j][v]);
        }
      float out[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        out[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) out[v] = fmaf(w[W - 1 - j][v], gw[j][v], out[v]);
      }
      SeqVecA<T, V> o;
      if (dnew && p >= len - (W - 1) && p < t1) {
        o.load(dnew + (p - len + (W - 1)) * ns);
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] += o[v];
      }
      o.put(out);
      if (p >= t0 && p < t1)
        o.store(dx + p * pdx.stride);
      else if (t0 == 0 && p < 0 && dstate)
        o.store(dstate + (p + W - 1) * ds);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      db[v] += group_b[v];
#pragma unroll
      for (int j = 0; j < W; ++j) dw[j][v] += group_w[j][v];
    }
  }
  float* part = a.part + (size_t)unit * (W + 1) * a.channels + c;
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    SeqVecA<float, V> o;
    o.put(j < W ? dw[j < W ? j : 0] : db);
    o.store(part + (size_t)j * a.channels);
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
  run[w][lane] = i < n ? nb2_sum_units(part + i, n, n_units, w) : 0.0f;
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

template <typename K, typename A>
static cudaError_t conv_run(K kernel, dim3 grid, int smem, cudaStream_t s, const A& a, int tiles) {
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  return nb2_launch(kernel, grid, dim3(CONV_THREADS), smem, s, a, tiles);
}

template <typename T, int V, bool SILU>
static cudaError_t conv_launch(cudaStream_t s, const nb2_causal_conv_args& a) {
  const int tiles = (a.channels + V * CONV_THREADS - 1) / (V * CONV_THREADS);
  const dim3 grid((unsigned)a.n_units * tiles);
#define NB2_CASE(W) \
  case W: return conv_run(nb2_causal_conv_kernel<T, V, W, SILU>, grid, ConvRows<T, V, 8, 1>::bytes() + 4 * ConvWeights<V, W>::kFloats, s, a, tiles)
  switch (a.taps) {
    NB2_CASE(1); NB2_CASE(2); NB2_CASE(3); NB2_CASE(4); NB2_CASE(5); NB2_CASE(6); NB2_CASE(7);
    default: return conv_run(nb2_causal_conv_kernel<T, V, 8, SILU>, grid, ConvRows<T, V, 8, 1>::bytes() + 4 * ConvWeights<V, 8>::kFloats, s, a, tiles);
  }
#undef NB2_CASE
}

template <typename T, int V, bool SILU>
static cudaError_t conv_grad_launch(cudaStream_t s, const nb2_causal_conv_grad_args& a) {
  const int tiles = (a.channels + V * CONV_THREADS - 1) / (V * CONV_THREADS);
  const dim3 grid((unsigned)a.n_units * tiles);
#define NB2_CASE(W) \
  case W: return conv_run(nb2_causal_conv_grad_kernel<T, V, W, SILU>, grid, ConvRows<T, V, 4, 2>::bytes() + 4 * ConvWeights<V, W>::kFloats, s, a, tiles)
  switch (a.taps) {
    NB2_CASE(1); NB2_CASE(2); NB2_CASE(3); NB2_CASE(4); NB2_CASE(5); NB2_CASE(6); NB2_CASE(7);
    default: return conv_run(nb2_causal_conv_grad_kernel<T, V, 8, SILU>, grid, ConvRows<T, V, 4, 2>::bytes() + 4 * ConvWeights<V, 8>::kFloats, s, a, tiles);
  }
#undef NB2_CASE
}

// Four channels to a thread whatever the type: the windows, the weights and (backward) their sums fill the registers.
template <typename T>
static cudaError_t conv_dispatch(cudaStream_t s, const nb2_causal_conv_args& a) {
  if (a.vec) return a.silu ? conv_launch<T, 4, true>(s, a) : conv_launch<T, 4, false>(s, a);
  return a.silu ? conv_launch<T, 1, true>(s, a) : conv_launch<T, 1, false>(s, a);
}
template <typename T>
static cudaError_t conv_dispatch(cudaStream_t s, const nb2_causal_conv_grad_args& a) {
  if (a.vec) return a.silu ? conv_grad_launch<T, 4, true>(s, a) : conv_grad_launch<T, 4, false>(s, a);
  return a.silu ? conv_grad_launch<T, 1, true>(s, a) : conv_grad_launch<T, 1, false>(s, a);
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
  NB2_SEQ_DTYPE(a.dtype, NB2_CUDA(conv_dispatch<T>(nb2_stream(stream), a)));
  return NB2_OK;
}

extern "C" int nb2_causal_conv_grad(void* stream, const nb2_causal_conv_grad_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_causal_conv_grad_args& a = *args;
  if (int e = conv_check(a)) return e;
  NB2_REQUIRE(a.dy && a.dx && a.dw && a.part, "null pointer");
  NB2_SEQ_DTYPE(a.dtype, NB2_CUDA(conv_dispatch<T>(nb2_stream(stream), a)));
  const int64_t n = (int64_t)(a.taps + 1) * a.channels;
  NB2_CUDA(nb2_launch(nb2_conv_grad_sum_kernel, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, nb2_stream(stream), a.part,
                      a.n_units, a.taps, a.channels, a.dw, a.dbias));
  return NB2_OK;
}
