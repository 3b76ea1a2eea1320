// Selective state space scan along the rows of sequences: the linear filter whose step size, input
// and output weights depend on the row.  Per channel c with states n (B, C shared by a group of channels):
//   s = softplus(dt + dt_bias),  a[n] = exp(s A[n]),  h[n] = a[n] h[n] + s x B[n],
//   y = (sum_n C[n] h[n] + D x) silu(z)
//
// Four states to a lane, S = 1 .. 32 lanes to a channel (S = the power of two that covers the states),
// so a warp carries 32 / S channels and walks the rows S at a time: lane j of a channel prepares row
// t + j (step size, scaled input, gate) and hands it to the others by shuffles; the S partial sums over
// the states that every lane forms are then transposed and added in S - 1 shuffles, which leaves row
// t + j's output with lane j.
#include "nb2_sequence.cuh"

#define SCAN_WARPS 4
#define SCAN_THREADS (32 * SCAN_WARPS)
#define LOG2E 1.4426950408889634f

template <int S>
struct ScanTile {
  static constexpr int kChannels = 32 / S;                // of a warp
  static constexpr int kBlock = kChannels * SCAN_WARPS;   // of a block
};

static int scan_lanes(int n_states) {
  int s = 1;
  while (4 * s < n_states) s *= 2;
  return s;
}

struct ScanPlace {
  int64_t start, stride;
};
__device__ __forceinline__ ScanPlace scan_place(const int64_t* table, int n_seq, int array, int k) {
  return {table[(size_t)(1 + 2 * array) * n_seq + k], table[(size_t)(2 + 2 * array) * n_seq + k]};
}

__device__ __forceinline__ float scan_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// log(1 + e^v); above 20 the difference to v is less than half a step of v
__device__ __forceinline__ float scan_softplus(float v) { return v > 20.0f ? v : log1pf(__expf(v)); }

// The lane's four states of a row (n0 .. n0 + 3 of n), zeros past the last one.
template <typename T>
__device__ __forceinline__ void scan_load4(const T* p, int n0, int n, int vec, float (&out)[4]) {
  if (vec && n0 + 4 <= n) {
    SeqVecA<T, 4> r;
    r.load(p + n0);
#pragma unroll
    for (int m = 0; m < 4; ++m) out[m] = r[m];
  } else {
#pragma unroll
    for (int m = 0; m < 4; ++m) out[m] = n0 + m < n ? nb2_to_float(p[n0 + m]) : 0.0f;
  }
}
__device__ __forceinline__ void scan_store4(float* p, int n0, int n, int vec, const float (&v)[4]) {
  if (vec && n0 + 4 <= n)
    *reinterpret_cast<float4*>(p + n0) = make_float4(v[0], v[1], v[2], v[3]);
  else
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (n0 + m < n) p[n0 + m] = v[m];
}

// Lane j of S neighbours gets the sum over the S lanes of their p[j].
template <int S>
__device__ __forceinline__ float scan_transpose_sum(float (&p)[S], int j) {
#pragma unroll
  for (int w = S / 2; w >= 1; w /= 2) {
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const bool up = j & w;
      const float keep = up ? p[i + w] : p[i], send = up ? p[i] : p[i + w];
      p[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
    }
  }
  return p[0];
}

// Which channel a lane works on.  Blocks are (sequence, group, channel tile of the group).
template <int S>
struct ScanLane {
  int k, group, tile, c, j, n0;
  bool valid;
  __device__ ScanLane(int channels, int groups) {
    const int per = channels / groups, tiles = (per + ScanTile<S>::kBlock - 1) / ScanTile<S>::kBlock;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x % (tiles * groups);
    k = blockIdx.x / (tiles * groups);
    group = b / tiles;
    tile = b - group * tiles;
    const int in = tile * ScanTile<S>::kBlock + warp * ScanTile<S>::kChannels + lane / S;
    valid = in < per;
    c = group * per + min(in, per - 1);  // (a lane without a channel computes the last one's and stores nothing)
    j = lane % S;
    n0 = 4 * j;
  }
};

template <typename T, int S>
__global__ void __launch_bounds__(SCAN_THREADS) nb2_selective_scan_kernel(const nb2_selective_scan_args a) {
  nb2_pdl_enter();
  const ScanLane<S> l(a.channels, a.groups);
  const int n = a.n_states;
  const int64_t len = a.table[l.k];
  const ScanPlace px = scan_place(a.table, a.n_seq, 0, l.k), pt = scan_place(a.table, a.n_seq, 1, l.k),
                  pb = scan_place(a.table, a.n_seq, 2, l.k), pc = scan_place(a.table, a.n_seq, 3, l.k),
                  py = scan_place(a.table, a.n_seq, 4, l.k), pz = scan_place(a.table, a.n_seq, 5, l.k);
  const T* x = (const T*)a.x + px.start + l.c;
  const T* dt = (const T*)a.dt + pt.start + l.c;
  const T* B = (const T*)a.B + pb.start + (int64_t)l.group * n;
  const T* C = (const T*)a.C + pc.start + (int64_t)l.group * n;
  T* y = (T*)a.y + py.start + l.c;
  const T* z = a.z ? (const T*)a.z + pz.start + l.c : nullptr;
  float A2[4], h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  scan_load4(a.A + (int64_t)l.c * n, l.n0, n, 0, A2);
#pragma unroll
  for (int m = 0; m < 4; ++m) A2[m] *= LOG2E;
  if (a.state) {
    const ScanPlace p = scan_place(a.table, a.n_seq, 6, l.k);
    scan_load4(a.state + p.start + l.c * p.stride, l.n0, n, a.state_vec, h);
  }
  const float D = a.D ? a.D[l.c] : 0.0f, bias = a.dt_bias ? a.dt_bias[l.c] : 0.0f;
  float* keep = a.keep ? a.keep + (a.table[(size_t)17 * a.n_seq + l.k] * a.channels + l.c) * n : nullptr;
  const int base = threadIdx.x & 31 & ~(S - 1);
  for (int64_t tb = 0; tb < len; tb += S) {
    if (keep && tb % NB2_SCAN_KEEP == 0) {
      if (l.valid) scan_store4(keep, l.n0, n, n % 4 == 0, h);
      keep += (int64_t)a.channels * n;
    }
    const int64_t t = tb + l.j;
    const bool in = t < len;
    float s = 0.0f, xv = 0.0f;
    if (in) {
      s = nb2_to_float(dt[t * pt.stride]) + bias;
      xv = nb2_to_float(x[t * px.stride]);
      if (a.softplus) s = scan_softplus(s);
    }
    const float sx = s * xv;
    float p[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
      p[i] = 0.0f;
      const float si = __shfl_sync(0xffffffffu, s, base + i), xi = __shfl_sync(0xffffffffu, sx, base + i);
      if (tb + i < len) {
        float b4[4], c4[4];
        scan_load4(B + (tb + i) * pb.stride, l.n0, n, a.vec, b4);
        scan_load4(C + (tb + i) * pc.stride, l.n0, n, a.vec, c4);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          h[m] = fmaf(scan_exp2(si * A2[m]), h[m], xi * b4[m]);
          p[i] = fmaf(c4[m], h[m], p[i]);
        }
      }
    }
    float o = fmaf(D, xv, scan_transpose_sum<S>(p, l.j));
    if (in && l.valid) {
      if (z) {
        const float zv = nb2_to_float(z[t * pz.stride]);
        o *= zv * nb2_sigmoid(zv);
      }
      y[t * py.stride] = nb2_from_float<T>(o);
    }
  }
  if (a.new_state && l.valid) {
    const ScanPlace p = scan_place(a.table, a.n_seq, 7, l.k);
    scan_store4(a.new_state + p.start + l.c * p.stride, l.n0, n, a.state_vec, h);
  }
}

// Backward.  With dp = dy silu(z), g[t] = C dp + a[t+1] g[t+1] (at the end: dnew_state):
//   dz = dy p silu'(z), u = sum_n g B, dx = D dp + s u, ds = x u + sum_n g a h[t-1] A,
//   ddt = ds softplus', dA = sum_t g a h[t-1] s, dB = sum_c g s x, dC = sum_c dp h, dstate = a[0] g[0].
// A block walks the NB2_SCAN_KEEP-row stretches of its sequence from the last to the first: it
// recomputes a stretch's states from the kept one into shared memory, then goes back through its rows.
template <int S>
struct ScanGradSmem {
  static constexpr int kPitch = 8 * S;  // dB, dC of one row, all lanes' states
  float4 h[NB2_SCAN_KEEP][SCAN_THREADS];
  float red[NB2_SCAN_KEEP][SCAN_WARPS][kPitch];
};

template <typename T, int S>
__global__ void __launch_bounds__(SCAN_THREADS) nb2_selective_scan_grad_kernel(const nb2_selective_scan_grad_args a) {
  extern __shared__ __align__(16) char smem_raw[];
  ScanGradSmem<S>& sm = *reinterpret_cast<ScanGradSmem<S>*>(smem_raw);
  constexpr int kKeep = NB2_SCAN_KEEP;
  nb2_pdl_enter();
  const ScanLane<S> l(a.channels, a.groups);
  const int n = a.n_states, tid = threadIdx.x, warp = tid >> 5;
  const int64_t len = a.table[l.k];
  const ScanPlace px = scan_place(a.table, a.n_seq, 0, l.k), pt = scan_place(a.table, a.n_seq, 1, l.k),
                  pb = scan_place(a.table, a.n_seq, 2, l.k), pc = scan_place(a.table, a.n_seq, 3, l.k),
                  pz = scan_place(a.table, a.n_seq, 4, l.k), pdy = scan_place(a.table, a.n_seq, 5, l.k),
                  pdx = scan_place(a.table, a.n_seq, 6, l.k), pdt = scan_place(a.table, a.n_seq, 7, l.k),
                  pdz = scan_place(a.table, a.n_seq, 10, l.k);
  const T* x = (const T*)a.x + px.start + l.c;
  const T* dt = (const T*)a.dt + pt.start + l.c;
  const T* B = (const T*)a.B + pb.start + (int64_t)l.group * n;
  const T* C = (const T*)a.C + pc.start + (int64_t)l.group * n;
  const T* z = a.z ? (const T*)a.z + pz.start + l.c : nullptr;
  const T* dy = (const T*)a.dy + pdy.start + l.c;
  T* dx = (T*)a.dx + pdx.start + l.c;
  T* ddt = (T*)a.ddt + pdt.start + l.c;
  T* dz = a.dz ? (T*)a.dz + pdz.start + l.c : nullptr;
  const float* keep = a.keep + (a.table[(size_t)27 * a.n_seq + l.k] * a.channels + l.c) * n;
  const int64_t row0 = a.table[(size_t)28 * a.n_seq + l.k];
  float A[4], carry[4] = {0.0f, 0.0f, 0.0f, 0.0f}, dA[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  scan_load4(a.A + (int64_t)l.c * n, l.n0, n, 0, A);
  if (a.dnew_state && l.valid) {
    const ScanPlace p = scan_place(a.table, a.n_seq, 12, l.k);
    scan_load4(a.dnew_state + p.start + l.c * p.stride, l.n0, n, a.state_vec, carry);
  }
  const float D = a.D ? a.D[l.c] : 0.0f, bias = a.dt_bias ? a.dt_bias[l.c] : 0.0f;
  float dD = 0.0f, dbias = 0.0f;
  const int base = tid & 31 & ~(S - 1);
  for (int64_t q = (len + kKeep - 1) / kKeep - 1; q >= 0; --q) {
    const int64_t tq = q * kKeep;
    const int rows = (int)min((int64_t)kKeep, len - tq);
    float h0[4], h[4];
    scan_load4(keep + q * a.channels * n, l.n0, n, n % 4 == 0, h0);
#pragma unroll
    for (int m = 0; m < 4; ++m) h[m] = h0[m];
    for (int r = 0; r < rows; r += S) {
      const int64_t t = tq + r + l.j;
      const bool in = t < len;
      float s = 0.0f, xv = 0.0f;
      if (in) {
        s = nb2_to_float(dt[t * pt.stride]) + bias;
        xv = nb2_to_float(x[t * px.stride]);
        if (a.softplus) s = scan_softplus(s);
      }
      const float sx = s * xv;
      float p[S];
#pragma unroll
      for (int i = 0; i < S; ++i) {
        p[i] = 0.0f;
        const float si = __shfl_sync(0xffffffffu, s, base + i), xi = __shfl_sync(0xffffffffu, sx, base + i);
        if (r + i < rows) {
          float b4[4], c4[4];
          scan_load4(B + (tq + r + i) * pb.stride, l.n0, n, a.vec, b4);
          scan_load4(C + (tq + r + i) * pc.stride, l.n0, n, a.vec, c4);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            h[m] = fmaf(scan_exp2(si * (A[m] * LOG2E)), h[m], xi * b4[m]);
            p[i] = fmaf(c4[m], h[m], p[i]);
          }
          sm.h[r + i][tid] = make_float4(h[0], h[1], h[2], h[3]);
        }
      }
      if (dz) {
        const float o = fmaf(D, xv, scan_transpose_sum<S>(p, l.j));
        if (in && l.valid)
          dz[t * pdz.stride] = nb2_from_float<T>(nb2_to_float(dy[t * pdy.stride]) * o *
                                                 nb2_silu_slope(nb2_to_float(z[t * pz.stride])));
      }
    }
    for (int r = (rows - 1) / S * S; r >= 0; r -= S) {
      const int64_t t = tq + r + l.j;
      const bool in = t < len;
      float s = 0.0f, xv = 0.0f, raw = 0.0f, dp = 0.0f;
      if (in) {
        raw = nb2_to_float(dt[t * pt.stride]) + bias;
        xv = nb2_to_float(x[t * px.stride]);
        s = a.softplus ? scan_softplus(raw) : raw;
        if (l.valid) {
          dp = nb2_to_float(dy[t * pdy.stride]);
          if (z) {
            const float zv = nb2_to_float(z[t * pz.stride]);
            dp *= zv * nb2_sigmoid(zv);
          }
        }
      }
      const float sx = s * xv;
      float pu[S], pe[S];
#pragma unroll
      for (int i = S - 1; i >= 0; --i) {
        pu[i] = pe[i] = 0.0f;
        const float si = __shfl_sync(0xffffffffu, s, base + i), xi = __shfl_sync(0xffffffffu, sx, base + i),
                    di = __shfl_sync(0xffffffffu, dp, base + i);
        if (r + i < rows) {
          float b4[4], c4[4], out[8];
          scan_load4(B + (tq + r + i) * pb.stride, l.n0, n, a.vec, b4);
          scan_load4(C + (tq + r + i) * pc.stride, l.n0, n, a.vec, c4);
          const float4 ht = sm.h[r + i][tid];
          const float4 hp = r + i > 0 ? sm.h[r + i - 1][tid] : make_float4(h0[0], h0[1], h0[2], h0[3]);
          const float hv[4] = {ht.x, ht.y, ht.z, ht.w}, hq[4] = {hp.x, hp.y, hp.z, hp.w};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float g = fmaf(c4[m], di, carry[m]);
            carry[m] = g * scan_exp2(si * (A[m] * LOG2E));
            const float ga = carry[m] * hq[m];
            pu[i] = fmaf(g, b4[m], pu[i]);
            pe[i] = fmaf(ga, A[m], pe[i]);
            dA[m] = fmaf(ga, si, dA[m]);
            out[m] = g * xi;
            out[4 + m] = di * hv[m];
          }
          // over the warp's channels
#pragma unroll
          for (int m = 0; m < 8; ++m)
#pragma unroll
            for (int w = S; w < 32; w *= 2) out[m] += __shfl_xor_sync(0xffffffffu, out[m], w);
          if ((tid & 31) < S) {
            float* red = sm.red[r + i][warp];
            *reinterpret_cast<float4*>(red + l.n0) = make_float4(out[0], out[1], out[2], out[3]);
            *reinterpret_cast<float4*>(red + 4 * S + l.n0) = make_float4(out[4], out[5], out[6], out[7]);
          }
        }
      }
      const float u = scan_transpose_sum<S>(pu, l.j), e = scan_transpose_sum<S>(pe, l.j);
      if (in && l.valid) {
        float ds = fmaf(xv, u, e);
        if (a.softplus) ds *= nb2_sigmoid(raw);
        dx[t * pdx.stride] = nb2_from_float<T>(fmaf(D, dp, s * u));
        ddt[t * pdt.stride] = nb2_from_float<T>(ds);
        dD = fmaf(dp, xv, dD);
        dbias += ds;
      }
    }
    __syncthreads();
    // the block's share of dB and dC: warps in order
    for (int i = tid; i < rows * 2 * n; i += SCAN_THREADS) {
      const int r = i / (2 * n), m = i - r * 2 * n;
      const int col = m < n ? m : 4 * S + m - n;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < SCAN_WARPS; ++w) sum += sm.red[r][w][col];
      a.part_bc[(((int64_t)l.tile * a.total_rows + row0 + tq + r) * a.groups + l.group) * 2 * n + m] = sum;
    }
    __syncthreads();
  }
#pragma unroll
  for (int w = 1; w < S; w *= 2) {
    dD += __shfl_xor_sync(0xffffffffu, dD, w);
    dbias += __shfl_xor_sync(0xffffffffu, dbias, w);
  }
  if (l.valid) {
    const int64_t at = (int64_t)l.k * a.channels + l.c;
    scan_store4(a.part_a + at * n, l.n0, n, 0, dA);
    if (l.j == 0) {
      if (a.dD) a.part_d[at] = dD;
      if (a.ddt_bias) a.part_s[at] = dbias;
    }
    if (a.dstate) {
      const ScanPlace p = scan_place(a.table, a.n_seq, 11, l.k);
      scan_store4(a.dstate + p.start + l.c * p.stride, l.n0, n, a.state_vec, carry);
    }
  }
}

// dB and dC of every row: the channel tiles' shares added in order.
template <typename T>
__global__ void __launch_bounds__(256) nb2_scan_grad_bc_kernel(const nb2_selective_scan_grad_args a, int tiles) {
  nb2_pdl_enter();
  const int n = a.n_states, wide = a.groups * 2 * n;
  const int64_t all = a.total_rows * wide;
  const int k = blockIdx.y;
  const int64_t len = a.table[k], row0 = a.table[(size_t)28 * a.n_seq + k];
  const ScanPlace pb = scan_place(a.table, a.n_seq, 8, k), pc = scan_place(a.table, a.n_seq, 9, k);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < len * wide; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / wide;
    const int rest = (int)(i - r * wide), group = rest / (2 * n), m = rest - group * 2 * n;
    float sum = 0.0f;
    for (int u = 0; u < tiles; ++u) sum += a.part_bc[u * all + (row0 + r) * wide + rest];
    if (m < n)
      ((T*)a.dB)[pb.start + r * pb.stride + group * n + m] = nb2_from_float<T>(sum);
    else
      ((T*)a.dC)[pc.start + r * pc.stride + group * n + m - n] = nb2_from_float<T>(sum);
  }
}

template <typename A>
static int scan_check(const A& a) {
  NB2_REQUIRE(a.table && a.x && a.dt && a.B && a.C && a.A, "null pointer");
  NB2_REQUIRE(a.dtype >= NB2_F32 && a.dtype <= NB2_BF16, "dtype");
  NB2_REQUIRE(a.n_seq >= 1 && a.channels >= 1 && a.groups >= 1 && a.channels % a.groups == 0, "shape");
  NB2_REQUIRE(a.n_states >= 1 && a.n_states <= NB2_SCAN_MAX_STATES, "n_states");
  NB2_REQUIRE((int64_t)a.n_seq * (a.channels + a.groups) < (1ll << 31), "too many sequences x channels");
  NB2_REQUIRE_DEVICE(a.device);
  return NB2_OK;
}

static int scan_tiles(int channels, int groups, int lanes) {
  const int per = channels / groups, block = SCAN_THREADS / lanes;
  return (per + block - 1) / block;
}

template <typename T, int S>
static cudaError_t scan_launch(cudaStream_t s, const nb2_selective_scan_args& a) {
  const unsigned blocks = (unsigned)a.n_seq * a.groups * scan_tiles(a.channels, a.groups, S);
  return nb2_launch(nb2_selective_scan_kernel<T, S>, dim3(blocks), dim3(SCAN_THREADS), 0, s, a);
}

template <typename T, int S>
static cudaError_t scan_grad_launch(cudaStream_t s, const nb2_selective_scan_grad_args& a) {
  const unsigned blocks = (unsigned)a.n_seq * a.groups * scan_tiles(a.channels, a.groups, S);
  const size_t smem = sizeof(ScanGradSmem<S>);
  cudaError_t e = cudaFuncSetAttribute(nb2_selective_scan_grad_kernel<T, S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem);
  if (e != cudaSuccess) return e;
  return nb2_launch(nb2_selective_scan_grad_kernel<T, S>, dim3(blocks), dim3(SCAN_THREADS), smem, s, a);
}

#define SCAN_BY_LANES(lanes, launch)             \
  switch (lanes) {                               \
    case 1: NB2_CUDA((launch<T, 1>(s, a))); break;   \
    case 2: NB2_CUDA((launch<T, 2>(s, a))); break;   \
    case 4: NB2_CUDA((launch<T, 4>(s, a))); break;   \
    case 8: NB2_CUDA((launch<T, 8>(s, a))); break;   \
    case 16: NB2_CUDA((launch<T, 16>(s, a))); break; \
    default: NB2_CUDA((launch<T, 32>(s, a))); break; \
  }

extern "C" int nb2_selective_scan_tile(int n_states) {
  NB2_REQUIRE(n_states >= 1 && n_states <= NB2_SCAN_MAX_STATES, "n_states");
  return SCAN_THREADS / scan_lanes(n_states);
}

extern "C" int nb2_selective_scan(void* stream, const nb2_selective_scan_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_selective_scan_args& a = *args;
  if (int e = scan_check(a)) return e;
  NB2_REQUIRE(a.y, "null pointer");
  cudaStream_t s = nb2_stream(stream);
  NB2_SEQ_DTYPE(a.dtype, SCAN_BY_LANES(scan_lanes(a.n_states), scan_launch));
  return NB2_OK;
}

extern "C" int nb2_selective_scan_grad(void* stream, const nb2_selective_scan_grad_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_selective_scan_grad_args& a = *args;
  if (int e = scan_check(a)) return e;
  NB2_REQUIRE(a.dy && a.dx && a.ddt && a.dB && a.dC && a.dA && a.keep && a.part_bc && a.part_a, "null pointer");
  NB2_REQUIRE((!a.dz || a.z) && (!a.dD || (a.D && a.part_d)) && (!a.ddt_bias || (a.dt_bias && a.part_s)), "gradients");
  NB2_REQUIRE(a.n_seq <= 65535, "too many sequences");
  cudaStream_t s = nb2_stream(stream);
  const int tiles = scan_tiles(a.channels, a.groups, scan_lanes(a.n_states));
  NB2_SEQ_DTYPE(a.dtype, SCAN_BY_LANES(scan_lanes(a.n_states), scan_grad_launch));
  if (a.total_rows > 0) {
    const int64_t wide = (a.total_rows * a.groups * 2 * a.n_states + 255) / 256;
    const int64_t per = (wide + a.n_seq - 1) / a.n_seq;
    const dim3 grid((unsigned)(per < 8192 ? per : 8192), (unsigned)a.n_seq);
    NB2_SEQ_DTYPE(a.dtype, NB2_CUDA(nb2_launch(nb2_scan_grad_bc_kernel<T>, grid, dim3(256), 0, s, a, tiles)));
  }
  NB2_CUDA(nb2_seq_sum_parts(s, a.part_a, a.n_seq, (int64_t)a.channels * a.n_states, a.dA));
  if (a.dD) NB2_CUDA(nb2_seq_sum_parts(s, a.part_d, a.n_seq, a.channels, a.dD));
  if (a.ddt_bias) NB2_CUDA(nb2_seq_sum_parts(s, a.part_s, a.n_seq, a.channels, a.ddt_bias));
  return NB2_OK;
}
