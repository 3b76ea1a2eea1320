// Selective state space scan along the rows of sequences: the linear filter whose step size, input
// and output weights depend on the row.  Per channel c with states n (B, C shared by a group of channels):
//   s = softplus(dt + dt_bias),  a[n] = exp(s A[n]),  h[n] = a[n] h[n] + s x B[n],
//   y = (sum_n C[n] h[n] + D x) silu(z)
//
// Four states to a lane, S = 1 .. 32 lanes to a channel (S = the power of two that covers the states),
// so a warp carries 32 / S channels.  The partial sums over the states that every lane forms for RB rows
// are transposed and added in RB - 1 shuffles, which leaves row j's sum with lane j.
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

// Which channel a lane works on.  Blocks are (unit, group, channel tile of the group); a unit is a stretch
// of a sequence's rows, or without `units` a sequence.
template <int S>
struct ScanLane {
  int unit, k, first, group, tile, width, c0, c, j, n0, in_block;
  bool valid;
  __device__ ScanLane(int channels, int groups, const int* units) {
    const int per = channels / groups, tiles = (per + ScanTile<S>::kBlock - 1) / ScanTile<S>::kBlock;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x % (tiles * groups);
    unit = blockIdx.x / (tiles * groups);
    k = units ? units[2 * unit] : unit;
    first = units ? units[2 * unit + 1] : 0;
    group = b / tiles;
    tile = b - group * tiles;
    width = min(per - tile * ScanTile<S>::kBlock, ScanTile<S>::kBlock);  // channels of this tile
    c0 = group * per + tile * ScanTile<S>::kBlock;
    in_block = warp * ScanTile<S>::kChannels + lane / S;
    valid = in_block < width;
    c = c0 + min(in_block, width - 1);  // (a lane without a channel computes with the last one's and stores nothing)
    j = lane % S;
    n0 = 4 * j;
  }
};

// ---- two floats at a time: the fused multiply-add unit's packed form halves the issue slots -------------
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 exp2x2(f32x2 v) {
  float a, b;
  unpack2(v, a, b);
  return pack2(scan_exp2(a), scan_exp2(b));
}

__device__ __forceinline__ void scan_cp_async(void* smem, const void* gmem, int bytes) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  if (bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(gmem) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(s), "l"(gmem) : "memory");
}
__device__ __forceinline__ void scan_cp_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// What a block stages in shared memory: R rows of its channels of NA arrays in their own type, and the
// rows' weights B, C in float32 (converted once for all its channels), padded with zeros to 4 S states.
template <typename T, int S, int R, int NA>
struct ScanStage {
  static constexpr int kChannels = SCAN_THREADS / S, kRows = R;
  // rows that a warp's lanes read at the same time start in different banks
  static constexpr int kPitch = ((kChannels + 32 / S) * (int)sizeof(T) + 15) / 16 * 16 / (int)sizeof(T);
  static constexpr int kStates = 4 * S;
  static constexpr int kBytes = kChannels * (int)sizeof(T) < 16 ? kChannels * (int)sizeof(T) : 16;
  alignas(16) T in[NA][R][kPitch];
  alignas(16) float bc[R][2][kStates];
};

// A tile's prepared rows: (s, s x) of every channel
template <int S, int R>
struct ScanRows {
  static constexpr int kPitch = SCAN_THREADS / S + (S < 16 ? 16 / S : 1);
  float2 sx[R][kPitch];
};

// rows x channels of one array, asynchronously (VEC) or element by element
template <bool VEC, typename T, int ROWS, int PITCH, int CHANNELS, int BYTES>
__device__ __forceinline__ void scan_fetch(T (&to)[ROWS][PITCH], const T* from, int64_t stride, int rows, int channels) {
  if constexpr (VEC) {
    constexpr int kPer = BYTES / sizeof(T), kChunks = CHANNELS / kPer;
#pragma unroll
    for (int i = 0; i < (ROWS * kChunks + SCAN_THREADS - 1) / SCAN_THREADS; ++i) {
      const int at = threadIdx.x + i * SCAN_THREADS, r = at / kChunks, c = at % kChunks * kPer;
      if (r < rows && c < channels) scan_cp_async(&to[r][c], from + r * stride + c, BYTES);
    }
  } else {
    for (int at = threadIdx.x; at < rows * CHANNELS; at += SCAN_THREADS) {
      const int r = at / CHANNELS, c = at % CHANNELS;
      if (c < channels) to[r][c] = from[r * stride + c];
    }
  }
}

// B and C of a tile's rows, on their way through registers from the arrays' type to float32; rows past the
// end become zeros
template <bool VEC, typename T, int S, int R>
struct ScanWeights {
  static constexpr int kPer = VEC ? 16 / (int)sizeof(T) : 1;
  static constexpr int kCount = (R * 8 * S / kPer + SCAN_THREADS - 1) / SCAN_THREADS;
  SeqVecA<T, kPer> v[kCount];
  // entry i of the thread: (row, B or C, first state); false past the tile
  static __device__ __forceinline__ bool at(int i, int n, int& r, int& which, int& m) {
    const int per = n / kPer, e = threadIdx.x + i * SCAN_THREADS;
    r = e / (2 * per);
    const int rest = e - r * 2 * per;
    which = rest >= per;
    m = (rest - which * per) * kPer;
    return r < R;
  }
  __device__ __forceinline__ void load(const T* B, int64_t bs, const T* C, int64_t cs, int n, int rows) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      int r, which, m;
      v[i].zero();
      if (at(i, n, r, which, m) && r < rows) v[i].load((which ? C + r * cs : B + r * bs) + m);
    }
  }
  __device__ __forceinline__ void store(float (&bc)[R][2][4 * S], int n) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      int r, which, m;
      if (at(i, n, r, which, m))
#pragma unroll
        for (int e = 0; e < kPer; ++e) bc[r][which][m + e] = v[i][e];
    }
  }
};

template <typename Stage>
__device__ __forceinline__ void scan_clear_weights(Stage* stages, int count) {
  constexpr int kEach = Stage::kRows * 2 * Stage::kStates;
  for (int i = threadIdx.x; i < count * kEach; i += SCAN_THREADS) (&stages[i / kEach].bc[0][0][0])[i % kEach] = 0.0f;
}

// A[c][n0 ..] log2(e), two states to a register pair.  Held finite: a row past a sequence's end counts as a
// step of zero, which has to leave the state as it is (0 * inf would not).
__device__ __forceinline__ void scan_rates(const float* A, int n0, int n, f32x2 (&A2)[2]) {
  float v[4];
  scan_load4(A, n0, n, 0, v);
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const float r = v[m] * LOG2E;
    v[m] = r > 3e38f ? 3e38f : r < -3e38f ? -3e38f : r;
  }
  A2[0] = pack2(v[0], v[1]);
  A2[1] = pack2(v[2], v[3]);
}

// Units are stretches of unit_rows rows of a sequence.  One unit to a sequence: the block starts from its
// state and walks it to the end.  More (a long sequence of few channels): ENDS first leaves the state that
// every unit would reach from zero and the sum of its steps, nb2_scan_join_kernel turns these into the
// states that the units start from, and the second walk (ENDS false) starts there.
//
// A tile of R rows is worked in three phases, each a warp's own: its lanes prepare (s, s x) of the tile's rows
// for their channels, walk the rows through the states, and finish the outputs.
template <typename T, int S, bool VEC, bool ENDS>
__global__ void __launch_bounds__(SCAN_THREADS) nb2_selective_scan_kernel(const nb2_selective_scan_args a) {
  constexpr int R = S <= 4 ? 32 : 16, RB = S < 8 ? S : 8;
  using Stage = ScanStage<T, S, R, 3>;
  extern __shared__ __align__(16) char smem_raw[];
  Stage* stages = reinterpret_cast<Stage*>(smem_raw);
  ScanRows<S, R>& ready = *reinterpret_cast<ScanRows<S, R>*>(smem_raw + 2 * sizeof(Stage));
  nb2_pdl_wait();
  const ScanLane<S> l(a.channels, a.groups, a.units);
  const int n = a.n_states;
  const int64_t len = a.table[l.k], t0 = l.first, t1 = min(t0 + a.unit_rows, len);
  if (ENDS && t1 == len) return;  // nothing starts from the last unit's end
  const int64_t nk = a.n_seq;
  const ScanPlace px = scan_place(a.table, nk, 0, l.k), pt = scan_place(a.table, nk, 1, l.k),
                  pb = scan_place(a.table, nk, 2, l.k), pc = scan_place(a.table, nk, 3, l.k),
                  py = scan_place(a.table, nk, 4, l.k), pz = scan_place(a.table, nk, 5, l.k);
  const T* x = (const T*)a.x + px.start + t0 * px.stride + l.c0;
  const T* dt = (const T*)a.dt + pt.start + t0 * pt.stride + l.c0;
  const T* z = !ENDS && a.z ? (const T*)a.z + pz.start + t0 * pz.stride + l.c0 : nullptr;
  const T* B = (const T*)a.B + pb.start + t0 * pb.stride + (int64_t)l.group * n;
  const T* C = (const T*)a.C + pc.start + t0 * pc.stride + (int64_t)l.group * n;
  T* y = (T*)a.y + py.start + t0 * py.stride + l.c;
  f32x2 A2[2], h[2];
  scan_rates(a.A + (int64_t)l.c * n, l.n0, n, A2);
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (!ENDS) {
    if (a.ends)
      scan_load4(a.ends + ((int64_t)l.unit * a.channels + l.c) * n, l.n0, n, n % 4 == 0, v);
    else if (a.state) {
      const ScanPlace p = scan_place(a.table, nk, 6, l.k);
      scan_load4(a.state + p.start + l.c * p.stride, l.n0, n, a.state_vec, v);
    }
  }
  h[0] = pack2(v[0], v[1]);
  h[1] = pack2(v[2], v[3]);
  const float D = !ENDS && a.D ? a.D[l.c] : 0.0f, bias = a.dt_bias ? a.dt_bias[l.c] : 0.0f;
  float* keep = !ENDS && a.keep
                    ? a.keep + ((a.table[17 * nk + l.k] + t0 / NB2_SCAN_KEEP) * a.channels + l.c) * n
                    : nullptr;
  const int j = l.j % RB, mine = l.in_block;
  float total = 0.0f;

  scan_clear_weights(stages, 2);  // the padding states' stay zero: only the real ones are written
  __syncthreads();
  ScanWeights<VEC, T, S, R> weights;
  auto fetch = [&](Stage& st, int64_t from, int rows) {
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[0], dt + from * pt.stride, pt.stride, rows, l.width);
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[1], x + from * px.stride, px.stride, rows, l.width);
    if (z)
      scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[2], z + from * pz.stride, pz.stride, rows, l.width);
    weights.load(B + from * pb.stride, pb.stride, C + from * pc.stride, pc.stride, n, rows);
  };
  const int64_t all = t1 - t0;
  if (all > 0) {
    fetch(stages[0], 0, (int)min((int64_t)R, all));
    weights.store(stages[0].bc, n);
  }
  int cur = 0;
  for (int64_t tb = 0; tb < all; tb += R, cur ^= 1) {
    const int rows = (int)min((int64_t)R, all - tb), next = (int)min((int64_t)R, all - tb - rows);
    scan_cp_wait();
    __syncthreads();
    const Stage& st = stages[cur];
    if (next > 0) fetch(stages[cur ^ 1], tb + R, next);
    if (l.j < RB) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RB) {
        const int r = r0 + j;
        float2 o = make_float2(0.0f, 0.0f);
        if (r < rows) {
          o.x = nb2_to_float(st.in[0][r][mine]) + bias;
          if (a.softplus) o.x = scan_softplus(o.x);
          o.y = o.x * nb2_to_float(st.in[1][r][mine]);
        }
        if (ENDS) total += o.x;
        ready.sx[r][mine] = o;
      }
    }
    __syncwarp();
    float out[R / RB];
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += RB) {
      if (keep && r0 % NB2_SCAN_KEEP == 0 && r0 < rows) {
        unpack2(h[0], v[0], v[1]);
        unpack2(h[1], v[2], v[3]);
        if (l.valid) scan_store4(keep, l.n0, n, n % 4 == 0, v);
        keep += (int64_t)a.channels * n;
      }
      float p[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const float2 sx = ready.sx[r0 + i][mine];
        const f32x2 s2 = pack2(sx.x, sx.x), x2 = pack2(sx.y, sx.y);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[r0 + i][0][l.n0]);
        h[0] = fma2(exp2x2(mul2(s2, A2[0])), h[0], mul2(x2, b.x));
        h[1] = fma2(exp2x2(mul2(s2, A2[1])), h[1], mul2(x2, b.y));
        if (!ENDS) {
          const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&st.bc[r0 + i][1][l.n0]);
          float lo, hi;
          unpack2(fma2(c.y, h[1], mul2(c.x, h[0])), lo, hi);
          p[i] = lo + hi;
        }
      }
      if (!ENDS) {
        float o = scan_transpose_sum<RB>(p, j);
#pragma unroll
        for (int w = RB; w < S; w *= 2) o += __shfl_xor_sync(0xffffffffu, o, w);
        out[r0 / RB] = o;
      }
    }
    if (!ENDS && l.valid && l.j < RB) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RB) {
        const int r = r0 + j;
        if (r < rows) {
          float o = fmaf(D, nb2_to_float(st.in[1][r][mine]), out[r0 / RB]);
          if (z) {
            const float zv = nb2_to_float(st.in[2][r][mine]);
            o *= zv * nb2_sigmoid(zv);
          }
          y[(tb + r) * py.stride] = nb2_from_float<T>(o);
        }
      }
    }
    if (next > 0) weights.store(stages[cur ^ 1].bc, n);
  }
  unpack2(h[0], v[0], v[1]);
  unpack2(h[1], v[2], v[3]);
  if (ENDS) {
#pragma unroll
    for (int w = 1; w < RB; w *= 2) total += __shfl_xor_sync(0xffffffffu, total, w);
    if (l.valid) {
      const int64_t at = (int64_t)l.unit * a.channels + l.c;
      scan_store4(a.ends + at * n, l.n0, n, n % 4 == 0, v);
      if (l.j == 0) a.sums[at] = total;
    }
  } else if (a.new_state && l.valid && t1 == len) {
    const ScanPlace p = scan_place(a.table, nk, 7, l.k);
    scan_store4(a.new_state + p.start + l.c * p.stride, l.n0, n, a.state_vec, v);
  }
}

// From what the units reach from zero to what they start from, in order of time (the states) or against it
// (the gradients): start' = exp(A sum s) start + end.  A thread per (sequence, channel, state).
struct ScanJoin {
  const int64_t* table;
  int n_seq, n_states, unit_rows, backwards;
  int64_t channels, per_seq, first_unit_field;
  const float* A;
  const float* from;  // where the walk starts: rows of n_states at (start, stride) of `from_array`; NULL: zeros
  int from_array;
  float* ends;
  const float* sums;
};
__global__ void __launch_bounds__(256) nb2_scan_join_kernel(const ScanJoin a) {
  nb2_pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int k = (int)(i / a.per_seq);
  if (k >= a.n_seq) return;
  const int64_t cn = i - k * a.per_seq, c = cn / a.n_states, len = a.table[k];
  const int64_t u0 = a.table[a.first_unit_field * a.n_seq + k], units = max((len + a.unit_rows - 1) / a.unit_rows, (int64_t)1);
  const float A2 = a.A[cn] * LOG2E;
  float h = 0.0f;
  if (a.from) {
    const ScanPlace p = scan_place(a.table, a.n_seq, a.from_array, k);
    h = a.from[p.start + c * p.stride + (cn - c * a.n_states)];
  }
  const int64_t first = a.backwards ? u0 + units - 1 : u0, step = a.backwards ? -1 : 1;
  float* ends = a.ends + first * a.per_seq + cn;
  const float* sums = a.sums + first * a.channels + c;
  constexpr int kAhead = 8;
  for (int64_t u = 0; u < units; u += kAhead) {
    float e[kAhead], s[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const bool more = u + q + 1 < units;
      e[q] = more ? ends[(u + q) * step * a.per_seq] : 0.0f;
      s[q] = more ? sums[(u + q) * step * a.channels] : 0.0f;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (u + q >= units) break;
      ends[(u + q) * step * a.per_seq] = h;
      h = fmaf(scan_exp2(s[q] * A2), h, e[q]);
    }
  }
}

// Single tokens and a few rows: the state is most of the traffic.  No staging; a lane loads the next
// channel's state while it works, rows are read straight from memory.
template <typename T, int S>
__global__ void __launch_bounds__(SCAN_THREADS) nb2_selective_scan_token_kernel(const nb2_selective_scan_args a, int tiles,
                                                                                int per_block) {
  constexpr int kWarp = 32 / S, kBlock = kWarp * SCAN_WARPS, kUnroll = 4;
  nb2_pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = a.n_states;
  const int k = blockIdx.x / tiles, j = lane % S, n0 = 4 * j;
  const int per = a.channels / a.groups;
  const int64_t len = a.table[k], nk = a.n_seq;
  const ScanPlace px = scan_place(a.table, nk, 0, k), pt = scan_place(a.table, nk, 1, k),
                  pb = scan_place(a.table, nk, 2, k), pc = scan_place(a.table, nk, 3, k),
                  py = scan_place(a.table, nk, 4, k), pz = scan_place(a.table, nk, 5, k),
                  ps = scan_place(a.table, nk, 6, k), pn = scan_place(a.table, nk, 7, k);
  const T* x = (const T*)a.x + px.start;
  const T* dt = (const T*)a.dt + pt.start;
  const T* B = (const T*)a.B + pb.start;
  const T* C = (const T*)a.C + pc.start;
  T* y = (T*)a.y + py.start;
  const T* z = (const T*)a.z + pz.start;
  const int c0 = (blockIdx.x - k * tiles) * per_block, c1 = min(c0 + per_block, a.channels);
  for (int cb = c0 + warp * kWarp + lane / S; cb - lane / S < c1; cb += kBlock * kUnroll) {
    float h[kUnroll][4], A2[kUnroll][4], b[4], c4[4], tv[kUnroll], xv[kUnroll], zv[kUnroll], D[kUnroll], bias[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int c = min(cb + u * kBlock, a.channels - 1);
#pragma unroll
      for (int m = 0; m < 4; ++m) h[u][m] = 0.0f;
      if (a.state) scan_load4(a.state + ps.start + c * ps.stride, n0, n, a.state_vec, h[u]);
      scan_load4(a.A + (int64_t)c * n, n0, n, n % 4 == 0 && a.a_vec, A2[u]);
      D[u] = a.D ? a.D[c] : 0.0f;
      bias[u] = a.dt_bias ? a.dt_bias[c] : 0.0f;
    }
    for (int64_t t = 0; t < len; ++t) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = min(cb + u * kBlock, a.channels - 1);
        tv[u] = nb2_to_float(dt[t * pt.stride + c]);
        xv[u] = nb2_to_float(x[t * px.stride + c]);
        zv[u] = a.z ? nb2_to_float(z[t * pz.stride + c]) : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int c = min(cb + u * kBlock, a.channels - 1), g = c / per;
        scan_load4(B + t * pb.stride + g * n, n0, n, a.vec, b);
        scan_load4(C + t * pc.stride + g * n, n0, n, a.vec, c4);
        float s = tv[u] + bias[u], o = 0.0f;
        if (a.softplus) s = scan_softplus(s);
        const float sx = s * xv[u];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          h[u][m] = fmaf(scan_exp2(s * (A2[u][m] * LOG2E)), h[u][m], sx * b[m]);
          o = fmaf(c4[m], h[u][m], o);
        }
#pragma unroll
        for (int w = 1; w < S; w *= 2) o += __shfl_xor_sync(0xffffffffu, o, w);
        o = fmaf(D[u], xv[u], o);
        if (a.z) o *= zv[u] * nb2_sigmoid(zv[u]);
        if (j == 0 && cb + u * kBlock < c1) y[t * py.stride + c] = nb2_from_float<T>(o);
      }
    }
    if (a.new_state)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (cb + u * kBlock < c1) scan_store4(a.new_state + pn.start + (cb + u * kBlock) * pn.stride, n0, n, a.state_vec, h[u]);
  }
}

// Backward.  With dp = dy silu(z), g[t] = C dp + a[t+1] g[t+1] (at the end: dnew_state):
//   dz = dy p silu'(z), u = sum_n g B, dx = D dp + s u, ds = x u + sum_n g a h[t-1] A,
//   ddt = ds softplus', dA = sum_t g a h[t-1] s, dB = sum_c g s x, dC = sum_c dp h, dstate = a[0] g[0].
// A block walks its unit's NB2_SCAN_KEEP-row tiles from the last to the first: it recomputes a tile's decays
// and states from the kept state into registers, then goes back through its rows.  Units as in the forward
// pass, run through from the last: nb2_scan_grad_ends_kernel leaves the gradient that each would hand on if it
// received zero.
template <int S>
struct ScanGradSmem {
  static constexpr int R = NB2_SCAN_KEEP;
  ScanRows<S, R> ready;
  float dp[R][ScanRows<S, R>::kPitch];
  alignas(16) float red[R][SCAN_WARPS][8 * S];  // dB, dC of a row: a warp's channels added
};

// Sums over the warp's channels (the lane bits S, 2 S ..) of eight values: transposed while there are values
// to share, so lane bits choose which of them a lane ends up with (at, at + 1, .. of `kLeft`), then plain.
template <int S>
struct ScanChannelSum {
  static constexpr int kStages = S == 32 ? 0 : S == 16 ? 1 : S == 8 ? 2 : 3;
  static constexpr int kLeft = 8 >> kStages;
  static __device__ __forceinline__ void sum(float (&v)[8], int lane) {
    int w = S;
#pragma unroll
    for (int half = 4; half >= kLeft; half /= 2, w *= 2) {
      const bool up = lane & w;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float keep = up ? v[i + half] : v[i], send = up ? v[i] : v[i + half];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
      }
    }
#pragma unroll
    for (int b = S << kStages; b < 32; b *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], b);
  }
  static __device__ __forceinline__ int at(int lane) {
    int i = 0;
#pragma unroll
    for (int q = 0; q < kStages; ++q)
      if (lane & (S << q)) i += 4 >> q;
    return i;
  }
  static __device__ __forceinline__ bool writes(int lane) { return lane < (S << kStages); }
};

template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(SCAN_THREADS) nb2_scan_grad_ends_kernel(const nb2_selective_scan_grad_args a) {
  constexpr int R = NB2_SCAN_KEEP, RB = S < 8 ? S : 8;
  using Stage = ScanStage<T, S, R, 3>;
  extern __shared__ __align__(16) char smem_raw[];
  Stage* stages = reinterpret_cast<Stage*>(smem_raw);
  ScanRows<S, R>& ready = *reinterpret_cast<ScanRows<S, R>*>(smem_raw + 2 * sizeof(Stage));
  nb2_pdl_wait();
  const ScanLane<S> l(a.channels, a.groups, a.units);
  const int n = a.n_states;
  const int64_t len = a.table[l.k], t0 = l.first, t1 = min(t0 + a.unit_rows, len), nk = a.n_seq;
  if (t0 == 0) return;  // nothing comes before the first unit
  const ScanPlace pt = scan_place(a.table, nk, 1, l.k), pb = scan_place(a.table, nk, 2, l.k),
                  pc = scan_place(a.table, nk, 3, l.k), pz = scan_place(a.table, nk, 4, l.k),
                  pdy = scan_place(a.table, nk, 5, l.k);
  const T* dt = (const T*)a.dt + pt.start + t0 * pt.stride + l.c0;
  const T* z = a.z ? (const T*)a.z + pz.start + t0 * pz.stride + l.c0 : nullptr;
  const T* dy = (const T*)a.dy + pdy.start + t0 * pdy.stride + l.c0;
  const T* B = (const T*)a.B + pb.start + t0 * pb.stride + (int64_t)l.group * n;
  const T* C = (const T*)a.C + pc.start + t0 * pc.stride + (int64_t)l.group * n;
  f32x2 A2[2], g[2] = {0, 0};
  scan_rates(a.A + (int64_t)l.c * n, l.n0, n, A2);
  const float bias = a.dt_bias ? a.dt_bias[l.c] : 0.0f;
  const int j = l.j % RB, mine = l.in_block;
  float total = 0.0f;
  scan_clear_weights(stages, 2);
  __syncthreads();
  ScanWeights<VEC, T, S, R> weights;
  auto fetch = [&](Stage& st, int64_t from, int rows) {
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[0], dt + from * pt.stride, pt.stride, rows, l.width);
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[1], dy + from * pdy.stride, pdy.stride, rows, l.width);
    if (z)
      scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[2], z + from * pz.stride, pz.stride, rows, l.width);
    weights.load(B + from * pb.stride, pb.stride, C + from * pc.stride, pc.stride, n, rows);
  };
  const int64_t all = t1 - t0, last = (all - 1) / R * R;
  fetch(stages[0], last, (int)(all - last));
  weights.store(stages[0].bc, n);
  int cur = 0;
  for (int64_t tb = last; tb >= 0; tb -= R, cur ^= 1) {
    const int rows = (int)min((int64_t)R, all - tb);
    scan_cp_wait();
    __syncthreads();
    const Stage& st = stages[cur];
    if (tb > 0) fetch(stages[cur ^ 1], tb - R, R);
    if (l.j < RB) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RB) {
        const int r = r0 + j;
        float2 o = make_float2(0.0f, 0.0f);  // (s, dp)
        if (r < rows) {
          o.x = nb2_to_float(st.in[0][r][mine]) + bias;
          if (a.softplus) o.x = scan_softplus(o.x);
          o.y = nb2_to_float(st.in[1][r][mine]);
          if (z) {
            const float zv = nb2_to_float(st.in[2][r][mine]);
            o.y *= zv * nb2_sigmoid(zv);
          }
        }
        total += o.x;
        ready.sx[r][mine] = o;
      }
    }
    __syncwarp();
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      const float2 sd = ready.sx[r][mine];
      const f32x2 s2 = pack2(sd.x, sd.x), d2 = pack2(sd.y, sd.y);
      const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&st.bc[r][1][l.n0]);
      g[0] = mul2(exp2x2(mul2(s2, A2[0])), fma2(c.x, d2, g[0]));
      g[1] = mul2(exp2x2(mul2(s2, A2[1])), fma2(c.y, d2, g[1]));
    }
    if (tb > 0) weights.store(stages[cur ^ 1].bc, n);
  }
#pragma unroll
  for (int w = 1; w < RB; w *= 2) total += __shfl_xor_sync(0xffffffffu, total, w);
  if (l.valid) {
    float v[4];
    unpack2(g[0], v[0], v[1]);
    unpack2(g[1], v[2], v[3]);
    const int64_t at = (int64_t)l.unit * a.channels + l.c;
    scan_store4(a.ends + at * n, l.n0, n, n % 4 == 0, v);
    if (l.j == 0) a.sums[at] = total;
  }
}

template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(SCAN_THREADS) nb2_selective_scan_grad_kernel(const nb2_selective_scan_grad_args a) {
  constexpr int R = NB2_SCAN_KEEP, RB = S < 8 ? S : 8;
  using Stage = ScanStage<T, S, R, 4>;
  using Sum = ScanChannelSum<S>;
  extern __shared__ __align__(16) char smem_raw[];
  Stage* stages = reinterpret_cast<Stage*>(smem_raw);
  ScanGradSmem<S>& sm = *reinterpret_cast<ScanGradSmem<S>*>(smem_raw + 2 * sizeof(Stage));
  nb2_pdl_wait();
  const ScanLane<S> l(a.channels, a.groups, a.units);
  const int n = a.n_states, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t len = a.table[l.k], t0 = l.first, t1 = min(t0 + a.unit_rows, len), nk = a.n_seq;
  const ScanPlace px = scan_place(a.table, nk, 0, l.k), pt = scan_place(a.table, nk, 1, l.k),
                  pb = scan_place(a.table, nk, 2, l.k), pc = scan_place(a.table, nk, 3, l.k),
                  pz = scan_place(a.table, nk, 4, l.k), pdy = scan_place(a.table, nk, 5, l.k),
                  pdx = scan_place(a.table, nk, 6, l.k), pdt = scan_place(a.table, nk, 7, l.k),
                  pdz = scan_place(a.table, nk, 10, l.k);
  const T* x = (const T*)a.x + px.start + t0 * px.stride + l.c0;
  const T* dt = (const T*)a.dt + pt.start + t0 * pt.stride + l.c0;
  const T* z = a.z ? (const T*)a.z + pz.start + t0 * pz.stride + l.c0 : nullptr;
  const T* dy = (const T*)a.dy + pdy.start + t0 * pdy.stride + l.c0;
  const T* B = (const T*)a.B + pb.start + t0 * pb.stride + (int64_t)l.group * n;
  const T* C = (const T*)a.C + pc.start + t0 * pc.stride + (int64_t)l.group * n;
  T* dx = (T*)a.dx + pdx.start + t0 * pdx.stride + l.c;
  T* ddt = (T*)a.ddt + pdt.start + t0 * pdt.stride + l.c;
  T* dz = a.dz ? (T*)a.dz + pdz.start + t0 * pdz.stride + l.c : nullptr;
  const float* keep = a.keep + ((a.table[27 * nk + l.k] + t0 / R) * a.channels + l.c) * n;
  const int64_t row0 = a.table[28 * nk + l.k] + t0;
  f32x2 A2[2], A[2], carry[2], dA[2] = {0, 0};
  float v[4];
  scan_rates(a.A + (int64_t)l.c * n, l.n0, n, A2);
  scan_load4(a.A + (int64_t)l.c * n, l.n0, n, 0, v);
  A[0] = pack2(v[0], v[1]);
  A[1] = pack2(v[2], v[3]);
#pragma unroll
  for (int m = 0; m < 4; ++m) v[m] = 0.0f;
  if (l.valid) {
    if (a.ends)
      scan_load4(a.ends + ((int64_t)l.unit * a.channels + l.c) * n, l.n0, n, n % 4 == 0, v);
    else if (a.dnew_state) {
      const ScanPlace p = scan_place(a.table, nk, 12, l.k);
      scan_load4(a.dnew_state + p.start + l.c * p.stride, l.n0, n, a.state_vec, v);
    }
  }
  carry[0] = pack2(v[0], v[1]);
  carry[1] = pack2(v[2], v[3]);
  const float D = a.D ? a.D[l.c] : 0.0f, bias = a.dt_bias ? a.dt_bias[l.c] : 0.0f;
  const int j = l.j % RB, mine = l.in_block;
  float dD = 0.0f, dbias = 0.0f, h0[4];
  scan_clear_weights(stages, 2);
  __syncthreads();
  ScanWeights<VEC, T, S, R> weights;
  auto fetch = [&](Stage& st, int64_t from, int rows) {
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[0], dt + from * pt.stride, pt.stride, rows, l.width);
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[1], x + from * px.stride, px.stride, rows, l.width);
    scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[2], dy + from * pdy.stride, pdy.stride, rows, l.width);
    if (z)
      scan_fetch<VEC, T, R, Stage::kPitch, Stage::kChannels, Stage::kBytes>(st.in[3], z + from * pz.stride, pz.stride, rows, l.width);
    weights.load(B + from * pb.stride, pb.stride, C + from * pc.stride, pc.stride, n, rows);
    scan_load4(keep + from / R * a.channels * n, l.n0, n, n % 4 == 0, h0);
  };
  const int64_t all = t1 - t0, last = (all - 1) / R * R;
  if (all > 0) {
    fetch(stages[0], last, (int)(all - last));
    weights.store(stages[0].bc, n);
  }
  int cur = 0;
  for (int64_t tb = all > 0 ? last : -1; tb >= 0; tb -= R, cur ^= 1) {
    const int rows = (int)min((int64_t)R, all - tb);
    scan_cp_wait();
    __syncthreads();
    const Stage& st = stages[cur];
    const f32x2 start[2] = {pack2(h0[0], h0[1]), pack2(h0[2], h0[3])};
    if (tb > 0) fetch(stages[cur ^ 1], tb - R, R);
    if (l.j < RB) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RB) {
        const int r = r0 + j;
        float2 o = make_float2(0.0f, 0.0f);
        float dp = 0.0f;
        if (r < rows) {
          o.x = nb2_to_float(st.in[0][r][mine]) + bias;
          if (a.softplus) o.x = scan_softplus(o.x);
          o.y = o.x * nb2_to_float(st.in[1][r][mine]);
          if (l.valid) {  // (a lane without a channel adds nothing to dB, dC)
            dp = nb2_to_float(st.in[2][r][mine]);
            if (z) {
              const float zv = nb2_to_float(st.in[3][r][mine]);
              dp *= zv * nb2_sigmoid(zv);
            }
          } else {
            o = make_float2(0.0f, 0.0f);
          }
        }
        sm.ready.sx[r][mine] = o;
        sm.dp[r][mine] = dp;
      }
    }
    __syncwarp();
    f32x2 h[R][2], dec[R][2];
    float out[R / RB], du[R / RB], de[R / RB];
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += RB) {
      float p[RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int r = r0 + i;
        const float2 sx = sm.ready.sx[r][mine];
        const f32x2 s2 = pack2(sx.x, sx.x), x2 = pack2(sx.y, sx.y);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[r][0][l.n0]);
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&st.bc[r][1][l.n0]);
        dec[r][0] = exp2x2(mul2(s2, A2[0]));
        dec[r][1] = exp2x2(mul2(s2, A2[1]));
        h[r][0] = fma2(dec[r][0], r ? h[r ? r - 1 : 0][0] : start[0], mul2(x2, b.x));
        h[r][1] = fma2(dec[r][1], r ? h[r ? r - 1 : 0][1] : start[1], mul2(x2, b.y));
        float lo, hi;
        unpack2(fma2(c.y, h[r][1], mul2(c.x, h[r][0])), lo, hi);
        p[i] = lo + hi;
      }
      out[r0 / RB] = 0.0f;
      if (dz) {
        float o = scan_transpose_sum<RB>(p, j);
#pragma unroll
        for (int w = RB; w < S; w *= 2) o += __shfl_xor_sync(0xffffffffu, o, w);
        out[r0 / RB] = o;
      }
    }
#pragma unroll
    for (int r0 = R - RB; r0 >= 0; r0 -= RB) {
      float pu[RB], pe[RB];
#pragma unroll
      for (int i = RB - 1; i >= 0; --i) {
        const int r = r0 + i;
        const float2 sx = sm.ready.sx[r][mine];
        const float dp = sm.dp[r][mine];
        const f32x2 s2 = pack2(sx.x, sx.x), x2 = pack2(sx.y, sx.y), d2 = pack2(dp, dp);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[r][0][l.n0]);
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&st.bc[r][1][l.n0]);
        const f32x2 g0 = fma2(c.x, d2, carry[0]), g1 = fma2(c.y, d2, carry[1]);
        carry[0] = mul2(g0, dec[r][0]);
        carry[1] = mul2(g1, dec[r][1]);
        const f32x2 q0 = mul2(carry[0], r ? h[r ? r - 1 : 0][0] : start[0]);
        const f32x2 q1 = mul2(carry[1], r ? h[r ? r - 1 : 0][1] : start[1]);
        dA[0] = fma2(q0, s2, dA[0]);
        dA[1] = fma2(q1, s2, dA[1]);
        float lo, hi;
        unpack2(fma2(g1, b.y, mul2(g0, b.x)), lo, hi);
        pu[i] = lo + hi;
        unpack2(fma2(q1, A[1], mul2(q0, A[0])), lo, hi);
        pe[i] = lo + hi;
        float w[8];
        unpack2(mul2(g0, x2), w[0], w[1]);
        unpack2(mul2(g1, x2), w[2], w[3]);
        unpack2(mul2(d2, h[r][0]), w[4], w[5]);
        unpack2(mul2(d2, h[r][1]), w[6], w[7]);
        Sum::sum(w, lane);
        if (Sum::writes(lane)) {
          const int at = Sum::at(lane);
#pragma unroll
          for (int m = 0; m < Sum::kLeft; ++m) sm.red[r][warp][((at + m) >> 2) * 4 * S + l.n0 + ((at + m) & 3)] = w[m];
        }
      }
      float u = scan_transpose_sum<RB>(pu, j), e = scan_transpose_sum<RB>(pe, j);
#pragma unroll
      for (int w = RB; w < S; w *= 2) {
        u += __shfl_xor_sync(0xffffffffu, u, w);
        e += __shfl_xor_sync(0xffffffffu, e, w);
      }
      du[r0 / RB] = u;
      de[r0 / RB] = e;
    }
    if (l.valid && l.j < RB) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RB) {
        const int r = r0 + j;
        if (r < rows) {
          const float raw = nb2_to_float(st.in[0][r][mine]) + bias, xv = nb2_to_float(st.in[1][r][mine]);
          const float dp = sm.dp[r][mine], u = du[r0 / RB];
          float ds = fmaf(xv, u, de[r0 / RB]);
          if (a.softplus) ds *= nb2_sigmoid(raw);
          dx[(tb + r) * pdx.stride] = nb2_from_float<T>(fmaf(D, dp, sm.ready.sx[r][mine].x * u));
          ddt[(tb + r) * pdt.stride] = nb2_from_float<T>(ds);
          if (dz)
            dz[(tb + r) * pdz.stride] = nb2_from_float<T>(nb2_to_float(st.in[2][r][mine]) * fmaf(D, xv, out[r0 / RB]) *
                                                          nb2_silu_slope(nb2_to_float(st.in[3][r][mine])));
          dD = fmaf(dp, xv, dD);
          dbias += ds;
        }
      }
    }
    if (tb > 0) weights.store(stages[cur ^ 1].bc, n);
    __syncthreads();
    // the block's share of dB and dC: warps in order
    for (int i = tid; i < rows * 2 * n; i += SCAN_THREADS) {
      const int r = i / (2 * n), m = i - r * 2 * n;
      const int col = m < n ? m : 4 * S + m - n;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < SCAN_WARPS; ++w) sum += sm.red[r][w][col];
      a.part_bc[(((int64_t)l.tile * a.total_rows + row0 + tb + r) * a.groups + l.group) * 2 * n + m] = sum;
    }
  }
#pragma unroll
  for (int w = 1; w < RB; w *= 2) {
    dD += __shfl_xor_sync(0xffffffffu, dD, w);
    dbias += __shfl_xor_sync(0xffffffffu, dbias, w);
  }
  if (l.valid) {
    const int64_t at = (int64_t)l.unit * a.channels + l.c;
    unpack2(dA[0], v[0], v[1]);
    unpack2(dA[1], v[2], v[3]);
    scan_store4(a.part_a + at * n, l.n0, n, 0, v);
    if (l.j == 0) {
      if (a.dD) a.part_d[at] = dD;
      if (a.ddt_bias) a.part_s[at] = dbias;
    }
    if (a.dstate && t0 == 0) {
      const ScanPlace p = scan_place(a.table, nk, 11, l.k);
      unpack2(carry[0], v[0], v[1]);
      unpack2(carry[1], v[2], v[3]);
      scan_store4(a.dstate + p.start + l.c * p.stride, l.n0, n, a.state_vec, v);
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

template <typename K>
static cudaError_t scan_allow_smem(K kernel, size_t smem) {
  return smem > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
}
#define SCAN_TRY(call)                       \
  do {                                       \
    cudaError_t e__ = (call);                \
    if (e__ != cudaSuccess) return e__;      \
  } while (0)

static cudaError_t scan_join(cudaStream_t s, ScanJoin j) {
  j.per_seq = j.channels * j.n_states;
  return nb2_launch(nb2_scan_join_kernel, dim3((unsigned)((j.per_seq * j.n_seq + 255) / 256)), dim3(256), 0, s, j);
}

template <typename T, int S, bool VEC>
static cudaError_t scan_launch_units(cudaStream_t s, const nb2_selective_scan_args& a) {
  constexpr int R = S <= 4 ? 32 : 16;
  const dim3 grid((unsigned)a.n_units * a.groups * scan_tiles(a.channels, a.groups, S)), block(SCAN_THREADS);
  const size_t smem = 2 * sizeof(ScanStage<T, S, R, 3>) + sizeof(ScanRows<S, R>);
  if (a.ends) {
    SCAN_TRY(scan_allow_smem(nb2_selective_scan_kernel<T, S, VEC, true>, smem));
    SCAN_TRY(nb2_launch(nb2_selective_scan_kernel<T, S, VEC, true>, grid, block, smem, s, a));
    SCAN_TRY(scan_join(s, ScanJoin{a.table, a.n_seq, a.n_states, a.unit_rows, 0, a.channels, 0, 18, a.A, a.state, 6, a.ends, a.sums}));
  }
  SCAN_TRY(scan_allow_smem(nb2_selective_scan_kernel<T, S, VEC, false>, smem));
  return nb2_launch(nb2_selective_scan_kernel<T, S, VEC, false>, grid, block, smem, s, a);
}

template <typename T, int S, bool VEC>
static cudaError_t scan_grad_units(cudaStream_t s, const nb2_selective_scan_grad_args& a) {
  constexpr int R = NB2_SCAN_KEEP;
  const dim3 grid((unsigned)a.n_units * a.groups * scan_tiles(a.channels, a.groups, S)), block(SCAN_THREADS);
  if (a.ends) {
    const size_t smem = 2 * sizeof(ScanStage<T, S, R, 3>) + sizeof(ScanRows<S, R>);
    SCAN_TRY(scan_allow_smem(nb2_scan_grad_ends_kernel<T, S, VEC>, smem));
    SCAN_TRY(nb2_launch(nb2_scan_grad_ends_kernel<T, S, VEC>, grid, block, smem, s, a));
    SCAN_TRY(scan_join(s, ScanJoin{a.table, a.n_seq, a.n_states, a.unit_rows, 1, a.channels, 0, 29, a.A, a.dnew_state, 12, a.ends, a.sums}));
  }
  const size_t smem = 2 * sizeof(ScanStage<T, S, R, 4>) + sizeof(ScanGradSmem<S>);
  SCAN_TRY(scan_allow_smem(nb2_selective_scan_grad_kernel<T, S, VEC>, smem));
  return nb2_launch(nb2_selective_scan_grad_kernel<T, S, VEC>, grid, block, smem, s, a);
}

template <typename T, int S>
static cudaError_t scan_launch(cudaStream_t s, const nb2_selective_scan_args& a) {
  if (a.tokens) {
    const int block = SCAN_THREADS / S, per_block = 4 * block, tiles = (a.channels + per_block - 1) / per_block;
    return nb2_launch(nb2_selective_scan_token_kernel<T, S>, dim3((unsigned)a.n_seq * tiles), dim3(SCAN_THREADS), 0, s, a,
                      tiles, per_block);
  }
  return a.rows_vec && a.vec ? scan_launch_units<T, S, true>(s, a) : scan_launch_units<T, S, false>(s, a);
}

template <typename T, int S>
static cudaError_t scan_grad_launch(cudaStream_t s, const nb2_selective_scan_grad_args& a) {
  return a.rows_vec && a.vec ? scan_grad_units<T, S, true>(s, a) : scan_grad_units<T, S, false>(s, a);
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
  if (a.tokens) {
    NB2_REQUIRE(!a.keep, "rows are kept by the walk over units only");
  } else {
    NB2_REQUIRE(a.units && a.n_units >= a.n_seq && a.unit_rows >= 1 && a.unit_rows % NB2_SCAN_KEEP == 0, "units");
    NB2_REQUIRE((int64_t)a.n_units * (a.channels + a.groups) < (1ll << 31), "too many units x channels");
    NB2_REQUIRE(!a.ends || a.sums, "null pointer");
    NB2_REQUIRE(a.ends || a.n_units == a.n_seq, "units of a sequence need their states");
    NB2_REQUIRE(!a.ends || (int64_t)a.n_seq * a.channels * a.n_states < (1ll << 38), "too many states");
  }
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
  NB2_REQUIRE(a.units && a.n_units >= a.n_seq && a.unit_rows >= 1 && a.unit_rows % NB2_SCAN_KEEP == 0, "units");
  NB2_REQUIRE((int64_t)a.n_units * (a.channels + a.groups) < (1ll << 31), "too many units x channels");
  NB2_REQUIRE(!a.ends || a.sums, "null pointer");
  NB2_REQUIRE(a.ends || a.n_units == a.n_seq, "units of a sequence need their gradients");
  cudaStream_t s = nb2_stream(stream);
  const int tiles = scan_tiles(a.channels, a.groups, scan_lanes(a.n_states));
  NB2_SEQ_DTYPE(a.dtype, SCAN_BY_LANES(scan_lanes(a.n_states), scan_grad_launch));
  if (a.total_rows > 0) {
    const int64_t wide = (a.total_rows * a.groups * 2 * a.n_states + 255) / 256;
    const int64_t per = (wide + a.n_seq - 1) / a.n_seq;
    const dim3 grid((unsigned)(per < 8192 ? per : 8192), (unsigned)a.n_seq);
    NB2_SEQ_DTYPE(a.dtype, NB2_CUDA(nb2_launch(nb2_scan_grad_bc_kernel<T>, grid, dim3(256), 0, s, a, tiles)));
  }
  NB2_CUDA(nb2_seq_sum_parts(s, a.part_a, a.n_units, (int64_t)a.channels * a.n_states, a.dA));
  if (a.dD) NB2_CUDA(nb2_seq_sum_parts(s, a.part_d, a.n_units, a.channels, a.dD));
  if (a.ddt_bias) NB2_CUDA(nb2_seq_sum_parts(s, a.part_s, a.n_units, a.channels, a.ddt_bias));
  return NB2_OK;
}
