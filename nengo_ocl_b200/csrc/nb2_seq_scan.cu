// Forward pass of the selective scan: the walk over units of rows, and the kernel for single tokens.
#include "nb2_seq_scan.cuh"

// Units are stretches of unit_rows rows of a sequence.  One unit to a sequence: the block starts from its
// state and walks it to the end.  More (a long sequence of few channels): ENDS first leaves the state that
// every unit would reach from zero and the sum of its steps, nb2_scan_join_kernel turns these into the
// states that the units start from, and the second walk (ENDS false) starts there.
//
// A tile of R rows is worked in three phases, each a warp's own: its lanes prepare (s, s x) of the tile's rows
// for their channels, walk the rows through the states, and finish the outputs.
//
// Bound by the special function unit: n + 4 results a row and channel at 16 a cycle and multiprocessor, 19 us for
// 4096 rows x 1024 channels x 16 states and walk where memory needs 10 (float32).  Measured (B200): 48 x 256 rows x 4096
// channels 326 us, 0.7 of the unit busy (225 us of it at full rate); 4097 rows of 4 uneven prompts, split, 225 us.  Bounds
// of six blocks a multiprocessor (80 registers; float32's shared memory, 41 KB, holds five, 16 bits' 28 KB six) against
// five and four: 225 / 230 / 231 us, one bfloat16 prompt of 16384 x 1024 210 / 210 / 213; rows copied element by element
// need more registers: four.
#define SCAN_P 2
#define SCAN_TOKEN_BLOCKS 16
template <typename T, int S, bool VEC, bool ENDS>
__global__ void __launch_bounds__(SCAN_THREADS, VEC ? 6 : 4) nb2_selective_scan_kernel(const nb2_selective_scan_args a) {
  constexpr int P = SCAN_P, R = NB2_SCAN_KEEP, RB = S < 4 ? S : 4;
  constexpr int NA = 3;
  using Stage = ScanStage<T, S, P, R, NA>;
  extern __shared__ __align__(16) char smem_raw[];
  Stage* stages = reinterpret_cast<Stage*>(smem_raw);
  ScanRows<S, P, R>& ready = *reinterpret_cast<ScanRows<S, P, R>*>(smem_raw + 2 * sizeof(Stage));
  enum { kDt, kX, kZ, kB, kC, kY, kArrays };
  __shared__ ScanArray arrays[kArrays];
  nb2_pdl_wait();
  const ScanLane<S, P> l(a.channels, a.groups, a.units);
  const int n = a.n_states;
  const int64_t len = a.table[l.k], t0 = l.first, t1 = min(t0 + a.unit_rows, len);
  if (ENDS && t1 == len) return;  // nothing starts from the last unit's end
  const int64_t nk = a.n_seq;
  if (threadIdx.x < kArrays) {
    const int field[kArrays] = {1, 0, 5, 2, 3, 4};
    const void* const base[kArrays] = {a.dt, a.x, a.z, a.B, a.C, a.y};
#pragma unroll
    for (int q = 0; q < kArrays; ++q)
      if (threadIdx.x == q) {
        const ScanPlace p = scan_place(a.table, nk, field[q], l.k);
        const int64_t column = q == kB || q == kC ? (int64_t)l.group * n : l.c0;
        arrays[q].p = (char*)base[q] + (p.start + t0 * p.stride + column) * (int64_t)sizeof(T);
        arrays[q].stride = p.stride;
      }
  }
  const bool gate = !ENDS && a.z;
  f32x2 A2[P][2], h[P][2];
  float D[P], bias[P], total[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = l.channel(p);
    scan_rates(a.A + (int64_t)c * n, l.n0, n, A2[p]);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!ENDS) {
      if (a.ends)
        scan_load4(a.ends + ((int64_t)l.unit * a.channels + c) * n, l.n0, n, n % 4 == 0, v);
      else if (a.state) {
        const ScanPlace ps = scan_place(a.table, nk, 6, l.k);
        scan_load4(a.state + ps.start + c * ps.stride, l.n0, n, a.state_vec, v);
      }
    }
    h[p][0] = pack2(v[0], v[1]);
    h[p][1] = pack2(v[2], v[3]);
    D[p] = !ENDS && a.D ? a.D[c] : 0.0f;
    bias[p] = a.dt_bias ? a.dt_bias[c] : 0.0f;
    total[p] = 0.0f;
  }
  float* keep = !ENDS && a.keep ? a.keep + (a.table[17 * nk + l.k] + t0 / R) * a.channels * n : nullptr;
  const int j = l.j % RB, mine = l.in_block;
  const int stores = l.j < RB ? l.width - mine : 0;  // of the lane's channels

  scan_clear_weights(stages, 2);  // the padding states' stay zero: only the real ones are written
  __syncthreads();
  ScanWeights<VEC, T, S, R> weights(n);
  ScanCopy<VEC, T, Stage> copy[NA];
  auto fetch = [&](Stage& st, int64_t from, int rows) {
#pragma unroll
    for (int q = 0; q < NA; ++q)
      if (q != kZ || gate) {
        const ScanArray r = arrays[q];
        copy[q].load(st.in[q], (const T*)r.p + from * r.stride, r.stride, rows, l.width);
      }
    const ScanArray b = arrays[kB], c = arrays[kC];
    weights.load((const T*)b.p + from * b.stride, b.stride, (const T*)c.p + from * c.stride, c.stride, n, rows);
  };
  auto arrive = [&](Stage& st) {
    weights.store(st.bc);
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (i != kZ || gate) copy[i].store(st.in[i]);
  };
  const int64_t all = t1 - t0;
  if (all > 0) {
    fetch(stages[0], 0, (int)min((int64_t)R, all));
    arrive(stages[0]);
  }
  int cur = 0;
  for (int64_t tb = 0; tb < all; tb += R, cur ^= 1) {
    const int rows = (int)min((int64_t)R, all - tb), next = (int)min((int64_t)R, all - tb - rows);
    scan_cp_wait();
    __syncthreads();
    const Stage& st = stages[cur];
    if (next > 0) fetch(stages[cur ^ 1], tb + R, next);
    if (keep) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float v[4];
        unpack2(h[p][0], v[0], v[1]);
        unpack2(h[p][1], v[2], v[3]);
        if (l.valid(p)) scan_store4(keep + (int64_t)l.channel(p) * n, l.n0, n, n % 4 == 0, v);
      }
      keep += (int64_t)a.channels * n;
    }
    scan_switch(a.softplus, [&](auto soft) {
#pragma unroll
      for (int r0 = 0; r0 < R; r0 += RB) {
        const int r = r0 + j;
        float s[P], xv[P];
        scan_get<T, P>(&st.in[0][r][mine], s);
        scan_get<T, P>(&st.in[1][r][mine], xv);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          s[p] += bias[p];
          if (decltype(soft)::value) s[p] = scan_softplus(s[p]);
          xv[p] *= s[p];
          if (r >= rows) s[p] = xv[p] = 0.0f;  // (whatever lies past the end: read, not used)
          if (ENDS) total[p] += s[p];
        }
        if (RB == S || l.j < RB) ready.put(r, mine, s, xv);
      }
    });
    __syncwarp();
    // Blocks of RB rows; what does not wait for the state (decays, inputs) is computed a block ahead.
    float out[R / RB][P];
    f32x2 dec[2][RB][P][2], in[2][RB][P][2];
    auto ahead = [&](int r0, f32x2 (&d)[RB][P][2], f32x2 (&u)[RB][P][2]) {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        f32x2 s2[P], x2[P];
        ready.get(r0 + i, mine, s2, x2);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[r0 + i][0][l.n0]);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          d[i][p][0] = scan_decay2(s2[p], A2[p][0]);
          d[i][p][1] = scan_decay2(s2[p], A2[p][1]);
          u[i][p][0] = mul2(x2[p], b.x);
          u[i][p][1] = mul2(x2[p], b.y);
        }
      }
    };
    ahead(0, dec[0], in[0]);
#pragma unroll
    for (int q = 0; q < R / RB; ++q) {
      float sum[P][RB];
#pragma unroll
      for (int i = 0; i < RB; ++i) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          h[p][0] = fma2(dec[q & 1][i][p][0], h[p][0], in[q & 1][i][p][0]);
          h[p][1] = fma2(dec[q & 1][i][p][1], h[p][1], in[q & 1][i][p][1]);
        }
        if (!ENDS) {
          const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&st.bc[q * RB + i][1][l.n0]);
#pragma unroll
          for (int p = 0; p < P; ++p) {
            float lo, hi;
            unpack2(fma2(c.y, h[p][1], mul2(c.x, h[p][0])), lo, hi);
            sum[p][i] = lo + hi;
          }
        }
      }
      if (q + 1 < R / RB) ahead((q + 1) * RB, dec[(q + 1) & 1], in[(q + 1) & 1]);
      if (!ENDS) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
          float o = scan_transpose_sum<RB>(sum[p], j);
#pragma unroll
          for (int w = RB; w < S; w *= 2) o += __shfl_xor_sync(0xffffffffu, o, w);
          out[q][p] = o;
        }
      }
    }
    if (!ENDS) {
      const ScanArray to = arrays[kY];
      T* y = (T*)to.p + mine;
      scan_switch(gate, [&](auto gated) {
#pragma unroll
        for (int q = 0; q < R / RB; ++q) {
          const int r = q * RB + j;
          float xv[P], o[P], zv[P];
          scan_get<T, P>(&st.in[1][r][mine], xv);
          if (decltype(gated)::value) scan_get<T, P>(&st.in[2][r][mine], zv);
#pragma unroll
          for (int p = 0; p < P; ++p) {
            o[p] = fmaf(D[p], xv[p], out[q][p]);
            if (decltype(gated)::value) o[p] *= zv[p] * nb2_sigmoid(zv[p]);
          }
          if (r < rows) scan_put<VEC, T, P>(y + (tb + r) * to.stride, o, stores);
        }
      });
    }
    if (next > 0) arrive(stages[cur ^ 1]);
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float v[4];
    unpack2(h[p][0], v[0], v[1]);
    unpack2(h[p][1], v[2], v[3]);
    const int c = l.channel(p);
    if (ENDS) {
#pragma unroll
      for (int w = 1; w < RB; w *= 2) total[p] += __shfl_xor_sync(0xffffffffu, total[p], w);
      if (l.valid(p)) {
        const int64_t at = (int64_t)l.unit * a.channels + c;
        scan_store4(a.ends + at * n, l.n0, n, n % 4 == 0, v);
        if (l.j == 0) a.sums[at] = total[p];
      }
    } else if (a.new_state && l.valid(p) && t1 == len) {
      const ScanPlace ps = scan_place(a.table, nk, 7, l.k);
      scan_store4(a.new_state + ps.start + c * ps.stride, l.n0, n, a.state_vec, v);
    }
  }
}

// From what the units reach from zero to what they start from, in order of time (the states) or against it
// (the gradients): start' = exp(A sum s) start + end.  A thread per (sequence, channel, state).
__global__ void __launch_bounds__(256) nb2_scan_join_kernel(const ScanJoin a) {
  nb2_pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int k = (int)(i / a.per_seq);
  if (k >= a.n_seq) return;
  const int64_t cn = i - k * a.per_seq, c = cn / a.n_states, len = a.table[k];
  const int64_t u0 = a.table[a.first_unit_field * a.n_seq + k], units = max((len + a.unit_rows - 1) / a.unit_rows, (int64_t)1);
  const float A2 = scan_rate(a.A[cn]);
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
      // row by row a growing state reaches infinity only where it is: nothing comes of zero, and half the exponent at
      // a time a small start does not meet a factor past the range
      const float half = scan_exp2(0.5f * (s[q] * A2));
      h = h == 0.0f ? e[q] : fmaf(half, half * h, e[q]);
    }
  }
}

cudaError_t nb2_scan_join(cudaStream_t s, ScanJoin j) {
  j.per_seq = j.channels * j.n_states;
  return nb2_launch(nb2_scan_join_kernel, dim3((unsigned)((j.per_seq * j.n_seq + 255) / 256)), dim3(256), 0, s, j);
}

// Single tokens and a few rows: the states are most of the traffic, one read and one write of each.  A block keeps
// its channels' parameters and takes one sequence after the other, the next one's state and first row on their
// way while it works.  Bound by memory, 8 bytes a state; measured 50 us = 2.9 TB/s for 256 tokens x 4096 channels x 16
// states, with the table read from memory per sequence 58, one block per sequence and 128 channels 81; eight blocks a
// multiprocessor (64 registers) against six: 51 / 59 us; channels of a lane 1 / 2 / 4: 60 / 51 / 74 us.
constexpr int kTokenUnroll = 2;  // channels of a lane, SCAN_THREADS / S apart
constexpr int kTokenSequences = 64, kTokenFields = 17;  // of a block; of the table: the length and eight (start, stride)
template <typename T, int S>
struct ScanToken {
  float h[kTokenUnroll][4], b[4], c[4], dt[kTokenUnroll], x[kTokenUnroll], z[kTokenUnroll];
  // seq: the sequence's fields of the table
  __device__ __forceinline__ void row(const nb2_selective_scan_args& a, const int64_t* seq, int64_t t,
                                      const int (&ch)[kTokenUnroll], int group, int n0) {
    const int n = a.n_states;
    scan_load4((const T*)a.B + seq[5] + t * seq[6] + (int64_t)group * n, n0, n, a.vec, b);
    scan_load4((const T*)a.C + seq[7] + t * seq[8] + (int64_t)group * n, n0, n, a.vec, c);
    const T* xr = (const T*)a.x + seq[1] + t * seq[2];
    const T* tr = (const T*)a.dt + seq[3] + t * seq[4];
    const T* zr = a.z ? (const T*)a.z + seq[11] + t * seq[12] : nullptr;
#pragma unroll
    for (int u = 0; u < kTokenUnroll; ++u) {
      dt[u] = nb2_to_float(tr[ch[u]]);
      x[u] = nb2_to_float(xr[ch[u]]);
      z[u] = zr ? nb2_to_float(zr[ch[u]]) : 0.0f;
    }
  }
  __device__ __forceinline__ void load(const nb2_selective_scan_args& a, const int64_t* seq, const int (&ch)[kTokenUnroll],
                                       int group, int n0) {
#pragma unroll
    for (int u = 0; u < kTokenUnroll; ++u) {
#pragma unroll
      for (int m = 0; m < 4; ++m) h[u][m] = 0.0f;
      if (a.state) scan_load4(a.state + seq[13] + ch[u] * seq[14], n0, a.n_states, a.state_vec, h[u]);
    }
    if (seq[0] > 0) row(a, seq, 0, ch, group, n0);
  }
};

template <typename T, int S>
__global__ void __launch_bounds__(SCAN_THREADS, 8) nb2_selective_scan_token_kernel(const nb2_selective_scan_args a, int tiles, int each) {
  constexpr int U = kTokenUnroll, kStep = SCAN_THREADS / S;
  __shared__ int64_t table[kTokenSequences][kTokenFields];
  nb2_pdl_enter();
  const int j = threadIdx.x % S, n0 = 4 * j, n = a.n_states, per = a.channels / a.groups;
  const int tile = blockIdx.x % tiles, group = tile / (tiles / a.groups), in = (tile - group * (tiles / a.groups)) * kStep * U;
  const int64_t k0 = (int64_t)(blockIdx.x / tiles) * each, k1 = min(k0 + each, (int64_t)a.n_seq);
  for (int i = threadIdx.x; i < (k1 - k0) * kTokenFields; i += SCAN_THREADS)
    table[i / kTokenFields][i % kTokenFields] = a.table[(int64_t)(i % kTokenFields) * a.n_seq + k0 + i / kTokenFields];
  int ch[U];
  bool valid[U];
  float A2[U][4], D[U], bias[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int at = in + u * kStep + threadIdx.x / S;
    valid[u] = at < per;
    ch[u] = group * per + min(at, per - 1);
    scan_load4(a.A + (int64_t)ch[u] * n, n0, n, n % 4 == 0 && a.a_vec, A2[u]);
#pragma unroll
    for (int m = 0; m < 4; ++m) A2[u][m] = scan_rate(A2[u][m]);
    D[u] = a.D ? a.D[ch[u]] : 0.0f;
    bias[u] = a.dt_bias ? a.dt_bias[ch[u]] : 0.0f;
  }
  __syncthreads();
  auto work = [&](ScanToken<T, S>& s, const int64_t* seq) {
    for (int64_t t = 0; t < seq[0]; ++t) {
      if (t > 0) s.row(a, seq, t, ch, group, n0);
      T* yr = (T*)a.y + seq[9] + t * seq[10];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float step = s.dt[u] + bias[u], o = 0.0f;
        if (a.softplus) step = scan_softplus(step);
        const float sx = step * s.x[u];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          s.h[u][m] = fmaf(scan_decay(step, A2[u][m]), s.h[u][m], sx * s.b[m]);
          o = fmaf(s.c[m], s.h[u][m], o);
        }
#pragma unroll
        for (int w = 1; w < S; w *= 2) o += __shfl_xor_sync(0xffffffffu, o, w);
        o = fmaf(D[u], s.x[u], o);
        if (a.z) o *= s.z[u] * nb2_sigmoid(s.z[u]);
        if (j == 0 && valid[u]) yr[ch[u]] = nb2_from_float<T>(o);
      }
    }
    if (a.new_state)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (valid[u]) scan_store4(a.new_state + seq[15] + ch[u] * seq[16], n0, n, a.state_vec, s.h[u]);
  };
  ScanToken<T, S> even, odd;
  const int count = (int)(k1 - k0);
  if (count > 0) even.load(a, table[0], ch, group, n0);
  for (int k = 0; k < count; k += 2) {
    if (k + 1 < count) odd.load(a, table[k + 1], ch, group, n0);
    work(even, table[k]);
    if (k + 2 < count) even.load(a, table[k + 2], ch, group, n0);
    if (k + 1 < count) work(odd, table[k + 1]);
  }
}

template <typename T, int S, bool VEC>
static cudaError_t scan_launch_units(cudaStream_t s, const nb2_selective_scan_args& a) {
  constexpr int P = SCAN_P, R = NB2_SCAN_KEEP;
  const dim3 grid((unsigned)a.n_units * a.groups * scan_tiles(a.channels, a.groups, ScanLane<S, P>::kBlock)), block(SCAN_THREADS);
  const size_t smem = 2 * sizeof(ScanStage<T, S, P, R, 3>) + sizeof(ScanRows<S, P, R>);
  if (a.ends) {
    SCAN_TRY(scan_allow_smem(nb2_selective_scan_kernel<T, S, VEC, true>, smem));
    SCAN_TRY(nb2_launch(nb2_selective_scan_kernel<T, S, VEC, true>, grid, block, smem, s, a));
    SCAN_TRY(nb2_scan_join(s, ScanJoin{a.table, a.n_seq, a.n_states, a.unit_rows, 0, a.channels, 0, 18, a.A, a.state, 6, a.ends, a.sums}));
  }
  SCAN_TRY(scan_allow_smem(nb2_selective_scan_kernel<T, S, VEC, false>, smem));
  return nb2_launch(nb2_selective_scan_kernel<T, S, VEC, false>, grid, block, smem, s, a);
}

template <typename T, int S>
static cudaError_t scan_launch(cudaStream_t s, const nb2_selective_scan_args& a) {
  if (a.tokens) {
    // as many blocks to a tile of channels as fill the GPU a few times, each with its share of the sequences
    const int tiles = a.groups * scan_tiles(a.channels, a.groups, SCAN_THREADS / S * kTokenUnroll);
    const int blocks = max(1, min(a.n_seq, SCAN_TOKEN_BLOCKS * NB2_NUM_SMS / tiles)), each = min((a.n_seq + blocks - 1) / blocks, kTokenSequences);
    return nb2_launch(nb2_selective_scan_token_kernel<T, S>, dim3((unsigned)tiles * ((a.n_seq + each - 1) / each)),
                      dim3(SCAN_THREADS), 0, s, a, tiles, each);
  }
  return a.rows_vec && a.vec ? scan_launch_units<T, S, true>(s, a) : scan_launch_units<T, S, false>(s, a);
}

extern "C" int nb2_selective_scan_tile(int n_states, int backward) {
  NB2_REQUIRE(n_states >= 1 && n_states <= NB2_SCAN_MAX_STATES, "n_states");
  return SCAN_THREADS / scan_lanes(n_states) * (backward ? 1 : SCAN_P);
}

extern "C" int nb2_selective_scan(void* stream, const nb2_selective_scan_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_selective_scan_args& a = *args;
  if (int e = scan_check(a)) return e;
  NB2_REQUIRE(a.y, "null pointer");
  if (a.tokens)
    NB2_REQUIRE(!a.keep, "rows are kept by the walk over units only");
  else if (int e = scan_check_units(a))
    return e;
  cudaStream_t s = nb2_stream(stream);
  NB2_SEQ_DTYPE(a.dtype, SCAN_BY_LANES(scan_lanes(a.n_states), scan_launch));
  return NB2_OK;
}
