// Backward pass of the selective scan.
#include "nb2_seq_scan.cuh"

// Backward.  With dp = dy silu(z), g[t] = C dp + a[t+1] g[t+1] (at the end: dnew_state):
//   dz = dy p silu'(z), u = sum_n g B, dx = D dp + s u, ds = x u + sum_n g a h[t-1] A,
//   ddt = ds softplus', dA = sum_t g a h[t-1] s, dB = sum_c g s x, dC = sum_c dp h, dstate = a[0] g[0].
// A block walks its unit's NB2_SCAN_KEEP-row tiles from the last to the first: it recomputes a tile's decays
// and states from the kept state into registers, then goes back through its rows.  Units as in the forward
// pass, run through from the last: nb2_scan_grad_ends_kernel leaves the gradient that each would hand on if it
// received zero.
//
// Bound by shared-memory words and issue slots: a lane reads 26 words a row (B and C twice, the prepared rows) and the
// sums over channels and states are 9 shuffles.  Measured (B200, 2 x 2048 rows x 2048 channels x 16 states, float32): both
// passes 424 us, of which this walk about 225; 16 x 512 rows 652.  Four blocks a multiprocessor against three and five:
// 424 / 456 / 483 us; above 32 states three (64 states 2.22 ms against 2.27 with four).  Two channels to a lane spilled,
// which an earlier form of this walk paid with a tenth.
enum ScanGradArrays { kDt, kX, kDy, kZ, kB, kC, kDx, kDdt, kDz, kArrays };
template <int S>
struct ScanGradSmem {
  static constexpr int R = NB2_SCAN_KEEP;
  ScanArray arrays[kArrays];
  ScanRows<S, 1, R> ready;
  float dp[R][ScanRows<S, 1, R>::kPitch];
  float4 kept[2][SCAN_THREADS];  // the lanes' states before a tile, of this one and the next
  float4 sums[R][SCAN_THREADS / S];  // over the states: g B, g a h[t-1] A log2(e), C h
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
  constexpr int R = NB2_SCAN_KEEP, RB = S < 4 ? S : 4;
  constexpr int NA = 3;
  using Stage = ScanStage<T, S, 1, R, NA>;
  extern __shared__ __align__(16) char smem_raw[];
  Stage* stages = reinterpret_cast<Stage*>(smem_raw);
  ScanRows<S, 1, R>& ready = *reinterpret_cast<ScanRows<S, 1, R>*>(smem_raw + 2 * sizeof(Stage));
  nb2_pdl_wait();
  const ScanLane<S, 1> l(a.channels, a.groups, a.units);
  const int n = a.n_states, c = l.channel(0);
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
  scan_rates(a.A + (int64_t)c * n, l.n0, n, A2);
  const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f;
  const int j = l.j % RB, mine = l.in_block;
  float total = 0.0f;
  scan_clear_weights(stages, 2);
  __syncthreads();
  ScanWeights<VEC, T, S, R> weights(n);
  ScanCopy<VEC, T, Stage> copy[NA];
  auto fetch = [&](Stage& st, int64_t from, int rows) {
    copy[0].load(st.in[0], dt + from * pt.stride, pt.stride, rows, l.width);
    copy[1].load(st.in[1], dy + from * pdy.stride, pdy.stride, rows, l.width);
    if (z)
      copy[2].load(st.in[2], z + from * pz.stride, pz.stride, rows, l.width);
    weights.load(B + from * pb.stride, pb.stride, C + from * pc.stride, pc.stride, n, rows);
  };
  auto arrive = [&](Stage& st) {
    weights.store(st.bc);
#pragma unroll
    for (int i = 0; i < NA; ++i) copy[i].store(st.in[i]);
  };
  const int64_t all = t1 - t0, last = (all - 1) / R * R;
  fetch(stages[0], last, (int)(all - last));
  arrive(stages[0]);
  int cur = 0;
  for (int64_t tb = last; tb >= 0; tb -= R, cur ^= 1) {
    const int rows = (int)min((int64_t)R, all - tb);
    scan_cp_wait();
    __syncthreads();
    const Stage& st = stages[cur];
    if (tb > 0) fetch(stages[cur ^ 1], tb - R, R);
    scan_switch(a.softplus, [&](auto soft) {
      scan_switch(z != nullptr, [&](auto gated) {
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += RB) {
          const int r = r0 + j;
          float2 o;  // (s, dp)
          o.x = nb2_to_float(st.in[0][r][mine]) + bias;
          if (decltype(soft)::value) o.x = scan_softplus(o.x);
          o.y = nb2_to_float(st.in[1][r][mine]);
          if (decltype(gated)::value) {
            const float zv = nb2_to_float(st.in[2][r][mine]);
            o.y *= zv * nb2_sigmoid(zv);
          }
          if (r >= rows) o = make_float2(0.0f, 0.0f);
          total += o.x;
          if (RB == S || l.j < RB) ready.sx[r][mine] = o;
        }
      });
    });
    __syncwarp();
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      const float2 sd = ready.sx[r][mine];
      const f32x2 s2 = pack2(sd.x, sd.x), d2 = pack2(sd.y, sd.y);
      const ulonglong2 cw = *reinterpret_cast<const ulonglong2*>(&st.bc[r][1][l.n0]);
      g[0] = mul2(scan_decay2(s2, A2[0]), fma2(cw.x, d2, g[0]));
      g[1] = mul2(scan_decay2(s2, A2[1]), fma2(cw.y, d2, g[1]));
    }
    if (tb > 0) arrive(stages[cur ^ 1]);
  }
#pragma unroll
  for (int w = 1; w < RB; w *= 2) total += __shfl_xor_sync(0xffffffffu, total, w);
  if (l.valid(0)) {
    float v[4];
    unpack2(g[0], v[0], v[1]);
    unpack2(g[1], v[2], v[3]);
    const int64_t at = (int64_t)l.unit * a.channels + c;
    scan_store4(a.ends + at * n, l.n0, n, n % 4 == 0, v);
    if (l.j == 0) a.sums[at] = total;
  }
}

template <typename T, int S, bool VEC>
__global__ void __launch_bounds__(SCAN_THREADS, S < 16 ? 4 : 3) nb2_selective_scan_grad_kernel(const nb2_selective_scan_grad_args a) {
  constexpr int R = NB2_SCAN_KEEP, RB = S < 4 ? S : 4;
  constexpr int NA = 4;
  using Stage = ScanStage<T, S, 1, R, NA, true>;
  using Sum = ScanChannelSum<S>;
  extern __shared__ __align__(16) char smem_raw[];
  Stage* stages = reinterpret_cast<Stage*>(smem_raw);
  ScanGradSmem<S>& sm = *reinterpret_cast<ScanGradSmem<S>*>(smem_raw + 2 * sizeof(Stage));
  nb2_pdl_wait();
  const ScanLane<S, 1> l(a.channels, a.groups, a.units);
  const int n = a.n_states, c = l.channel(0), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t len = a.table[l.k], t0 = l.first, t1 = min(t0 + a.unit_rows, len), nk = a.n_seq;
  if (tid < kArrays) {
    const int field[kArrays] = {1, 0, 5, 4, 2, 3, 6, 7, 10};
    const void* const base[kArrays] = {a.dt, a.x, a.dy, a.z, a.B, a.C, a.dx, a.ddt, a.dz};
#pragma unroll
    for (int q = 0; q < kArrays; ++q)
      if (tid == q) {
        const ScanPlace p = scan_place(a.table, nk, field[q], l.k);
        const int64_t column = q == kB || q == kC ? (int64_t)l.group * n : l.c0;
        sm.arrays[q].p = (char*)base[q] + (p.start + t0 * p.stride + column) * (int64_t)sizeof(T);
        sm.arrays[q].stride = p.stride;
      }
  }
  const bool gate = a.z != nullptr, dgate = a.dz != nullptr;
  const float* keep = a.keep + ((a.table[27 * nk + l.k] + t0 / R) * a.channels + c) * n;
  const int64_t row0 = a.table[28 * nk + l.k] + t0;
  f32x2 A2[2], carry[2], dA[2] = {0, 0};
  float v[4];
  scan_rates(a.A + (int64_t)c * n, l.n0, n, A2);
#pragma unroll
  for (int m = 0; m < 4; ++m) v[m] = 0.0f;
  if (l.valid(0)) {
    if (a.ends)
      scan_load4(a.ends + ((int64_t)l.unit * a.channels + c) * n, l.n0, n, n % 4 == 0, v);
    else if (a.dnew_state) {
      const ScanPlace p = scan_place(a.table, nk, 12, l.k);
      scan_load4(a.dnew_state + p.start + c * p.stride, l.n0, n, a.state_vec, v);
    }
  }
  carry[0] = pack2(v[0], v[1]);
  carry[1] = pack2(v[2], v[3]);
  const float D = a.D ? a.D[c] : 0.0f, bias = a.dt_bias ? a.dt_bias[c] : 0.0f;
  const int j = l.j % RB, mine = l.in_block;
  const bool stores = l.valid(0) && l.j < RB;
  // A lane without a channel adds nothing to dB and dC: steps, gradients, weights and states of zero.
  const int bc0 = l.valid(0) ? l.n0 : 4 * S;
  float dD = 0.0f, dbias = 0.0f;
  sm.kept[0][tid] = sm.kept[1][tid] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // (only real states are written)
  scan_clear_weights(stages, 2);
  __syncthreads();
  ScanWeights<VEC, T, S, R> weights(n);
  ScanCopy<VEC, T, Stage> copy[NA];
  auto fetch = [&](Stage& st, int64_t from, int rows) {
#pragma unroll
    for (int q = 0; q < NA; ++q)
      if (q != kZ || gate) {
        const ScanArray r = sm.arrays[q];
        copy[q].load(st.in[q], (const T*)r.p + from * r.stride, r.stride, rows, l.width);
      }
    const ScanArray b = sm.arrays[kB], c = sm.arrays[kC];
    weights.load((const T*)b.p + from * b.stride, b.stride, (const T*)c.p + from * c.stride, c.stride, n, rows);
    if (l.valid(0)) {
      const float* k = keep + from / R * a.channels * n + l.n0;
      float* to = reinterpret_cast<float*>(&sm.kept[&st - stages][tid]);
      if (n % 4 == 0) {
        if (l.n0 < n) scan_cp_async(to, k, 16);
      } else {
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (l.n0 + m < n) scan_cp_async4(to + m, k + m);
      }
    }
  };
  auto arrive = [&](Stage& st) {
    weights.store(st.bc);
#pragma unroll
    for (int i = 0; i < NA; ++i) copy[i].store(st.in[i]);
  };
  auto put = [&](int q, int64_t row, float v) {
    const ScanArray r = sm.arrays[q];
    ((T*)r.p)[row * r.stride + mine] = nb2_from_float<T>(v);
  };
  const int64_t all = t1 - t0, last = (all - 1) / R * R;
  if (all > 0) {
    fetch(stages[0], last, (int)(all - last));
    arrive(stages[0]);
  }
  int cur = 0;
  for (int64_t tb = all > 0 ? last : -1; tb >= 0; tb -= R, cur ^= 1) {
    const int rows = (int)min((int64_t)R, all - tb);
    scan_cp_wait();
    __syncthreads();
    const Stage& st = stages[cur];
    const ulonglong2& start = *reinterpret_cast<const ulonglong2*>(&sm.kept[cur][tid]);
    if (tb > 0) fetch(stages[cur ^ 1], tb - R, R);
    scan_switch(a.softplus, [&](auto soft) {
      scan_switch(gate, [&](auto gated) {
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += RB) {
          const int r = r0 + j;
          float2 o;
          o.x = nb2_to_float(st.in[0][r][mine]) + bias;
          if (decltype(soft)::value) o.x = scan_softplus(o.x);
          o.y = o.x * nb2_to_float(st.in[1][r][mine]);
          float dp = nb2_to_float(st.in[2][r][mine]);
          if (decltype(gated)::value) {
            const float zv = nb2_to_float(st.in[3][r][mine]);
            dp *= zv * nb2_sigmoid(zv);
          }
          if (r >= rows || !l.valid(0)) {
            o = make_float2(0.0f, 0.0f);
            dp = 0.0f;
          }
          if (RB == S || l.j < RB) {
            sm.ready.sx[r][mine] = o;
            sm.dp[r][mine] = dp;
          }
        }
      });
    });
    __syncwarp();
    // Half a tile at a time, the later one first: its decays and states stay in registers for the way back.
    // (The later half's start costs its rows' decays once more, which the registers for 16 rows would cost in
    // resident warps.)
    constexpr int H = R / 2;
    f32x2 mid[2] = {start.x, start.y};
    if (rows > H)
#pragma unroll
      for (int r = 0; r < H; ++r) {
        f32x2 s2[1], x2[1];
        sm.ready.get(r, mine, s2, x2);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[r][0][bc0]);
        mid[0] = fma2(scan_decay2(s2[0], A2[0]), mid[0], mul2(x2[0], b.x));
        mid[1] = fma2(scan_decay2(s2[0], A2[1]), mid[1], mul2(x2[0], b.y));
      }
#pragma unroll 1
    for (int rb = rows > H ? H : 0; rb >= 0; rb -= H) {
      const f32x2 from[2] = {rb ? mid[0] : start.x, rb ? mid[1] : start.y};
      f32x2 h[H][2], dec[H][2];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        f32x2 s2[1], x2[1];
        sm.ready.get(rb + i, mine, s2, x2);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[rb + i][0][bc0]);
        dec[i][0] = scan_decay2(s2[0], A2[0]);
        dec[i][1] = scan_decay2(s2[0], A2[1]);
        h[i][0] = fma2(dec[i][0], i ? h[i ? i - 1 : 0][0] : from[0], mul2(x2[0], b.x));
        h[i][1] = fma2(dec[i][1], i ? h[i ? i - 1 : 0][1] : from[1], mul2(x2[0], b.y));
      }
#pragma unroll
      for (int q = H - RB; q >= 0; q -= RB) {
        float pu[RB], pe[RB], ps[RB];
#pragma unroll
        for (int i = RB - 1; i >= 0; --i) {
          const int r = rb + q + i;
          f32x2 s2[1], x2[1];
          sm.ready.get(r, mine, s2, x2);
          const float dp = sm.dp[r][mine];
          const f32x2 d2 = pack2(dp, dp);
          const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&st.bc[r][0][bc0]);
          const ulonglong2 cw = *reinterpret_cast<const ulonglong2*>(&st.bc[r][1][bc0]);
          const f32x2 h0 = h[q + i][0], h1 = h[q + i][1];
          const f32x2 g0 = fma2(cw.x, d2, carry[0]), g1 = fma2(cw.y, d2, carry[1]);
          carry[0] = mul2(g0, dec[q + i][0]);
          carry[1] = mul2(g1, dec[q + i][1]);
          const f32x2 q0 = mul2(carry[0], q + i ? h[q + i ? q + i - 1 : 0][0] : from[0]);
          const f32x2 q1 = mul2(carry[1], q + i ? h[q + i ? q + i - 1 : 0][1] : from[1]);
          if (r < rows) {  // (past the end the last state stands before the row: infinite, times a step of zero)
            dA[0] = fma2(q0, s2[0], dA[0]);
            dA[1] = fma2(q1, s2[0], dA[1]);
          }
          float lo, hi;
          unpack2(fma2(g1, b.y, mul2(g0, b.x)), lo, hi);
          pu[i] = lo + hi;
          unpack2(fma2(q1, A2[1], mul2(q0, A2[0])), lo, hi);
          pe[i] = lo + hi;
          unpack2(fma2(cw.y, h1, mul2(cw.x, h0)), lo, hi);
          ps[i] = lo + hi;
          float w[8];
          unpack2(mul2(g0, x2[0]), w[0], w[1]);
          unpack2(mul2(g1, x2[0]), w[2], w[3]);
          unpack2(mul2(d2, h0), w[4], w[5]);
          unpack2(mul2(d2, h1), w[6], w[7]);
          Sum::sum(w, lane);
          if (Sum::writes(lane)) {
            const int at = Sum::at(lane);
#pragma unroll
            for (int m = 0; m < Sum::kLeft; ++m) sm.red[r][warp][((at + m) >> 2) * 4 * S + l.n0 + ((at + m) & 3)] = w[m];
          }
        }
        float u = scan_transpose_sum<RB>(pu, j), e = scan_transpose_sum<RB>(pe, j), o = scan_transpose_sum<RB>(ps, j);
#pragma unroll
        for (int w = RB; w < S; w *= 2) {
          u += __shfl_xor_sync(0xffffffffu, u, w);
          e += __shfl_xor_sync(0xffffffffu, e, w);
          o += __shfl_xor_sync(0xffffffffu, o, w);
        }
        if (RB == S || l.j < RB) sm.sums[rb + q + j][mine] = make_float4(u, e, o, 0.0f);
      }
    }
    __syncwarp();
    float tile_D = 0.0f, tile_s = 0.0f;  // (a tile's rows apart, then the tiles: shorter chains of additions)
    scan_switch(a.softplus, [&](auto soft) {
      scan_switch(dgate, [&](auto gated) {
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += RB) {
          const int r = r0 + j;
          const float raw = nb2_to_float(st.in[0][r][mine]) + bias, xv = nb2_to_float(st.in[1][r][mine]);
          const float4 sum = sm.sums[r][mine];
          const float dp = sm.dp[r][mine], u = sum.x;
          float ds = fmaf(xv, u, sum.y * LN2), gz = 0.0f;
          if (decltype(soft)::value) ds *= nb2_sigmoid(raw);
          if (decltype(gated)::value)
            gz = nb2_to_float(st.in[2][r][mine]) * fmaf(D, xv, sum.z) * nb2_silu_slope(nb2_to_float(st.in[3][r][mine]));
          if (r < rows && stores) {
            put(kDx, tb + r, fmaf(D, dp, sm.ready.sx[r][mine].x * u));
            put(kDdt, tb + r, ds);
            if (decltype(gated)::value) put(kDz, tb + r, gz);
            tile_D = fmaf(dp, xv, tile_D);
            tile_s += ds;
          }
        }
      });
    });
    dD += tile_D;
    dbias += tile_s;
    if (tb > 0) arrive(stages[cur ^ 1]);
    __syncthreads();
    // the block's share of dB and dC: warps in order
    for (int i = tid; i < rows * 8 * S; i += SCAN_THREADS) {
      const int r = i / (8 * S), col = i % (8 * S), state = col % (4 * S), m = col < 4 * S ? state : n + state;
      if (state >= n) continue;
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
  if (l.valid(0)) {
    const int64_t at = (int64_t)l.unit * a.channels + c;
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
      scan_store4(a.dstate + p.start + c * p.stride, l.n0, n, a.state_vec, v);
    }
  }
}

// dB and dC of every row: the channel tiles' shares added in order.  A thread per value, rows of all sequences in one.
template <typename T>
__global__ void __launch_bounds__(256) nb2_scan_grad_bc_kernel(const nb2_selective_scan_grad_args a, int tiles) {
  nb2_pdl_wait();
  const int n = a.n_states, wide = a.groups * 2 * n;
  const int64_t all = a.total_rows * wide, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  float sum = 0.0f;
#pragma unroll 16
  for (int u = 0; u < tiles; ++u) sum += a.part_bc[u * all + i];
  const int64_t row = i / wide;
  const int rest = (int)(i - row * wide), group = rest / (2 * n), m = rest - group * 2 * n;
  const int64_t* before = a.table + (size_t)28 * a.n_seq;  // rows of the sequences before each
  int k = 0;
  for (int span = a.n_seq; span > 1;) {  // the last sequence that begins at or before the row (and is not empty)
    const int half = span / 2;
    if (before[k + half] <= row) k += half, span -= half;
    else span = half;
  }
  const ScanPlace p = scan_place(a.table, a.n_seq, m < n ? 8 : 9, k);
  ((T*)(m < n ? a.dB : a.dC))[p.start + (row - before[k]) * p.stride + group * n + (m < n ? m : m - n)] = nb2_from_float<T>(sum);
}

// Gradients of A, D and dt_bias: the units' shares added in order within eight interleaved runs.  A block owns 32
// columns of [channels x n_states | channels | channels].
__global__ void __launch_bounds__(256) nb2_scan_grad_sum_kernel(const nb2_selective_scan_grad_args a) {
  nb2_pdl_wait();
  __shared__ float run[8][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t states = (int64_t)a.channels * a.n_states, i = (int64_t)blockIdx.x * 32 + lane;
  const float* part = nullptr;
  float* out = nullptr;
  int64_t n = a.channels, at = i;
  if (i < states)
    part = a.part_a, out = a.dA, n = states;
  else if (i < states + a.channels)
    part = a.part_d, out = a.dD, at = i - states;
  else if (i < states + 2 * a.channels)
    part = a.part_s, out = a.ddt_bias, at = i - states - a.channels;
  run[w][lane] = out ? nb2_sum_units(part + at, n, a.n_units, w) : 0.0f;
  __syncthreads();
  if (w == 0 && out) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; ++r) sum += run[r][lane];
    out[at] = sum;
  }
}

template <typename T, int S, bool VEC>
static cudaError_t scan_grad_units(cudaStream_t s, const nb2_selective_scan_grad_args& a) {
  constexpr int R = NB2_SCAN_KEEP;
  const dim3 grid((unsigned)a.n_units * a.groups * scan_tiles(a.channels, a.groups, ScanLane<S, 1>::kBlock)), block(SCAN_THREADS);
  if (a.ends) {
    const size_t smem = 2 * sizeof(ScanStage<T, S, 1, R, 3>) + sizeof(ScanRows<S, 1, R>);
    SCAN_TRY(scan_allow_smem(nb2_scan_grad_ends_kernel<T, S, VEC>, smem));
    SCAN_TRY(nb2_launch(nb2_scan_grad_ends_kernel<T, S, VEC>, grid, block, smem, s, a));
    SCAN_TRY(nb2_scan_join(s, ScanJoin{a.table, a.n_seq, a.n_states, a.unit_rows, 1, a.channels, 0, 29, a.A, a.dnew_state, 12, a.ends, a.sums}));
  }
  const size_t smem = 2 * sizeof(ScanStage<T, S, 1, R, 4, true>) + sizeof(ScanGradSmem<S>);
  SCAN_TRY(scan_allow_smem(nb2_selective_scan_grad_kernel<T, S, VEC>, smem));
  return nb2_launch(nb2_selective_scan_grad_kernel<T, S, VEC>, grid, block, smem, s, a);
}

template <typename T, int S>
static cudaError_t scan_grad_launch(cudaStream_t s, const nb2_selective_scan_grad_args& a) {
  return a.rows_vec && a.vec ? scan_grad_units<T, S, true>(s, a) : scan_grad_units<T, S, false>(s, a);
}

extern "C" int nb2_selective_scan_grad(void* stream, const nb2_selective_scan_grad_args* args) {
  NB2_REQUIRE(args, "args");
  const nb2_selective_scan_grad_args& a = *args;
  if (int e = scan_check(a)) return e;
  NB2_REQUIRE(a.dy && a.dx && a.ddt && a.dB && a.dC && a.dA && a.keep && a.part_bc && a.part_a, "null pointer");
  NB2_REQUIRE((!a.dz || a.z) && (!a.dD || (a.D && a.part_d)) && (!a.ddt_bias || (a.dt_bias && a.part_s)), "gradients");
  if (int e = scan_check_units(a)) return e;
  cudaStream_t s = nb2_stream(stream);
  const int tiles = scan_tiles(a.channels, a.groups, SCAN_THREADS / scan_lanes(a.n_states));
  NB2_SEQ_DTYPE(a.dtype, SCAN_BY_LANES(scan_lanes(a.n_states), scan_grad_launch));
  if (a.total_rows > 0) {
    const int64_t blocks = (a.total_rows * a.groups * 2 * a.n_states + 255) / 256;
    NB2_REQUIRE(blocks < (1ll << 31), "too many rows");
    NB2_SEQ_DTYPE(a.dtype, NB2_CUDA(nb2_launch(nb2_scan_grad_bc_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, a, tiles)));
  }
  const int64_t columns = (int64_t)a.channels * (a.n_states + 2);
  NB2_CUDA(nb2_launch(nb2_scan_grad_sum_kernel, dim3((unsigned)((columns + 31) / 32)), dim3(256), 0, s, a));
  return NB2_OK;
}
