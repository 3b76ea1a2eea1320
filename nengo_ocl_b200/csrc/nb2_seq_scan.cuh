// Selective state space scan along the rows of sequences: the linear filter whose step size, input
// and output weights depend on the row.  Per channel c with states n (B, C shared by a group of channels):
//   s = softplus(dt + dt_bias),  a[n] = exp(s A[n]),  h[n] = a[n] h[n] + s x B[n],
//   y = (sum_n C[n] h[n] + D x) silu(z)
//
// Four states to a lane, S = 1 .. 32 lanes to a channel (S = the power of two that covers the states) and P
// neighbouring channels to a lane.  Shared memory delivers 32 words a cycle whatever they are, so every row
// of B and C that a lane loads serves its P channels.  The partial sums over the states that every lane forms for RB rows
// are transposed and added in RB - 1 shuffles, which leaves row j's sum with lane j.
#pragma once
#include "nb2_sequence.cuh"

#define SCAN_WARPS 4
#define SCAN_THREADS (32 * SCAN_WARPS)
#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f
// Added to a decay's exponent.  The hardware's exponential is on average 0.3 * 2^-24 too small just below zero (measured
// on a B200: 0.09 at exponents of -0.002 to 0, 0.25 to 0.5 at -0.5 to -0.004), and a state that remembers hundreds of rows
// adds that up; with the exponent moved by this much its mean is within 0.2 of the value (just above zero, A > 0, where it
// was 0.3 too large, 0.6: a growing state's own error grows with it).  A step of zero still leaves
// the state: the exponential of anything up to 1.1e-7 is 1.  4096 x 2048 x 16 training, relative errors without / with it:
// dA 1.6e-6 / 6.3e-7, dB and dC 4.8e-7 / 2.8e-7, ddt 4.6e-7 / 2.4e-7; states after 4097 rows of prompts 4.6e-7 / 2.5e-7
// (elementary float32 operations: 1.2e-6, 3.3e-7, 3.2e-7; 1.4e-6).  A correctly rounded exponential: 3.8e-7, 2.4e-7, 1.8e-7;
// 1.6e-7.  The multiplication it joins was there: no time.
#define SCAN_CENTRE 2.6e-8f

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

// The hardware's exponential: 2 units in the last place, results below 2^-126 are zero (a state that decays by that in
// a row has forgotten).
__device__ __forceinline__ float scan_exp2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// log(1 + e^v) = max(v, 0) + log1p(e), e = exp(-|v|) in [0, 1], without a branch, so that a lane's rows overlap.
// log1p(e) = 2 atanh(w), w = e / (2 + e) <= 1/3: the series in w^2 <= 1/9 to w^12 leaves 2e-8 of it, and small e
// (a step size of 0.001 is log1p(0.001)) keep their digits.  The argument's rounding in base 2 makes e uncertain by
// |v| * 2^-24; expf in its place leaves every output's error as it is and costs 6 us of 225 (4097 rows of prompts x 4096
// channels x 16 states) and 8 of 423 (training, 4096 x 2048 x 16).
__device__ __forceinline__ float scan_softplus(float v) {
  const float e = scan_exp2(-LOG2E * fabsf(v));
  const float w = __fdividef(e, 2.0f + e), q = w * w;
  float s = 1.0f / 13.0f;
  s = fmaf(s, q, 1.0f / 11.0f);
  s = fmaf(s, q, 1.0f / 9.0f);
  s = fmaf(s, q, 1.0f / 7.0f);
  s = fmaf(s, q, 1.0f / 5.0f);
  s = fmaf(s, q, 1.0f / 3.0f);
  s = fmaf(s, q, 1.0f);
  return fmaf(2.0f * w, s, fmaxf(v, 0.0f));
}

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

// f(true) or f(false) with the flag known at compile time: a loop inside has no branch on it
template <bool V>
struct ScanFlag {
  static constexpr bool value = V;
};
template <typename F>
__device__ __forceinline__ void scan_switch(bool flag, F f) {
  if (flag)
    f(ScanFlag<true>());
  else
    f(ScanFlag<false>());
}

// Which channels a lane works on.  Blocks are (unit, group, channel tile of the group); a unit is a stretch
// of a sequence's rows.
template <int S, int P>
struct ScanLane {
  static constexpr int kBlock = SCAN_THREADS / S * P;  // channels of a block
  int unit, k, first, group, tile, width, c0, j, n0, in_block;
  __device__ ScanLane(int channels, int groups, const int* units) {
    const int per = channels / groups, tiles = (per + kBlock - 1) / kBlock;
    const int b = blockIdx.x % (tiles * groups);
    unit = blockIdx.x / (tiles * groups);
    k = units[2 * unit];
    first = units[2 * unit + 1];
    group = b / tiles;
    tile = b - group * tiles;
    width = min(per - tile * kBlock, kBlock);  // channels of this tile
    c0 = group * per + tile * kBlock;
    in_block = threadIdx.x / S * P;  // the lane's first channel in the tile
    j = threadIdx.x % S;
    n0 = 4 * j;
  }
  __device__ bool valid(int p) const { return in_block + p < width; }
  // (a lane without a channel computes with the last one's and stores nothing)
  __device__ int channel(int p) const { return c0 + min(in_block + p, width - 1); }
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

// exp(s A) of two states, A2 = A log2(e); see SCAN_CENTRE
__device__ __forceinline__ f32x2 scan_decay2(f32x2 s2, f32x2 A2) {
  return exp2x2(fma2(s2, A2, pack2(SCAN_CENTRE, SCAN_CENTRE)));
}
__device__ __forceinline__ float scan_decay(float s, float A2) { return scan_exp2(fmaf(s, A2, SCAN_CENTRE)); }

__device__ __forceinline__ void scan_cp_async(void* smem, const void* gmem, int bytes) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  if (bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(gmem) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(s), "l"(gmem) : "memory");
}
__device__ __forceinline__ void scan_cp_async4(void* smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void scan_cp_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Where an array's rows of the unit begin: in shared memory, since nine of them would fill 36 registers (backward), six 24.
struct ScanArray {
  char* p;
  int64_t stride;
};

// What a block stages in shared memory: R rows of its channels of NA arrays in their own type, and the
// rows' weights B, C in float32 (converted once for all its channels), padded with zeros to 4 S states and, for
// sums over channels (ZEROS), four zeros more: those of a lane without a channel, whatever B and C hold.
template <typename T, int S, int P, int R, int NA, bool ZEROS = false>
struct ScanStage {
  static constexpr int kChannels = SCAN_THREADS / S * P, kRows = R;
  // rows that a warp's lanes read at the same time start in different banks
  static constexpr int kPad = (P * (int)sizeof(T) < 4 ? P * (int)sizeof(T) : 4) * 32 / S;
  static constexpr int kPitch = (kChannels * (int)sizeof(T) + kPad + 15) / 16 * 16 / (int)sizeof(T);
  static constexpr int kStates = 4 * S + (ZEROS ? 4 : 0);
  static constexpr int kBytes = kChannels * (int)sizeof(T) < 16 ? kChannels * (int)sizeof(T) : 16;
  alignas(16) T in[NA][R][kPitch];
  alignas(16) float bc[R][2][kStates];
};

// A tile's prepared rows: (s, s x) of every channel
template <int S, int P, int R>
struct ScanRows {
  static constexpr int kPad = 16 / S > 2 ? 16 / S : 2;
  static constexpr int kPitch = SCAN_THREADS / S * P + kPad;
  alignas(16) float2 sx[R][kPitch];
  __device__ __forceinline__ void put(int r, int c, const float (&s)[P], const float (&x)[P]) {
    if constexpr (P == 2)
      *reinterpret_cast<float4*>(&sx[r][c]) = make_float4(s[0], x[0], s[1], x[1]);
    else
      sx[r][c] = make_float2(s[0], x[0]);
  }
  // each value twice, for both halves of a register pair
  __device__ __forceinline__ void get(int r, int c, f32x2 (&s)[P], f32x2 (&x)[P]) const {
    if constexpr (P == 2) {
      const float4 v = *reinterpret_cast<const float4*>(&sx[r][c]);
      s[0] = pack2(v.x, v.x), x[0] = pack2(v.y, v.y), s[P - 1] = pack2(v.z, v.z), x[P - 1] = pack2(v.w, v.w);
    } else {
      const float2 v = sx[r][c];
      s[0] = pack2(v.x, v.x), x[0] = pack2(v.y, v.y);
    }
  }
};

// The lane's P values of a row
template <typename T, int P>
__device__ __forceinline__ void scan_get(const T* from, float (&v)[P]) {
  SeqVecA<T, P> r;
  r.load(from);
#pragma unroll
  for (int p = 0; p < P; ++p) v[p] = r[p];
}
// ... and to memory: one access if VEC (then all P are valid or none), else the valid ones
template <bool VEC, typename T, int P>
__device__ __forceinline__ void scan_put(T* to, const float (&v)[P], int valid) {
  if constexpr (VEC) {
    SeqVecA<T, P> r;
    r.put(v);
    if (valid > 0) r.store(to);
  } else {
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p < valid) to[p] = nb2_from_float<T>(v[p]);
  }
}

// rows x channels of one array on their way to shared memory: asynchronously (VEC), or element by element through
// registers, loaded (load) before a tile is worked on and stored (store) after it
template <bool VEC, typename T, typename Stage>
struct ScanCopy {
  static constexpr int R = Stage::kRows, kChannels = Stage::kChannels, kPer = VEC ? Stage::kBytes / (int)sizeof(T) : 1;
  static constexpr int kCount = (R * kChannels / kPer + SCAN_THREADS - 1) / SCAN_THREADS;
  T v[VEC ? 1 : kCount];
  __device__ __forceinline__ void load(T (&to)[R][Stage::kPitch], const T* from, int64_t stride, int rows, int channels) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int at = threadIdx.x + i * SCAN_THREADS, r = at / (kChannels / kPer), c = at % (kChannels / kPer) * kPer;
      if constexpr (VEC) {
        if (r < rows && c < channels) scan_cp_async(&to[r][c], from + r * stride + c, Stage::kBytes);
      } else {
        v[i] = r < rows && c < channels ? from[r * stride + c] : nb2_from_float<T>(0.0f);
      }
    }
  }
  __device__ __forceinline__ void store(T (&to)[R][Stage::kPitch]) const {
    if constexpr (!VEC)
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const int at = threadIdx.x + i * SCAN_THREADS;
        if (at < R * kChannels) to[at / kChannels][at % kChannels] = v[i];
      }
  }
};

// B and C of a tile's rows, on their way through registers from the arrays' type to float32; rows past the
// end become zeros
template <bool VEC, typename T, int S, int R>
struct ScanWeights {
  static constexpr int kPer = VEC ? 16 / (int)sizeof(T) : 1;
  static constexpr int kCount = (R * 8 * S / kPer + SCAN_THREADS - 1) / SCAN_THREADS;
  SeqVecA<T, kPer> v[kCount];
  int to[kCount];  // place of entry i in [R][B, C][4 S], -1 past the tile (the same for every tile)
  __device__ __forceinline__ explicit ScanWeights(int n) {
    const int per = n / kPer;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int e = threadIdx.x + i * SCAN_THREADS, row = e / per, m = (e - row * per) * kPer;
      to[i] = row < 2 * R ? row * 4 * S + m : -1;
    }
  }
  __device__ __forceinline__ void load(const T* B, int64_t bs, const T* C, int64_t cs, int n, int rows) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int r = to[i] / (8 * S), m = to[i] % (4 * S);
      v[i].zero();
      if (to[i] >= 0 && r < rows) v[i].load((to[i] & (4 * S) ? C + r * cs : B + r * bs) + m);
    }
  }
  template <int PITCH>
  __device__ __forceinline__ void store(float (&bc)[R][2][PITCH]) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      if (to[i] >= 0)
#pragma unroll
        for (int e = 0; e < kPer; ++e) (&bc[0][0][0])[to[i] / (4 * S) * (PITCH - 4 * S) + to[i] + e] = v[i][e];
  }
};

template <typename Stage>
__device__ __forceinline__ void scan_clear_weights(Stage* stages, int count) {
  constexpr int kEach = Stage::kRows * 2 * Stage::kStates;
  for (int i = threadIdx.x; i < count * kEach; i += SCAN_THREADS) (&stages[i / kEach].bc[0][0][0])[i % kEach] = 0.0f;
}

// A log2(e), held finite: a step of zero (a masked row, or one past a sequence's end) has to leave the state as it
// is, which 0 * inf would not.
__device__ __forceinline__ float scan_rate(float A) {
  const float r = A * LOG2E;
  return r > 3e38f ? 3e38f : r < -3e38f ? -3e38f : r;
}

// A[c][n0 ..] log2(e), two states to a register pair
__device__ __forceinline__ void scan_rates(const float* A, int n0, int n, f32x2 (&A2)[2]) {
  float v[4];
  scan_load4(A, n0, n, 0, v);
#pragma unroll
  for (int m = 0; m < 4; ++m) v[m] = scan_rate(v[m]);
  A2[0] = pack2(v[0], v[1]);
  A2[1] = pack2(v[2], v[3]);
}

#define SCAN_TRY(call)                  \
  do {                                  \
    cudaError_t e__ = (call);           \
    if (e__ != cudaSuccess) return e__; \
  } while (0)

template <typename K>
static cudaError_t scan_allow_smem(K kernel, size_t smem) {
  return smem > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
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
template <typename A>
static int scan_check_units(const A& a) {
  NB2_REQUIRE(a.units && a.n_units >= a.n_seq && a.unit_rows >= 1 && a.unit_rows % NB2_SCAN_KEEP == 0, "units");
  NB2_REQUIRE((int64_t)a.n_units * (a.channels + a.groups) < (1ll << 31), "too many units x channels");
  NB2_REQUIRE(!a.ends || a.sums, "null pointer");
  NB2_REQUIRE(a.ends || a.n_units == a.n_seq, "units of a sequence need what they start from");
  NB2_REQUIRE(!a.ends || (int64_t)a.n_seq * a.channels * a.n_states < (1ll << 38), "too many states");
  return NB2_OK;
}

static int scan_tiles(int channels, int groups, int block) { return (channels / groups + block - 1) / block; }

// Launches that both passes share; see nb2_scan_join_kernel.
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
cudaError_t nb2_scan_join(cudaStream_t s, ScanJoin j);

#define SCAN_BY_LANES(lanes, launch)                 \
  switch (lanes) {                                   \
    case 1: NB2_CUDA((launch<T, 1>(s, a))); break;   \
    case 2: NB2_CUDA((launch<T, 2>(s, a))); break;   \
    case 4: NB2_CUDA((launch<T, 4>(s, a))); break;   \
    case 8: NB2_CUDA((launch<T, 8>(s, a))); break;   \
    case 16: NB2_CUDA((launch<T, 16>(s, a))); break; \
    default: NB2_CUDA((launch<T, 32>(s, a))); break; \
  }
