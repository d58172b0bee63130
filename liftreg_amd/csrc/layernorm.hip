// layernorm.hip — layer norm over the last axis, LeakyReLU in the same pass, and its gradient with the reduction of the weight's.
//
//   xhat = (x - mean) rstd,  z = xhat w + b,  y = z >= 0 ? z : slope z
//   g = gy (z >= 0 ? 1 : slope),  h = g w,  gx = rstd (h - mean(h) - xhat mean(h xhat))
//   gw[c] = sum over rows of g xhat,  gb[c] = sum over rows of g
//
// Bound by memory: x and y once forward; x, gy and gx once backward.  Two forms, by the length of a row:
//  * up to kResident columns a row lives in the registers of a group of G lanes (four for the 16 channels of a voxel, two waves for
//    the head's 800 features, a workgroup above 1024 columns), 16 bytes a lane and load.  Mean and variance are two
//    passes over registers.  Backward recomputes them: x is there anyway, and 8 bytes of saved statistics a row would be 1/8 of a
//    16-channel row forward and again backward.  A lane keeps its columns over all its rows, so the weight's gradient grows in
//    registers; groups, then waves add theirs, each workgroup leaves one partial row, a second kernel adds those in a fixed order.
//  * longer rows are cut into chunks (few rows would leave most CUs idle): per-chunk mean and variance (Chan's update), joined per row,
//    then one pass that normalises; backward the same with the sums of h and h xhat, where a workgroup of the last pass owns columns
//    and walks down the rows, so the weight's gradient needs no atomics either.
#include "lr_common.h"

namespace {

constexpr int kResident = 16384;       // longest row that is held in registers: 1024 lanes of 16 elements
// arrays from this size on pass the caches by: no line of them would be there when it is read next (the last-level cache holds 256 MB; 1 GB
// arrays forward + backward 997 us through the caches, 948 past them)
constexpr int64_t kStream = (int64_t)256 << 20;

template <class T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
  struct Raw {             // a vector as it is fetched; four registers of their own: one that is put together from elements waits for each
    float e[4];
    __device__ __forceinline__ float& operator[](int i) { return e[i]; }
  };
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
  static __device__ __forceinline__ V pack(const float* r) { return V{r[0], r[1], r[2], r[3]}; }
};
template <> struct Vec<uint16_t> {     // bfloat16
  static constexpr int N = 8;
  typedef uint16_t V __attribute__((ext_vector_type(8), aligned(2)));
  typedef V Raw;
  static __device__ __forceinline__ float up(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t down(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }   // nearest even
  static __device__ __forceinline__ V pack(const float* r) {      // two in an instruction
    typedef float F __attribute__((ext_vector_type(8)));
    typedef __bf16 B __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(V, __builtin_convertvector((F{r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]}), B));
  }
};

// N elements from column c of a row of C (past the end: 0, not written).  A row may start at any element: gfx950 takes 16-byte
// accesses at any address.  RAGGED = false: C is a multiple of N.  The last, partial vector of a ragged row is loaded element by
// element, which in a wave waits for the others' whole vectors, or, SHIFT (C >= N), as the row's last N elements, which unpack()
// shifts down: backward, where rows are fetched ahead, 30000 x 801 fp32 71 us by element and 58 shifted, 44739 x 1500 bf16 209 and 155;
// forward the shifts cost more than they save (100000 x 801 fp32 128 and 160).  fetch() and unpack() are two steps so that rows
// fetched ahead wait as they are: 4 registers of 8 bf16, no conversion that waits for them.
template <bool RAGGED = true, bool SHIFT = false, bool STREAM = false, class T>
__device__ __forceinline__ typename Vec<T>::Raw fetch(const T* row, int64_t c, int64_t C) {
  constexpr int N = Vec<T>::N;
  typedef typename Vec<T>::V V;
  typename Vec<T>::Raw r;
  if (RAGGED && SHIFT && C >= N) {
    const V v = *reinterpret_cast<const V*>(row + (c < C - N ? c : C - N));
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = v[e];
  } else if (RAGGED ? c + N <= C : c < C) {
    const V* at = reinterpret_cast<const V*>(row + c);
    const V v = STREAM ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = RAGGED && c + e < C ? row[c + e] : (T)0;
  }
  return r;
}
template <bool RAGGED = true, bool SHIFT = false, class T = float>
__device__ __forceinline__ void unpack(typename Vec<T>::Raw v, int64_t c, int64_t C, float* r) {
  constexpr int N = Vec<T>::N;
  if constexpr (RAGGED && SHIFT) {
    if (C >= N) {
      const int d = c < C - N ? 0 : (int)min(c - (C - N), (int64_t)N);
      if constexpr (N == 8) {
        typedef uint64_t Q __attribute__((ext_vector_type(2)));
        Q t;
        __builtin_memcpy(&t, &v, sizeof t);
        const int n = 16 * (d & 3);
        uint64_t lo = d & 4 ? t[1] : t[0], hi = d & 4 ? 0 : t[1];
        lo = n ? lo >> n | hi << (64 - n) : lo;
        hi >>= n;
        if (d >= 8) lo = hi = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          r[e] = Vec<T>::up((uint16_t)(lo >> (16 * e)));
          r[e + 4] = Vec<T>::up((uint16_t)(hi >> (16 * e)));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = e < 3 && d & 1 ? v[e < 3 ? e + 1 : 3] : v[e];
        r[3] = d & 1 ? 0.f : r[3];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = d & 2 ? (e < 2 ? r[e < 2 ? e + 2 : 3] : 0.f) : r[e];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = d & 4 ? 0.f : r[e];
      }
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) r[e] = Vec<T>::up(v[e]);
}
template <bool RAGGED = true, bool STREAM = false, class T>
__device__ __forceinline__ void load(const T* row, int64_t c, int64_t C, float* r) {
  unpack<RAGGED, false, T>(fetch<RAGGED, false, STREAM>(row, c, C), c, C, r);
}
template <bool RAGGED = true, bool STREAM = false, class T>
__device__ __forceinline__ void store(T* row, int64_t c, int64_t C, const float* r) {
  constexpr int N = Vec<T>::N;
  if (c + N <= C) {
    const typename Vec<T>::V v = Vec<T>::pack(r);
    typename Vec<T>::V* at = reinterpret_cast<typename Vec<T>::V*>(row + c);
    if (STREAM) __builtin_nontemporal_store(v, at);
    else *at = v;
  } else if (RAGGED) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < C) row[c + e] = Vec<T>::down(r[e]);
  }
}
template <int N>
__device__ __forceinline__ void load_f(const float* a, int64_t c, int64_t C, float other, float* r) {
#pragma unroll
  for (int e = 0; e < N; ++e) r[e] = other;
  if (!a) return;
  if (c + N <= C) {
#pragma unroll
    for (int q = 0; q < N; q += 4) load<false>(a, c + q, C, r + q);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < C) r[e] = a[c + e];
  }
}

template <int N>
__device__ __forceinline__ void store_f(float* a, int64_t c, int64_t C, const float* r) {
#pragma unroll
  for (int q = 0; q < N; q += 4) store<true>(a, c + q, C, r + q);
}

template <int CTRL>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, true));
}
// x + the x of the lane 16 (32) further on, modulo 32 (64): gfx950's row swaps, a tenth of a cross-lane read through LDS
__device__ __forceinline__ float add_row(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// the same of both words of an fp64 number
__device__ __forceinline__ double words(uint32_t lo, uint32_t hi) { return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo)); }
__device__ __forceinline__ uint32_t low(double x) { return (uint32_t)__double_as_longlong(x); }
__device__ __forceinline__ uint32_t high(double x) { return (uint32_t)(__double_as_longlong(x) >> 32); }
template <int CTRL>
__device__ __forceinline__ double add_dpp(double x) {
  return x + words((uint32_t)__builtin_amdgcn_mov_dpp((int)low(x), CTRL, 0xf, 0xf, true), (uint32_t)__builtin_amdgcn_mov_dpp((int)high(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ double add_row(double x) {
  const auto l = __builtin_amdgcn_permlane16_swap(low(x), low(x), false, false), h = __builtin_amdgcn_permlane16_swap(high(x), high(x), false, false);
  return words(l[0], h[0]) + words(l[1], h[1]);
}
__device__ __forceinline__ double add_half(double x) {
  const auto l = __builtin_amdgcn_permlane32_swap(low(x), low(x), false, false), h = __builtin_amdgcn_permlane32_swap(high(x), high(x), false, false);
  return words(l[0], h[0]) + words(l[1], h[1]);
}
// sum over aligned groups of G lanes, in every lane
template <int G, class F>
__device__ __forceinline__ F lane_sum(F x) {
  if (G >= 2) x = add_dpp<0xB1>(x);      // neighbour
  if (G >= 4) x = add_dpp<0x4E>(x);      // pair
  if (G >= 8) x = add_dpp<0x141>(x);     // mirrored half row of 8
  if (G >= 16) x = add_dpp<0x140>(x);    // mirrored row of 16
  if (G >= 32) x = add_row(x);
  if (G >= 64) x = add_half(x);
  return x;
}
// sum over the lanes of a wave that are equal modulo G, in every lane: rotations within a row of 16, then the rows
template <int G>
__device__ __forceinline__ float stride_sum(float x) {
  if (G <= 8) x = add_dpp<0x128>(x);
  if (G <= 4) x = add_dpp<0x124>(x);
  if (G <= 2) x = add_dpp<0x122>(x);
  if (G <= 1) x = add_dpp<0x121>(x);
  if (G <= 16) x = add_row(x);
  if (G <= 32) x = add_half(x);
  return x;
}

// sums over the G lanes of a row.  Above a wave: through LDS, two buffers in turn, one barrier a sum.
template <int G, int NT>
struct Group {
  static constexpr int W = G / 64;       // waves of a row
  float (*red)[2][NT / 64];
  int turn;
  __device__ __forceinline__ explicit Group(float (*r)[2][NT / 64]) : red(r), turn(0) {}
  __device__ __forceinline__ float sum(float x) { return across(lane_sum<(G < 64 ? G : 64)>(x)); }
  // x: a wave's sum, in every lane.  A lane takes one wave's and lanes are added up: all of them in every lane would take W registers.
  template <class F>
  __device__ __forceinline__ F across(F x) {
    if (G <= 64) return x;
    F* buf = reinterpret_cast<F*>(red[turn]);
    turn ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) buf[wave] = x;
    __syncthreads();
    constexpr int M = W > 0 ? W : 1;
    return lane_sum<M>(buf[wave / M * M + threadIdx.x % M]);
  }
  __device__ __forceinline__ void sum2(float& a, float& b) {
    a = lane_sum<(G < 64 ? G : 64)>(a);
    b = lane_sum<(G < 64 ? G : 64)>(b);
    if (G <= 64) return;
    float (*buf)[NT / 64] = red[turn];
    turn ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      buf[0][wave] = a;
      buf[1][wave] = b;
    }
    __syncthreads();
    const int first = W > 0 ? wave / (W > 0 ? W : 1) * W : 0;
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a += buf[0][first + w];
      b += buf[1][first + w];
    }
  }
};

// x[0] + ... + x[N-1], N a power of two, by halves: equal numbers add up without rounding
template <int N>
__device__ __forceinline__ float halves(const float* x) {
  float t[N];
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = x[i];
#pragma unroll
  for (int o = N / 2; o > 0; o /= 2)
#pragma unroll
    for (int i = 0; i < o; ++i) t[i] += t[i + o];
  return t[0];
}
// mean and rstd of a row held as x[K * N]; RAGGED: cols is no multiple of N.  A constant row has its own value as mean, which a sum in
// fp32 misses (16384 times 1000.1: xhat 0.096 with eps = 1e-5 and not 0).  Equal numbers add up by halves without rounding: so do rows that
// fill their lanes, and waves of longer rows that the row fills.  Elsewhere vectors are added up by halves, the rest in fp64; a row's one
// partial vector is off by at most 2^-24 of itself, which counts where a row has few vectors: there pairs go to fp64.
template <int K, int N, int G, bool RAGGED, class Gr>
__device__ __forceinline__ void row_stats(Gr& gr, const float* x, int lane, int C, double inv, float inv32, float eps, float& mean,
                                          float& rstd) {
  constexpr int L = G < 64 ? G : 64, V = RAGGED && G < 16 ? 2 : N;
  const int end = __builtin_amdgcn_readfirstlane(((K - 1) * G + (lane | (L - 1)) + 1) * N);      // of the columns that the wave can hold
  double s;
  if ((!RAGGED || G > 64) && end <= C) {
    s = (double)lane_sum<L>(halves<K * N>(x) * 0x1p-10f) * 0x1p10;      // scaled: at most 1024 numbers, no further overflow
  } else {
    s = (double)halves<V>(x);
#pragma unroll
    for (int i = V; i < K * N; i += V) s += (double)halves<V>(x + i);
    s = lane_sum<L>(s);
  }
  mean = (float)(gr.across(s) * inv);
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * G + lane) * N;
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = x[k * N + e] - mean;
      t = fmaf(d, (!RAGGED || c + e < C) ? d : 0.f, t);
    }
    q += RAGGED || c < C ? t : 0.f;
  }
  const float v = fmaf(gr.sum(q), inv32, eps);
  rstd = v < 0x1p-100f ? __builtin_amdgcn_rsqf(v * 0x1p60f) * 0x1p30f : __builtin_amdgcn_rsqf(v);   // v_rsq_f32 takes no subnormals
}

// STREAM: x, gy, y and gx past the caches (kStream).
template <class T, int G, int K, int NT, bool RAGGED, bool STREAM>
__global__ __launch_bounds__(NT) void fwd_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                 T* __restrict__ y, float* __restrict__ stats, int64_t rows, int C, double inv,
                                                 float inv32, float eps, float slope) {
  constexpr int N = Vec<T>::N, RPB = NT / G;
  __shared__ __attribute__((aligned(8))) float red[2][2][NT / 64];
  Group<G, NT> gr(red);
  const int lane = threadIdx.x % G;
  float wv[K * N], bv[K * N];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_f<N>(w, (k * G + lane) * N, C, 1.f, wv + k * N);
    load_f<N>(b, (k * G + lane) * N, C, 0.f, bv + k * N);
  }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
    const int64_t r = r0 + threadIdx.x / G;
    const int cols = r < rows ? C : 0;      // all lanes stay for the sums
    const T* xr = x + r * C;
    float v[K * N];
#pragma unroll
    for (int k = 0; k < K; ++k) load<RAGGED, STREAM>(xr, (k * G + lane) * N, cols, v + k * N);
    float mean, rstd;
    row_stats<K, N, G, RAGGED>(gr, v, lane, C, inv, inv32, eps, mean, rstd);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float z = fmaf((v[k * N + e] - mean) * rstd, wv[k * N + e], bv[k * N + e]);
        v[k * N + e] = z >= 0.f ? z : z * slope;
      }
      store<RAGGED, STREAM>(y + r * C, (k * G + lane) * N, cols, v + k * N);
    }
    if (stats && lane == 0 && r < rows) {
      stats[2 * r] = mean;
      stats[2 * r + 1] = rstd;
    }
  }
}

// gx (if set), and this workgroup's sums of g xhat and g at sw, sb (if set) + blockIdx.x * stride.  ACT: there is a LeakyReLU mask
// (without it b is not needed).  The next rows are loaded before these rows' sums (three dependent reductions), up to 8 elements a
// lane: beyond that the registers are worth more as occupancy.  (Of a workgroup of 1024 with several rows at a time only fp32's:
// 8192 x 800 19.0 us ahead, 20.8 without; bf16 16.5 and 16.3.)  Four waves a SIMD, at most 128 registers: one ragged form took 129
// (22362 x 3001 fp32 230 us, 170 with 128).
template <class T, int G, int K, int NT, bool RAGGED, bool ACT, bool STREAM>
__global__ __launch_bounds__(NT, 4) void bwd_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                 const T* __restrict__ gy, T* __restrict__ gx, float* __restrict__ sw, float* __restrict__ sb,
                                                 int64_t stride, int64_t rows, int C, double inv, float inv32, float eps,
                                                 float slope) {
  constexpr int N = Vec<T>::N, RPB = NT / G, E = K * N;
  constexpr bool SHIFT = N == 8 || E <= 8;      // 16 fp32 elements a lane: 1000 x 16001 66 us shifted, 52 by element
  constexpr bool AHEAD = E <= 8 && (NT < 1024 || G == NT || N == 4);
  __shared__ __attribute__((aligned(8))) float red[2][2][NT / 64];
  Group<G, NT> gr(red);
  const int lane = threadIdx.x % G;
  const int64_t step = (int64_t)gridDim.x * RPB;
  constexpr bool HOLD = ACT && E <= 8;      // b in registers; 16 elements a lane spill then (4096 x 10000 fp32 654 us): fetched for each row (135)
  float wv[E], bv[HOLD ? E : 1], aw[E], ab[E], v[E], g[E];
  typename Vec<T>::Raw nv[K], ng[K];
  int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
  auto get = [&](int64_t at) {
    const int cols = at < rows ? C : 0;
#pragma unroll
    for (int k = 0; k < K; ++k) nv[k] = fetch<RAGGED, SHIFT, STREAM>(x + at * C, (k * G + lane) * N, cols);
#pragma unroll
    for (int k = 0; k < K; ++k) ng[k] = fetch<RAGGED, SHIFT, STREAM>(gy + at * C, (k * G + lane) * N, cols);
  };
  if (AHEAD) get(r);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_f<N>(w, (k * G + lane) * N, C, 1.f, wv + k * N);
    if (HOLD) load_f<N>(b, (k * G + lane) * N, C, 0.f, bv + (HOLD ? k * N : 0));
  }
#pragma unroll
  for (int i = 0; i < E; ++i) aw[i] = ab[i] = 0.f;
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += step, r += step) {
    const int cols = r < rows ? C : 0;
    if (!AHEAD) get(r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack<RAGGED, SHIFT, T>(nv[k], (k * G + lane) * N, C, v + k * N);
      unpack<RAGGED, SHIFT, T>(ng[k], (k * G + lane) * N, C, g + k * N);
    }
    if (AHEAD) get(r + step);
    float mean, rstd;
    row_stats<K, N, G, RAGGED>(gr, v, lane, C, inv, inv32, eps, mean, rstd);
    if (r >= rows) rstd = 0.f;        // no row: xhat = 0 even where eps = 0
    float s1 = 0.f, s2 = 0.f;
    const float* bp = b;
    if (ACT && !HOLD) asm volatile("" : "+s"(bp));      // not out of the loop again
#pragma unroll
    for (int k = 0; k < K; ++k) {     // past the end g and xhat are 0 (mean rstd may be beyond fp32): nothing is added
      float bk[N];
      if (ACT && !HOLD) load_f<N>(bp, (k * G + lane) * N, C, 0.f, bk);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = k * N + e, c = (k * G + lane) * N + (RAGGED ? e : 0);
        const float xh = (v[i] - mean) * (c < C ? rstd : 0.f);
        float gg = g[i];
        if (ACT) gg = fmaf(xh, wv[i], HOLD ? bv[HOLD ? i : 0] : bk[e]) >= 0.f ? gg : gg * slope;
        aw[i] = fmaf(gg, xh, aw[i]);
        ab[i] += gg;
        const float h = gg * wv[i];
        s1 += h;
        s2 = fmaf(h, xh, s2);
        v[i] = xh;
        g[i] = h;
      }
    }
    gr.sum2(s1, s2);
    if (gx) {
      s1 *= inv32;
      s2 *= inv32;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int i = k * N + e;
          v[i] = rstd * (g[i] - fmaf(v[i], s2, s1));
        }
        store<RAGGED, STREAM>(gx + r * C, (k * G + lane) * N, cols, v + k * N);
      }
    }
  }
  if (!sw && !sb) return;
  // groups of a wave, then waves
#pragma unroll
  for (int i = 0; i < E; ++i) {
    aw[i] = stride_sum<G>(aw[i]);
    ab[i] = stride_sum<G>(ab[i]);
  }
  const int64_t at0 = (int64_t)blockIdx.x * stride;
  if (G == NT) {         // one row at a time: every column has one lane
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * G + lane) * N;
      if (sw) store_f<N>(sw + at0, c, C, aw + k * N);
      if (sb) store_f<N>(sb + at0, c, C, ab + k * N);
    }
    return;
  }
  constexpr int W = G == NT ? 1 : G <= 64 ? NT / 64 : NT / G, L = G == NT ? 1 : G * E;      // sums to add, columns
  __shared__ float cols[W][L];
  const int set = threadIdx.x / (G <= 64 ? 64 : G), at = threadIdx.x % (G <= 64 ? 64 : G);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float* part = which ? ab : aw;
    float* out = which ? sb : sw;
    if (!out) continue;
    __syncthreads();
    if (at < G) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) cols[set % W][((k * G + at) * N + e) % L] = part[k * N + e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += NT) {
      float s = 0.f;
      for (int q = 0; q < W; ++q) s += cols[q][c % L];
      out[at0 + c] = s;
    }
  }
}

// gw = sum of the first halves of the partial rows [n][2 C], gb of the second, in a fixed order; LANES rows at a time: 32 where there
// are many rows, one (a column a thread) where there are few and long ones (2 rows of 1 M: 142 us with 32, 7 with one)
template <int LANES>
__global__ __launch_bounds__(LANES == 1 ? 256 : 1024) void finish_kernel(const float* __restrict__ part, int n, int64_t C,
                                                                         float* __restrict__ gw, float* __restrict__ gb) {
  constexpr int COLS = LANES == 1 ? 256 : 1024 / LANES;
  const int64_t c = (int64_t)blockIdx.x * COLS + threadIdx.x % COLS;
  const int j = threadIdx.x / COLS;
  float s = 0.f;
  if (c < 2 * C)
#pragma unroll 8
    for (int i = j; i < n; i += LANES) s += part[(int64_t)i * 2 * C + c];
  if (LANES > 1) {
    __shared__ float red[LANES][COLS + 1];
    red[j][threadIdx.x % COLS] = s;
    __syncthreads();
    for (int o = LANES / 2; o > 0; o >>= 1) {
      if (j < o) red[j][threadIdx.x % COLS] += red[j + o][threadIdx.x % COLS];
      __syncthreads();
    }
    s = red[0][threadIdx.x % COLS];
  }
  if (j == 0 && c < 2 * C) {
    float* out = c < C ? gw : gb;
    if (out) out[c < C ? c : c - C] = s;
  }
}

// ---------------------------------------------------------------- rows that are cut into chunks
// Chan's update.  The weight goes into the difference before the square: an empty side's mean is 0, so where one side is empty d is the
// other's whole mean, whose square may leave fp32, and the weight 0.
struct Part { float n, mean, m2; };
__device__ __forceinline__ Part join(Part a, Part b) {
  Part r;
  r.n = a.n + b.n;
  const float d = b.mean - a.mean, f = r.n > 0.f ? b.n / r.n : 0.f;
  r.mean = fmaf(d, f, a.mean);
  r.m2 = fmaf(d * (a.n * f), d, a.m2 + b.m2);
  return r;
}
__device__ __forceinline__ Part block_join(Part p) {     // 256 threads; in every thread
  __shared__ Part red[4];
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    Part q = {__shfl_xor(p.n, o, 64), __shfl_xor(p.mean, o, 64), __shfl_xor(p.m2, o, 64)};
    p = join(p, q);
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = p;
  __syncthreads();
  return join(join(red[0], red[1]), join(red[2], red[3]));
}

// mean and variance of chunk blockIdx.x (`len` columns) of row blockIdx.y
template <class T>
__global__ __launch_bounds__(256) void chunk_stats_kernel(const T* __restrict__ x, float* __restrict__ part, int chunks, int64_t C,
                                                          int64_t len, int64_t row0) {
  if ((int)blockIdx.x >= chunks) return;
  constexpr int N = Vec<T>::N, K = 16 / N;
  const int64_t row = row0 + blockIdx.y, lo = blockIdx.x * len, hi = min(C, lo + len);
  const T* xr = x + row * C;
  Part p = {0.f, 0.f, 0.f};
  for (int64_t at = lo; at < hi; at += 256 * 16) {
    float v[16];
    int have = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = at + (k * 256 + threadIdx.x) * N;
      load(xr, c, hi, v + k * N);
      have += (int)max((int64_t)0, min((int64_t)N, hi - c));
    }
    float q = 0.f;
    Part t;
    t.n = (float)have;
    t.mean = halves<16>(v) * 0.0625f;
    if (have < 16) {         // as exact where all are equal, which halves are not
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += (double)v[i];
      t.mean = have ? (float)(s / (double)have) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = at + (k * 256 + threadIdx.x) * N + e < hi ? v[k * N + e] - t.mean : 0.f;
        q = fmaf(d, d, q);
      }
    t.m2 = q;
    p = join(p, t);
  }
  p = block_join(p);
  if (threadIdx.x == 0) {
    float* o = part + (row * chunks + blockIdx.x) * 2;
    o[0] = p.mean;
    o[1] = p.m2 / p.n;
  }
}

// f(c, end, whether the vector at c ends behind `end`) for a workgroup's vectors of [lo, hi): the whole ones four in flight, without the
// element loads of a part, then the part
struct Whole { static constexpr bool value = false; };
struct Partial { static constexpr bool value = true; };
template <int N, class F>
__device__ __forceinline__ void whole_then_part(int64_t lo, int64_t hi, F f) {
  int64_t c = lo + threadIdx.x * N;
#pragma unroll 4
  for (; c + N <= hi; c += 256 * N) f(c, c + N, Whole());
  if (c < hi) f(c, hi, Partial());
}

// mean and rstd of a row from its chunks, by a whole workgroup.  A chunk counts as its share of the row: the sum is then the variance and not
// C times it, which leaves fp32 sooner.
__device__ __forceinline__ void join_stats(const float* part, int64_t row, int chunks, int64_t C, int64_t len, float eps, float& mean,
                                           float& rstd) {
  const float inv = 1.0f / (float)C;
  Part p = {0.f, 0.f, 0.f};
  for (int i = threadIdx.x; i < chunks; i += 256) {
    const float* o = part + (row * chunks + i) * 2;
    const float n = (float)min(len, C - i * len) * inv;
    p = join(p, {n, o[0], o[1] * n});
  }
  p = block_join(p);
  mean = p.mean;
  rstd = 1.0f / sqrtf(p.m2 / p.n + eps);
}

__global__ __launch_bounds__(256) void join_stats_kernel(const float* __restrict__ part, int chunks, int64_t C, int64_t len,
                                                         float eps, float* __restrict__ stats, int64_t row0) {
  const int64_t row = row0 + blockIdx.x;
  float mean, rstd;
  join_stats(part, row, chunks, C, len, eps, mean, rstd);
  if (threadIdx.x == 0) {
    stats[2 * row] = mean;
    stats[2 * row + 1] = rstd;
  }
}

// every workgroup joins its row's statistics again (at most 8 KB from L2): a launch of its own for them takes 4.6 us
template <class T>
__global__ __launch_bounds__(256) void chunk_fwd_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                        T* __restrict__ y, const float* __restrict__ part, float* __restrict__ stats,
                                                        int chunks, int64_t C, int64_t len, float eps, float slope, int64_t row0) {
  if ((int)blockIdx.x >= chunks) return;
  constexpr int N = Vec<T>::N;
  const int64_t row = row0 + blockIdx.y, lo = blockIdx.x * len, hi = min(C, lo + len);
  float mean, rstd;
  join_stats(part, row, chunks, C, len, eps, mean, rstd);
  if (stats && blockIdx.x == 0 && threadIdx.x == 0) {
    stats[2 * row] = mean;
    stats[2 * row + 1] = rstd;
  }
  whole_then_part<N>(lo, hi, [&](int64_t c, int64_t end, auto part) {
    float v[N], wv[N], bv[N];
    load<decltype(part)::value>(x + row * C, c, end, v);
    load_f<N>(w, c, end, 1.f, wv);
    load_f<N>(b, c, end, 0.f, bv);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float z = fmaf((v[e] - mean) * rstd, wv[e], bv[e]);
      v[e] = z >= 0.f ? z : z * slope;
    }
    store<true, true>(y + row * C, c, end, v);
  });
}

// sums of h and h xhat over a chunk of a row
template <class T, bool ACT>
__global__ __launch_bounds__(256) void chunk_sums_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                         const T* __restrict__ gy, const float* __restrict__ stats,
                                                         float* __restrict__ part, int chunks, int64_t C, int64_t len, float slope,
                                                         int64_t row0) {
  if ((int)blockIdx.x >= chunks) return;
  constexpr int N = Vec<T>::N;
  __shared__ float red[4][2];
  const int64_t row = row0 + blockIdx.y, lo = blockIdx.x * len, hi = min(C, lo + len);
  const float mean = stats[2 * row], rstd = stats[2 * row + 1];
  float s1 = 0.f, s2 = 0.f;
  whole_then_part<N>(lo, hi, [&](int64_t c, int64_t end, auto part) {
    float v[N], g[N], wv[N], bv[N];
    load<decltype(part)::value>(x + row * C, c, end, v);
    load<decltype(part)::value>(gy + row * C, c, end, g);
    load_f<N>(w, c, end, 1.f, wv);
    if (ACT) load_f<N>(b, c, end, 0.f, bv);
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float xh = (v[e] - mean) * rstd;
      const float h = (!ACT || fmaf(xh, wv[e], bv[e]) >= 0.f ? g[e] : g[e] * slope) * wv[e];
      t1 += h;
      t2 = c + e < end ? fmaf(h, xh, t2) : t2;
    }
    s1 += t1;
    s2 += t2;
  });
  s1 = lane_sum<64>(s1);
  s2 = lane_sum<64>(s2);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = s1;
    red[threadIdx.x >> 6][1] = s2;
  }
  __syncthreads();
  if (threadIdx.x < 2)
    part[(row * chunks + blockIdx.x) * 2 + threadIdx.x] =
        (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// sums[row] = the row's means of h and h xhat
__global__ __launch_bounds__(256) void join_sums_kernel(const float* __restrict__ part, int chunks, int64_t C, float* __restrict__ sums,
                                                        int64_t row0) {
  __shared__ float red[4][2];
  const int64_t row = row0 + blockIdx.x;
  float s1 = 0.f, s2 = 0.f;
  for (int i = threadIdx.x; i < chunks; i += 256) {
    s1 += part[(row * chunks + i) * 2];
    s2 += part[(row * chunks + i) * 2 + 1];
  }
  s1 = lane_sum<64>(s1);
  s2 = lane_sum<64>(s2);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = s1;
    red[threadIdx.x >> 6][1] = s2;
  }
  __syncthreads();
  if (threadIdx.x < 2)
    sums[row * 2 + threadIdx.x] =
        ((red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x])) / (float)C;
}

// columns of a workgroup, rows [row0 + blockIdx.y * span, + span) below row1: gx, and the columns' sums over these rows (`more`: on top of
// what is there).  JOIN: the rows' sums of h and h xhat are added up from their chunks here, a wave a row (span rows of `chunks` chunks,
// at most kJoin in all: 2 x 8.4 M columns save a launch of 4.7 us); else `sums` holds the means.
constexpr int kJoin = 2048;
template <class T, bool JOIN, bool ACT>
__global__ __launch_bounds__(256) void chunk_bwd_kernel(const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                        const T* __restrict__ gy, const float* __restrict__ stats,
                                                        const float* __restrict__ sums, T* __restrict__ gx, float* __restrict__ gw,
                                                        float* __restrict__ gb, int64_t stride, int64_t row0, int64_t row1, int64_t span,
                                                        int chunks, int64_t C, float slope, bool more) {
  constexpr int N = Vec<T>::N;
  __shared__ float joined[JOIN ? kJoin : 1][2];
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  const int64_t lo = row0 + blockIdx.y * span, hi = min(row1, lo + span);
  if (JOIN) {
    for (int64_t r = lo + (threadIdx.x >> 6); r < hi; r += 4) {
      float s1 = 0.f, s2 = 0.f;
      for (int i = threadIdx.x & 63; i < chunks; i += 64) {
        s1 += sums[(r * chunks + i) * 2];
        s2 += sums[(r * chunks + i) * 2 + 1];
      }
      s1 = lane_sum<64>(s1);
      s2 = lane_sum<64>(s2);
      if ((threadIdx.x & 63) == 0) {
        joined[r - lo][0] = s1 / (float)C;
        joined[r - lo][1] = s2 / (float)C;
      }
    }
    __syncthreads();
  }
  if (c >= C) return;
  float wv[N], bv[N], aw[N], ab[N];
  load_f<N>(w, c, C, 1.f, wv);
  if (ACT) load_f<N>(b, c, C, 0.f, bv);
#pragma unroll
  for (int e = 0; e < N; ++e) aw[e] = ab[e] = 0.f;
#pragma unroll 2
  for (int64_t r = lo; r < hi; ++r) {
    float v[N], g[N];
    load(x + r * C, c, C, v);
    load(gy + r * C, c, C, g);
    const float mean = stats[2 * r], rstd = stats[2 * r + 1];
    const float s1 = JOIN ? joined[r - lo][0] : sums[2 * r], s2 = JOIN ? joined[r - lo][1] : sums[2 * r + 1];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float xh = (v[e] - mean) * rstd;
      const float gg = !ACT || fmaf(xh, wv[e], bv[e]) >= 0.f ? g[e] : g[e] * slope;
      aw[e] = fmaf(gg, xh, aw[e]);
      ab[e] += gg;
      v[e] = rstd * (gg * wv[e] - fmaf(xh, s2, s1));
    }
    if (gx) store<true, true>(gx + r * C, c, C, v);
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (c + e < C) {
      const int64_t at = blockIdx.y * stride + c + e;
      if (gw) gw[at] = more ? gw[at] + aw[e] : aw[e];
      if (gb) gb[at] = more ? gb[at] + ab[e] : ab[e];
    }
}

// ---------------------------------------------------------------- host
// Rows of one launch: at most 32768 (a grid's y extent).  Forward also at most 144 MB of x where there is more, so that the second read
// of a row comes from the last-level cache (256 MB): 13422 x 20000 fp32 625 us in one go, 557 in eight, bf16 420 and 354.  Backward,
// where the second pass reads and writes as much again, it costs: 67 x 1000000 bf16 124 us in one go, 147 in two.
int64_t rows_at_once(int64_t rows, int64_t row_bytes) {
  int64_t parts = (rows * row_bytes + ((int64_t)144 << 20) - 1) / ((int64_t)144 << 20);
  if (parts < 1) parts = 1;
  const int64_t n = (rows + parts - 1) / parts;
  return n < 32768 ? n : 32768;
}

// Chunks of 8192 columns where a row has at most 128 of them (3948 x 17000 fp32 forward 135 us, 176 with 16384, whose join reads fewer:
// 2 x 8.4 M 46 us, 56 with 8192), of 4096 where there would be fewer than 1024 workgroups.  Where w and b (8 bytes a column) may not
// stay in an L2 of 4 MB, a grid's row is a multiple of eight: workgroups go to the 8 XCDs in turn, and with it the same columns' w
// and b to the same L2 (67 x 1000000 bf16 forward 73 us, 99 without; 671 x 100000, where 3 of 16 idle, 85 and 72).
struct Plan {
  int64_t most;             // rows at a time
  int64_t len, chunks;      // columns of a chunk (a multiple of 4096), chunks of a row (at most 1024)
  unsigned grid;            // workgroups of a row
  int64_t groups, span;     // row groups of the last backward pass: enough workgroups for the chip, at least 4 rows each
};
Plan plan_of(int64_t rows, int64_t cols, int64_t size, bool backward) {
  auto over = [](int64_t n, int64_t d) { return (n + d - 1) / d; };
  Plan p;
  p.most = rows_at_once(rows, backward ? 0 : cols * size);
  p.len = over(cols, 8192) > 128 ? 16384 : 8192;
  while (p.len > 4096 && p.most * over(cols, p.len) < 1024) p.len >>= 1;
  if (over(cols, p.len) > 1024) p.len = over(over(cols, 1024), 4096) * 4096;
  p.chunks = over(cols, p.len);
  p.grid = (unsigned)(cols > 1 << 18 ? over(p.chunks, 8) * 8 : p.chunks);
  const int64_t wide = (cols + 1023) / 1024;
  p.groups = (1024 + wide - 1) / wide;
  if (p.groups > p.most / 4) p.groups = p.most / 4;
  p.groups = p.groups < 1 ? 1 : p.groups > 256 ? 256 : p.groups;
  p.span = (p.most + p.groups - 1) / p.groups;
  return p;
}

// Lanes of a row: the fewest that hold it with 16 bytes each, up to a wave; then 8 elements a lane (backward holds five arrays of that
// length, and on few rows fewer loads in a row are shorter: 4099 x 801 forward 10.4 us with 16 elements, 7.5 with 8), until 1024 lanes
// are not enough.  NT: lanes of a workgroup.  Backward few rows are one workgroup's, which then writes the weight's gradient itself, no
// partial rows and no second launch: up to four rounds of 256 lanes, or of 1024 two where a row takes more than a wave (8 x 800: 7.7 us
// in four rounds, 4.9 in one; 128 x 16: 3.2 us with 256 lanes, 3.5 with 1024).
// More rows, up to four rounds of 256 such workgroups, take 1024 lanes too: a quarter of the partial rows (4099 x 801 fp32 18.3 and 16.5 us,
// bf16 17.1 and 15.2; 100000 x 800 bf16 142 and 119; with 512 lanes a row in bf16 only: 1024 x 4000 16.5 and 14.6, fp32 15.4 and 15.9).
// `most` workgroups at once: DRAM serves a few long streams faster than many short ones, and backward each leaves a partial row of
// 2 cols numbers.  Of 256 lanes, backward 512 in fp32 (16.8 M x 16 555 us, 671 with 2048; 100000 x 800 164 and 190), where the two
// waves of a SIMD wait for less arithmetic than bf16's or a ragged row's, which take 1024 (16.8 M x 16 bf16 295, 339 with 512, 308
// with 2048).  Forward 2048; fp32 of 64 MB and more 1024 (16.8 M x 16 384 and 392 us, 100000 x 800 111 and 122).
struct Shape { int G, E, NT, most; };
Shape shape_of(int64_t rows, int64_t cols, int vec, bool backward) {
  Shape s = {0, 0, 256, 2048};
  for (int G = 1; G <= 64 && !s.G; G *= 2)
    if (cols <= (int64_t)G * vec) s.G = G, s.E = vec;
  for (int G = 64; G <= 1024 && !s.G; G *= 2)
    for (int E = 8; E <= (G < 1024 ? 8 : 16) && !s.G; E *= 2)
      if (cols <= (int64_t)G * E) s.G = G, s.E = E;
  if (s.G > 256) s.NT = s.G;
  const int64_t lanes = rows * s.G;
  if (backward && s.G > 64 && (lanes <= 2 * 1024 || (lanes >= 128 * 1024 && lanes <= 1024 * 1024 && s.G <= (vec == 4 ? 256 : 512)))) s.NT = 1024;
  const bool plain = vec == 4 && cols % vec == 0;
  if (backward) s.most = plain ? 512 : 1024;
  else if (plain && rows * cols >= 1 << 24) s.most = 1024;
  s.most = s.most * 256 / s.NT;
  if (s.most < 256) s.most = 256;
  return s;
}
bool one_workgroup(int64_t rows, const Shape& s) { return rows * s.G <= (s.G > 64 ? 2 * 1024 : 4 * 256); }
// Backward four rounds of rows each where that leaves a workgroup for every CU.
int64_t resident_blocks(int64_t rows, const Shape& s, bool backward) {
  const int64_t rpb = s.NT / s.G, need = (rows + rpb - 1) / rpb;
  int64_t n = need;
  if (backward) {
    if (one_workgroup(rows, s)) return 1;
    if (n > 256) n = need / 4 > 256 ? need / 4 : 256;
  }
  return n < s.most ? n : s.most;
}

bool sizes_ok(int64_t rows, int64_t cols) { return rows >= 0 && cols >= 1 && cols <= (int64_t)1 << 31 && rows <= ((int64_t)1 << 44) / cols; }

int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }

template <class T, int G, int K, int NT>
void launch_fwd(const T* x, const float* w, const float* b, T* y, float* stats, int64_t rows, int64_t cols, float eps, float slope,
                int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)blocks);
  const double inv = 1.0 / (double)cols;
#define LR_GO(RAGGED, STREAM) \
  hipLaunchKernelGGL((fwd_kernel<T, G, K, NT, RAGGED, STREAM>), grid, dim3(NT), 0, st, x, w, b, y, stats, rows, (int)cols, inv, (float)inv, eps, slope)
  if (cols % Vec<T>::N) LR_GO(true, false);
  else if (rows * cols * (int64_t)sizeof(T) >= kStream) LR_GO(false, true);
  else LR_GO(false, false);
#undef LR_GO
}
template <class T, int G, int K, int NT>
void launch_bwd(const T* x, const float* w, const float* b, const T* gy, T* gx, float* sw, float* sb, int64_t stride, int64_t rows,
                int64_t cols, float eps, float slope, int64_t blocks, hipStream_t st) {
  const dim3 grid((unsigned)blocks);
  const double inv = 1.0 / (double)cols;
#define LR_GO(RAGGED, ACT, STREAM) \
  hipLaunchKernelGGL((bwd_kernel<T, G, K, NT, RAGGED, ACT, STREAM>), grid, dim3(NT), 0, st, x, w, b, gy, gx, sw, sb, stride, rows, (int)cols, inv, (float)inv, eps, slope)
  const bool ragged = cols % Vec<T>::N, act = slope != 1.0f, stream = rows * cols * (int64_t)sizeof(T) >= kStream;
  if (ragged && act) LR_GO(true, true, false);
  else if (ragged) LR_GO(true, false, false);
  else if (act && stream) LR_GO(false, true, true);
  else if (act) LR_GO(false, true, false);
  else if (stream) LR_GO(false, false, true);
  else LR_GO(false, false, false);
#undef LR_GO
}

// CALL(lanes, vectors a lane, workgroup) for shape s
#define LR_LN_SHAPES(CALL)                                                        \
  if (s.G == 1) CALL(1, 1, 256);                                                  \
  else if (s.G == 2) CALL(2, 1, 256);                                             \
  else if (s.G == 4) CALL(4, 1, 256);                                             \
  else if (s.G == 8) CALL(8, 1, 256);                                             \
  else if (s.G == 16) CALL(16, 1, 256);                                           \
  else if (s.G == 32) CALL(32, 1, 256);                                           \
  else if (s.G == 64 && s.E == N) CALL(64, 1, 256);                               \
  else if (s.G == 64) CALL(64, 8 / N, 256);                                       \
  else if (s.G == 128 && s.NT == 256) CALL(128, 8 / N, 256);                      \
  else if (s.G == 256 && s.NT == 256) CALL(256, 8 / N, 256);                      \
  else if (s.G == 512 && s.NT == 512) CALL(512, 8 / N, 512);                      \
  else if (s.G == 1024 && s.E == 8) CALL(1024, 8 / N, 1024);                      \
  else if (s.G == 1024) CALL(1024, 16 / N, 1024)

template <class T>
int fwd(const T* x, const float* w, const float* b, T* y, float* stats, float* ws, int64_t rows, int64_t cols, float eps, float slope,
        hipStream_t st) {
  if (cols <= kResident) {
    constexpr int N = Vec<T>::N;
    const Shape s = shape_of(rows, cols, N, false);
#define LR_CALL(G, K, NT) launch_fwd<T, G, K, NT>(x, w, b, y, stats, rows, cols, eps, slope, resident_blocks(rows, s, false), st)
    LR_LN_SHAPES(LR_CALL);
#undef LR_CALL
    return lr_launch_status();
  }
  const Plan p = plan_of(rows, cols, sizeof(T), false);
  const int64_t len = p.len, most = p.most;
  const int chunks = (int)p.chunks;
  for (int64_t r = 0; r < rows; r += most) {
    const unsigned k = (unsigned)(rows - r < most ? rows - r : most);
    hipLaunchKernelGGL((chunk_stats_kernel<T>), dim3(p.grid, k), dim3(256), 0, st, x, ws, chunks, cols, len, r);
    hipLaunchKernelGGL((chunk_fwd_kernel<T>), dim3(p.grid, k), dim3(256), 0, st, x, w, b, y, ws, stats, chunks, cols, len, eps, slope, r);
    const int rc = lr_launch_status();
    if (rc != LR_OK) return rc;
  }
  return LR_OK;
}

int finish(const float* part, int64_t n, int64_t cols, float* gw, float* gb, hipStream_t st) {
  if (n <= 16) hipLaunchKernelGGL((finish_kernel<1>), dim3((unsigned)((2 * cols + 255) / 256)), dim3(256), 0, st, part, (int)n, cols, gw, gb);
  else hipLaunchKernelGGL((finish_kernel<32>), dim3((unsigned)((2 * cols + 31) / 32)), dim3(1024), 0, st, part, (int)n, cols, gw, gb);
  return lr_launch_status();
}

template <class T>
int bwd(const T* x, const float* w, const float* b, const T* gy, const float* stats, T* gx, float* gw, float* gb, float* ws,
        int64_t rows, int64_t cols, float eps, float slope, hipStream_t st) {
  if (cols <= kResident) {
    constexpr int N = Vec<T>::N;
    const Shape s = shape_of(rows, cols, N, true);
    const int64_t blocks = resident_blocks(rows, s, true);
    const bool part = blocks > 1 && (gw || gb);
    float *sw = part ? ws : gw, *sb = part ? ws + cols : gb;
    const int64_t stride = part ? 2 * cols : 0;
#define LR_CALL(G, K, NT) launch_bwd<T, G, K, NT>(x, w, b, gy, gx, sw, sb, stride, rows, cols, eps, slope, blocks, st)
    LR_LN_SHAPES(LR_CALL);
    else if (s.G == 128) LR_CALL(128, 8 / N, 1024);
    else if (s.G == 256) LR_CALL(256, 8 / N, 1024);
    else LR_CALL(512, 8 / N, 1024);
#undef LR_CALL
    const int rc = lr_launch_status();
    if (rc != LR_OK || !part) return rc;
    return finish(ws, blocks, cols, gw, gb, st);
  }
  const Plan p = plan_of(rows, cols, sizeof(T), true);
  const int64_t len = p.len, most = p.most, groups = p.groups, span = p.span;
  const int chunks = (int)p.chunks;
  const bool inside = span * chunks <= kJoin, direct = groups == 1;
  float* sums = ws + 2 * rows * p.chunks;
  float* own = sums + up16(2 * rows);
  float* part = own + up16(2 * rows);
  const dim3 grid((unsigned)((cols + 256 * Vec<T>::N - 1) / (256 * Vec<T>::N)), (unsigned)groups);
  float *sw = direct ? gw : part, *sb = direct ? gb : part + cols;
  const int64_t stride = direct ? 0 : 2 * cols;
  const float* sv = stats ? stats : own;
  const bool act = slope != 1.0f;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t end = r + most < rows ? r + most : rows;
    const unsigned k = (unsigned)(end - r);
    if (!stats) {
      hipLaunchKernelGGL((chunk_stats_kernel<T>), dim3(p.grid, k), dim3(256), 0, st, x, ws, chunks, cols, len, r);
      hipLaunchKernelGGL(join_stats_kernel, dim3(k), dim3(256), 0, st, ws, chunks, cols, len, eps, own, r);
    }
    if (act) hipLaunchKernelGGL((chunk_sums_kernel<T, true>), dim3(p.grid, k), dim3(256), 0, st, x, w, b, gy, sv, ws, chunks, cols, len, slope, r);
    else hipLaunchKernelGGL((chunk_sums_kernel<T, false>), dim3(p.grid, k), dim3(256), 0, st, x, w, b, gy, sv, ws, chunks, cols, len, slope, r);
    if (!inside) hipLaunchKernelGGL(join_sums_kernel, dim3(k), dim3(256), 0, st, ws, chunks, cols, sums, r);
#define LR_GO(JOIN, ACT)                                                                                                              \
  hipLaunchKernelGGL((chunk_bwd_kernel<T, JOIN, ACT>), grid, dim3(256), 0, st, x, w, b, gy, sv, inside ? ws : sums, gx, sw, sb, stride, r, \
                     end, span, chunks, cols, slope, r > 0)
    if (inside && act) LR_GO(true, true);
    else if (inside) LR_GO(true, false);
    else if (act) LR_GO(false, true);
    else LR_GO(false, false);
#undef LR_GO
    const int rc = lr_launch_status();
    if (rc != LR_OK) return rc;
  }
  if (direct || !(gw || gb)) return LR_OK;
  return finish(part, groups, cols, gw, gb, st);
}

__global__ __launch_bounds__(256) void zero_kernel(float* a, float* b, int64_t n) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    if (a) a[i] = 0.f;
    if (b) b[i] = 0.f;
  }
}

}  // namespace

extern "C" int64_t lr_layer_norm_resident_cols(void) { return kResident; }

extern "C" int64_t lr_layer_norm_workspace(int64_t rows, int64_t cols, int backward) {
  if (!sizes_ok(rows, cols)) return LR_EINVAL;
  if (rows == 0) return 0;
  if (cols <= kResident) {
    if (!backward) return 0;
    // the larger of the two types' launches
    const int64_t a = resident_blocks(rows, shape_of(rows, cols, 4, true), true), b = resident_blocks(rows, shape_of(rows, cols, 8, true), true);
    return a == 1 && b == 1 ? 0 : 4 * 2 * cols * (a > b ? a : b);
  }
  const Plan p = plan_of(rows, cols, 2, backward), q = plan_of(rows, cols, 4, backward);      // the larger of the two types'
  const int64_t words = 2 * rows * (p.chunks > q.chunks ? p.chunks : q.chunks), groups = p.groups > q.groups ? p.groups : q.groups;
  return 4 * (words + (backward ? 2 * up16(2 * rows) + (groups > 1 ? 2 * cols * groups : 0) : 0));
}

extern "C" int lr_layer_norm(const void* x, const float* w, const float* b, void* y, float* stats, void* workspace, int64_t rows,
                             int64_t cols, int bf16, float eps, float slope, void* stream) {
  if (!sizes_ok(rows, cols) || !(eps >= 0.f)) return LR_EINVAL;
  if (rows == 0) return LR_OK;
  if (!x || !y || (cols > kResident && !workspace)) return LR_ENULL;
  hipStream_t st = lr_stream(stream);
  float* ws = static_cast<float*>(workspace);
  if (bf16) return fwd(static_cast<const uint16_t*>(x), w, b, static_cast<uint16_t*>(y), stats, ws, rows, cols, eps, slope, st);
  return fwd(static_cast<const float*>(x), w, b, static_cast<float*>(y), stats, ws, rows, cols, eps, slope, st);
}

extern "C" int lr_layer_norm_bwd(const void* x, const float* w, const float* b, const void* gy, const float* stats, void* gx, float* gw,
                                 float* gb, void* workspace, int64_t rows, int64_t cols, int bf16, float eps, float slope, void* stream) {
  if (!sizes_ok(rows, cols) || !(eps >= 0.f)) return LR_EINVAL;
  hipStream_t st = lr_stream(stream);
  if (rows == 0) {
    if (!gw && !gb) return LR_OK;
    hipLaunchKernelGGL(zero_kernel, dim3((unsigned)((cols + 255) / 256 < 1024 ? (cols + 255) / 256 : 1024)), dim3(256), 0, st, gw, gb, cols);
    return lr_launch_status();
  }
  if (!gx && !gw && !gb) return LR_OK;
  if (!x || !gy || (!workspace && lr_layer_norm_workspace(rows, cols, 1))) return LR_ENULL;
  float* ws = static_cast<float*>(workspace);
  if (bf16)
    return bwd(static_cast<const uint16_t*>(x), w, b, static_cast<const uint16_t*>(gy), stats, static_cast<uint16_t*>(gx), gw, gb, ws, rows,
               cols, eps, slope, st);
  return bwd(static_cast<const float*>(x), w, b, static_cast<const float*>(gy), stats, static_cast<float*>(gx), gw, gb, ws, rows, cols, eps,
             slope, st);
}
