// optim.hip — the update of the network's parameters: the AdamW step over all the tensors of a model (64 tensors a launch, 61 with
// 8-bit states), with 32-bit or block-scaled 8-bit states, and the global norm of the gradients it clips by.
//
// The reference trains with torch.optim.Adam (src/liftreg/networks/RegistrationNet.py:245); with weight_decay = 0 this is its step.
//   g = grad * c,  c = min(1, max_norm / (|grad|_2 + 1e-6))         (c = 1 without clipping)
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit states: 32 consecutive elements of a tensor share a power-of-two scale 2^(s - 127) (one byte, e8m0); m / scale is held in
// e4m3, v / scale in e5m2.  Both are rounded stochastically: a step moves v by (1 - b2) = 0.1 % of itself while neighbouring codes
// are 12 ... 25 % apart, so rounding to nearest would leave v where it is for ever; rounding up with the probability of the
// remainder keeps the expected state equal to the unrounded one.  A v that is not zero never rounds to zero (m / eps would follow).
// The block's largest magnitude is placed in [2^7, 2^8) of e4m3's 448 and in [2^14, 2^15) of e5m2's 57344: rounding up cannot
// overflow.  The 16 + 16 random bits of an element are a hash of (seed, step, position), so a step can be repeated bit for bit.
// 32-bit states are formed with the separate fp32 roundings of the formula above (no contraction), 8-bit ones in fp64 before their one
// rounding; the update itself uses v_sqrt_f32 / v_rcp_f32 (1 ulp each, of a number that is lr times smaller than p).
#include "lr_common.h"

namespace {

constexpr int kThreads = 256;
// A workgroup takes chunks of ROUNDS * 1024 elements (whole 32-element scale blocks): four rounds where there is work for every wave
// slot of the chip, one where the launch is latency and more workgroups shorten it (0.55 M elements: 6.4 us with four, 4.8 with one).
constexpr int kRound = kThreads * 4;
constexpr int kTensors = 64;                        // tensors of one launch: a lane each in the search for a chunk's tensor
constexpr int kBlocks = 2048;                       // four waves each: every wave slot of the 256 CUs
constexpr int kNormBlocks = 1024;                    // of the norm: each leaves a number that every workgroup of the step adds up again

// tensors of one launch, by value in the kernel arguments (at most 4 KB): nothing to upload, nothing that a captured graph could
// outlive
struct Table32 {
  static constexpr int kMax = kTensors;
  void* p[kMax];
  const void* g[kMax];
  float* m[kMax];
  float* v[kMax];
  int64_t n[kMax];
  uint32_t end[kMax];   // chunks of this launch up to and including this tensor
  int count;
};
struct Table8 {
  static constexpr int kMax = 61;
  void* p[kMax];
  const void* g[kMax];
  uint8_t* m[kMax];
  uint8_t* v[kMax];
  uint8_t* ms[kMax];
  uint8_t* vs[kMax];
  int64_t n[kMax];
  uint32_t end[kMax];
  uint32_t pos[kMax];   // position of the tensor's first element in the concatenation padded to whole scale blocks, mod 2^32
  int count;
};
struct TableG {
  static constexpr int kMax = 3 * kTensors;      // three tensors a lane
  const void* g[kMax];
  int64_t n[kMax];
  uint32_t end[kMax];
  int count;
};

struct Rates {               // what a step derives from its hyperparameters
  float size, rbc2, keep;
  uint32_t key;
};
struct Hyper {
  double b1, b2, lr, eps, wd;
  Rates r;                   // of (lr, step); derived on the device where one of them lives there
  const float* lr_dev;       // if set: the learning rate
  const int64_t* step_dev;   // if set: the step
  int64_t step;
  const double* sumsq;       // partial sums of squares of the gradients (n_sumsq of them), or NULL
  const float* norm_in;      // the gradients' norm, or NULL
  float* norm_out;
  int n_sumsq;
  float max_norm;
  uint64_t seed;
};

static_assert(sizeof(Table32) + sizeof(Hyper) <= 4096 && sizeof(Table8) + sizeof(Hyper) <= 4096 && sizeof(TableG) + 8 <= 4096,
              "a launch's arguments are at most 4 KB");

// the alignment of a tensor that is a view into a flat buffer is its element's: gfx950 loads 16 bytes from any dword (or byte)
// address in one instruction, aligned or not at the same rate where the access is contiguous over the wave
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u1 __attribute__((aligned(1)));

struct F32 { float x[4]; };

__device__ __forceinline__ float bf_to_f(uint16_t u) { return __uint_as_float((uint32_t)u << 16); }
__device__ __forceinline__ uint16_t f_to_bf(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }   // nearest even

// 4 elements at i of an array of n (elements past the end read as 0 and are not written).  ONCE: they are not wanted again before the
// next step and leave the caches to the gradients, which the norm has read just before (13.5 M parameters with clipping 86 us without,
// 73 with; 44.6 M without clipping 243 and 225).
template <bool ONCE>
__device__ __forceinline__ F32 load4(const float* a, int64_t i, int64_t n) {
  F32 r = {{0.f, 0.f, 0.f, 0.f}};
  if (i + 4 <= n) {
    const f4* at = reinterpret_cast<const f4*>(a + i);
    const f4 t = ONCE ? __builtin_nontemporal_load(at) : *at;
    r.x[0] = t[0]; r.x[1] = t[1]; r.x[2] = t[2]; r.x[3] = t[3];
  } else {
    for (int k = 0; k < 3; ++k)
      if (i + k < n) r.x[k] = a[i + k];
  }
  return r;
}
template <bool ONCE>
__device__ __forceinline__ F32 load4(const uint16_t* a, int64_t i, int64_t n) {
  F32 r = {{0.f, 0.f, 0.f, 0.f}};
  if (i + 4 <= n) {
    const h4* at = reinterpret_cast<const h4*>(a + i);
    const h4 t = ONCE ? __builtin_nontemporal_load(at) : *at;
    for (int k = 0; k < 4; ++k) r.x[k] = bf_to_f(t[k]);
  } else {
    for (int k = 0; k < 3; ++k)
      if (i + k < n) r.x[k] = bf_to_f(a[i + k]);
  }
  return r;
}
__device__ __forceinline__ void store4(float* a, int64_t i, int64_t n, const F32& r) {
  if (i + 4 <= n) {
    f4 t = {r.x[0], r.x[1], r.x[2], r.x[3]};
    __builtin_nontemporal_store(t, reinterpret_cast<f4*>(a + i));
  } else {
    for (int k = 0; k < 3; ++k)
      if (i + k < n) a[i + k] = r.x[k];
  }
}
__device__ __forceinline__ void store4(uint16_t* a, int64_t i, int64_t n, const F32& r) {
  if (i + 4 <= n) {
    typedef float F __attribute__((ext_vector_type(4)));
    typedef __bf16 B __attribute__((ext_vector_type(4)));
    const h4 t = __builtin_bit_cast(h4, __builtin_convertvector((F{r.x[0], r.x[1], r.x[2], r.x[3]}), B));      // two in an instruction
    __builtin_nontemporal_store(t, reinterpret_cast<h4*>(a + i));
  } else {
    for (int k = 0; k < 3; ++k)
      if (i + k < n) a[i + k] = f_to_bf(r.x[k]);
  }
}
__device__ __forceinline__ uint32_t load4b(const uint8_t* a, int64_t i, int64_t n) {
  if (i + 4 <= n) return *reinterpret_cast<const u1*>(a + i);
  uint32_t r = 0;
  for (int k = 0; k < 3; ++k)
    if (i + k < n) r |= (uint32_t)a[i + k] << (8 * k);
  return r;
}
__device__ __forceinline__ void store4b(uint8_t* a, int64_t i, int64_t n, uint32_t r) {
  if (i + 4 <= n) *reinterpret_cast<u1*>(a + i) = r;
  else
    for (int k = 0; k < 3; ++k)
      if (i + k < n) a[i + k] = (uint8_t)(r >> (8 * k));
}

// The table as the lanes of a wave hold it, lane k tensor k: all of it is fetched at once (kernel arguments are a miss of about a
// microsecond), and a chunk's tensor is a ballot and a few readlanes away.
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int k) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), k) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, k);
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int k) { return (uint32_t)__builtin_amdgcn_readlane((int)v, k); }
template <class P>
__device__ __forceinline__ P* lane_ptr(uint64_t v, int k) { return reinterpret_cast<P*>(lane_of(v, k)); }

struct Sizes {               // every table's, 64 tensors of it
  uint64_t n;
  uint32_t end;
  template <class T>
  __device__ __forceinline__ void fetch(const T& t, int first) {
    const int lane = threadIdx.x & 63, i = min(first + lane, t.count - 1);
    n = (uint64_t)t.n[i];
    end = first + lane < t.count ? t.end[i] : 0xffffffffu;
  }
  __device__ __forceinline__ int before(uint32_t c) const { return (int)__popcll(__ballot(end <= c)); }      // tensors that end there
  // the tensor that chunk c belongs to, its size and the chunk's first element
  __device__ __forceinline__ int find(uint32_t c, int64_t chunk, int64_t& size, int64_t& base) const {
    const int k = __builtin_amdgcn_readfirstlane(before(c));
    size = (int64_t)lane_of(n, k);
    base = (int64_t)(c - (k ? lane_of(end, k - 1) : 0u)) * chunk;
    return k;
  }
};
template <class T> struct Held;
template <> struct Held<TableG> {
  Sizes z0, z1, z2;
  uint64_t g0, g1, g2;
  __device__ __forceinline__ explicit Held(const TableG& t) {
    const int lane = threadIdx.x & 63, last = t.count - 1;
    z0.fetch(t, 0);
    z1.fetch(t, 64);
    z2.fetch(t, 128);
    g0 = (uint64_t)t.g[min(lane, last)];
    g1 = (uint64_t)t.g[min(64 + lane, last)];
    g2 = (uint64_t)t.g[min(128 + lane, last)];
  }
  // readlane from all three, then a scalar choice
  template <class V>
  static __device__ __forceinline__ V of(V a, V b, V c, int k) {
    const V x = lane_of(a, k & 63), y = lane_of(b, k & 63), z = lane_of(c, k & 63);
    return k < 64 ? x : k < 128 ? y : z;
  }
  template <class G>
  __device__ __forceinline__ const G* find(uint32_t c, int64_t chunk, int64_t& size, int64_t& base) const {
    const int k = __builtin_amdgcn_readfirstlane(z0.before(c) + z1.before(c) + z2.before(c));
    size = (int64_t)of(z0.n, z1.n, z2.n, k);
    base = (int64_t)(c - (k ? of(z0.end, z1.end, z2.end, k - 1) : 0u)) * chunk;
    return reinterpret_cast<const G*>(of(g0, g1, g2, k));
  }
};
template <> struct Held<Table32> {
  Sizes z;
  uint64_t p, g, m, v;
  __device__ __forceinline__ explicit Held(const Table32& t) {
    const int i = min((int)(threadIdx.x & 63), t.count - 1);
    z.fetch(t, 0);
    p = (uint64_t)t.p[i];
    g = (uint64_t)t.g[i];
    m = (uint64_t)t.m[i];
    v = (uint64_t)t.v[i];
  }
};
template <> struct Held<Table8> {
  Sizes z;
  uint64_t p, g, m, v, ms, vs;
  uint32_t pos;
  __device__ __forceinline__ explicit Held(const Table8& t) {
    const int i = min((int)(threadIdx.x & 63), t.count - 1);
    z.fetch(t, 0);
    p = (uint64_t)t.p[i];
    g = (uint64_t)t.g[i];
    m = (uint64_t)t.m[i];
    v = (uint64_t)t.v[i];
    ms = (uint64_t)t.ms[i];
    vs = (uint64_t)t.vs[i];
    pos = t.pos[i];
  }
};

__device__ __forceinline__ double block_sum(double s) {   // the same order in every block: the same bits
  __shared__ double red[kThreads / 64];
  s = lr_wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// ---------------------------------------------------------------- the gradients' norm
// fp64 accumulators: 13 M squares of numbers that span decades; the conversion and the fma hide under the read.
template <class G, int ROUNDS>
__global__ __launch_bounds__(kThreads) void sumsq_kernel(TableG t, double* __restrict__ partial) {
  const Held<TableG> held(t);
  const uint32_t chunks = t.end[t.count - 1];
  double s = 0.0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int64_t n, base;
    const G* g = held.find<G>(c, ROUNDS * kRound, n, base);
    F32 x[ROUNDS];
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) x[j] = load4<false>(g, base + (j * kThreads + threadIdx.x) * 4, n);
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fma((double)x[j].x[e], (double)x[j].x[e], s);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double* __restrict__ partial, int n, float* __restrict__ out) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += partial[i];
  s = block_sum(s);
  if (threadIdx.x == 0) *out = (float)sqrt(s);
}

// ---------------------------------------------------------------- 8-bit states
__host__ __device__ inline uint32_t mix(uint32_t x) {   // xor-shift and odd multiplication, twice: a bijection of 32 bits
  x ^= x >> 16;
  x *= 0x0A00F875u;
  x ^= x >> 15;
  x *= 0x517B5965u;
  return x ^ (x >> 16);
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true));
}
// over the 8 lanes that hold a scale block: neighbours, pairs, then the mirrored half row
__device__ __forceinline__ uint32_t max8(uint32_t x) { return max_dpp<0x141>(max_dpp<0x4E>(max_dpp<0xB1>(x))); }

__device__ __forceinline__ float scale_of(uint32_t s) {   // 2^(s - 127); 255 is NaN, 0 the subnormal 2^-127
  const uint32_t b = s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23;
  return __uint_as_float(b);
}

__device__ __forceinline__ uint32_t high(double x) { return (uint32_t)(__double_as_longlong(x) >> 32); }
__device__ __forceinline__ double pow2(int e) { return __longlong_as_double((int64_t)(e + 1023) << 52); }

// the exponent byte of the block's scale: its peak lands in [2^top, 2^(top+1)); 255 where it is beyond fp32 or no number
template <int TOP>
__device__ __forceinline__ uint32_t block_scale(const double (&a)[4]) {
  uint32_t u = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) u = max(u, high(a[e]) & 0x7fffffffu);
  const int ex = (int)(max8(u) >> 20) - (1023 - 127);
  return ex > 254 ? 255u : (uint32_t)max(ex - TOP, 1);
}

// |x| / scale in MAN mantissa bits, exponent bias BIAS, rounded up with the probability of what is cut off, for 4 elements.  The random
// bits end above the low word, which therefore cannot carry.  Below the smallest normal number the steps are even; few waves meet one.
template <int MAN, int BIAS>
__device__ __forceinline__ void codes_of(const double (&x)[4], double inv, const uint32_t (&r)[4], uint32_t (&c)[4]) {
  constexpr uint32_t NORMAL = (1024u - BIAS) << 20;
  double y[4];
  bool low = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = fabs(x[e]) * inv;
    low |= high(y[e]) < NORMAL;
    c[e] = ((high(y[e]) + (r[e] << (20 - MAN - 16))) >> (20 - MAN)) - ((1023u - BIAS) << MAN);
  }
  if (__builtin_expect(__any(low), 0)) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (high(y[e]) < NORMAL) c[e] = (uint32_t)(int)fma(y[e], (double)(1u << (BIAS - 1 + MAN)), (double)r[e] * 0x1p-16);
  }
}

typedef float f2 __attribute__((ext_vector_type(2)));

template <class T>
struct State;   // how a step reads and writes the two moments of 4 elements; At: where those of a tensor are

template <>
struct State<Table32> {
  struct At {
    float *m, *v;
    __device__ __forceinline__ At(const Held<Table32>& h, int k) : m(lane_ptr<float>(h.m, k)), v(lane_ptr<float>(h.v, k)) {}
  };
  typedef float R;           // what the moments are formed in
  R m[4], v[4];
  __device__ __forceinline__ void load(const At& t, int64_t i, int64_t n) {
    const F32 a = load4<true>(t.m, i, n), b = load4<true>(t.v, i, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = a.x[e];
      v[e] = b.x[e];
    }
  }
  __device__ __forceinline__ void open() {}
  __device__ __forceinline__ void store(const At& t, int64_t i, int64_t n, uint32_t) {
    store4(t.m, i, n, {{m[0], m[1], m[2], m[3]}});
    store4(t.v, i, n, {{v[0], v[1], v[2], v[3]}});
  }
};

template <>
struct State<Table8> {
  struct At {
    uint8_t *m, *v, *ms, *vs;
    uint32_t pos;
    __device__ __forceinline__ At(const Held<Table8>& h, int k)
        : m(lane_ptr<uint8_t>(h.m, k)), v(lane_ptr<uint8_t>(h.v, k)), ms(lane_ptr<uint8_t>(h.ms, k)), vs(lane_ptr<uint8_t>(h.vs, k)),
          pos(lane_of(h.pos, k)) {}
  };
  // fp64 runs at fp32's rate here: the stochastic rounding then starts from the moments themselves and not from their fp32 neighbours,
  // which land on the other side of a code now and then
  typedef double R;
  R m[4], v[4];
  uint32_t mq, vq, ms, vs;
  __device__ __forceinline__ void load(const At& t, int64_t i, int64_t n) {
    mq = load4b(t.m, i, n);
    vq = load4b(t.v, i, n);
    ms = i < n ? t.ms[i >> 5] : 1u;
    vs = i < n ? t.vs[i >> 5] : 1u;
  }
  __device__ __forceinline__ void open() {
    const float a = scale_of(ms), b = scale_of(vs);
    const f2 m0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mq, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mq, true);
    const f2 v0 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vq, false), v1 = __builtin_amdgcn_cvt_pk_f32_bf8((int)vq, true);
    m[0] = m0[0] * a; m[1] = m0[1] * a; m[2] = m1[0] * a; m[3] = m1[1] * a;
    v[0] = v0[0] * b; v[1] = v0[1] * b; v[2] = v1[0] * b; v[3] = v1[1] * b;
  }
  // every lane of the wave comes here (elements past the end are zeros): the scale is a maximum over 8 lanes
  __device__ __forceinline__ void store(const At& t, int64_t i, int64_t n, uint32_t key) {
    ms = block_scale<7>(m);
    vs = block_scale<14>(v);
    const double a = pow2(127 - (int)ms), b = pow2(127 - (int)vs);
    uint32_t rm[4], rv[4], cm[4], cv[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t r = mix((t.pos + (uint32_t)i + e) ^ key);
      rm[e] = r & 0xffffu;
      rv[e] = r >> 16;
      if (ms == 255u) m[e] = 0.0;      // a block that is not finite: scale NaN, codes 0
      if (vs == 255u) v[e] = 0.0;
    }
    codes_of<3, 7>(m, a, rm, cm);
    codes_of<2, 15>(v, b, rv, cv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cm[e] |= high(m[e]) >> 24 & 0x80u;
      if (v[e] > 0.0) cv[e] = max(cv[e], 1u);
    }
    store4b(t.m, i, n, cm[0] | cm[1] << 8 | cm[2] << 16 | cm[3] << 24);
    store4b(t.v, i, n, cv[0] | cv[1] << 8 | cv[2] << 16 | cv[3] << 24);
    if ((threadIdx.x & 7) == 0 && i < n) {
      t.ms[i >> 5] = (uint8_t)ms;
      t.vs[i >> 5] = (uint8_t)vs;
    }
  }
};

__host__ __device__ inline double ipow(double b, int64_t t) {   // b^t, t >= 0
  double r = 1.0;
  for (; t > 0; t >>= 1) {
    if (t & 1) r *= b;
    b *= b;
  }
  return r;
}
__host__ __device__ inline Rates rates(const Hyper& h, double lr, int64_t step) {
  Rates r;
  r.size = (float)(lr / (1.0 - ipow(h.b1, step)));
  r.rbc2 = (float)(1.0 / sqrt(1.0 - ipow(h.b2, step)));
  r.keep = (float)(1.0 - lr * h.wd);
  r.key = mix(mix(mix((uint32_t)step) ^ (uint32_t)(h.seed >> 32)) ^ (uint32_t)h.seed);
  return r;
}

// Bound by memory: 28 bytes an element with 32-bit states and fp32 parameters, 16 with 8-bit ones.
template <class P, class T, int ROUNDS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(T t, Hyper h) {
  const Held<T> held(t);
  const uint32_t chunks = lane_of(held.z.end, t.count - 1);
  Rates r = h.r;
  if (h.lr_dev || h.step_dev) r = rates(h, h.lr_dev ? (double)*h.lr_dev : h.lr, h.step_dev ? *h.step_dev : h.step);
  typedef typename State<T>::R R;
  const R b1 = (R)h.b1, b2 = (R)h.b2, c1 = (R)(1.0 - h.b1), c2 = (R)(1.0 - h.b2);
  const float eps = (float)h.eps;
  // v_sqrt_f32 takes subnormals as 0.  Their roots, below 2^-63, are less than half a step of a larger eps; next to such a one v is scaled
  // (always: 2.5 % more time with 8-bit states)
  const bool tiny = __builtin_amdgcn_readfirstlane(eps < r.rbc2 * 0x1p-38f);
  R coef = 1;
  if (h.sumsq || h.norm_in) {
    R norm;
    if (h.sumsq) {
      double s = 0.0;
      for (int i = threadIdx.x; i < h.n_sumsq; i += kThreads) s += h.sumsq[i];
      norm = (R)sqrt(block_sum(s));
      if (blockIdx.x == 0 && threadIdx.x == 0 && h.norm_out) *h.norm_out = (float)norm;
    } else {
      norm = *h.norm_in;
    }
    coef = (R)h.max_norm / (norm + (R)1e-6);
    coef = coef > (R)1 ? (R)1 : coef;     // NaN stays NaN
  }
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    int64_t n, base;
    const int k = held.z.find(c, ROUNDS * kRound, n, base);
    P* pp = lane_ptr<P>(held.p, k);
    const P* gp = lane_ptr<const P>(held.g, k);
    const typename State<T>::At at(held, k);
    // rounds in flight: with 8-bit states one (61 registers, eight waves a SIMD) beats two (89, five): 13.5 M bf16 parameters 35 and 38 us;
    // 32-bit states 57 us either way, 44.6 M 246 with one and 243 with two
    constexpr int Q = ROUNDS < 2 || T::kMax < kTensors ? 1 : 2;
#pragma unroll
    for (int j = 0; j < ROUNDS; j += Q) {
      F32 p[Q], g[Q];
      State<T> s[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int64_t i = base + ((j + q) * kThreads + threadIdx.x) * 4;
        g[q] = load4<false>(gp, i, n);
        s[q].load(at, i, n);
        p[q] = load4<true>(pp, i, n);
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int64_t i = base + ((j + q) * kThreads + threadIdx.x) * 4;
        s[q].open();
        float root[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const R x = (R)g[q].x[e] * coef;
          const R m = s[q].m[e] * b1 + x * c1, v = s[q].v[e] * b2 + x * x * c2;
          s[q].m[e] = m;
          s[q].v[e] = v;
          root[e] = __builtin_amdgcn_sqrtf((float)v);
        }
        if (tiny) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((float)s[q].v[e] < 0x1p-96f) root[e] = __builtin_amdgcn_sqrtf((float)s[q].v[e] * 0x1p64f) * 0x1p-32f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float den = fmaf(root[e], r.rbc2, eps);
          p[q].x[e] = p[q].x[e] * r.keep - r.size * ((float)s[q].m[e] * __builtin_amdgcn_rcpf(den));
        }
        store4(pp, i, n, p[q]);
        s[q].store(at, i, n, r.key);
      }
    }
  }
}

// ---------------------------------------------------------------- host
bool sizes_ok(const int64_t* numel, int n) {
  if (n < 1) return false;
  for (int i = 0; i < n; ++i)
    if (numel[i] < 0 || numel[i] > (int64_t)1 << 40) return false;
  return true;
}

// v_rcp_f32 takes subnormals as 0, and where g and v are 0 the denominator is eps
bool eps_ok(double eps) { return eps == 0.0 || eps >= 0x1p-126; }

// Calls f(first, last, rounds, chunks) for each run of at most `most` tensors with elements; rounds of a chunk (see kRound): four where
// that leaves at least `blocks` chunks of one round.
template <class F>
int for_launches(const int64_t* numel, int n, int most, int64_t blocks, F f) {
  int first = 0;
  while (first < n) {
    int last = first, held = 0;
    int64_t chunks1 = 0, chunks4 = 0;
    while (last < n && held < most) {
      const int64_t one = (numel[last] + kRound - 1) / kRound, four = (numel[last] + 4 * kRound - 1) / (4 * kRound);
      if (chunks4 + four > 0x7fffffff) break;
      chunks1 += one;
      chunks4 += four;
      held += numel[last] > 0;
      ++last;
    }
    const bool small = chunks1 <= blocks;
    if (held) {
      const int rc = f(first, last, small ? 1 : 4, (uint32_t)(small ? chunks1 : chunks4));
      if (rc != LR_OK) return rc;
    }
    first = last;
  }
  return LR_OK;
}

// t's sizes and chunk ends of tensors [first, last), calling put(slot, tensor) for each that has elements
template <class T, class F>
void fill(T& t, const int64_t* numel, int first, int last, int rounds, F put) {
  int k = 0;
  uint32_t end = 0;
  for (int i = first; i < last; ++i) {
    if (!numel[i]) continue;
    put(k, i);
    t.n[k] = numel[i];
    t.end[k++] = end += (uint32_t)((numel[i] + rounds * kRound - 1) / (rounds * kRound));
  }
  t.count = k;
}

unsigned norm_blocks(uint32_t chunks) { return chunks < (uint32_t)kNormBlocks ? chunks : (unsigned)kNormBlocks; }

int sumsq_launches(const void* const* grads, const int64_t* numel, int n, int bf16, double* partial, hipStream_t st) {
  int used = 0;
  return for_launches(numel, n, TableG::kMax, kNormBlocks, [&](int first, int last, int rounds, uint32_t chunks) {
    TableG t;
    fill(t, numel, first, last, rounds, [&](int k, int i) { t.g[k] = grads[i]; });
    const dim3 nb(norm_blocks(chunks));
    double* out = partial + used;
    used += (int)nb.x;
    if (bf16 && rounds == 1) hipLaunchKernelGGL((sumsq_kernel<uint16_t, 1>), nb, dim3(kThreads), 0, st, t, out);
    else if (bf16) hipLaunchKernelGGL((sumsq_kernel<uint16_t, 4>), nb, dim3(kThreads), 0, st, t, out);
    else if (rounds == 1) hipLaunchKernelGGL((sumsq_kernel<float, 1>), nb, dim3(kThreads), 0, st, t, out);
    else hipLaunchKernelGGL((sumsq_kernel<float, 4>), nb, dim3(kThreads), 0, st, t, out);
    return lr_launch_status();
  });
}

template <class T>
int launch_step(const T& t, const Hyper& h, uint32_t chunks, int rounds, int bf16, hipStream_t st) {
  const dim3 grid(chunks < (uint32_t)kBlocks ? chunks : (uint32_t)kBlocks);
  if (bf16 && rounds == 1) hipLaunchKernelGGL((adamw_kernel<uint16_t, T, 1>), grid, dim3(kThreads), 0, st, t, h);
  else if (bf16) hipLaunchKernelGGL((adamw_kernel<uint16_t, T, 4>), grid, dim3(kThreads), 0, st, t, h);
  else if (rounds == 1) hipLaunchKernelGGL((adamw_kernel<float, T, 1>), grid, dim3(kThreads), 0, st, t, h);
  else hipLaunchKernelGGL((adamw_kernel<float, T, 4>), grid, dim3(kThreads), 0, st, t, h);
  return lr_launch_status();
}

}  // namespace

extern "C" int64_t lr_grad_norm_partials(const int64_t* numel, int n) {
  if (!numel) return LR_ENULL;
  if (!sizes_ok(numel, n)) return LR_EINVAL;
  int64_t used = 0;
  for_launches(numel, n, TableG::kMax, kNormBlocks, [&](int, int, int, uint32_t chunks) {
    used += norm_blocks(chunks);
    return LR_OK;
  });
  return used;
}

extern "C" int lr_grad_norm(const void* const* grads, const int64_t* numel, int n, int bf16, double* partial, float* norm,
                            void* stream) {
  if (!grads || !numel || !partial || !norm) return LR_ENULL;
  const int64_t used = lr_grad_norm_partials(numel, n);
  if (used < 0) return (int)used;
  for (int i = 0; i < n; ++i)
    if (numel[i] && !grads[i]) return LR_ENULL;
  hipStream_t st = lr_stream(stream);
  const int rc = sumsq_launches(grads, numel, n, bf16, partial, st);
  if (rc != LR_OK) return rc;
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, partial, (int)used, norm);
  return lr_launch_status();
}

extern "C" int lr_adamw_step(void* const* params, const void* const* grads, void* const* exp_avg, void* const* exp_avg_sq,
                             void* const* exp_avg_scale, void* const* exp_avg_sq_scale, const int64_t* numel, int n, int bf16,
                             double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                             const float* lr_dev, const int64_t* step_dev, float max_norm, const float* norm_in,
                             double* partial, float* norm_out, uint64_t seed, void* stream) {
  if (!params || !grads || !exp_avg || !exp_avg_sq || !numel) return LR_ENULL;
  if (!exp_avg_scale != !exp_avg_sq_scale) return LR_ENULL;
  if (!sizes_ok(numel, n)) return LR_EINVAL;
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps_ok(eps)) || (!step_dev && step < 1)) return LR_EINVAL;
  if ((norm_in || partial) && !(max_norm > 0)) return LR_EINVAL;
  if (norm_in && partial) return LR_EINVAL;
  const bool eight = exp_avg_scale != nullptr;
  for (int i = 0; i < n; ++i)
    if (numel[i] && (!params[i] || !grads[i] || !exp_avg[i] || !exp_avg_sq[i] || (eight && (!exp_avg_scale[i] || !exp_avg_sq_scale[i]))))
      return LR_ENULL;
  hipStream_t st = lr_stream(stream);
  Hyper h = {beta1, beta2, lr, eps, weight_decay, {}, lr_dev, step_dev, step, partial, norm_in, norm_out, 0, max_norm, seed};
  h.r = rates(h, lr, step_dev ? 1 : step);
  if (partial) {
    h.n_sumsq = (int)lr_grad_norm_partials(numel, n);
    const int rc = sumsq_launches(grads, numel, n, bf16, partial, st);
    if (rc != LR_OK) return rc;
    if (!h.n_sumsq && norm_out) {     // no element at all: the norm is 0
      hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, partial, 0, norm_out);
      return lr_launch_status();
    }
  }
  if (!eight)
    return for_launches(numel, n, Table32::kMax, kBlocks, [&](int first, int last, int rounds, uint32_t chunks) {
      Table32 t;
      fill(t, numel, first, last, rounds, [&](int k, int i) {
        t.p[k] = params[i];
        t.g[k] = grads[i];
        t.m[k] = static_cast<float*>(exp_avg[i]);
        t.v[k] = static_cast<float*>(exp_avg_sq[i]);
      });
      return launch_step(t, h, chunks, rounds, bf16, st);
    });
  uint32_t pos = 0;
  return for_launches(numel, n, Table8::kMax, kBlocks, [&](int first, int last, int rounds, uint32_t chunks) {
    Table8 t;
    fill(t, numel, first, last, rounds, [&](int k, int i) {
      t.p[k] = params[i];
      t.g[k] = grads[i];
      t.m[k] = static_cast<uint8_t*>(exp_avg[i]);
      t.v[k] = static_cast<uint8_t*>(exp_avg_sq[i]);
      t.ms[k] = static_cast<uint8_t*>(exp_avg_scale[i]);
      t.vs[k] = static_cast<uint8_t*>(exp_avg_sq_scale[i]);
      t.pos[k] = pos;
      pos += (uint32_t)((numel[i] + 31) & ~(int64_t)31);
    });
    return launch_step(t, h, chunks, rounds, bf16, st);
  });
}
