// Operators over many tensors in one launch: the AdamW step with 32-bit or 8-bit states, the common norm of a list of
// gradients, and their clipping (include/pdes_hip.h: pdes_adamw_step, pdes_grad_norm, pdes_clip_grads).
//
// One workgroup walks over chunks of the concatenated list.  The list itself (addresses, lengths) travels BY VALUE in the
// kernel arguments, up to 96 tensors a launch: nothing to copy, no buffer that a later call could overwrite while an
// earlier launch still reads it, and a captured graph holds its own copy.
//
// This file is compiled with -ffp-contract=off: every product and sum below rounds once, in the order written, so that a
// step on equal inputs gives equal bits whichever kernel, chunk or launch an element falls into, and the 8-bit codes and the
// kept low halves can be compared exactly with any other computation of the same formulas.
#include <math.h>
#include "pdes_common.h"
#include "../../include/pdes_hip.h"

namespace pdes {

constexpr int MT_BLOCK = PDES_MT_BLOCK;      // elements that share a scale; every tensor's state starts at a multiple of it
constexpr int MT_MAX = 96;                   // tensors of one launch
constexpr int MT_CLASSES = PDES_MT_CLASSES;  // different sets of hyper-parameters of one launch
constexpr int MT_ROWS = PDES_MT_ROWS;        // partial sums of the norm
constexpr long long MT_LONGEST = 1ll << 40;  // elements of a list: chunks are counted in 32 bits
constexpr int MT_TILE = 2048;                // elements that a workgroup of the step takes at a time: the unit of a chunk

typedef float f32x4 __attribute__((ext_vector_type(4)));
// parameters and gradients are views anywhere in their buffers: their vector accesses need the element's alignment only
// (one 16-byte access on gfx950, whatever the alignment)
typedef float f32x4_e __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_e __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));

struct MtRef {            // one tensor of a launch (32 bytes)
  void* p;
  void* g;
  uint32_t n_lo;
  uint16_t n_hi, cls;
  uint32_t block0, ordinal;
};
struct MtHyper {          // the constants of a step: computed in double, rounded once
  float decay, step, rc2, eps, b1, ob1, b2, ob2;
  uint32_t key;
};
struct StepArgs {
  MtRef t[MT_MAX];
  uint32_t chunk0[MT_MAX];      // first chunk of each tensor; unused entries hold 0xffffffff
  MtHyper h[MT_CLASSES];
  const MtHyper* hdev;          // captured steps: the same table in device memory
  const double* partials;       // not NULL: clip by the norm that these rows add up to
  float* norm_out;
  void* m;
  void* v;
  float* ms;
  float* rs;
  int16_t* low;
  uint32_t chunks, tiles;       // chunks of this launch; tiles of a chunk
  float limit, sign;
};
static_assert(sizeof(StepArgs) <= 4096, "kernel arguments");

constexpr int NORM_MAX = 160;
struct NormArgs {
  void* g[NORM_MAX];
  long long n[NORM_MAX];
  uint32_t chunk0[NORM_MAX];
  const double* in;             // rows of an earlier launch of the same norm, added to this launch's
  double* out;
  float* norm_out;
  uint32_t chunks;
  float limit;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// index of the tensor that chunk `c` belongs to: every lane compares a few of the table's first chunks, so the look-up
// costs two or three ballots and no chain of dependent loads
template <int N>
struct Finder {
  uint32_t mine[(N + 63) / 64];
  __device__ __forceinline__ explicit Finder(const uint32_t* first) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < (N + 63) / 64; ++k) mine[k] = 64 * k + lane < N ? first[64 * k + lane] : 0xffffffffu;
  }
  __device__ __forceinline__ int operator()(uint32_t c) const {
    int at = -1;
#pragma unroll
    for (int k = 0; k < (N + 63) / 64; ++k) at += __popcll(__ballot(mine[k] <= c));
    return at;
  }
};

// ---- element types -----------------------------------------------------------------------------------------------------
struct F32 {
  typedef float E;
  static __device__ __forceinline__ float up(E x) { return x; }
  static __device__ __forceinline__ E down(float x) { return x; }
};
struct BF16 {
  typedef uint16_t E;
  static __device__ __forceinline__ float up(E x) { return __uint_as_float((uint32_t)x << 16); }
  static __device__ __forceinline__ E down(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }      // to nearest, ties to even
};
struct F16 {
  typedef uint16_t E;
  static __device__ __forceinline__ float up(E x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ E down(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};

// N consecutive elements of which `cnt` exist (the others read as zero and are not written)
template <class T, int N>
__device__ __forceinline__ void load(const typename T::E* p, long long cnt, typename T::E (&x)[N]) {
  if (cnt >= N) {
    if constexpr (sizeof(typename T::E) == 4) {
#pragma unroll
      for (int k = 0; k < N / 4; ++k) {
        const f32x4_e w = reinterpret_cast<const f32x4_e*>(p)[k];
        x[4 * k] = w[0]; x[4 * k + 1] = w[1]; x[4 * k + 2] = w[2]; x[4 * k + 3] = w[3];
      }
    } else if constexpr (N == 4) {
      const u32x2_e w = *reinterpret_cast<const u32x2_e*>(p);
#pragma unroll
      for (int k = 0; k < 2; ++k) { x[2 * k] = (uint16_t)w[k]; x[2 * k + 1] = (uint16_t)(w[k] >> 16); }
    } else {
#pragma unroll
      for (int j = 0; j < N / 8; ++j) {
        const u32x4_e w = reinterpret_cast<const u32x4_e*>(p)[j];
#pragma unroll
        for (int k = 0; k < 4; ++k) { x[8 * j + 2 * k] = (uint16_t)w[k]; x[8 * j + 2 * k + 1] = (uint16_t)(w[k] >> 16); }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = k < cnt ? p[k] : (typename T::E)0;
  }
}
template <class T, int N>
__device__ __forceinline__ void store(typename T::E* p, long long cnt, const typename T::E (&x)[N]) {
  if (cnt >= N) {
    if constexpr (sizeof(typename T::E) == 4) {
#pragma unroll
      for (int k = 0; k < N / 4; ++k) {
        const f32x4_e w = {x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
        reinterpret_cast<f32x4_e*>(p)[k] = w;
      }
    } else if constexpr (N == 4) {
      const u32x2_e w = {x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16};
      *reinterpret_cast<u32x2_e*>(p) = w;
    } else {
#pragma unroll
      for (int j = 0; j < N / 8; ++j) {
        u32x4_e w;
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = x[8 * j + 2 * k] | (uint32_t)x[8 * j + 2 * k + 1] << 16;
        reinterpret_cast<u32x4_e*>(p)[j] = w;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < cnt) p[k] = x[k];
  }
}

// ---- the norm ----------------------------------------------------------------------------------------------------------
// kind 2: sum of squares; kind 0: largest magnitude, NaN if any element is.  Sums are fp64 throughout (the squares of fp32
// numbers neither overflow nor vanish there), every row adds its elements in a fixed order and the rows are added in a fixed
// order: the same gradients give the same norm bit for bit.
template <int KIND>
__device__ __forceinline__ double join(double a, double b) {
  if (KIND == 2) return a + b;
  return a != a ? a : (b > a || b != b) ? b : a;
}
template <int KIND, int WAVES>
__device__ __forceinline__ double block_join(double x, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = join<KIND>(x, __shfl_xor(x, o, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) x = join<KIND>(x, lds[w]);
  return x;
}
// the norm from its rows (every thread of a workgroup of 256 calls it), as fp32
template <int KIND>
__device__ __forceinline__ float whole_norm(const double* rows, double* lds) {
  static_assert(MT_ROWS == 256, "one row a thread");
  const double s = block_join<KIND, 4>(rows[threadIdx.x], lds);
  return (float)(KIND == 2 ? sqrt(s) : s);
}
// what the gradients are multiplied by: limit / (norm + 1e-6), rounded the way torch.nn.utils.clip_grad_norm_ rounds it
// (a reciprocal, then a product); NaN stays NaN
__device__ __forceinline__ float clip_factor(float norm, float limit) {
  const float c = 1.f / (norm + 1e-6f) * limit;
  return c > 1.f ? 1.f : c;
}

constexpr int NORM_THREADS = 512;
template <class T, int KIND>
__global__ __launch_bounds__(NORM_THREADS) void grad_norm_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(typename T::E);
  constexpr int TILE = NORM_THREADS * V;       // one 16-byte access of every thread: a chunk is four of them
  __shared__ double lds[NORM_THREADS / 64];
  const Finder<NORM_MAX> find(a.chunk0);
  double acc = 0.0;
  for (uint32_t c = blockIdx.x; c < a.chunks; c += MT_ROWS) {
    const int at = __builtin_amdgcn_readfirstlane(find(c));
    const typename T::E* g = static_cast<const typename T::E*>(a.g[at]);
    const long long n = a.n[at], base = (long long)(c - a.chunk0[at]) * (4 * TILE) + (int)threadIdx.x * V;
    typename T::E x[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load<T, V>(g + base + u * TILE, n - base - u * TILE, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const double d = (double)T::up(x[u][k]);
        acc = KIND == 2 ? fma(d, d, acc) : join<0>(acc, fabs(d));
      }
  }
  const double s = block_join<KIND, NORM_THREADS / 64>(acc, lds);
  if (threadIdx.x == 0) a.out[blockIdx.x] = a.in ? join<KIND>(a.in[blockIdx.x], s) : s;
}

// gradients times the clipping factor; where that is 1 nothing is read or written
template <class T, int KIND>
__global__ __launch_bounds__(256) void clip_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(typename T::E);
  constexpr int TILE = 256 * V;
  __shared__ double lds[4];
  const float norm = whole_norm<KIND>(a.in, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm_out) *a.norm_out = norm;
  if (a.limit == INFINITY) return;             // the norm alone was asked for
  const float f = clip_factor(norm, a.limit);
  if (f == 1.f) return;
  const Finder<NORM_MAX> find(a.chunk0);
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int at = __builtin_amdgcn_readfirstlane(find(c));
    typename T::E* g = static_cast<typename T::E*>(a.g[at]);
    const long long n = a.n[at], base = (long long)(c - a.chunk0[at]) * (4 * TILE) + (int)threadIdx.x * V;
    typename T::E x[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load<T, V>(g + base + u * TILE, n - base - u * TILE, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int k = 0; k < V; ++k) x[u][k] = T::down(T::up(x[u][k]) * f);
      store<T, V>(g + base + u * TILE, n - base - u * TILE, x[u]);
    }
  }
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
// w of an element: a parameter, or a bf16 parameter and the 16 bits below it (see narrow())
template <class T, bool LOW>
__device__ __forceinline__ float widen(typename T::E p, int16_t low) {
  if constexpr (!LOW) {
    return T::up(p);
  } else {
    int bits = (int)((uint32_t)p << 16);
    const uint32_t mag = p & 0x7fffu;
    // a parameter that the program has changed by itself keeps its value: nothing is added to an infinity or NaN, and
    // nothing taken from a zero
    const bool odd = mag >= 0x7f80u || (mag == 0 && low < 0);
    return __int_as_float(bits + (odd ? 0 : (int)low));
  }
}
// The upper half is w rounded to bf16 with ties AWAY from zero: with that rule the distance to w, counted in w's last place,
// is -0x8000 .. 0x7fff and fits the lower half exactly (ties to even would also need +0x8000).
template <class T, bool LOW>
__device__ __forceinline__ typename T::E narrow(float w, int16_t& low) {
  if constexpr (!LOW) {
    return T::down(w);
  } else {
    const int bits = __float_as_int(w);
    const int high = (int)((uint32_t)bits + 0x8000u) >> 16;
    low = (int16_t)(bits - (int)((uint32_t)high << 16));
    if (w != w) low = 0;
    return w != w ? (uint16_t)0x7fc0 : (uint16_t)high;
  }
}

__device__ __forceinline__ float new_weight(float w, float m, float r, const MtHyper& h) {
  const float u = m / (r * h.rc2 + h.eps);
  return w * h.decay - u * h.step;
}

// factor of the gradients: -1 to maximise, times the clipping factor
template <bool CLIP>
__device__ __forceinline__ float grad_factor(const StepArgs& a, double* lds) {
  if constexpr (!CLIP) return a.sign;
  const float norm = whole_norm<2>(a.partials, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm_out) *a.norm_out = norm;
  return a.sign * clip_factor(norm, a.limit);
}

template <class T, bool LOW, bool CLIP>
__global__ __launch_bounds__(256) void adamw32_kernel(const StepArgs a) {
  typedef typename T::E E;
  __shared__ double lds[4];
  const float gf = grad_factor<CLIP>(a, lds);
  const Finder<MT_MAX> find(a.chunk0);
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int at = __builtin_amdgcn_readfirstlane(find(c));
    const MtRef t = a.t[at];
    const MtHyper h = a.hdev ? a.hdev[t.cls] : a.h[t.cls];
    const long long n = (long long)((uint64_t)t.n_hi << 32 | t.n_lo), s0 = (long long)t.block0 * MT_BLOCK;
    const long long base = (long long)(c - a.chunk0[at]) * a.tiles * MT_TILE;
    E* const p = static_cast<E*>(t.p) + base;
    const E* const g = static_cast<const E*>(t.g) + base;
    float* const m = static_cast<float*>(a.m) + s0 + base;
    float* const v = static_cast<float*>(a.v) + s0 + base;
    int16_t* const low = LOW ? a.low + s0 + base : nullptr;
    const long long left = n - base;
    const int end = (int)(left < (long long)a.tiles * MT_TILE ? left : (long long)a.tiles * MT_TILE);
    for (int i = threadIdx.x * 4; i < end; i += 1024) {
      E pe[4], ge[4];
      int16_t lw[4] = {};
      load<T, 4>(p + i, end - i, pe);
      load<T, 4>(g + i, end - i, ge);
      f32x4 mv = *reinterpret_cast<const f32x4*>(m + i), vv = *reinterpret_cast<const f32x4*>(v + i);   // (states are padded to a block)
      if constexpr (LOW) {
        const uint2 w = *reinterpret_cast<const uint2*>(low + i);
        lw[0] = (int16_t)w.x; lw[1] = (int16_t)(w.x >> 16); lw[2] = (int16_t)w.y; lw[3] = (int16_t)(w.y >> 16);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gk = T::up(ge[k]) * gf;
        mv[k] = mv[k] * h.b1 + gk * h.ob1;
        vv[k] = vv[k] * h.b2 + gk * gk * h.ob2;
        const float w = new_weight(widen<T, LOW>(pe[k], lw[k]), mv[k], sqrtf(vv[k]), h);
        pe[k] = narrow<T, LOW>(w, lw[k]);
      }
      store<T, 4>(p + i, end - i, pe);
      *reinterpret_cast<f32x4*>(m + i) = mv;
      *reinterpret_cast<f32x4*>(v + i) = vv;
      if constexpr (LOW) {
        const uint2 w = make_uint2((uint16_t)lw[0] | (uint32_t)(uint16_t)lw[1] << 16, (uint16_t)lw[2] | (uint32_t)(uint16_t)lw[3] << 16);
        *reinterpret_cast<uint2*>(low + i) = w;
      }
    }
  }
}

// 8-bit states.  Blocks of 256 elements of one tensor share an fp32 scale = (largest value) / 448, and m and r = sqrt(v) are
// held as e4m3 numbers of value / scale.  r and not v: the root halves the range that the eight bits have to cover, and it is
// r that the step divides by.  Rounding is stochastic: (1 - beta2) moves r by 5e-4 of itself in a step, far under half of
// e4m3's spacing (2^-4 of the value), so rounding to nearest would hold r where it is for good; rounding down after
// adding a number from [0, 1) spacings is right on average.  r > 0 is never held as zero (smallest code instead): a lost
// second moment would turn the next step of its element into m / eps.  Values that are not finite are held as NaN and leave
// the scale of their block alone, so one of them spoils one element, as it does with 32-bit states.
constexpr uint32_t GOLD = 0x9E3779B9u;       // fractions of the golden ratio, sqrt 2 and sqrt 3 (odd)
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  x ^= x >> 16;
  return x;
}
// the largest magnitude among the 32 lanes of a half wave, as fp32 bits
__device__ __forceinline__ uint32_t half_max(uint32_t x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint32_t y = (uint32_t)__shfl_xor((int)x, o, 64);
    x = x > y ? x : y;
  }
  return x;
}
// scale of a block and what its values are multiplied by, from its largest value
__device__ __forceinline__ void scales(uint32_t top_bits, float& scale, float& inverse) {
  const float top = __uint_as_float(top_bits);
  const bool live = top >= 0x1p-100f;          // under that the scale's own arithmetic would be subnormal: held as zeros
  scale = live ? top * (1.f / 448.f) : 0.f;
  inverse = live ? 448.f / top : 0.f;
}
// e4m3 code of |x| * inverse, rounded down after `noise` / 2^20 of a spacing was added.  The product with 2^-120 puts e4m3's
// exponents (bias 7) where fp32's lie (bias 127), its subnormal range included: the code is the upper bits.
__device__ __forceinline__ uint32_t to_code(uint32_t mag_bits, float inverse, uint32_t noise) {
  const float y = __uint_as_float(mag_bits) * inverse * 0x1p-120f;
  const uint32_t code = (__float_as_uint(y) + noise) >> 20;
  return code < 0x7Eu ? code : 0x7Eu;
}
__device__ __forceinline__ void unpack8(uint32_t w, float scale, float* x) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a[0] * scale; x[1] = a[1] * scale; x[2] = b[0] * scale; x[3] = b[1] * scale;
}

template <class T, bool LOW, bool CLIP>
__global__ __launch_bounds__(256) void adamw8_kernel(const StepArgs a) {
  typedef typename T::E E;
  __shared__ double lds[4];
  const float gf = grad_factor<CLIP>(a, lds);
  const Finder<MT_MAX> find(a.chunk0);
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 5;       // a half wave takes a block, a lane eight elements of it
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int at = __builtin_amdgcn_readfirstlane(find(c));
    const MtRef t = a.t[at];
    const MtHyper h = a.hdev ? a.hdev[t.cls] : a.h[t.cls];
    const long long n = (long long)((uint64_t)t.n_hi << 32 | t.n_lo);
    const uint32_t blocks = (uint32_t)((n + MT_BLOCK - 1) / MT_BLOCK), first = (c - a.chunk0[at]) * a.tiles * (MT_TILE / MT_BLOCK);
    const uint32_t many = a.tiles * (MT_TILE / MT_BLOCK), stop = blocks - first < many ? blocks : first + many;
    const uint32_t tensor_key = mix(h.key + GOLD * (t.ordinal + 1));
    for (uint32_t b = first + half; b < stop; b += 8) {
      const long long i = (long long)b * MT_BLOCK + lane * 8, cnt = n - i;
      const long long sb = (long long)t.block0 + b, s = sb * MT_BLOCK + lane * 8;
      E* const p = static_cast<E*>(t.p) + i;
      E pe[8], ge[8];
      int16_t lw[8] = {};
      load<T, 8>(p, cnt, pe);
      load<T, 8>(static_cast<const E*>(t.g) + i, cnt, ge);
      const uint2 mq = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + s);
      const uint2 rq = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + s);
      const float ms = a.ms[sb], rs = a.rs[sb];
      if constexpr (LOW) {
        const uint4 w = *reinterpret_cast<const uint4*>(a.low + s);
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) { lw[2 * k] = (int16_t)q[k]; lw[2 * k + 1] = (int16_t)(q[k] >> 16); }
      }
      float m[8], r[8];
      unpack8(mq.x, ms, m); unpack8(mq.y, ms, m + 4);
      unpack8(rq.x, rs, r); unpack8(rq.y, rs, r + 4);
      uint32_t mb[8], rb[8], mtop = 0, rtop = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float gk = T::up(ge[k]) * gf;
        m[k] = m[k] * h.b1 + gk * h.ob1;
        r[k] = sqrtf(r[k] * r[k] * h.b2 + gk * gk * h.ob2);
        pe[k] = narrow<T, LOW>(new_weight(widen<T, LOW>(pe[k], lw[k]), m[k], r[k], h), lw[k]);
        mb[k] = __float_as_uint(m[k]) & 0x7fffffffu;
        rb[k] = __float_as_uint(r[k]) & 0x7fffffffu;
        mtop = mb[k] > mtop ? mb[k] : mtop;
        rtop = rb[k] > rtop ? rb[k] : rtop;
      }
      store<T, 8>(p, cnt, pe);
      if constexpr (LOW) {
        uint32_t q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = (uint16_t)lw[2 * k] | (uint32_t)(uint16_t)lw[2 * k + 1] << 16;
        *reinterpret_cast<uint4*>(a.low + s) = make_uint4(q[0], q[1], q[2], q[3]);
      }
      mtop = half_max(mtop);
      rtop = half_max(rtop);
      const bool bad = mtop >= 0x7f800000u || rtop >= 0x7f800000u;         // the same in all lanes of the half wave
      if (bad) {
        mtop = rtop = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (mb[k] < 0x7f800000u && mb[k] > mtop) mtop = mb[k];
          if (rb[k] < 0x7f800000u && rb[k] > rtop) rtop = rb[k];
        }
        mtop = half_max(mtop);
        rtop = half_max(rtop);
      }
      float nms, mi, nrs, ri;
      scales(mtop, nms, mi);
      scales(rtop, nrs, ri);
      const uint32_t key = mix(tensor_key + GOLD * b);
      uint32_t mc[8], rc[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t z = mix(key + GOLD * (uint32_t)(lane * 8 + k));
        mc[k] = to_code(mb[k], mi, z >> 12);
        rc[k] = to_code(rb[k], ri, z & 0xfffffu);
        rc[k] = rc[k] ? rc[k] : rb[k] ? 1u : 0u;
        if (bad) {
          if (mb[k] >= 0x7f800000u) mc[k] = 0x7fu;
          if (rb[k] >= 0x7f800000u) rc[k] = 0x7fu;
        }
        mc[k] |= (__float_as_uint(m[k]) >> 24) & 0x80u;
      }
      const uint2 mo = make_uint2(mc[0] | mc[1] << 8 | mc[2] << 16 | mc[3] << 24, mc[4] | mc[5] << 8 | mc[6] << 16 | mc[7] << 24);
      const uint2 ro = make_uint2(rc[0] | rc[1] << 8 | rc[2] << 16 | rc[3] << 24, rc[4] | rc[5] << 8 | rc[6] << 16 | rc[7] << 24);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.m) + s) = mo;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v) + s) = ro;
      if (lane == 0) { a.ms[sb] = nms; a.rs[sb] = nrs; }
    }
  }
}

// ---- captured steps: the step counts live on the device ---------------------------------------------------------------
struct ClassArgs {
  double lr[MT_CLASSES], b1[MT_CLASSES], b2[MT_CLASSES], eps[MT_CLASSES], wd[MT_CLASSES];
  const float* lr_dev[MT_CLASSES];
  float* step_dev[MT_CLASSES];
  MtHyper* out;
  uint32_t seed;
  int n;
};
__host__ __device__ __forceinline__ MtHyper constants(double lr, double b1, double b2, double eps, double wd, long long t, uint32_t seed) {
  MtHyper h;
  h.decay = (float)(1.0 - lr * wd);
  h.step = (float)(lr / (1.0 - pow(b1, (double)t)));
  h.rc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  h.eps = (float)eps;
  h.b1 = (float)b1; h.ob1 = (float)(1.0 - b1);
  h.b2 = (float)b2; h.ob2 = (float)(1.0 - b2);
  h.key = mix(seed + GOLD * (uint32_t)t);
  return h;
}
__global__ __launch_bounds__(64) void adamw_count_kernel(const ClassArgs a) {
  const int k = threadIdx.x;
  if (k >= a.n) return;
  const float t = *a.step_dev[k] + 1.f;
  *a.step_dev[k] = t;
  a.out[k] = constants(a.lr_dev[k] ? (double)*a.lr_dev[k] : a.lr[k], a.b1[k], a.b2[k], a.eps[k], a.wd[k], (long long)t, a.seed);
}

static int item_size(int dtype) { return dtype == PDES_MT_F32 ? 4 : 2; }

// one launch over grads[at .. at + count): fills the table, returns the number of tensors that went into it or an error
static int fill(NormArgs& a, const unsigned long long* grads, const long long* sizes, int count, int dtype, long long chunk, int& taken) {
  a.chunks = 0;
  taken = 0;
  int k = 0;
  long long total = 0;
  for (; taken < count && k < NORM_MAX; ++taken) {
    const long long n = sizes[taken];
    if (n < 0 || n >= MT_LONGEST - total) return PDES_EINVAL;
    if (n == 0) continue;
    total += n;
    if (!grads[taken]) return PDES_EINVAL;
    if (grads[taken] % item_size(dtype)) return PDES_EALIGN;
    a.g[k] = reinterpret_cast<void*>(grads[taken]);
    a.n[k] = n;
    a.chunk0[k++] = a.chunks;
    a.chunks += (uint32_t)((n + chunk - 1) / chunk);
  }
  for (; k < NORM_MAX; ++k) a.chunk0[k] = 0xffffffffu;
  return PDES_OK;
}

template <class T>
static void launch_norm(int kind, const NormArgs& a, hipStream_t st) {
  if (kind == 2)
    hipLaunchKernelGGL((grad_norm_kernel<T, 2>), dim3(MT_ROWS), dim3(NORM_THREADS), 0, st, a);
  else
    hipLaunchKernelGGL((grad_norm_kernel<T, 0>), dim3(MT_ROWS), dim3(NORM_THREADS), 0, st, a);
}
template <class T>
static void launch_clip(int kind, const NormArgs& a, hipStream_t st) {
  const unsigned grid = a.limit == INFINITY || a.chunks == 0 ? 1 : a.chunks < 2048 ? a.chunks : 2048;
  if (kind == 2)
    hipLaunchKernelGGL((clip_kernel<T, 2>), dim3(grid), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((clip_kernel<T, 0>), dim3(grid), dim3(256), 0, st, a);
}

template <class T, bool LOW>
static void launch_step(int bits, const StepArgs& a, unsigned grid, hipStream_t st) {
  if (bits == 32) {
    if (a.partials)
      hipLaunchKernelGGL((adamw32_kernel<T, LOW, true>), dim3(grid), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((adamw32_kernel<T, LOW, false>), dim3(grid), dim3(256), 0, st, a);
  } else {
    if (a.partials)
      hipLaunchKernelGGL((adamw8_kernel<T, LOW, true>), dim3(grid), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((adamw8_kernel<T, LOW, false>), dim3(grid), dim3(256), 0, st, a);
  }
}

}  // namespace pdes

using namespace pdes;

extern "C" int pdes_grad_norm(const unsigned long long* grads, const long long* sizes, int count, int dtype, int kind,
                              double* rows, int add, void* stream) {
  if (count < 0 || (count && (!grads || !sizes)) || !rows || dtype < 0 || dtype > 2 || (kind != 0 && kind != 2)) return PDES_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  NormArgs a;
  a.out = rows; a.norm_out = nullptr; a.limit = 0.f;
  int done = 0;
  do {                            // (an empty list still writes its rows)
    int taken;
    const int rc = fill(a, grads + done, sizes + done, count - done, dtype, 4ll * NORM_THREADS * (16 / item_size(dtype)), taken);
    if (rc) return rc;
    a.in = add || done ? rows : nullptr;
    done += taken;
    if (dtype == PDES_MT_F32) launch_norm<F32>(kind, a, st);
    else if (dtype == PDES_MT_BF16) launch_norm<BF16>(kind, a, st);
    else launch_norm<F16>(kind, a, st);
    PDES_LAUNCH_CHECK();
  } while (done < count);
  return PDES_OK;
}

extern "C" int pdes_clip_grads(const unsigned long long* grads, const long long* sizes, int count, int dtype, int kind,
                               const double* rows, float limit, float* norm_out, void* stream) {
  if (count < 0 || (count && (!grads || !sizes)) || !rows || dtype < 0 || dtype > 2 || (kind != 0 && kind != 2) || !(limit >= 0.f))
    return PDES_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  NormArgs a;
  a.in = rows; a.out = nullptr; a.limit = limit; a.norm_out = norm_out;
  int done = 0;
  do {
    int taken;
    const int rc = fill(a, grads + done, sizes + done, count - done, dtype, 4ll * 256 * (16 / item_size(dtype)), taken);
    if (rc) return rc;
    if (limit == INFINITY) taken = count - done;      // one launch writes the norm
    done += taken;
    if (dtype == PDES_MT_F32) launch_clip<F32>(kind, a, st);
    else if (dtype == PDES_MT_BF16) launch_clip<BF16>(kind, a, st);
    else launch_clip<F16>(kind, a, st);
    PDES_LAUNCH_CHECK();
  } while (done < count);
  return PDES_OK;
}

extern "C" int pdes_adamw_step(const unsigned long long* params, const unsigned long long* grads, const pdes_mt_tensor* tensors,
                               int count, const pdes_adamw_class* classes, int nclasses, const pdes_adamw_state* state,
                               void* stream) {
  if (count < 0 || !state || nclasses <= 0 || nclasses > MT_CLASSES || !classes || (count && (!params || !grads || !tensors))) return PDES_EINVAL;
  const pdes_adamw_state& s = *state;
  if (s.dtype < 0 || s.dtype > 2 || (s.bits != 32 && s.bits != 8) || (s.low && s.dtype != PDES_MT_BF16)) return PDES_EINVAL;
  if (s.blocks < 0 || s.blocks > 0xffffffffll || (s.norm_rows && !(s.limit >= 0.f))) return PDES_EINVAL;
  if (s.blocks && (!s.exp_avg || !s.exp_avg_sq || (s.bits == 8 && (!s.exp_avg_scale || !s.rms_scale)))) return PDES_EINVAL;
  if (!aligned16(s.exp_avg) || !aligned16(s.exp_avg_sq) || !aligned16(s.low)) return PDES_EALIGN;
  const bool captured = classes[0].step_dev != nullptr;
  if (captured && !s.hyper) return PDES_EINVAL;
  for (int k = 0; k < nclasses; ++k) {
    const pdes_adamw_class& c = classes[k];
    if (!(c.beta1 >= 0.0 && c.beta1 < 1.0 && c.beta2 >= 0.0 && c.beta2 < 1.0 && c.eps >= 0.0)) return PDES_EINVAL;
    if ((c.step_dev != nullptr) != captured || (!captured && (c.step < 1 || c.lr_dev))) return PDES_EINVAL;
  }
  const int size = item_size(s.dtype);
  long long total = 0;
  for (int k = 0; k < count; ++k) {
    const pdes_mt_tensor& t = tensors[k];
    if (t.n < 0 || t.n >= MT_LONGEST - total || t.block0 < 0 || t.cls < 0 || t.cls >= nclasses) return PDES_EINVAL;
    if (t.block0 + (t.n + MT_BLOCK - 1) / MT_BLOCK > s.blocks) return PDES_EINVAL;
    if (t.n && (!params[k] || !grads[k])) return PDES_EINVAL;
    if (params[k] % size || grads[k] % size) return PDES_EALIGN;
    total += t.n;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  StepArgs a;
  if (captured) {
    ClassArgs ca;
    ca.n = nclasses; ca.seed = s.seed; ca.out = static_cast<MtHyper*>(s.hyper);
    for (int k = 0; k < nclasses; ++k) {
      ca.lr[k] = classes[k].lr; ca.b1[k] = classes[k].beta1; ca.b2[k] = classes[k].beta2;
      ca.eps[k] = classes[k].eps; ca.wd[k] = classes[k].weight_decay;
      ca.lr_dev[k] = classes[k].lr_dev; ca.step_dev[k] = classes[k].step_dev;
    }
    hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(64), 0, st, ca);
    PDES_LAUNCH_CHECK();
  } else {
    for (int k = 0; k < nclasses; ++k)
      a.h[k] = constants(classes[k].lr, classes[k].beta1, classes[k].beta2, classes[k].eps, classes[k].weight_decay, classes[k].step, s.seed);
  }
  a.hdev = captured ? static_cast<const MtHyper*>(s.hyper) : nullptr;
  a.partials = s.norm_rows; a.norm_out = s.norm_out;
  a.m = s.exp_avg; a.v = s.exp_avg_sq; a.ms = s.exp_avg_scale; a.rs = s.rms_scale; a.low = s.low;
  a.limit = s.limit; a.sign = s.maximize ? -1.f : 1.f;
  // small lists are cut finely so that every CU has work; long ones into chunks that make the look-up disappear
  a.tiles = total < (8ll << 20) ? 1 : 4;
  const long long chunk = (long long)a.tiles * MT_TILE;
  for (int done = 0; done < count;) {
    int k = 0;
    a.chunks = 0;
    for (; done < count && k < MT_MAX; ++done) {
      const pdes_mt_tensor& t = tensors[done];
      if (t.n == 0) continue;
      a.t[k] = {reinterpret_cast<void*>(params[done]), reinterpret_cast<void*>(grads[done]), (uint32_t)t.n, (uint16_t)(t.n >> 32),
                (uint16_t)t.cls, (uint32_t)t.block0, (uint32_t)t.ordinal};
      a.chunk0[k++] = a.chunks;
      a.chunks += (uint32_t)((t.n + chunk - 1) / chunk);
    }
    for (; k < MT_MAX; ++k) a.chunk0[k] = 0xffffffffu;
    if (a.chunks == 0) continue;
    const unsigned grid = a.chunks < 2048 ? a.chunks : 2048;
    if (s.dtype == PDES_MT_F32) launch_step<F32, false>(s.bits, a, grid, st);
    else if (s.dtype == PDES_MT_F16) launch_step<F16, false>(s.bits, a, grid, st);
    else if (s.low) launch_step<BF16, true>(s.bits, a, grid, st);
    else launch_step<BF16, false>(s.bits, a, grid, st);
    PDES_LAUNCH_CHECK();
  }
  return PDES_OK;
}
