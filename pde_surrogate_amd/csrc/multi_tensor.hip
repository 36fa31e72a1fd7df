// Operators over many tensors in one launch: the AdamW step with 32-bit or 8-bit states, the common norm of a list of
// gradients, and their clipping (include/pdes_hip.h: pdes_adamw_step, pdes_grad_norm, pdes_clip_grads).  Where a comment compares
// two ways, both were built from this file and timed in turn on one MI355X; 332 M and 217 M
// are 332,410,880 and 216,545,280 elements, any other M is 2^20.
//
// The list is cut into chunks, each inside one tensor; a workgroup of a step takes one.  The list itself (addresses, lengths) travels BY VALUE in the
// kernel arguments, up to 96 tensors a launch: nothing to copy, no buffer that a later call could overwrite while an
// earlier launch still reads it, and a captured graph holds its own copy.
//
// This file is compiled with -ffp-contract=off: every product and sum below rounds once, in the order written, so that a
// step on equal inputs gives equal bits whichever kernel, chunk or launch an element falls into, and the moments, the 8-bit codes
// and the kept low halves can be compared exactly with any other computation of the same formulas.  One exception: with 8-bit states
// the new value of a 16-bit weight without a low half (new_weight_16).
#include <math.h>
#include "pdes_common.h"
#include "../../include/pdes_hip.h"

namespace pdes {

constexpr int MT_BLOCK = PDES_MT_BLOCK;      // elements that share a scale; every tensor's state starts at a multiple of it
constexpr int MT_MAX = 96;                   // tensors of one launch
constexpr int MT_CLASSES = PDES_MT_CLASSES;  // different sets of hyper-parameters of one launch
constexpr int MT_ROWS = PDES_MT_ROWS;        // partial sums of the norm
constexpr long long MT_LONGEST = 1ll << 40;  // elements of a list: chunks are counted in 32 bits
constexpr int MT_TILE = 2048;                // elements that a workgroup of the step takes at a time: eight a thread

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
  const double* rows;           // clipping by the norm that these rows make (NULL: `norm` holds it already)
  float* norm;                  // NULL: no clipping
  void* m;
  void* v;
  float* ms;
  float* rs;
  int16_t* low;
  uint32_t chunks, tiles;       // chunks of this launch, a workgroup each; tiles of a chunk
  float limit;
};
static_assert(sizeof(StepArgs) <= 4096, "kernel arguments");
static_assert(sizeof(MtHyper) * MT_CLASSES == PDES_MT_HYPER_BYTES, "pdes_adamw_state.hyper");

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

// Global accesses.  NT: streaming ones, for lists that are larger than the caches and will be gone from them before anybody asks
// again (STEP_STREAMS, NORM_STREAMS).
#define PDES_GLOBAL __attribute__((address_space(1)))
template <bool NT, class W>
__device__ __forceinline__ W get(const void* p, int k = 0) {
  const PDES_GLOBAL W* q = (const PDES_GLOBAL W*)p + k;
  if constexpr (NT) return __builtin_nontemporal_load(q);
  return *q;
}
template <bool NT, class W>
__device__ __forceinline__ void put(void* p, W w, int k = 0) {
  PDES_GLOBAL W* q = (PDES_GLOBAL W*)p + k;
  if constexpr (NT) __builtin_nontemporal_store(w, q);
  else *q = w;
}
// N consecutive elements.  ALL: they exist; otherwise `cnt` of them do (the others read as zero and are not written).  The
// whole-vector form is a plain global access without a branch, so that a thread's loads are all under way at once (norm of 332 M
// fp32 elements: 224 us with a branch at each load, 195 without; fp16 121 and 102)
template <class T, int N, bool ALL, bool NT>
__device__ __forceinline__ void load(const typename T::E* p, long long cnt, typename T::E (&x)[N]) {
  typedef typename T::E E;
  if constexpr (!ALL) {
    if (cnt >= N) return load<T, N, true, NT>(p, cnt, x);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = k < cnt ? get<false, E>(p, k) : (E)0;
  } else if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const f32x4_e w = get<NT, f32x4_e>(p, k);
      x[4 * k] = w[0]; x[4 * k + 1] = w[1]; x[4 * k + 2] = w[2]; x[4 * k + 3] = w[3];
    }
  } else if constexpr (N == 4) {
    const u32x2_e w = get<NT, u32x2_e>(p);
#pragma unroll
    for (int k = 0; k < 2; ++k) { x[2 * k] = (uint16_t)w[k]; x[2 * k + 1] = (uint16_t)(w[k] >> 16); }
  } else {
    static_assert(N == 8, "one 16-byte access");
    const u32x4_e w = get<NT, u32x4_e>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) { x[2 * k] = (uint16_t)w[k]; x[2 * k + 1] = (uint16_t)(w[k] >> 16); }
  }
}
template <class T, int N, bool ALL, bool NT>
__device__ __forceinline__ void store(typename T::E* p, long long cnt, const typename T::E (&x)[N]) {
  typedef typename T::E E;
  if constexpr (!ALL) {
    if (cnt >= N) return store<T, N, true, NT>(p, cnt, x);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < cnt) put<false, E>(p, x[k], k);
  } else if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int k = 0; k < N / 4; ++k) {
      const f32x4_e w = {x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
      put<NT>(p, w, k);
    }
  } else if constexpr (N == 4) {
    const u32x2_e w = {x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16};
    put<NT>(p, w);
  } else {
    static_assert(N == 8, "one 16-byte access");
    u32x4_e w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = x[2 * k] | (uint32_t)x[2 * k + 1] << 16;
    put<NT>(p, w);
  }
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
// (a reciprocal, then a product); NaN stays NaN.  Without a limit nothing is changed, whatever the norm
__device__ __forceinline__ float clip_factor(float norm, float limit) {
  if (limit == INFINITY) return 1.f;
  const float c = 1.f / (norm + 1e-6f) * limit;
  return c > 1.f ? 1.f : c;
}

template <class T, int KIND, int THREADS, int U, bool NT, bool ALL>
__device__ __forceinline__ void norm_chunk(const typename T::E* g, long long left, double (&acc)[4]) {
  constexpr int V = 16 / sizeof(typename T::E), TILE = THREADS * V;
  typename T::E x[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) load<T, V, ALL, NT>(g + u * TILE, left - u * TILE, x[u]);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const double d = (double)T::up(x[u][k]);
      acc[k & 3] = KIND == 2 ? fma(d, d, acc[k & 3]) : join<0>(acc[k & 3], fabs(d));
    }
}
// One workgroup a CU and row; a thread has U accesses of 16 bytes under way.  Bound by reading: 332 M elements of fp32 192 us =
// 6.9 TB/s, of bf16 99 us = 6.7 TB/s (a call 195 and 101 us; 216 and 114 through the caches).  The maximum norm has three fp64
// comparisons an element: 197 and 117 us.
template <class T, int KIND, int THREADS, int U, bool NT>
__global__ __launch_bounds__(THREADS) void grad_norm_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(typename T::E), CHUNK = THREADS * V * U;
  __shared__ double lds[THREADS / 64];
  const Finder<NORM_MAX> find(a.chunk0);
  double acc[4] = {0.0, 0.0, 0.0, 0.0};        // (four chains: one would wait for itself)
  for (uint32_t c = blockIdx.x; c < a.chunks; c += MT_ROWS) {
    const int at = __builtin_amdgcn_readfirstlane(find(c));
    const long long base = (long long)(c - a.chunk0[at]) * CHUNK, left = a.n[at] - base;
    const int mine = (int)threadIdx.x * V;
    const typename T::E* g = static_cast<const typename T::E*>(a.g[at]) + base + mine;
    if (left >= CHUNK) norm_chunk<T, KIND, THREADS, U, NT, true>(g, left - mine, acc);
    else norm_chunk<T, KIND, THREADS, U, NT, false>(g, left - mine, acc);
  }
  const double x = join<KIND>(join<KIND>(acc[0], acc[1]), join<KIND>(acc[2], acc[3]));
  const double s = block_join<KIND, THREADS / 64>(x, lds);
  if (threadIdx.x == 0) a.out[blockIdx.x] = a.in ? join<KIND>(a.in[blockIdx.x], s) : s;
}
// the norm of the rows, for steps of many workgroups
__global__ __launch_bounds__(MT_ROWS) void norm_kernel(const double* rows, float* norm) {
  __shared__ double lds[4];
  const float x = whole_norm<2>(rows, lds);
  if (threadIdx.x == 0) *norm = x;
}

// Gradients times the clipping factor; where that is 1 nothing is read or written.  332 M elements of fp32 483 us, of bf16 240 us, both
// 5.5 TB/s (half of it writes); 20 M fp32, found in the cache by the norm in front, 26 us.
template <class T, bool ALL>
__device__ __forceinline__ void clip_chunk(typename T::E* g, long long left, float f) {
  constexpr int V = 16 / sizeof(typename T::E), TILE = 256 * V;
  typename T::E x[4][V];
#pragma unroll
  for (int u = 0; u < 4; ++u) load<T, V, ALL, false>(g + u * TILE, left - u * TILE, x[u]);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
#pragma unroll
    for (int k = 0; k < V; ++k) x[u][k] = T::down(T::up(x[u][k]) * f);
    store<T, V, ALL, false>(g + u * TILE, left - u * TILE, x[u]);
  }
}
template <class T, int KIND>
__global__ __launch_bounds__(256) void clip_kernel(const NormArgs a) {
  constexpr int V = 16 / sizeof(typename T::E), CHUNK = 4 * 256 * V;
  __shared__ double lds[4];
  const float norm = whole_norm<KIND>(a.in, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.norm_out) *a.norm_out = norm;
  const float f = clip_factor(norm, a.limit);
  if (f == 1.f) return;
  const Finder<NORM_MAX> find(a.chunk0);
  for (uint32_t c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    const int at = __builtin_amdgcn_readfirstlane(find(c));
    const long long base = (long long)(c - a.chunk0[at]) * CHUNK, left = a.n[at] - base;
    const int mine = (int)threadIdx.x * V;
    typename T::E* g = static_cast<typename T::E*>(a.g[at]) + base + mine;
    if (left >= CHUNK) clip_chunk<T, true>(g, left - mine, f);
    else clip_chunk<T, false>(g, left - mine, f);
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
// The same in the 8-bit kernel for weights of 16 bits (see EXACT there): the quotient from the reciprocal instruction; the fix-up
// gives the quotients of zeros, infinities and NaN
__device__ __forceinline__ float new_weight_16(float w, float m, float r, const MtHyper& h) {
  const float den = fmaf(r, h.rc2, h.eps);
  const float u = __builtin_amdgcn_div_fixupf(m * __builtin_amdgcn_rcpf(den), den, m);
  return fmaf(-u, h.step, w * h.decay);
}

// what clipping multiplies the gradients by
__device__ __forceinline__ float grad_factor(const StepArgs& a, double* lds) {
  if (!a.norm) return 1.f;
  if (!a.rows) return clip_factor(*(const PDES_GLOBAL float*)a.norm, a.limit);
  const float norm = whole_norm<2>(a.rows, lds);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
  return clip_factor(norm, a.limit);
}
__device__ __forceinline__ MtHyper hyper_of(const StepArgs& a, int cls) {
  if (!a.hdev) return a.h[cls];
  MtHyper h;
  const PDES_GLOBAL MtHyper* d = (const PDES_GLOBAL MtHyper*)a.hdev + cls;
  h.decay = d->decay; h.step = d->step; h.rc2 = d->rc2; h.eps = d->eps;
  h.b1 = d->b1; h.ob1 = d->ob1; h.b2 = d->b2; h.ob2 = d->ob2; h.key = d->key;
  return h;
}

// a thread's share of a tile: twice four consecutive elements, 1024 elements apart.  All of its loads come first
constexpr int V32 = MT_TILE / 1024;
template <class T, bool LOW, bool NT, bool ALL>
__device__ __forceinline__ void step32(typename T::E* p, const typename T::E* g, float* m, float* v, int16_t* low, int cnt, float gf,
                                       const MtHyper& h) {
  typename T::E pe[V32][4], ge[V32][4];
  f32x4 mv[V32], vv[V32];
  u32x2 lw[V32];
#pragma unroll
  for (int u = 0; u < V32; ++u) {
    const int i = 1024 * u, left = cnt - i;
    if (!ALL && left <= 0) continue;
    load<T, 4, ALL, NT>(p + i, left, pe[u]);
    load<T, 4, ALL, NT>(g + i, left, ge[u]);
    mv[u] = get<NT, f32x4>(m + i);                         // (states are padded to a block)
    vv[u] = get<NT, f32x4>(v + i);
    if constexpr (LOW) lw[u] = get<NT, u32x2>(low + i);
  }
#pragma unroll
  for (int u = 0; u < V32; ++u) {
    const int i = 1024 * u, left = cnt - i;
    if (!ALL && left <= 0) continue;
    int16_t lo[4] = {};
    if constexpr (LOW) { lo[0] = (int16_t)lw[u][0]; lo[1] = (int16_t)(lw[u][0] >> 16); lo[2] = (int16_t)lw[u][1]; lo[3] = (int16_t)(lw[u][1] >> 16); }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // (a factor that is NaN stays out of the padding)
      const float gk = !ALL && k >= left ? 0.f : T::up(ge[u][k]) * gf;
      mv[u][k] = mv[u][k] * h.b1 + gk * h.ob1;
      vv[u][k] = vv[u][k] * h.b2 + gk * gk * h.ob2;
      pe[u][k] = narrow<T, LOW>(new_weight(widen<T, LOW>(pe[u][k], lo[k]), mv[u][k], sqrtf(vv[u][k]), h), lo[k]);
    }
    store<T, 4, ALL, NT>(p + i, left, pe[u]);
    put<NT>(m + i, mv[u]);
    put<NT>(v + i, vv[u]);
    if constexpr (LOW) {
      const u32x2 w = {(uint16_t)lo[0] | (uint32_t)(uint16_t)lo[1] << 16, (uint16_t)lo[2] | (uint32_t)(uint16_t)lo[3] << 16};
      put<NT>(low + i, w);
    }
  }
}
template <class T, bool LOW, bool NT>
__global__ __launch_bounds__(256) void adamw32_kernel(const StepArgs a) {
  typedef typename T::E E;
  __shared__ double lds[4];
  const float gf = grad_factor(a, lds);
  const Finder<MT_MAX> find(a.chunk0);
  const int at = __builtin_amdgcn_readfirstlane(find(blockIdx.x));
  const MtRef t = a.t[at];
  const MtHyper h = hyper_of(a, t.cls);
  const long long n = (long long)((uint64_t)t.n_hi << 32 | t.n_lo), base = (long long)(blockIdx.x - a.chunk0[at]) * MT_TILE, left = n - base;
  const long long s = (long long)t.block0 * MT_BLOCK + base;
  const uint32_t mine = threadIdx.x * 4;
  E* const p = static_cast<E*>(t.p) + base + mine;
  const E* const g = static_cast<const E*>(t.g) + base + mine;
  float* const m = static_cast<float*>(a.m) + s + mine;
  float* const v = static_cast<float*>(a.v) + s + mine;
  int16_t* const low = LOW ? a.low + s + mine : nullptr;
  if (left >= MT_TILE) step32<T, LOW, NT, true>(p, g, m, v, low, MT_TILE, gf, h);
  else step32<T, LOW, NT, false>(p, g, m, v, low, (int)left - (int)mine, gf, h);
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
// The largest magnitudes of a half wave's block: a lane brings those of its m and r, as bits; lanes 0 .. 15 get the block's
// for m, lanes 16 .. 31 its for r.  One exchange of the rows sorts m into the first and r into the second, then both are
// reduced in their row at once (DPP); the scale and its inverse are found once in each row instead of twice in every lane.
__device__ __forceinline__ uint32_t row_tops(uint32_t m, uint32_t r) {
  const auto rows = __builtin_amdgcn_permlane16_swap(m, r, false, false);
  uint32_t x = rows[0] > rows[1] ? rows[0] : rows[1];
#define PDES_MAX_DPP(ctrl) { const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, ctrl, 0xf, 0xf, true); x = x > y ? x : y; }
  PDES_MAX_DPP(0xB1)       // lanes 1 0 3 2
  PDES_MAX_DPP(0x4E)       // lanes 2 3 0 1
  PDES_MAX_DPP(0x141)      // eight lanes mirrored
  PDES_MAX_DPP(0x140)      // sixteen lanes mirrored
#undef PDES_MAX_DPP
  return x;
}
// 448 / top, correctly rounded: the reciprocal, one step of Newton's for it and two corrections of the quotient.  (The division
// operator scales its operands besides; here they and all that is between are normal numbers: 2^-100 <= top <= 2^120.)
__device__ __forceinline__ float inverse_scale(float top) {
  float y = __builtin_amdgcn_rcpf(top);
  y = fmaf(fmaf(-top, y, 1.f), y, y);
  float q = 448.f * y;
  q = fmaf(fmaf(-q, top, 448.f), y, q);
  return fmaf(fmaf(-q, top, 448.f), y, q);
}
constexpr uint32_t TOP_LEAST = 0x0d800000u, TOP_MOST = 0x7b800000u;      // 2^-100 and 2^120 as bits
__device__ __forceinline__ void unpack8(uint32_t w, float scale, float* x) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = a[0] * scale; x[1] = a[1] * scale; x[2] = b[0] * scale; x[3] = b[1] * scale;
}
// sqrtf, correctly rounded, for x = 0 and 2^-102 <= x < infinity: from the reciprocal root and one correction by the residual.  (All
// 2^24 numbers of two neighbouring binades have been compared with sqrtf, at 2^0, 2^-60 and 2^-100; four times the number gives
// exactly twice the root.  Under 2^-102 the residual loses bits.)  NaN for infinity
__device__ __forceinline__ float root(float x) {
  const int bits = __float_as_int(x), least = 0x00800000;                      // (2^-126; x is not negative)
  const float y = __builtin_amdgcn_rsqf(__int_as_float(bits > least ? bits : least)), s = x * y;
  return fmaf(fmaf(-s, s, x), 0.5f * y, s);
}
constexpr uint32_t ROOT_LEAST = 0x0f800000u;                                   // 2^-96 as bits

// A half wave holds a block, a lane eight elements of it: consecutive ones of 16 bits, or twice four of 32 bits, 128 elements
// apart, so that each access of a wave covers whole lines (332 M fp32 parameters: 886 us; eight consecutive ones, two accesses to
// each half of a line: 1,130 us).
template <class T>
struct Share {
  static constexpr int PER = sizeof(typename T::E) == 4 ? 4 : 8, PARTS = 8 / PER, APART = 128;
  // the place of a lane's element k in its block
  static __device__ __forceinline__ uint32_t place(int lane, int k) { return lane * PER + k % PER + k / PER * APART; }
};
template <class T, bool ALL, bool NT>
__device__ __forceinline__ void load8(const typename T::E* p, long long cnt, typename T::E (&x)[8]) {
  constexpr int PER = Share<T>::PER;
#pragma unroll
  for (int j = 0; j < Share<T>::PARTS; ++j) {
    typename T::E part[PER];
    load<T, PER, ALL, NT>(p + j * Share<T>::APART, cnt - j * Share<T>::APART, part);
#pragma unroll
    for (int k = 0; k < PER; ++k) x[j * PER + k] = part[k];
  }
}
template <class T, bool ALL, bool NT>
__device__ __forceinline__ void store8(typename T::E* p, long long cnt, const typename T::E (&x)[8]) {
  constexpr int PER = Share<T>::PER;
#pragma unroll
  for (int j = 0; j < Share<T>::PARTS; ++j) {
    typename T::E part[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) part[k] = x[j * PER + k];
    store<T, PER, ALL, NT>(p + j * Share<T>::APART, cnt - j * Share<T>::APART, part);
  }
}
template <class T, bool NT>
__device__ __forceinline__ u32x2 get_codes(const uint8_t* q) {
  if constexpr (Share<T>::PARTS == 1) return get<NT, u32x2>(q);
  const u32x2 w = {get<NT, uint32_t>(q), get<NT, uint32_t>(q + Share<T>::APART)};
  return w;
}
template <class T, bool NT>
__device__ __forceinline__ void put_codes(uint8_t* q, u32x2 w) {
  if constexpr (Share<T>::PARTS == 1) {
    put<NT>(q, w);
  } else {
    put<NT, uint32_t>(q, w[0]);
    put<NT, uint32_t>(q + Share<T>::APART, w[1]);
  }
}

template <class T, bool LOW, bool CLIP, bool NT, bool ALL>
__device__ __forceinline__ void step8(typename T::E* p, const typename T::E* g, uint8_t* mq, uint8_t* rq, float* ms, float* rs, int16_t* low,
                                      long long cnt, float gf, const MtHyper& h, uint32_t key, int lane) {
  // Weights of 16 bits leave 10 bytes of traffic per element (332 M bf16: 562 us = 5.9 TB/s), about the time of this arithmetic.
  // There the weight itself is computed with fused sums and the reciprocal instruction, off by a few places of 2^-24 before it is
  // rounded by 2^-9 or 2^-12.  The moments are the same numbers for every type: which of two codes a value gets depends on their
  // last place, and so do later scales.
  constexpr bool EXACT = sizeof(typename T::E) == 4 || LOW;
  typename T::E pe[8], ge[8];
  int16_t lw[8] = {};
  load8<T, ALL, NT>(p, cnt, pe);
  load8<T, ALL, NT>(g, cnt, ge);
  const u32x2 mw = get_codes<T, NT>(mq), rw = get_codes<T, NT>(rq);
  const float m_scale = get<false, float>(ms), r_scale = get<false, float>(rs);
  if constexpr (LOW) {
    const u32x4 w = get<NT, u32x4>(low);
#pragma unroll
    for (int k = 0; k < 4; ++k) { lw[2 * k] = (int16_t)w[k]; lw[2 * k + 1] = (int16_t)(w[k] >> 16); }
  }
  float m[8], r[8], v[8];
  unpack8(mw[0], m_scale, m); unpack8(mw[1], m_scale, m + 4);
  unpack8(rw[0], r_scale, r); unpack8(rw[1], r_scale, r + 4);
  uint32_t mtop = 0, rtop = 0, least = ~0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    // (a factor that is NaN stays out of the padding)
    const bool there = ALL || k % Share<T>::PER + k / Share<T>::PER * Share<T>::APART < cnt;
    const float gk = !CLIP ? T::up(ge[k]) : there ? T::up(ge[k]) * gf : 0.f;
    m[k] = m[k] * h.b1 + gk * h.ob1;
    v[k] = r[k] * r[k] * h.b2 + gk * gk * h.ob2;
    r[k] = root(v[k]);
    const uint32_t mb = __float_as_uint(m[k]) & 0x7fffffffu, rb = __float_as_uint(r[k]), vb = __float_as_uint(v[k]) - 1u;
    mtop = mb > mtop ? mb : mtop;
    rtop = rb > rtop ? rb : rtop;              // (r is not negative; a NaN with the sign is the largest as well)
    least = vb < least ? vb : least;           // (of those that are not zero)
  }
  if (least < ROOT_LEAST - 1u || rtop >= 0x7f800000u) {      // numbers that root() is not for; for the others sqrtf is the same
    rtop = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      r[k] = sqrtf(v[k]);
      const uint32_t rb = __float_as_uint(r[k]);
      rtop = rb > rtop ? rb : rtop;
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float w = widen<T, LOW>(pe[k], lw[k]);
    pe[k] = narrow<T, LOW>(EXACT ? new_weight(w, m[k], r[k], h) : new_weight_16(w, m[k], r[k], h), lw[k]);
  }
  store8<T, ALL, NT>(p, cnt, pe);
  if constexpr (LOW) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint16_t)lw[2 * k] | (uint32_t)(uint16_t)lw[2 * k + 1] << 16;
    put<NT>(low, w);
  }
  uint32_t top = row_tops(mtop, rtop);
  const bool odd = __any(top > TOP_MOST);      // values that are not finite, or too large for inverse_scale
  float scale, inverse;
  if (!odd) {
    const bool live = top >= TOP_LEAST;        // under that the scale's own arithmetic would be subnormal: held as zeros
    scale = live ? __uint_as_float(top) * (1.f / 448.f) : 0.f;
    inverse = live ? inverse_scale(__uint_as_float(top)) : 0.f;
  } else {
    mtop = rtop = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t mb = __float_as_uint(m[k]) & 0x7fffffffu, rb = __float_as_uint(r[k]) & 0x7fffffffu;
      if (mb < 0x7f800000u && mb > mtop) mtop = mb;
      if (rb < 0x7f800000u && rb > rtop) rtop = rb;
    }
    top = row_tops(mtop, rtop);
    scale = top >= TOP_LEAST ? __uint_as_float(top) * (1.f / 448.f) : 0.f;
    inverse = top >= TOP_LEAST ? 448.f / __uint_as_float(top) : 0.f;
  }
  if ((lane & 15) == 0) put<false>(lane ? rs : ms, scale);
  const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(inverse), __float_as_uint(inverse), false, false);
  const float mi = __uint_as_float(both[0]), ri = __uint_as_float(both[1]);
  u32x2 mo = {0, 0}, ro = {0, 0};
  // the conversion drops 20 bits of the number (more under 2^-6) after the upper 20 bits of `z` have been added to them: rounding
  // down after z / 2^32 of a spacing was added, up to the bits behind 2^-29 of a number under 2^-6, which it cuts
#define PDES_HOLD(k, word, byte)                                                                                        \
  {                                                                                                                     \
    const uint32_t z = mix(key + GOLD * Share<T>::place(lane, k));                                                                 \
    mo[word] = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(__builtin_amdgcn_fmed3f(m[k] * mi, -448.f, 448.f), (int)z, (int)mo[word], byte); \
    ro[word] = (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(__builtin_amdgcn_fmed3f(r[k] * ri, r[k] > 0.f ? 0x1p-9f : 0.f, 448.f), (int)(z << 12), (int)ro[word], byte); \
  }
  PDES_HOLD(0, 0, 0) PDES_HOLD(1, 0, 1) PDES_HOLD(2, 0, 2) PDES_HOLD(3, 0, 3)
  PDES_HOLD(4, 1, 0) PDES_HOLD(5, 1, 1) PDES_HOLD(6, 1, 2) PDES_HOLD(7, 1, 3)
#undef PDES_HOLD
  if (odd) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t nan = 0x7fu << (8 * (k & 3)), sign = 0x80u << (8 * (k & 3));
      if ((__float_as_uint(m[k]) & 0x7fffffffu) >= 0x7f800000u)
        mo[k >> 2] = (mo[k >> 2] & ~sign) | nan | ((__float_as_uint(m[k]) >> 31) ? sign : 0u);
      if ((__float_as_uint(r[k]) & 0x7fffffffu) >= 0x7f800000u) ro[k >> 2] = (ro[k >> 2] & ~sign) | nan;
    }
  }
  put_codes<T, NT>(mq, mo);
  put_codes<T, NT>(rq, ro);
}

template <class T, bool LOW, bool CLIP, bool NT>
__global__ __launch_bounds__(256, sizeof(typename T::E) == 2 && !LOW ? 5 : 1) void adamw8_kernel(const StepArgs a) {
  typedef typename T::E E;
  __shared__ double lds[4];
  const float gf = CLIP ? grad_factor(a, lds) : 1.f;
  const Finder<MT_MAX> find(a.chunk0);
  const int lane = threadIdx.x & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = threadIdx.x >> 5;
  const uint32_t mine = half * MT_BLOCK + lane * Share<T>::PER;
  const int at = __builtin_amdgcn_readfirstlane(find(blockIdx.x));
  const MtRef t = a.t[at];
  const MtHyper h = hyper_of(a, t.cls);
  const long long n = (long long)((uint64_t)t.n_hi << 32 | t.n_lo);
  const uint32_t tensor_key = mix(h.key + GOLD * (t.ordinal + 1)), tile0 = (blockIdx.x - a.chunk0[at]) * a.tiles;
  for (uint32_t tile = tile0; tile < tile0 + a.tiles; ++tile) {
    const long long i = (long long)tile * MT_TILE, left = n - i;
    if (left <= 0) break;
    const uint32_t b = tile * (MT_TILE / MT_BLOCK) + 2 * wave;               // of the wave's lower half
    const uint32_t key0 = mix(tensor_key + GOLD * b), key1 = mix(tensor_key + GOLD * (b + 1)), key = half & 1 ? key1 : key0;
    const long long s = (long long)t.block0 * MT_BLOCK + i, sb = t.block0 + (long long)tile * (MT_TILE / MT_BLOCK) + half;
    E* const p = static_cast<E*>(t.p) + i + mine;
    const E* const g = static_cast<const E*>(t.g) + i + mine;
    uint8_t* const mq = static_cast<uint8_t*>(a.m) + s + mine;
    uint8_t* const rq = static_cast<uint8_t*>(a.v) + s + mine;
    int16_t* const low = LOW ? a.low + s + mine : nullptr;
    if (left >= MT_TILE) step8<T, LOW, CLIP, NT, true>(p, g, mq, rq, a.ms + sb, a.rs + sb, low, 8, gf, h, key, lane);
    else if (half * MT_BLOCK < (int)left)
      step8<T, LOW, CLIP, NT, false>(p, g, mq, rq, a.ms + sb, a.rs + sb, low, (int)left - (int)mine, gf, h, key, lane);
  }
}

// ---- captured steps: the step counts live on the device ---------------------------------------------------------------
struct ClassArgs {
  double lr[MT_CLASSES], b1[MT_CLASSES], b2[MT_CLASSES], eps[MT_CLASSES], wd[MT_CLASSES];
  const float* lr_dev[MT_CLASSES];
  float* step_dev[MT_CLASSES];
  MtHyper* out;
  uint32_t seed;
  int n, maximize, bits;
};
__host__ __device__ __forceinline__ MtHyper constants(double lr, double b1, double b2, double eps, double wd, bool maximize, int bits, long long t,
                                                       uint32_t seed) {
  MtHyper h;
  h.decay = (float)(1.0 - lr * wd);
  h.step = (float)(lr / (1.0 - pow(b1, (double)t)));
  h.rc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  h.eps = (float)(bits == 8 && eps < 0x1p-100 ? 0x1p-100 : eps);      // (r under 2^-100 is held as zero)
  h.b1 = (float)b1;
  h.ob1 = (float)(maximize ? b1 - 1.0 : 1.0 - b1);           // (of the gradient, only its sign in m differs)
  h.b2 = (float)b2; h.ob2 = (float)(1.0 - b2);
  h.key = mix(seed + GOLD * (uint32_t)t);
  return h;
}
__global__ __launch_bounds__(64) void adamw_count_kernel(const ClassArgs a) {
  const int k = threadIdx.x;
  if (k >= a.n) return;
  const float t = *a.step_dev[k] + 1.f;
  *a.step_dev[k] = t;
  a.out[k] = constants(a.lr_dev[k] ? (double)*a.lr_dev[k] : a.lr[k], a.b1[k], a.b2[k], a.eps[k], a.wd[k], a.maximize, a.bits, (long long)t, a.seed);
}

constexpr long long LONG_LIST = 8ll << 20;
// Tiles of a workgroup.  One, so that the workgroups walk through memory side by side (8-bit states of 332 M fp32 elements: 886 us,
// with two 937, with four 978).  16-bit elements with 8-bit states, where a workgroup's start (table, keys, clipping factor) weighs
// more: two from 8 M elements on, and four from 32 M on with clipping, whose factor each workgroup loads first (us with one / two /
// four: bf16 8 M 19.6 / 17.2 / 18.3, 64 M 117 / 117 / 134, 332 M 564 / 563 / 618; with low halves 332 M 839 / 795 / 834; clipped, with
// the norm, bf16 16 M 42.7 / 41.4 / 40.6, 64 M 159 / 141 / 139, 332 M 754 / 682 / 700, with low halves 150 M 459 / 431 / 425)
static uint32_t tiles_of(int bits, int size, bool clip, long long total) {
  if (bits == 32 || size == 4 || total < LONG_LIST) return 1;
  return clip && total >= 4 * LONG_LIST ? 4 : 2;
}
static int item_size(int dtype) { return dtype == PDES_MT_F32 ? 4 : 2; }

// whether a list can be taken, before any of its launches: a later one must not be refused when earlier ones have run
static int check(const unsigned long long* grads, const long long* sizes, int count, int dtype, long long& total) {
  total = 0;
  for (int k = 0; k < count; ++k) {
    if (sizes[k] < 0 || sizes[k] >= MT_LONGEST - total) return PDES_EINVAL;
    if (sizes[k] == 0) continue;
    total += sizes[k];
    if (!grads[k]) return PDES_EINVAL;
    if (grads[k] % item_size(dtype)) return PDES_EALIGN;
  }
  return PDES_OK;
}
// the table of one launch over the first tensors of a list; returns how many entries of the list went into it
static int fill(NormArgs& a, const unsigned long long* grads, const long long* sizes, int count, long long chunk) {
  a.chunks = 0;
  int taken = 0, k = 0;
  for (; taken < count && k < NORM_MAX; ++taken) {
    const long long n = sizes[taken];
    if (n == 0) continue;
    a.g[k] = reinterpret_cast<void*>(grads[taken]);
    a.n[k] = n;
    a.chunk0[k++] = a.chunks;
    a.chunks += (uint32_t)((n + chunk - 1) / chunk);
  }
  for (; k < NORM_MAX; ++k) a.chunk0[k] = 0xffffffffu;
  return taken;
}

// Lists up to 4 MiB, a pass of the chip: 256 threads and chunks of 16 KiB (0.7 M fp32 elements 3.2 us, 3.7 with the others' shape).
// Longer ones: 1024 threads and 64 KiB (332 M fp32: 196 us, 264 with the short ones' shape).  Streaming from 512 MiB on, twice the
// last-level cache: under it the optimiser's step that follows finds part of the gradients there (norm and step of fp32 elements,
// cached and streaming: 64 M 350 and 362 us, 100 M 545 and 555; from 200 M on both take the same, and the norm alone is faster by a
// tenth).
constexpr int LONG_THREADS = 1024, SHORT_THREADS = 256, NORM_U = 4;
constexpr long long SHORT_MOST = 16ll * MT_ROWS * SHORT_THREADS * NORM_U, NORM_STREAMS = 512ll << 20;
template <class T, int KIND>
static void launch_norm_kind(long long bytes, const NormArgs& a, hipStream_t st) {
  if (bytes > NORM_STREAMS)
    hipLaunchKernelGGL((grad_norm_kernel<T, KIND, LONG_THREADS, NORM_U, true>), dim3(MT_ROWS), dim3(LONG_THREADS), 0, st, a);
  else if (bytes > SHORT_MOST)
    hipLaunchKernelGGL((grad_norm_kernel<T, KIND, LONG_THREADS, NORM_U, false>), dim3(MT_ROWS), dim3(LONG_THREADS), 0, st, a);
  else
    hipLaunchKernelGGL((grad_norm_kernel<T, KIND, SHORT_THREADS, NORM_U, false>), dim3(MT_ROWS), dim3(SHORT_THREADS), 0, st, a);
}
template <class T>
static void launch_norm(int kind, long long bytes, const NormArgs& a, hipStream_t st) {
  if (kind == 2) launch_norm_kind<T, 2>(bytes, a, st);
  else launch_norm_kind<T, 0>(bytes, a, st);
}
template <class T>
static void launch_clip(int kind, const NormArgs& a, hipStream_t st) {
  const unsigned grid = a.limit == INFINITY || a.chunks == 0 ? 1 : a.chunks < 2048 ? a.chunks : 2048;
  if (kind == 2)
    hipLaunchKernelGGL((clip_kernel<T, 2>), dim3(grid), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((clip_kernel<T, 0>), dim3(grid), dim3(256), 0, st, a);
}

// Streaming accesses for steps that touch more than this.  With less, parts are still in the 256 MiB cache at the next step; with
// more, the rest of a training step has put other data there.  Four lists stepped in turn, through the caches and streaming (us):
//   32-bit states  fp32 4 M (64 MiB) 20.4 and 22.6, 6 M (96 MiB) 37.1 and 32.0, 16 M 92.2 and 78.4; bf16 6 M (72 MiB) 26.0 and 26.9,
//                  8 M (96 MiB) 37.6 and 34.6; low halves 4 M 18.6 and 22.2, 8 M (112 MiB) 45.6 and 40.9; fp16 as bf16
//   8-bit states   fp32 8 M (80 MiB) 27.4 and 24.9, 12 M (120 MiB) 40.6 and 35.3; bf16 8 M (48 MiB) 17.9 and 17.6, 16 M (96 MiB) 37.0
//                  and 32.4; low halves 8 M (64 MiB) 25.3 and 25.2, 12 M (96 MiB) 38.7 and 34.8; fp16 as bf16
// (One list alone, stepped again and again with nothing between, would stay cached up to 256 MiB: fp32 8 M 35.7 and 41.8.)
constexpr long long STEP_STREAMS = 96ll << 20;
// Streaming steps with 32-bit states run best with two (fp32) or three (16-bit) workgroups on a CU, 64 to 84 KiB of loads under
// way: the memory keeps fewer pages open (us with two / three / four / as many as the registers allow: 332 M fp32 1,505 / 1,564 / 1,601 /
// 1,637; bf16 1,317 / 1,166 / 1,208 / 1,308, fp16 the same; 217 M with low halves 962 / 956 / 983 / 1,019).  Unused LDS holds the
// others off.
constexpr unsigned HOLD_TWO = 80000, HOLD_THREE = 53000;
template <class T, bool LOW, bool NT>
static void launch_step(int bits, const StepArgs& a, hipStream_t st) {
  const unsigned hold = !NT ? 0 : sizeof(typename T::E) == 4 ? HOLD_TWO : HOLD_THREE;
  if (bits == 32)
    hipLaunchKernelGGL((adamw32_kernel<T, LOW, NT>), dim3(a.chunks), dim3(256), hold, st, a);
  else if (a.norm)
    hipLaunchKernelGGL((adamw8_kernel<T, LOW, true, NT>), dim3(a.chunks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((adamw8_kernel<T, LOW, false, NT>), dim3(a.chunks), dim3(256), 0, st, a);
}
template <class T, bool LOW>
static void launch_step(int bits, long long bytes, const StepArgs& a, hipStream_t st) {
  if (bytes > STEP_STREAMS) launch_step<T, LOW, true>(bits, a, st);
  else launch_step<T, LOW, false>(bits, a, st);
}

}  // namespace pdes

using namespace pdes;

extern "C" int pdes_grad_norm(const unsigned long long* grads, const long long* sizes, int count, int dtype, int kind,
                              double* rows, int add, void* stream) {
  if (count < 0 || (count && (!grads || !sizes)) || !rows || dtype < 0 || dtype > 2 || (kind != 0 && kind != 2)) return PDES_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  NormArgs a;
  a.out = rows; a.norm_out = nullptr; a.limit = 0.f;
  long long total;
  const int rc = check(grads, sizes, count, dtype, total);
  if (rc) return rc;
  const long long bytes = total * item_size(dtype),
                  chunk = (bytes > SHORT_MOST ? LONG_THREADS : SHORT_THREADS) * NORM_U * 16ll / item_size(dtype);
  int done = 0;
  do {                            // (an empty list still writes its rows)
    const int taken = fill(a, grads + done, sizes + done, count - done, chunk);
    a.in = add || done ? rows : nullptr;
    done += taken;
    if (dtype == PDES_MT_F32) launch_norm<F32>(kind, bytes, a, st);
    else if (dtype == PDES_MT_BF16) launch_norm<BF16>(kind, bytes, a, st);
    else launch_norm<F16>(kind, bytes, a, st);
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
  long long total;
  const int rc = check(grads, sizes, count, dtype, total);
  if (rc) return rc;
  int done = 0;
  do {
    int taken = fill(a, grads + done, sizes + done, count - done, 4ll * 256 * (16 / item_size(dtype)));
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
  if (s.blocks < 0 || s.blocks > 0xffffffffll || (s.norm_rows && (!s.norm_out || !(s.limit >= 0.f)))) return PDES_EINVAL;
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
  long long total = 0, chunks = 0;
  for (int k = 0; k < count; ++k) {
    const pdes_mt_tensor& t = tensors[k];
    if (t.n < 0 || t.n >= MT_LONGEST - total || t.block0 < 0 || t.cls < 0 || t.cls >= nclasses) return PDES_EINVAL;
    if (t.block0 > s.blocks || t.block0 + (t.n + MT_BLOCK - 1) / MT_BLOCK > s.blocks) return PDES_EINVAL;
    if (t.n && (!params[k] || !grads[k])) return PDES_EINVAL;
    if (params[k] % size || grads[k] % size) return PDES_EALIGN;
    total += t.n;
  }
  StepArgs a;
  const bool clip = s.norm_rows != nullptr;
  a.tiles = tiles_of(s.bits, size, clip, total);
  const long long chunk = (long long)a.tiles * MT_TILE;
  for (int k = 0; k < count; ++k) chunks += (tensors[k].n + chunk - 1) / chunk;
  if (chunks >= 1ll << 24) return PDES_ENOSUP;             // (a launch has under 2^32 threads)
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (captured) {
    ClassArgs ca;
    ca.n = nclasses; ca.maximize = s.maximize; ca.bits = s.bits; ca.seed = s.seed; ca.out = static_cast<MtHyper*>(s.hyper);
    for (int k = 0; k < nclasses; ++k) {
      ca.lr[k] = classes[k].lr; ca.b1[k] = classes[k].beta1; ca.b2[k] = classes[k].beta2;
      ca.eps[k] = classes[k].eps; ca.wd[k] = classes[k].weight_decay;
      ca.lr_dev[k] = classes[k].lr_dev; ca.step_dev[k] = classes[k].step_dev;
    }
    hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(64), 0, st, ca);
    PDES_LAUNCH_CHECK();
  } else {
    for (int k = 0; k < nclasses; ++k)
      a.h[k] = constants(classes[k].lr, classes[k].beta1, classes[k].beta2, classes[k].eps, classes[k].weight_decay, s.maximize != 0, s.bits,
                         classes[k].step, s.seed);
  }
  a.hdev = captured ? static_cast<const MtHyper*>(s.hyper) : nullptr;
  const long long bytes = total * (2 * size + (s.low ? 2 : 0) + (s.bits == 32 ? 8 : 2));
  a.rows = s.norm_rows; a.norm = clip ? s.norm_out : nullptr;
  a.m = s.exp_avg; a.v = s.exp_avg_sq; a.ms = s.exp_avg_scale; a.rs = s.rms_scale; a.low = s.low;
  a.limit = s.limit;
  if (clip && total > LONG_LIST) {
    // every workgroup of a step can add up the rows by itself, which saves a launch (1 M elements: 21.7 us a call for norm and step,
    // 24.6 with the launch); where they are many, that costs as much or more (200 M: fp32 with 8-bit states 683 us, 673 with the
    // launch; bf16 with 32-bit states 833 and 816; at 64 M both are within a per cent)
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(MT_ROWS), 0, st, a.rows, a.norm);
    PDES_LAUNCH_CHECK();
    a.rows = nullptr;
  }
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
    if (s.dtype == PDES_MT_F32) launch_step<F32, false>(s.bits, bytes, a, st);
    else if (s.dtype == PDES_MT_F16) launch_step<F16, false>(s.bits, bytes, a, st);
    else if (s.low) launch_step<BF16, true>(s.bits, bytes, a, st);
    else launch_step<BF16, false>(s.bits, bytes, a, st);
    PDES_LAUNCH_CHECK();
  }
  return PDES_OK;
}
