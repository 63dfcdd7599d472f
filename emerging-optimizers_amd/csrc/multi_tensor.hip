// Element-wise optimizer operators over whole lists of tensors: the AdamW step with moments in 32 or in 8 bits, the
// global 2-norm and the scaling that clips by it, and the conversions of 8-bit moments.
//
// One launch serves up to a few dozen tensors.  Their addresses and sizes travel in the kernel's argument block, so a
// call needs no table in device memory, no copy and no host wait, and a captured call replays with the addresses it was
// captured with.  The tensors of a launch are cut into chunks that are numbered through, one workgroup a chunk; a
// workgroup finds its tensor by bisection in the list of first chunks (uniform: scalar loads and scalar branches).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "../../include/mi_ns.h"
#include "launch.hpp"

namespace mi {
namespace {

constexpr int NT = 256;  // threads of a workgroup where nothing else is said
constexpr int BLOCK8 = 64;  // values that share a scale in the 8-bit form of a moment
// A launch's workgroup count stays below 2^24 (2^32 threads) with room to spare; a tensor of more chunks takes several
// launches.  Chunks of one tensor are numbered in 32 bits.
constexpr int64_t MAX_CHUNKS = (int64_t)1 << 23;
constexpr int64_t MAX_NUMEL = (int64_t)1 << 40;

// ---------------------------------------------------------------------------------------------
// Argument blocks (4 KB at most)
// ---------------------------------------------------------------------------------------------
struct AdamTensor {
  void* p;            // weights of record, updated in place
  const void* g;
  void* m;            // moments: float32 values, or the 8-bit form (codes, then the blocks' scales)
  void* v;
  const float* step;  // device step counter, or null (the call's own)
  int64_t n;
};
struct AdamTensorCopy : AdamTensor {
  void* low;  // 16-bit copy of the updated weights
};
struct AdamScalars {
  float b1, omb1, b2, omb2, eps, shrink, l2, step_size, inv_sqrt_bc2;
  // for a step counter or a learning rate on the device: bias corrections and decay are evaluated by the kernel
  int on_device, method;
  double lr, wd, ln_b1, ln_b2, step;
  const float* lr_dev;
  const float* grad_scale;
};
template <class T, int N>
struct TensorList {
  static constexpr int CAPACITY = N;
  T t[N];
  uint32_t first[N];  // number of the tensor's first chunk
  int count;
  uint32_t chunk0;  // number of the launch's first chunk
};
struct None {};  // no 16-bit copies
template <class LT>
struct AdamArgs {
  TensorList<AdamTensorCopy, 66> list;
  AdamScalars s;
};
template <>
struct AdamArgs<None> {
  TensorList<AdamTensor, 76> list;
  AdamScalars s;
};
static_assert(sizeof(AdamArgs<None>) <= 4096 && sizeof(AdamArgs<float>) <= 4096, "argument block");

struct ReadTensor {
  const void* x;
  int64_t n;
};
typedef TensorList<ReadTensor, 192> ReadList;
struct MoveTensor {
  const void* src;
  void* dst;
  int64_t n;
};
typedef TensorList<MoveTensor, 128> MoveList;
static_assert(sizeof(ReadList) <= 4000 && sizeof(MoveList) <= 4000, "argument block");

// Index of the tensor that chunk `b` belongs to: the last one whose first chunk is not behind it.
template <class L>
__host__ __device__ __forceinline__ int tensor_of(const L& l, uint32_t b) {
  int lo = 0, hi = l.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------------------------
// V values at a time, 4 of float32 or 8 where all types have 16 bits (16 bytes a lane).  Tensors need the alignment of
// their elements only: the vector types say so, and global loads and stores of any width take such addresses.  A step
// touches each value once and a list is far larger than the caches, so loads and stores are non-temporal: 268M float32
// weights with float32 moments in chunks of 4096 1395 -> 1294 us (5.4 -> 5.8 TB/s; loads alone 1351, stores alone 1414),
// the sum of squares of as many values 182 -> 160 us (6.7 TB/s).  Ten other pairs of cache policies gain nothing on them.
// ---------------------------------------------------------------------------------------------
template <class T, int V>
struct Pack {
  typedef T type __attribute__((ext_vector_type(V)));
  typedef type at __attribute__((aligned(sizeof(T))));
};
template <int V>
using Floats = typename Pack<float, V>::type;
template <int V, class T>
__device__ __forceinline__ Floats<V> load(const T* p) {
  typedef Pack<T, V> X;
  return __builtin_convertvector((typename X::type)__builtin_nontemporal_load(reinterpret_cast<const typename X::at*>(p)), Floats<V>);
}
template <int V, class T>
__device__ __forceinline__ void store(T* p, Floats<V> x) {
  typedef Pack<T, V> X;
  __builtin_nontemporal_store((typename X::at)__builtin_convertvector(x, typename X::type), reinterpret_cast<typename X::at*>(p));
}
// The values [k0, k) of V; zeros for the others.
template <int V, class T>
__device__ __forceinline__ Floats<V> load_part(const T* p, int k, int k0 = 0) {
  Floats<V> x = {};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i >= k0 && i < k) x[i] = (float)p[i];
  return x;
}
template <int V, class T>
__device__ __forceinline__ void store_part(T* p, Floats<V> x, int k, int k0 = 0) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i >= k0 && i < k) p[i] = (T)x[i];
}

// Chunks begin at multiples of 64 elements in memory, not of the tensor: a tensor that begins elsewhere has its first
// chunk begin that many places before it.  Otherwise the waves of a tensor at an odd place (in a bucket of tensors back to
// back) share the 128-byte lines at their ends, and lines written in two pieces cost 15 % of a step with 32-bit moments
// (268M float32 values: 1482 us one element behind a line, 1286 at one), 21 % with 16-bit copies; reading bfloat16 from an
// odd element costs 27 % of the norm.
template <class T>
__host__ __device__ __forceinline__ int places_before(const T* p) {
  return (int)((uintptr_t)p / sizeof(T) & 63);
}
// The part of a vector of V values that a tensor has: [k0, k1) of those at place `at`.
template <int V>
struct Part {
  int k0, k1;
  __device__ __forceinline__ Part(int64_t at, int64_t n)
      : k0(at < 0 ? (at > -V ? (int)-at : V) : 0), k1(n - at < V ? (n - at > 0 ? (int)(n - at) : 0) : V) {}
  __device__ __forceinline__ bool none() const { return k0 >= k1; }
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == V; }
};

// ---------------------------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------------------------
struct AdamCoef {
  float b1, omb1, b2, omb2, eps, shrink, l2, step_size, inv_sqrt_bc2, gscale;
};

enum { DECAY_DECOUPLED = 0, DECAY_INDEPENDENT = 1, DECAY_L2 = 2, DECAY_PALM = 3 };

// Share of the weight that goes, and multiple of the weight that joins the gradient, by decay method.  (The share and not
// what remains of the weight: 1 - 1e-7 has one digit of the share left in float32.)
__host__ __device__ inline void decay_terms(int method, double wd, double lr, float* shrink, float* l2) {
  *l2 = method == DECAY_L2 ? (float)wd : 0.0f;
  *shrink = (float)(method == DECAY_DECOUPLED ? wd * lr : method == DECAY_INDEPENDENT ? wd : method == DECAY_PALM ? wd * lr * lr : 0.0);
}
// lr / (1 - b1^t) and 1 / sqrt(1 - b2^t), in 64 bits: 1 - b^t loses its leading digits for small t and b near 1.
__host__ __device__ inline void bias_terms(double ln_b1, double ln_b2, double t, double lr, float* step_size, float* inv_sqrt_bc2) {
  *step_size = (float)(lr / -expm1(t * ln_b1));
  *inv_sqrt_bc2 = (float)(1.0 / sqrt(-expm1(t * ln_b2)));
}

__device__ __forceinline__ AdamCoef adam_coefficients(const AdamScalars& s, const float* step_dev) {
  AdamCoef c = {s.b1, s.omb1, s.b2, s.omb2, s.eps, s.shrink, s.l2, s.step_size, s.inv_sqrt_bc2, 1.0f};
  if (s.on_device) {
    const double lr = s.lr_dev ? (double)*s.lr_dev : s.lr;
    decay_terms(s.method, s.wd, lr, &c.shrink, &c.l2);
    bias_terms(s.ln_b1, s.ln_b2, step_dev ? (double)*step_dev : s.step, lr, &c.step_size, &c.inv_sqrt_bc2);
  }
  if (s.grad_scale) c.gscale = *s.grad_scale;
  return c;
}

// m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2,  p <- p - shrink p - step_size m / (sqrt(v) inv_sqrt_bc2 + eps)
//
// The coefficients are the same for all values; with a step count on the device every wave evaluates them for its 256 (512)
// values, about 90 64-bit instructions before the first load: nothing measurable beside 32-bit moments (0 to 4 %).
//
// FAST: square root and reciprocal of the hardware, each within one unit in the last place, for which a number below the
// smallest normal one is 0.  The correctly rounded sequences cost about 25 instructions a value: nothing beside 32-bit
// moments, where the memory sets the pace, and twice the time beside 8-bit ones (see below).
template <bool FAST>
__device__ __forceinline__ void adam_value(float& p, float g, float& m, float& v, const AdamCoef& c) {
  g *= c.gscale;
  if (c.l2 != 0.0f) g = fmaf(c.l2, p, g);
  m = fmaf(c.b1, m, c.omb1 * g);
  v = fmaf(c.b2, v, c.omb2 * g * g);
  const float den = fmaf(FAST ? __builtin_amdgcn_sqrtf(v) : sqrtf(v), c.inv_sqrt_bc2, c.eps);
  if (c.shrink != 0.0f) p = fmaf(-c.shrink, p, p);
  p = fmaf(-c.step_size, FAST ? m * __builtin_amdgcn_rcpf(den) : m / den, p);
}

// 32-bit moments.  Each value is read and written once: 28 bytes a value with float32 weights and gradients, 42
// instructions, so the memory bounds it: 269M values in 67 tensors take 1187 to 1240 us (6.1 to 6.3 TB/s; a large copy by
// torch reaches 4.9), 436M with bfloat16 gradients and copies 2.09 ms (5.8 TB/s).  A thread handles one vector of four and
// a workgroup 1024 values: chunks of 2048 and 4096 (more loads in flight a thread, fewer threads on a CU) take 2 to 4 %
// longer, 8 values a thread (32-byte pieces of float32) 14 %, workgroups of 128 threads 1 % (odd sizes: 8 %), of 512 and
// 1024 threads 2 to 6 %; handing each XCD a contiguous range of chunks takes up to 11 % longer.
constexpr int ADAM_V = 4;
constexpr int ADAM_CHUNK = NT * ADAM_V;

template <class PT, class GT, class LT>
__global__ __launch_bounds__(NT) void adamw_kernel(AdamArgs<LT> a) {
  constexpr int V = ADAM_V;
  typedef Floats<V> F;
  const uint32_t chunk = a.list.chunk0 + blockIdx.x;
  const int ti = tensor_of(a.list, chunk);
  const auto t = a.list.t[ti];
  // (the moments' places decide; weights and gradients in buckets of the same order have the same ones)
  const int64_t at = (int64_t)(chunk - a.list.first[ti]) * ADAM_CHUNK - places_before(static_cast<float*>(t.m)) + threadIdx.x * V;
  const Part<V> part(at, t.n);
  const AdamCoef c = adam_coefficients(a.s, t.step);
  if (part.none()) return;
  PT* __restrict__ p = static_cast<PT*>(t.p) + at;
  const GT* __restrict__ g = static_cast<const GT*>(t.g) + at;
  float* __restrict__ m = static_cast<float*>(t.m) + at;
  float* __restrict__ v = static_cast<float*>(t.v) + at;
  F pp, gg, mm, vv;
  if (part.whole()) {
    gg = load<V>(g);
    pp = load<V>(p);
    mm = load<V>(m);
    vv = load<V>(v);
  } else {
    gg = load_part<V>(g, part.k1, part.k0);
    pp = load_part<V>(p, part.k1, part.k0);
    mm = load_part<V>(m, part.k1, part.k0);
    vv = load_part<V>(v, part.k1, part.k0);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float pi = pp[i], mi = mm[i], vi = vv[i];
    adam_value<false>(pi, gg[i], mi, vi, c);
    pp[i] = pi;
    mm[i] = mi;
    vv[i] = vi;
  }
  if (part.whole()) {
    store<V>(p, pp);
    store<V>(m, mm);
    store<V>(v, vv);
    if constexpr (!__is_same(LT, None)) store<V>(static_cast<LT*>(t.low) + at, pp);
  } else {
    store_part<V>(p, pp, part.k1, part.k0);
    store_part<V>(m, mm, part.k1, part.k0);
    store_part<V>(v, vv, part.k1, part.k0);
    if constexpr (!__is_same(LT, None)) store_part<V>(static_cast<LT*>(t.low) + at, pp, part.k1, part.k0);
  }
}

// ---------------------------------------------------------------------------------------------
// 8-bit moments.  A tensor of n values is ceil(n / 64) blocks; its form is 64 bytes of codes for each block and behind
// them one float32 scale s for each, the largest magnitude of the block:
//   first moment    m = +- s (k / 127)^2   code +-k, k = round(127 sqrt(|m| / s))
//   second moment   v =    s (k / 255)^4   code   k, k = round(255 (v / s)^(1/4)), at least 1 for v > 0
// Roots space the codes finer towards 0, evenly in relative terms over a range of 1.6e4 in m and 6e4 in sqrt(v); a
// second moment over 0 never becomes 0, so no update divides by eps alone (linear codes of m and sqrt(v) and e4m3 let small
// second moments of a wide block become 0).
//
// To nearest is right for one conversion and wrong for a run of steps: a factor b changes code k of m by k (1 - b^(1/2))
// and of v by k (1 - b^(1/4)), and a code that a step changes by less than half never moves beside a scale that stays (at
// beta1 = 0.9 the codes up to 9, at beta2 = 0.999 all of v's).  So a run of steps takes DITHERED codes floor(y + u), with
// y = 127 sqrt(|m| / s) or 255 (v / s)^(1/4) and
//   u = fraction of (t c + i a)   for step t and place i of the tensor, c and a irrational, others for v than for m.
// For each place u rotates through its interval evenly, so a change of 0.01 of a code moves it every 100 steps, and the
// errors of consecutive steps cancel instead of adding up as independent random numbers' do.  Two rules beside it: codes of
// v below 6 round up (a root of v held at a fraction of itself blows the update up; so a root that falls stops at
// 1/1800 of its block's largest, which makes such a value's updates smaller, never larger), and the first four steps go to nearest
// (step t of a moving average changes a code by about 1 / (2 t) of itself, so nothing stands still yet).
// Simulated update error against 32-bit moments, gradients' scales spread as exp(N(0, sigma)), beta2 = 0.95 / 0.999:
//   sigma 0.5: nearest 2.3 / 5.6 %, independent random numbers 3.3 / 6.9 %, rotating 2.5 / 5.8 %
//   sigma 1.5: nearest 11 / 16 %, rotating 12 / 16 %;   sigma 2.5: nearest 84 / 94 %, rotating 40 / 42 %
//   half of each block's gradients fall to a tenth, beta2 = 0.999: sqrt(v) 4.6 times too large to nearest, 1.0 rotating.
// A block whose largest magnitude is below the smallest normal number is stored as 0, one that holds a value that is not
// finite as NaN.  Codes of places behind the last value are 0.
// ---------------------------------------------------------------------------------------------
__host__ __device__ inline int64_t blocks8(int64_t n) { return (n + BLOCK8 - 1) / BLOCK8; }

// Maximum over the lanes that hold a block: 16 with 4 values each, 8 with 8 (exchanges inside a row of 16 lanes; every
// lane of the block must be active).
template <int V>
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
  static_assert(V == 4 || V == 8, "lanes of a block");
#define MI_ROW_STEP(ctrl) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true))
  MI_ROW_STEP(0xB1);   // quad_perm [1, 0, 3, 2]
  MI_ROW_STEP(0x4E);   // quad_perm [2, 3, 0, 1]
  MI_ROW_STEP(0x141);  // row_half_mirror: the other quad of eight lanes
  if (V == 4) MI_ROW_STEP(0x140);  // row_mirror: the other half of the row
#undef MI_ROW_STEP
  return x;
}

// Scale of the block this lane's magnitudes belong to.  The bit patterns of magnitudes order as the numbers do, with
// infinities and then NaN above every finite one.
template <int V>
__device__ __forceinline__ float block_scale(Floats<V> x) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = block_max<V>(top);
  return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : top < 0x00800000u ? 0.0f : __uint_as_float(top);
}

template <int V>
using Codes = typename Pack<uint32_t, V / 4>::type;

// Codes of V values.  The product with 127 or 255 and the rounding to the nearest integer are one operation: the sum
// with 1.5 * 2^23 leaves the integer (two's complement for negative ones) in the lowest byte.  With the hardware's roots
// and reciprocal, a step of 268M bfloat16 weights with 8-bit moments takes 505 us instead of 875 with correctly rounded
// ones and a conversion to int.
template <int V, bool SIGNED>
__device__ __forceinline__ Codes<V> encode(Floats<V> x, float s) {
  float inv = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;  // (neither for 0 nor for NaN)
  if (__builtin_expect(s > 0x1p125f, 0)) inv = 1.0f / s;   // below the smallest normal number, which v_rcp_f32 makes 0
  const int least = s > 0.0f ? 1 : 0;
  uint32_t k[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float root = __builtin_amdgcn_sqrtf(fabsf(x[i]) * inv);
    if constexpr (SIGNED) {
      k[i] = __float_as_uint(fmaf(copysignf(root, x[i]), 127.0f, 12582912.0f));
    } else {
      k[i] = __float_as_uint(fmaf(__builtin_amdgcn_sqrtf(root), 255.0f, 12582912.0f));
      // 1 at least for a value over 0 (as integers -0.0 and negative values are below 0)
      k[i] = max(k[i], 0x4B400000u | (uint32_t)max(min(__float_as_int(x[i]), least), 0));
    }
  }
  Codes<V> codes;
#pragma unroll
  for (int i = 0; i < V; i += 4)
    codes[i / 4] = __builtin_amdgcn_perm(k[i + 1], k[i], 0x0c0c0400u) | __builtin_amdgcn_perm(k[i + 3], k[i + 2], 0x04000c0cu);
  return codes;
}

// Dithered codes: bits of u as fractions of 2^32, at the lane's first place and from one place to the next, and the root of
// v / s below which codes round up.
struct Dither {
  uint32_t m, v, m_place, v_place;
  float up;
};
constexpr uint32_t DITHER_M_STEP = 0x9E3779B9u;                                      // golden ratio
constexpr uint32_t DITHER_M_PLACE = 0x6A09E667u, DITHER_V_STEP = 0x6A09E667u;        // sqrt(2)
constexpr uint32_t DITHER_V_PLACE = 0xBB67AE85u;                                     // sqrt(3)
constexpr double DITHER_AFTER = 4.0;                                                 // steps to nearest
__device__ __forceinline__ Dither dither(const AdamScalars& s, const float* step_dev, uint32_t place) {
  const double t = step_dev ? (double)*step_dev : s.step;
  if (!(t > DITHER_AFTER)) return {0x80000000u, 0x80000000u, 0u, 0u, 0.0f};  // u = 1/2: to nearest
  const uint32_t n = (uint32_t)(uint64_t)t;
  return {n * DITHER_M_STEP + place * DITHER_M_PLACE, n * DITHER_V_STEP + place * DITHER_V_PLACE, DITHER_M_PLACE, DITHER_V_PLACE, 6.0f / 255};
}
template <int V, bool SIGNED>
__device__ __forceinline__ Codes<V> encode_dithered(Floats<V> x, float s, const Dither& d) {
  float inv = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;
  if (__builtin_expect(s > 0x1p125f, 0)) inv = 1.0f / s;
  uint32_t k[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float root = __builtin_amdgcn_sqrtf(fabsf(x[i]) * inv);
    if constexpr (!SIGNED) root = __builtin_amdgcn_sqrtf(root);
    const uint32_t bits = SIGNED ? d.m + i * d.m_place : d.v + i * d.v_place;
    float one_u = __uint_as_float(0x3f800000u | bits >> 9);                     // 1 + u
    if constexpr (!SIGNED) one_u = root < d.up ? 2.0f - 0x1p-8f : one_u;        // (1/256: the roots' own error is no step up)
    // at most the largest code, whatever the roots' last place is
    const uint32_t n = (uint32_t)fminf(fmaf(root, SIGNED ? 127.0f : 255.0f, one_u) - 1.0f, SIGNED ? 127.5f : 255.5f);
    k[i] = SIGNED ? (x[i] < 0.0f ? 0u - n : n) : max(n, x[i] > 0.0f && s > 0.0f ? 1u : 0u);
  }
  Codes<V> codes;
#pragma unroll
  for (int i = 0; i < V; i += 4)
    codes[i / 4] = __builtin_amdgcn_perm(k[i + 1], k[i], 0x0c0c0400u) | __builtin_amdgcn_perm(k[i + 3], k[i + 2], 0x04000c0cu);
  return codes;
}

template <int V, bool SIGNED>
__device__ __forceinline__ Floats<V> decode(Codes<V> codes, float s) {
  Floats<V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // the scale comes last: a share of it that is taken first would be denormal for scales far above the smallest number
    if constexpr (SIGNED) {
      const float k = (float)(int8_t)(codes[i / 4] >> (8 * (i % 4)));
      x[i] = k * fabsf(k) * (1.0f / (127 * 127)) * s;
    } else {
      const float k = (float)((codes[i / 4] >> (8 * (i % 4))) & 0xffu);
      const float k2 = k * k * (1.0f / (255 * 255));
      x[i] = k2 * k2 * s;
    }
  }
  return x;
}
template <int V>
__device__ __forceinline__ Codes<V> load_codes(const uint8_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const Codes<V>*>(p));
}
template <int V>
__device__ __forceinline__ void store_codes(uint8_t* p, Codes<V> codes) {
  __builtin_nontemporal_store(codes, reinterpret_cast<Codes<V>*>(p));
}

// The step itself: 16.25 bytes a value with float32 weights and gradients, 10.25 with 16-bit ones.  The values of a block
// sit in neighbouring lanes of one wave, so the new scale is a maximum over registers and three or four lane exchanges,
// and the moments never leave registers between reading and writing their codes.  269M float32 weights in 683 us (6.4
// TB/s), 268M bfloat16 ones in 435 us (6.3 TB/s); at first, with correctly rounded roots and quotients, 973 and 923 us,
// bound by the vector units.  Eight values a lane pay where weights and gradients have 16 bits (435 us; four: 464) and not
// with float32 (781 against 691 us).  Dithered codes take 17 to 18 instructions a value more (76 instead of 58 with float32, 70
// instead of 53 with 16 bits): nothing with float32 weights (688 us either way), 8 to 12 % with 16-bit ones (433 -> 469 us).
// A step count or a learning rate on the device adds the 64-bit coefficients to every wave: 4 to 33 % (688 -> 713 us and, dithered,
// 784; 433 -> 511 and, dithered, 469 -> 576).
template <class PT, class GT>
struct Adam8Shape {
  static constexpr int V = sizeof(PT) == 2 && sizeof(GT) == 2 ? 8 : 4, CHUNK = NT * V;
};

template <class PT, class GT, class LT, bool DITHERED>
__global__ __launch_bounds__(NT) void adamw8_kernel(AdamArgs<LT> a) {
  typedef Adam8Shape<PT, GT> S;
  constexpr int V = S::V;
  typedef Floats<V> F;
  const uint32_t chunk = a.list.chunk0 + blockIdx.x;
  const int ti = tensor_of(a.list, chunk);
  const auto t = a.list.t[ti];
  const int64_t base = (int64_t)(chunk - a.list.first[ti]) * S::CHUNK;
  PT* __restrict__ p = static_cast<PT*>(t.p) + base;
  const GT* __restrict__ g = static_cast<const GT*>(t.g) + base;
  const int64_t nb = blocks8(t.n);
  uint8_t* __restrict__ mc = static_cast<uint8_t*>(t.m) + base;
  uint8_t* __restrict__ vc = static_cast<uint8_t*>(t.v) + base;
  float* __restrict__ ms = reinterpret_cast<float*>(static_cast<uint8_t*>(t.m) + nb * BLOCK8) + base / BLOCK8;
  float* __restrict__ vs = reinterpret_cast<float*>(static_cast<uint8_t*>(t.v) + nb * BLOCK8) + base / BLOCK8;
  const int64_t left = t.n - base;
  const AdamCoef c = adam_coefficients(a.s, t.step);
  const int e = threadIdx.x * V;
  const int b = e / BLOCK8;
  if ((int64_t)b * BLOCK8 >= left) return;  // all lanes of the block together
  const int k = left - e >= V ? V : left - e > 0 ? (int)(left - e) : 0;
  F pp, gg;
  if (k == V) {
    pp = load<V>(p + e);
    gg = load<V>(g + e);
  } else {
    pp = load_part<V>(p + e, k);
    gg = load_part<V>(g + e, k);
  }
  F mm = decode<V, true>(load_codes<V>(mc + e), ms[b]), vv = decode<V, false>(load_codes<V>(vc + e), vs[b]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float pi = pp[i], mi = mm[i], vi = vv[i];
    adam_value<true>(pi, gg[i], mi, vi, c);
    pp[i] = pi;
    mm[i] = mi;
    vv[i] = vi;
  }
  if (k < V) {  // places behind the last value hold 0
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= k) mm[i] = vv[i] = 0.0f;
  }
  const float sm = block_scale<V>(mm), sv = block_scale<V>(vv);
  if constexpr (DITHERED) {
    const Dither d = dither(a.s, t.step, (uint32_t)(base + e));
    store_codes<V>(mc + e, encode_dithered<V, true>(mm, sm, d));
    store_codes<V>(vc + e, encode_dithered<V, false>(vv, sv, d));
  } else {
    store_codes<V>(mc + e, encode<V, true>(mm, sm));
    store_codes<V>(vc + e, encode<V, false>(vv, sv));
  }
  if (e % BLOCK8 == 0) {
    ms[b] = sm;
    vs[b] = sv;
  }
  if (k == V) {
    store<V>(p + e, pp);
    if constexpr (!__is_same(LT, None)) store<V>(static_cast<LT*>(t.low) + base + e, pp);
  } else {
    store_part<V>(p + e, pp, k);
    if constexpr (!__is_same(LT, None)) store_part<V>(static_cast<LT*>(t.low) + base + e, pp, k);
  }
}

// Conversions between a list of tensors and their 8-bit forms, bound by the memory: 268M values to 8 bits 202 us from
// float32 (6.7 TB/s) and 131 us from bfloat16 (5.8 to 6.5 TB/s), back to float32 226 us (6.0 TB/s) and to bfloat16 122 us
// (6.7 TB/s).  These move few bytes a value, so the cost of a workgroup shows (1024 values in one: 20 to 30 % longer):
// two vectors a thread, four where float32 is written; 128 threads are up to 5 % faster than 256.
template <class T, bool PACK>
struct MoveShape {
  static constexpr int V = sizeof(T) == 2 ? 8 : 4, U = sizeof(T) == 4 && !PACK ? 4 : 2, THREADS = 128;
  static constexpr int CHUNK = THREADS * V * U;
};

template <class T, bool SIGNED>
__global__ __launch_bounds__((MoveShape<T, true>::THREADS)) void pack8_kernel(MoveList l) {
  typedef MoveShape<T, true> S;
  constexpr int V = S::V;
  const uint32_t chunk = l.chunk0 + blockIdx.x;
  const int ti = tensor_of(l, chunk);
  const MoveTensor t = l.t[ti];
  const int64_t base = (int64_t)(chunk - l.first[ti]) * S::CHUNK;
  const T* __restrict__ x = static_cast<const T*>(t.src) + base;
  uint8_t* __restrict__ codes = static_cast<uint8_t*>(t.dst) + base;
  float* __restrict__ scales = reinterpret_cast<float*>(static_cast<uint8_t*>(t.dst) + blocks8(t.n) * BLOCK8) + base / BLOCK8;
  const int64_t left = t.n - base;
#pragma unroll
  for (int u = 0; u < S::U; ++u) {
    const int e = (u * S::THREADS + threadIdx.x) * V;
    const int b = e / BLOCK8;
    if ((int64_t)b * BLOCK8 >= left) return;  // all lanes of the block together
    const int k = left - e >= V ? V : left - e > 0 ? (int)(left - e) : 0;
    const Floats<V> xx = k == V ? load<V>(x + e) : load_part<V>(x + e, k);
    const float s = block_scale<V>(xx);
    store_codes<V>(codes + e, encode<V, SIGNED>(xx, s));
    if (e % BLOCK8 == 0) scales[b] = s;
  }
}

template <class T, bool SIGNED>
__global__ __launch_bounds__((MoveShape<T, false>::THREADS)) void unpack8_kernel(MoveList l) {
  typedef MoveShape<T, false> S;
  constexpr int V = S::V;
  const uint32_t chunk = l.chunk0 + blockIdx.x;
  const int ti = tensor_of(l, chunk);
  const MoveTensor t = l.t[ti];
  const int64_t base = (int64_t)(chunk - l.first[ti]) * S::CHUNK;
  const uint8_t* __restrict__ codes = static_cast<const uint8_t*>(t.src) + base;
  const float* __restrict__ scales = reinterpret_cast<const float*>(static_cast<const uint8_t*>(t.src) + blocks8(t.n) * BLOCK8) + base / BLOCK8;
  T* __restrict__ x = static_cast<T*>(t.dst) + base;
  const int64_t left = t.n - base;
#pragma unroll
  for (int u = 0; u < S::U; ++u) {
    const int e = (u * S::THREADS + threadIdx.x) * V;
    if (e >= left) return;
    const Floats<V> xx = decode<V, SIGNED>(load_codes<V>(codes + e), scales[e / BLOCK8]);
    if (left - e >= V) store<V>(x + e, xx);
    else store_part<V>(x + e, xx, (int)(left - e));
  }
}

// ---------------------------------------------------------------------------------------------
// Global norm and scaling
// ---------------------------------------------------------------------------------------------
constexpr int NORM_CHUNK = NT * 64;

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
  return x;
}
// Sum over the workgroup, in thread 0, in a fixed order.
template <int THREADS>
__device__ __forceinline__ double group_sum(double x) {
  __shared__ double part[THREADS / 64];
  x = wave_sum(x);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0.0;
  if (threadIdx.x == 0)
    for (int w = 0; w < THREADS / 64; ++w) s += part[w];
  return s;
}

// Global norm, one read of the list: 872 MB of bfloat16 in 128 us (6.8 TB/s).  Chunks of 16384 values; smaller ones pay for
// the reduction inside the workgroup (4096: 8 to 14 % longer), larger ones gain nothing.
//
// Sum of squares of every chunk, in 64 bits: squares of float32 values neither overflow nor vanish there, and sums over
// a whole model lose nothing.
template <class T>
__global__ __launch_bounds__(NT) void sumsq_list_kernel(ReadList l, double* __restrict__ partials) {
  const uint32_t chunk = l.chunk0 + blockIdx.x;
  const int ti = tensor_of(l, chunk);
  const T* const tensor = static_cast<const T*>(l.t[ti].x);
  const int64_t base = (int64_t)(chunk - l.first[ti]) * NORM_CHUNK - places_before(tensor), n = l.t[ti].n;
  const T* __restrict__ x = tensor + base;
  constexpr int V = 16 / sizeof(T);
  double sum = 0.0;
  if (base >= 0 && n - base >= NORM_CHUNK) {
#pragma unroll 4
    for (int e = threadIdx.x * V; e < NORM_CHUNK; e += NT * V) {
      const Floats<V> xx = load<V>(x + e);
#pragma unroll
      for (int i = 0; i < V; ++i) sum = fma((double)xx[i], (double)xx[i], sum);
    }
  } else {
    const int end = n - base < NORM_CHUNK ? (int)(n - base) : NORM_CHUNK;
#pragma unroll 4
    for (int e = threadIdx.x * V; e < end; e += NT * V) {
      const Part<V> part(base + e, n);
      const Floats<V> xx = part.whole() ? load<V>(x + e) : load_part<V>(x + e, part.k1, part.k0);
#pragma unroll
      for (int i = 0; i < V; ++i) sum = fma((double)xx[i], (double)xx[i], sum);
    }
  }
  sum = group_sum<NT>(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// A norm and the factor that clips to max_norm: min(1, max_norm / (norm + 1e-6)), NaN for a norm that is not a number.
struct NormAndFactor {
  float norm, factor;
};
__device__ __forceinline__ NormAndFactor norm_and_factor(double sum, float max_norm) {
  const float norm = (float)sqrt(sum);
  const float f = max_norm / (norm + 1e-6f);
  return {norm, f > 1.0f ? 1.0f : f};
}

// Sum of all partial sums, in thread 0.  The order depends on THREADS: a call with up to FEW_PARTIALS of them adds them
// up with NT threads, whoever does it.
constexpr int64_t FEW_PARTIALS = 2 * NT;
template <int THREADS>
__device__ __forceinline__ double sum_partials(const double* __restrict__ partials, int64_t count) {
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < count; i += THREADS) sum += partials[i];
  return group_sum<THREADS>(sum);
}

// out[0] = norm, out[1] = factor
template <int THREADS>
__global__ __launch_bounds__(THREADS) void norm_finish_kernel(const double* __restrict__ partials, int64_t count, float max_norm,
                                                              float* __restrict__ out) {
  const double sum = sum_partials<THREADS>(partials, count);
  if (threadIdx.x == 0) {
    const NormAndFactor r = norm_and_factor(sum, max_norm);
    out[0] = r.norm;
    out[1] = r.factor;
  }
}

// Scaling: 872 MB of bfloat16 read and written in 287 us (6.1 TB/s).  Reading in the opposite order of the norm, to meet what
// is left in the caches, changes nothing with or without non-temporal loads.
template <class T>
struct ScaleShape {
  static constexpr int V = 16 / sizeof(T), CHUNK = NT * V;
};

// x <- factor x; a factor of 1 changes nothing and reads nothing.  The factor is *factor, or, with FINISH, what the
// partial sums of a norm give: with few of them every workgroup adds them up itself (they come out of the cache), the
// first one stores norm and factor, and clipping takes two launches instead of three.
struct ScaleFactor {
  const float* factor;
  const double* partials;
  int64_t count;
  float max_norm;
  float* out;
};

template <class T, bool FINISH>
__global__ __launch_bounds__(NT) void scale_list_kernel(ReadList l, ScaleFactor sf) {
  typedef ScaleShape<T> S;
  constexpr int V = S::V;
  float f;
  if constexpr (FINISH) {
    __shared__ float shared_factor;
    const double sum = sum_partials<NT>(sf.partials, sf.count);
    if (threadIdx.x == 0) {
      const NormAndFactor r = norm_and_factor(sum, sf.max_norm);
      shared_factor = r.factor;
      if (blockIdx.x == 0) {
        sf.out[0] = r.norm;
        sf.out[1] = r.factor;
      }
    }
    __syncthreads();
    f = shared_factor;
  } else {
    f = *sf.factor;
  }
  if (f == 1.0f) return;
  const uint32_t chunk = l.chunk0 + blockIdx.x;
  const int ti = tensor_of(l, chunk);
  T* const tensor = static_cast<T*>(const_cast<void*>(l.t[ti].x));
  const int64_t at = (int64_t)(chunk - l.first[ti]) * S::CHUNK - places_before(tensor) + threadIdx.x * V;
  const Part<V> part(at, l.t[ti].n);
  if (part.none()) return;
  T* __restrict__ x = tensor + at;
  if (part.whole()) store<V>(x, load<V>(x) * f);
  else store_part<V>(x, load_part<V>(x, part.k1, part.k0) * f, part.k1, part.k0);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
// Walks a list of tensors and hands full argument blocks to `launch(list, chunks)`: empty tensors are left out, a block
// ends when it is full or its chunks would be too many, and a tensor with too many of them has launches of its own.
// `fill(i)` makes the entry of tensor i, `before(entry)` says how many places before the tensor its first chunk begins.
template <class L, class Fill, class Before, class Launch>
int for_each_list(int64_t count, const int64_t* numel, int64_t chunk, L& list, Fill fill, Before before, Launch launch) {
  int64_t chunks = 0;
  list.count = 0;
  list.chunk0 = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const auto entry = fill(i);
    const int64_t c = (numel[i] + before(entry) + chunk - 1) / chunk;
    if (list.count == L::CAPACITY || (list.count > 0 && chunks + c > MAX_CHUNKS)) {
      if (int rc = launch(list, chunks)) return rc;
      list.count = 0;
      chunks = 0;
    }
    list.first[list.count] = (uint32_t)chunks;
    list.t[list.count++] = entry;
    chunks += c;
    if (chunks > MAX_CHUNKS) {
      for (int64_t at = 0; at < c; at += MAX_CHUNKS) {
        list.chunk0 = (uint32_t)at;
        if (int rc = launch(list, std::min(MAX_CHUNKS, c - at))) return rc;
      }
      list.count = 0;
      list.chunk0 = 0;
      chunks = 0;
    }
  }
  return list.count ? launch(list, chunks) : MI_OK;
}

constexpr auto at_tensor = [](const auto&) { return 0; };  // chunks begin with the tensor
// Chunks begin at multiples of 64 elements (places_before).
template <class T>
constexpr auto at_line_of = [](const ReadTensor& t) { return places_before(static_cast<const T*>(t.x)); };

int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MI_OK : fail(MI_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
}

#ifdef MI_HOST_CHECK
// Every chunk of a launch falls into the tensor the bisection finds and reaches into it, and the chunks of a tensor
// reach its end (those of a tensor with launches of its own are walked launch by launch).
template <class L, class Before>
void walk(const L& l, int64_t chunks, int64_t chunk, Before before) {
  for (int64_t i = 0; i < chunks; i += (chunks > 4096 && i > 64 && i < chunks - 64) ? 61 : 1) {
    const int64_t b = l.chunk0 + i;
    const int ti = tensor_of(l, (uint32_t)b);
    if (b >> 32) host_check::fail("a chunk number past 32 bits");
    if (ti < 0 || ti >= l.count || l.first[ti] > b) host_check::fail("a chunk without a tensor");
    else if ((b - l.first[ti]) * chunk - before(l.t[ti]) >= l.t[ti].n) host_check::fail("a chunk behind the end of its tensor");
    else if ((b - l.first[ti] + 1) * chunk - before(l.t[ti]) <= 0) host_check::fail("a chunk before the start of its tensor");
  }
  for (int i = 0; i < l.count; ++i) {
    const int64_t end = i + 1 < l.count ? l.first[i + 1] : l.chunk0 + chunks;
    const bool last = i + 1 < l.count || chunks < MAX_CHUNKS;
    if (last && (end - l.first[i]) * chunk - before(l.t[i]) < l.t[i].n) host_check::fail("chunks that end before their tensor");
  }
}
#define MI_WALK(...) walk(__VA_ARGS__)
#else
#define MI_WALK(...) ((void)0)
#endif

int element_bytes(int dtype) { return dtype == MI_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == MI_DTYPE_F32 || dtype == MI_DTYPE_BF16 || dtype == MI_DTYPE_F16; }

// Memory of a call: no written range may meet any other.  The ranges come role by role (weights, gradients, ...); the
// addresses of a role mostly ascend already, so the roles are merged and only one that does not ascend is sorted.
struct Span {
  uintptr_t lo, hi;
};
struct Spans {
  static constexpr int MAX_ROLES = 5;
  std::vector<Span> all;
  size_t end[MAX_ROLES] = {};
  bool written[MAX_ROLES] = {};
  int roles = 0;

  void close_role(bool is_written) {
    const size_t begin = roles ? end[roles - 1] : 0;
    const auto before = [](const Span& a, const Span& b) { return a.lo < b.lo; };
    if (!std::is_sorted(all.begin() + begin, all.end(), before)) std::sort(all.begin() + begin, all.end(), before);
    written[roles] = is_written;
    end[roles++] = all.size();
  }
  bool conflict() const {
    size_t head[MAX_ROLES];
    for (int r = 0; r < roles; ++r) head[r] = r ? end[r - 1] : 0;
    uintptr_t end_any = 0, end_written = 0;
    for (;;) {
      int r = -1;
      for (int i = 0; i < roles; ++i)
        if (head[i] < end[i] && (r < 0 || all[head[i]].lo < all[head[r]].lo)) r = i;
      if (r < 0) return false;
      const Span& s = all[head[r]++];
      if (s.lo < (written[r] ? end_any : end_written)) return true;
      end_any = std::max(end_any, s.hi);
      if (written[r]) end_written = std::max(end_written, s.hi);
    }
  }
};

// Checks one list argument and adds its ranges.
int add_spans(const char* who, const char* what, Spans& spans, int64_t count, const void* const* ptrs, const int64_t* numel,
              int bytes, bool packed, bool written) {
  if (!ptrs && count > 0) return fail(MI_ERR_BAD_ARG, "%s: no list of %s", who, what);
  const uintptr_t align = packed ? 16 : (uintptr_t)bytes;
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(ptrs[i]);
    if (!lo) return fail(MI_ERR_BAD_ARG, "%s: %s %lld is null", who, what, (long long)i);
    if (lo % align) return fail(MI_ERR_BAD_ARG, "%s: %s %lld is not aligned to %d bytes", who, what, (long long)i, (int)align);
    spans.all.push_back({lo, lo + (packed ? mi_moment_8bit_bytes(numel[i]) : (size_t)numel[i] * bytes)});
  }
  spans.close_role(written);
  return MI_OK;
}

int check_numel(const char* who, int64_t count, const int64_t* numel) {
  if (count < 0 || (count > 0 && !numel)) return fail(MI_ERR_BAD_ARG, "%s: bad tensor count or no sizes", who);
  for (int64_t i = 0; i < count; ++i) {
    if (numel[i] < 0) return fail(MI_ERR_BAD_ARG, "%s: tensor %lld has a negative size", who, (long long)i);
    if (numel[i] > MAX_NUMEL)
      return fail(MI_ERR_UNSUPPORTED_SHAPE, "%s: tensor %lld has %lld elements, at most 2^40 are supported", who, (long long)i, (long long)numel[i]);
  }
  return MI_OK;
}

// LDS that a workgroup of the step with 32-bit moments holds without using it, so that fewer than eight of them share a CU:
// the memory does better with fewer rows open at once where 16-bit weights or copies are written beside 32-bit moments.
// Chosen by what is written, both sides measured (2^28 values in 16 tensors):
//   16-bit copies, five workgroups: bfloat16 gradients 1255 -> 1232 us, float32 ones 1450 -> 1418
//     (436M values in 19 tensors, clipped: 2280 us with eight, 2251 seven, 2216 six, 2197 five and four)
//   16-bit weights, six: bfloat16 gradients 956 -> 948 us, float32 ones 1035 -> 1025 (odd sizes 184 -> 187, 204 -> 202)
//   float32 weights alone, none: float32 gradients 1286 -> 1283 us with six and 1304 with five; bfloat16 ones 1143 -> 1122 with
//     six, but 140 -> 145 at 2^25 values.
// The other kernels gain nothing.
template <class PT, class LT>
constexpr unsigned idle_lds() {
  return !__is_same(LT, None) ? 160 * 1024 / 5 : sizeof(PT) == 2 ? 160 * 1024 / 6 / 512 * 512 : 0;
}

template <class PT, class GT, class LT>
int adam_launch(int bits, const AdamArgs<LT>& a, int64_t chunks, hipStream_t stream) {
  const dim3 grid((unsigned)chunks);
  [[maybe_unused]] constexpr unsigned idle = idle_lds<PT, LT>();
  if (bits == (8 | MI_DITHERED)) hipLaunchKernelGGL((adamw8_kernel<PT, GT, LT, true>), grid, dim3(NT), 0, stream, a);
  else if (bits == 8) hipLaunchKernelGGL((adamw8_kernel<PT, GT, LT, false>), grid, dim3(NT), 0, stream, a);
  else hipLaunchKernelGGL((adamw_kernel<PT, GT, LT>), grid, dim3(NT), idle, stream, a);
  return launched("mi_adamw_update");
}
template <class PT, class LT>
int adam_launch_grad(int grad_dtype, int bits, const AdamArgs<LT>& a, int64_t chunks, hipStream_t stream) {
  if (grad_dtype == MI_DTYPE_F32) return adam_launch<PT, float, LT>(bits, a, chunks, stream);
  if constexpr (!__is_same(PT, _Float16) && !__is_same(LT, _Float16))
    if (grad_dtype == MI_DTYPE_BF16) return adam_launch<PT, __bf16, LT>(bits, a, chunks, stream);
  if constexpr (!__is_same(PT, __bf16) && !__is_same(LT, __bf16))
    if (grad_dtype == MI_DTYPE_F16) return adam_launch<PT, _Float16, LT>(bits, a, chunks, stream);
  return fail(MI_ERR_BAD_ARG, "mi_adamw_update: bfloat16 and float16 do not go together");
}

int adam_impl(int64_t count, void* const* param, const void* const* grad, void* const* exp_avg, void* const* exp_avg_sq,
              void* const* model_param, const float* const* step_dev, const int64_t* numel, int param_dtype, int grad_dtype, int model_dtype,
              int moment_bits, double step, double lr, const float* lr_dev, double beta1, double beta2, double eps, double weight_decay,
              int decay_method, const float* grad_scale, hipStream_t stream) {
  const char* who = "mi_adamw_update";
  if (int rc = check_numel(who, count, numel)) return rc;
  if (!known_dtype(param_dtype) || !known_dtype(grad_dtype)) return fail(MI_ERR_BAD_ARG, "%s: unknown data type", who);
  if (model_param && (param_dtype != MI_DTYPE_F32 || (model_dtype != MI_DTYPE_BF16 && model_dtype != MI_DTYPE_F16)))
    return fail(MI_ERR_BAD_ARG, "%s: 16-bit copies go with float32 weights only", who);
  const int mixed = model_param ? model_dtype : param_dtype;
  if (mixed != MI_DTYPE_F32 && grad_dtype != MI_DTYPE_F32 && grad_dtype != mixed)
    return fail(MI_ERR_BAD_ARG, "%s: bfloat16 and float16 do not go together", who);
  if (moment_bits != 32 && moment_bits != 8 && moment_bits != (8 | MI_DITHERED)) return fail(MI_ERR_BAD_ARG, "%s: moments have 32 or 8 bits, got %d", who, moment_bits);
  // (comparisons that NaN fails)
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return fail(MI_ERR_BAD_ARG, "%s: betas must be in [0, 1)", who);
  if (!(eps >= 0.0)) return fail(MI_ERR_BAD_ARG, "%s: eps must not be negative", who);
  if (!step_dev && !(step >= 1.0)) return fail(MI_ERR_BAD_ARG, "%s: step must be at least 1", who);
  if (decay_method < DECAY_DECOUPLED || decay_method > DECAY_PALM) return fail(MI_ERR_BAD_ARG, "%s: unknown weight decay method %d", who, decay_method);
  const bool bits8 = moment_bits != 32;
  const int pb = element_bytes(param_dtype), gb = element_bytes(grad_dtype);
  {
    Spans spans;
    spans.all.reserve((size_t)count * (model_param ? 5 : 4));
    if (int rc = add_spans(who, "param", spans, count, const_cast<const void* const*>(param), numel, pb, false, true)) return rc;
    if (int rc = add_spans(who, "grad", spans, count, grad, numel, gb, false, false)) return rc;
    if (int rc = add_spans(who, "exp_avg", spans, count, const_cast<const void* const*>(exp_avg), numel, 4, bits8, true)) return rc;
    if (int rc = add_spans(who, "exp_avg_sq", spans, count, const_cast<const void* const*>(exp_avg_sq), numel, 4, bits8, true)) return rc;
    if (model_param)
      if (int rc = add_spans(who, "model_param", spans, count, const_cast<const void* const*>(model_param), numel, 2, false, true)) return rc;
    if (step_dev)
      for (int64_t i = 0; i < count; ++i)
        if (!step_dev[i] || reinterpret_cast<uintptr_t>(step_dev[i]) % 4) return fail(MI_ERR_BAD_ARG, "%s: step %lld is null or not aligned", who, (long long)i);
    if (spans.conflict()) return fail(MI_ERR_BAD_ARG, "%s: a tensor that is written overlaps another one of the call", who);
  }
  AdamScalars s = {};
  s.b1 = (float)beta1;
  s.omb1 = (float)(1.0 - beta1);
  s.b2 = (float)beta2;
  s.omb2 = (float)(1.0 - beta2);
  s.eps = (float)eps;
  s.on_device = step_dev || lr_dev;
  s.method = decay_method;
  s.lr = lr;
  s.wd = weight_decay;
  s.ln_b1 = log(beta1);
  s.ln_b2 = log(beta2);
  s.step = step;
  s.lr_dev = lr_dev;
  s.grad_scale = grad_scale;
  decay_terms(decay_method, weight_decay, lr, &s.shrink, &s.l2);
  if (!step_dev) bias_terms(s.ln_b1, s.ln_b2, step, lr, &s.step_size, &s.inv_sqrt_bc2);
  const int64_t chunk = !bits8 ? ADAM_CHUNK : pb == 2 && gb == 2 ? Adam8Shape<__bf16, __bf16>::CHUNK : Adam8Shape<float, float>::CHUNK;
  const auto entry = [&](int64_t i) { return AdamTensor{param[i], grad[i], exp_avg[i], exp_avg_sq[i], step_dev ? step_dev[i] : nullptr, numel[i]}; };
  const auto before = [&](const AdamTensor& t) { return bits8 ? 0 : places_before(static_cast<float*>(t.m)); };
  const auto state_footprints = [&](const auto& l, int64_t chunks) {
    MI_OTHER_LAUNCH();
    MI_WALK(l, chunks, chunk, before);
    for (int i = 0; i < l.count; ++i) {
      [[maybe_unused]] const AdamTensor& t = l.t[i];
      [[maybe_unused]] const int64_t moment = bits8 ? (int64_t)mi_moment_8bit_bytes(t.n) : t.n;
      MI_FOOTPRINT("weights", t.p, pb, 1, 0, 1, t.n, t.n);
      MI_FOOTPRINT("gradient", t.g, gb, 1, 0, 1, t.n, t.n);
      MI_FOOTPRINT("first moment", t.m, bits8 ? 1 : 4, 1, 0, 1, moment, moment);
      MI_FOOTPRINT("second moment", t.v, bits8 ? 1 : 4, 1, 0, 1, moment, moment);
    }
  };
  if (model_param) {
    const auto run = [&](auto* a, auto launch) {
      a->s = s;
      return for_each_list(
          count, numel, chunk, a->list, [&](int64_t i) { return AdamTensorCopy{entry(i), model_param[i]}; }, before,
          [&](const auto& l, int64_t chunks) -> int {
            state_footprints(l, chunks);
            for (int i = 0; i < l.count; ++i) MI_FOOTPRINT("16-bit copy", l.t[i].low, 2, 1, 0, 1, l.t[i].n, l.t[i].n);
            return launch(*a, chunks);
          });
    };
    if (model_dtype == MI_DTYPE_BF16) {
      AdamArgs<__bf16> a;
      return run(&a, [&](const auto& x, int64_t chunks) { return adam_launch_grad<float, __bf16>(grad_dtype, moment_bits, x, chunks, stream); });
    }
    AdamArgs<_Float16> a;
    return run(&a, [&](const auto& x, int64_t chunks) { return adam_launch_grad<float, _Float16>(grad_dtype, moment_bits, x, chunks, stream); });
  }
  AdamArgs<None> a;
  a.s = s;
  return for_each_list(count, numel, chunk, a.list, entry, before, [&](const auto& l, int64_t chunks) -> int {
    state_footprints(l, chunks);
    if (param_dtype == MI_DTYPE_F32) return adam_launch_grad<float, None>(grad_dtype, moment_bits, a, chunks, stream);
    if (param_dtype == MI_DTYPE_BF16) return adam_launch_grad<__bf16, None>(grad_dtype, moment_bits, a, chunks, stream);
    return adam_launch_grad<_Float16, None>(grad_dtype, moment_bits, a, chunks, stream);
  });
}

// Runs of equal data types are served by one launch each (as far as the argument block goes).
template <class Body>
int for_each_type(int64_t count, const int* dtype, Body body) {
  for (int64_t i = 0; i < count;) {
    int64_t j = i + 1;
    while (j < count && dtype[j] == dtype[i]) ++j;
    if (int rc = body(i, j - i, dtype[i])) return rc;
    i = j;
  }
  return MI_OK;
}

// Chunks of a list at most, wherever its tensors begin.
int64_t norm_chunks(int64_t count, const int64_t* numel) {
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) chunks += numel[i] ? (numel[i] + 63 + NORM_CHUNK - 1) / NORM_CHUNK : 0;
  return chunks;
}

int check_list(const char* who, int64_t count, const void* const* x, const int64_t* numel, const int* dtype) {
  if (int rc = check_numel(who, count, numel)) return rc;
  if (count > 0 && (!x || !dtype)) return fail(MI_ERR_BAD_ARG, "%s: no list of tensors or data types", who);
  for (int64_t i = 0; i < count; ++i) {
    if (!known_dtype(dtype[i])) return fail(MI_ERR_BAD_ARG, "%s: tensor %lld has an unknown data type", who, (long long)i);
    if (numel[i] > 0 && (!x[i] || reinterpret_cast<uintptr_t>(x[i]) % element_bytes(dtype[i])))
      return fail(MI_ERR_BAD_ARG, "%s: tensor %lld is null or not aligned to its elements", who, (long long)i);
  }
  return MI_OK;
}

// Partial sums of squares of a list, *total of them.
int sumsq_impl(const char* who, int64_t count, const void* const* x, const int64_t* numel, const int* dtype, double max_norm, double* partials,
               size_t partials_len, float* out, int64_t* total, hipStream_t stream) {
  if (int rc = check_list(who, count, x, numel, dtype)) return rc;
  if (!out) return fail(MI_ERR_BAD_ARG, "%s: no output", who);
  if (!(max_norm >= 0.0)) return fail(MI_ERR_BAD_ARG, "%s: max_norm must not be negative", who);
  const int64_t most = norm_chunks(count, numel);
  if (most > 0 && (!partials || partials_len < (size_t)most))
    return fail(MI_ERR_WORKSPACE, "%s: %lld partial sums are needed", who, (long long)most);
  MI_FOOTPRINT("norm and factor", out, 4, 1, 0, 1, 2, 2);
  int64_t& done = *total;
  done = 0;
  ReadList l;
  return for_each_type(count, dtype, [&](int64_t at, int64_t len, int dt) {
    const auto run = [&](auto before, auto kernel) {
      return for_each_list(
          len, numel + at, NORM_CHUNK, l, [&](int64_t i) { return ReadTensor{x[at + i], numel[at + i]}; }, before,
          [&](const ReadList& list, int64_t chunks) -> int {
            MI_OTHER_LAUNCH();
            MI_WALK(list, chunks, NORM_CHUNK, before);
            MI_FOOTPRINT("partial sums", partials + done, 8, 1, 0, 1, chunks, chunks);
            for (int i = 0; i < list.count; ++i) MI_FOOTPRINT("tensor", list.t[i].x, element_bytes(dt), 1, 0, 1, list.t[i].n, list.t[i].n);
            hipLaunchKernelGGL(kernel, dim3((unsigned)chunks), dim3(NT), 0, stream, list, partials + done);
            done += chunks;
            return launched(who);
          });
    };
    if (dt == MI_DTYPE_F32) return run(at_line_of<float>, sumsq_list_kernel<float>);
    if (dt == MI_DTYPE_BF16) return run(at_line_of<__bf16>, sumsq_list_kernel<__bf16>);
    return run(at_line_of<_Float16>, sumsq_list_kernel<_Float16>);
  });
}

int finish_impl(const char* who, const double* partials, int64_t total, double max_norm, float* out, hipStream_t stream) {
  MI_OTHER_LAUNCH();
  if (total <= FEW_PARTIALS) hipLaunchKernelGGL(norm_finish_kernel<NT>, dim3(1), dim3(NT), 0, stream, partials, total, (float)max_norm, out);
  else hipLaunchKernelGGL(norm_finish_kernel<1024>, dim3(1), dim3(1024), 0, stream, partials, total, (float)max_norm, out);
  return launched(who);
}

int overlap_impl(const char* who, int64_t count, const void* const* x, const int64_t* numel, const int* dtype) {
  Spans spans;
  spans.all.reserve((size_t)count);
  for (int64_t i = 0; i < count; ++i) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(x[i]);
    if (numel[i] > 0) spans.all.push_back({lo, lo + (size_t)numel[i] * element_bytes(dtype[i])});
  }
  spans.close_role(true);
  return spans.conflict() ? fail(MI_ERR_BAD_ARG, "%s: two of the tensors overlap", who) : MI_OK;
}

template <bool FINISH>
int scale_launches(const char* who, int64_t count, void* const* x, const int64_t* numel, const int* dtype, const ScaleFactor& sf, hipStream_t stream) {
  ReadList l;
  return for_each_type(count, dtype, [&](int64_t at, int64_t len, int dt) {
    const auto run = [&](int64_t chunk, auto before, auto kernel) {
      return for_each_list(
          len, numel + at, chunk, l, [&](int64_t i) { return ReadTensor{x[at + i], numel[at + i]}; }, before,
          [&](const ReadList& list, int64_t chunks) -> int {
            MI_OTHER_LAUNCH();
            MI_WALK(list, chunks, chunk, before);
            for (int i = 0; i < list.count; ++i) MI_FOOTPRINT("tensor", list.t[i].x, element_bytes(dt), 1, 0, 1, list.t[i].n, list.t[i].n);
            hipLaunchKernelGGL(kernel, dim3((unsigned)chunks), dim3(NT), 0, stream, list, sf);
            return launched(who);
          });
    };
    if (dt == MI_DTYPE_F32) return run(ScaleShape<float>::CHUNK, at_line_of<float>, scale_list_kernel<float, FINISH>);
    if (dt == MI_DTYPE_BF16) return run(ScaleShape<__bf16>::CHUNK, at_line_of<__bf16>, scale_list_kernel<__bf16, FINISH>);
    return run(ScaleShape<_Float16>::CHUNK, at_line_of<_Float16>, scale_list_kernel<_Float16, FINISH>);
  });
}

int norm_impl(int64_t count, const void* const* x, const int64_t* numel, const int* dtype, double max_norm, double* partials, size_t partials_len,
              float* out, hipStream_t stream) {
  const char* who = "mi_global_norm";
  int64_t total = 0;
  if (int rc = sumsq_impl(who, count, x, numel, dtype, max_norm, partials, partials_len, out, &total, stream)) return rc;
  return finish_impl(who, partials, total, max_norm, out, stream);
}

int scale_impl(int64_t count, void* const* x, const int64_t* numel, const int* dtype, const float* factor, hipStream_t stream) {
  const char* who = "mi_scale_tensors";
  if (int rc = check_list(who, count, x, numel, dtype)) return rc;
  if (!factor) return fail(MI_ERR_BAD_ARG, "%s: no factor", who);
  if (int rc = overlap_impl(who, count, x, numel, dtype)) return rc;
  return scale_launches<false>(who, count, x, numel, dtype, ScaleFactor{factor, nullptr, 0, 0.0f, nullptr}, stream);
}

int clip_impl(int64_t count, void* const* x, const int64_t* numel, const int* dtype, double max_norm, double* partials, size_t partials_len, float* out,
              hipStream_t stream) {
  const char* who = "mi_clip_by_global_norm";
  if (int rc = check_list(who, count, x, numel, dtype)) return rc;
  if (int rc = overlap_impl(who, count, x, numel, dtype)) return rc;
  int64_t total = 0;
  if (int rc = sumsq_impl(who, count, x, numel, dtype, max_norm, partials, partials_len, out, &total, stream)) return rc;
  if (total > 0 && total <= FEW_PARTIALS)
    return scale_launches<true>(who, count, x, numel, dtype, ScaleFactor{nullptr, partials, total, (float)max_norm, out}, stream);
  if (int rc = finish_impl(who, partials, total, max_norm, out, stream)) return rc;
  return scale_launches<false>(who, count, x, numel, dtype, ScaleFactor{out + 1, nullptr, 0, 0.0f, nullptr}, stream);
}

template <class T>
int move_launch(bool pack, bool second, const MoveList& l, int64_t chunks, hipStream_t stream, const char* who) {
  const dim3 grid((unsigned)chunks), packing(MoveShape<T, true>::THREADS), unpacking(MoveShape<T, false>::THREADS);
  if (pack && !second) hipLaunchKernelGGL((pack8_kernel<T, true>), grid, packing, 0, stream, l);
  else if (pack) hipLaunchKernelGGL((pack8_kernel<T, false>), grid, packing, 0, stream, l);
  else if (!second) hipLaunchKernelGGL((unpack8_kernel<T, true>), grid, unpacking, 0, stream, l);
  else hipLaunchKernelGGL((unpack8_kernel<T, false>), grid, unpacking, 0, stream, l);
  return launched(who);
}

int move_impl(bool pack, int64_t count, const void* const* src, void* const* dst, const int64_t* numel, int dtype, int second, hipStream_t stream) {
  const char* who = pack ? "mi_moments_8bit_pack" : "mi_moments_8bit_unpack";
  if (int rc = check_numel(who, count, numel)) return rc;
  if (!known_dtype(dtype)) return fail(MI_ERR_BAD_ARG, "%s: unknown data type", who);
  if (second != 0 && second != 1) return fail(MI_ERR_BAD_ARG, "%s: the moment is 0 (first) or 1 (second), got %d", who, second);
  {
    Spans spans;
    spans.all.reserve((size_t)count * 2);
    if (int rc = add_spans(who, "source", spans, count, src, numel, element_bytes(dtype), !pack, false)) return rc;
    if (int rc = add_spans(who, "destination", spans, count, const_cast<const void* const*>(dst), numel, element_bytes(dtype), pack, true)) return rc;
    if (spans.conflict()) return fail(MI_ERR_BAD_ARG, "%s: a tensor that is written overlaps another one of the call", who);
  }
  const int64_t chunk = dtype == MI_DTYPE_F32 ? (pack ? MoveShape<float, true>::CHUNK : MoveShape<float, false>::CHUNK) : MoveShape<__bf16, true>::CHUNK;
  static_assert(MoveShape<__bf16, true>::CHUNK == MoveShape<__bf16, false>::CHUNK, "one chunk for both directions");
  MoveList l;
  return for_each_list(
      count, numel, chunk, l, [&](int64_t i) { return MoveTensor{src[i], dst[i], numel[i]}; }, at_tensor,
      [&](const MoveList& list, int64_t chunks) -> int {
        MI_OTHER_LAUNCH();
        MI_WALK(list, chunks, chunk, at_tensor);
        for (int i = 0; i < list.count; ++i) {
          [[maybe_unused]] const MoveTensor& t = list.t[i];
          [[maybe_unused]] const int64_t bytes8 = (int64_t)mi_moment_8bit_bytes(t.n);
          MI_FOOTPRINT("8-bit form", pack ? t.dst : t.src, 1, 1, 0, 1, bytes8, bytes8);
          MI_FOOTPRINT("values", pack ? t.src : t.dst, element_bytes(dtype), 1, 0, 1, t.n, t.n);
        }
        if (dtype == MI_DTYPE_F32) return move_launch<float>(pack, second != 0, list, chunks, stream, who);
        if (dtype == MI_DTYPE_BF16) return move_launch<__bf16>(pack, second != 0, list, chunks, stream, who);
        return move_launch<_Float16>(pack, second != 0, list, chunks, stream, who);
      });
}

// The checks above keep vectors; nothing may be thrown across the C boundary.
template <class Body>
int guarded(const char* who, Body body) {
  try {
    return body();
  } catch (const std::exception& e) {
    return fail(MI_ERR_BAD_ARG, "%s: %s", who, e.what());
  }
}

}  // namespace
}  // namespace mi

#pragma GCC visibility push(default)
extern "C" {

size_t mi_moment_8bit_bytes(int64_t numel) { return numel <= 0 ? 0 : (size_t)mi::blocks8(numel) * (mi::BLOCK8 + 4); }

int mi_adamw_update(int64_t count, void* const* param, const void* const* grad, void* const* exp_avg, void* const* exp_avg_sq,
                    void* const* model_param, const float* const* step_dev, const int64_t* numel, int param_dtype, int grad_dtype,
                    int model_dtype, int moment_bits, double step, double lr, const float* lr_dev, double beta1, double beta2, double eps,
                    double weight_decay, int decay_method, const float* grad_scale, void* stream) {
  return mi::guarded("mi_adamw_update", [&] {
    return mi::adam_impl(count, param, grad, exp_avg, exp_avg_sq, model_param, step_dev, numel, param_dtype, grad_dtype, model_dtype, moment_bits, step,
                         lr, lr_dev, beta1, beta2, eps, weight_decay, decay_method, grad_scale, static_cast<hipStream_t>(stream));
  });
}

size_t mi_global_norm_partials_len(int64_t count, const int64_t* numel) {
  return count <= 0 || !numel ? 0 : (size_t)mi::norm_chunks(count, numel);
}

int mi_global_norm(int64_t count, const void* const* x, const int64_t* numel, const int* dtype, double max_norm, double* partials,
                   size_t partials_len, float* out, void* stream) {
  return mi::norm_impl(count, x, numel, dtype, max_norm, partials, partials_len, out, static_cast<hipStream_t>(stream));
}

int mi_clip_by_global_norm(int64_t count, void* const* x, const int64_t* numel, const int* dtype, double max_norm, double* partials,
                           size_t partials_len, float* out, void* stream) {
  return mi::guarded("mi_clip_by_global_norm",
                     [&] { return mi::clip_impl(count, x, numel, dtype, max_norm, partials, partials_len, out, static_cast<hipStream_t>(stream)); });
}

int mi_scale_tensors(int64_t count, void* const* x, const int64_t* numel, const int* dtype, const float* factor, void* stream) {
  return mi::guarded("mi_scale_tensors", [&] { return mi::scale_impl(count, x, numel, dtype, factor, static_cast<hipStream_t>(stream)); });
}

int mi_moments_8bit_pack(int64_t count, const void* const* src, void* const* packed, const int64_t* numel, int dtype, int second_moment, void* stream) {
  return mi::guarded("mi_moments_8bit_pack",
                     [&] { return mi::move_impl(true, count, src, packed, numel, dtype, second_moment, static_cast<hipStream_t>(stream)); });
}

int mi_moments_8bit_unpack(int64_t count, const void* const* packed, void* const* dst, const int64_t* numel, int dtype, int second_moment, void* stream) {
  return mi::guarded("mi_moments_8bit_unpack",
                     [&] { return mi::move_impl(false, count, packed, dst, numel, dtype, second_moment, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
#pragma GCC visibility pop
