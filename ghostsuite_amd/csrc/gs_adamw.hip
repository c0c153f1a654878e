// One step of AdamW over many tensors at once, its averages held in 32 or in 8 bits.
//
// Per element, t the steps taken with this one:
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = (1 - lr decay) p - lr / (1 - b1^t) m / ((v / (1 - b2^t))^(1/2) + eps)
// in fp32, p rounded once to its type.  Bound by memory: every array is read once and written once
// (GPT-2-small's 124 M bf16 parameters: 560 us with averages in 32 bits, 4.9 TB/s; 261 in 8 bits, 4.8 TB/s,
// where the vector units take as long).  In 8 bits every product, sum, root and quotient is rounded as fp32
// rounds it: with contraction and the hardware's approximate root and reciprocal (255 us) an average is a unit
// off, about one chance in 10^6 falls the other way and an element is held an eighth away, and where it is
// its block's largest on the next step, so is the block's scale.  What few elements need is apart: roots of
// numbers near the ends of fp32, values below 2^-6 of their scale (gradients over seven decades within a block:
// 355 us, before 300) and ones that are not finite; so all of them within each element took 288 us.
// A launch takes many tensors (their addresses travel in its arguments); its workgroups take runs
// of CHUNK elements, a tensor's last one shorter, and find their tensor by its first run (runs of 8192
// elements were 4% slower than runs of 2048: more workgroups at work at once, above all where a launch has
// few).
//
// In 8 bits, 256 consecutive elements (a block) share a scale, the largest magnitude over 448, and
// each holds its value over the scale as a float of 4 exponent and 3 mantissa bits.  Held are m and
// the root of v: the root halves v's range in powers of two, so that an element 2^-17 of its block's
// largest root still counts.  A nearest rounding would keep an average where it is whenever one
// step moves it by less than half of an eighth: with b2 = 0.999 nearly always.  So the rounding
// goes up or down by chance, with the odds that keep m and the root right on average: t + u rounded
// down, u spread evenly over [0, 1) by a hash of the element's place, the step and the seed, the
// same on every run.  (v, the root's square, comes out high by the rounding's variance: at most the
// sixteenth of its drift, a few hundredths of it where gradients are noise.)  A root that is not
// zero never becomes zero, nor less than half of itself, but for one below 2^-63, whose square leaves fp32:
// where the gradient stops, m is not divided by eps alone.  p is formed from m and v before their
// rounding.  A value that is not finite is held as NaN and has no part in its block's scale; p is NaN from
// the next step on.

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gs_common.h"

namespace gs {
namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int NT = 256, BLOCK = GS_ADAMW_BLOCK, VE = 8;
constexpr int CHUNK = NT * VE;       // elements of a workgroup, eight to a thread
constexpr int MOST = 64;             // tensors of a launch (3.8 KB of arguments)
constexpr int64_t MOST_RUNS = 1 << 23;   // runs of a launch: 2^31 threads
constexpr float TOP = 448.f;
// Blocks whose largest magnitude is below are held as zeros: where a gradient stops, m falls by b1 a step
// until 448 over it is infinite, which zero times is not a number.
constexpr float LEAST = 0x1p-100f;

struct Tensors {
  gs_adamw_tensor t[MOST];
  int32_t first[MOST + 1];           // each tensor's first run
  int count;
};
struct Factors {
  float keep, b1, b2, rest1, rest2;  // 1 - lr decay, b1, b2, 1 - b1, 1 - b2
  float step, root, eps;             // lr / (1 - b1^t), (1 - b2^t)^(-1/2)
  uint32_t key;
};

// The tensor of a run, by halves; uniform over the workgroup.
__device__ __forceinline__ int tensor_of(const Tensors& a, int run) {
  int lo = 0, hi = a.count;          // first[lo] <= run < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.first[mid] <= run) lo = mid; else hi = mid;
  }
  return lo;
}

template <class E>
struct Eight {
  float v[VE];
  __device__ __forceinline__ void load(const E* p, bool vec, int64_t left) {
    if (vec && left >= VE) {
      union { uint4 u[sizeof(E) / 2]; E e[VE]; } w;
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(E) / 2); ++i)
        w.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
      for (int i = 0; i < VE; ++i) v[i] = to_f32<E>(w.e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) v[i] = i < left ? to_f32<E>(p[i]) : 0.f;
    }
  }
  __device__ __forceinline__ void store(E* p, bool vec, int64_t left) const {
    if (vec && left >= VE) {
      union { uint4 u[sizeof(E) / 2]; E e[VE]; } w;
#pragma unroll
      for (int i = 0; i < VE; ++i) w.e[i] = from_f32<E>(v[i]);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(E) / 2); ++i)
        reinterpret_cast<uint4*>(p)[i] = w.u[i];
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (i < left) p[i] = from_f32<E>(v[i]);
    }
  }
};

template <class E>
__global__ void __launch_bounds__(NT) adamw_kernel(Tensors a, Factors f) {
  const int k = tensor_of(a, blockIdx.x);
  const gs_adamw_tensor& t = a.t[k];
  const int64_t first = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.first[k]) * CHUNK;
  const bool vec = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g) |
                     reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v)) & 15) == 0;
  float* tm = static_cast<float*>(t.m);
  float* tv = static_cast<float*>(t.v);
  const int64_t i = first + threadIdx.x * VE, left = t.n - i;
  if (left <= 0) return;
  Eight<E> p, g;
  Eight<float> m, v;
  p.load(static_cast<const E*>(t.p) + i, vec, left);
  g.load(static_cast<const E*>(t.g) + i, vec, left);
  m.load(tm + i, vec, left);
  v.load(tv + i, vec, left);
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    m.v[e] = f.b1 * m.v[e] + f.rest1 * g.v[e];
    v.v[e] = f.b2 * v.v[e] + f.rest2 * (g.v[e] * g.v[e]);
    p.v[e] = f.keep * p.v[e] - f.step * m.v[e] / (sqrtf(v.v[e]) * f.root + f.eps);
  }
  p.store(static_cast<E*>(t.p) + i, vec, left);
  m.store(tm + i, vec, left);
  v.store(tv + i, vec, left);
}

// The largest of 32 lanes (half a wave holds a block), in each of them: by row shifts, zeros beyond a row's
// first lane, and the broadcast of a row's last one.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true)));
}
__device__ __forceinline__ uint32_t half_max(uint32_t v) {
  v = max_dpp<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8: lane 15 holds its row's
  v = max_dpp<0x112, 0xf>(v);
  v = max_dpp<0x114, 0xf>(v);
  v = max_dpp<0x118, 0xf>(v);
  v = max_dpp<0x142, 0xa>(v);   // row_bcast 15 into rows 1 and 3: lanes 31 and 63
  const uint32_t lo = __builtin_amdgcn_readlane(v, 31), hi = __builtin_amdgcn_readlane(v, 63);
  return threadIdx.x & 32 ? hi : lo;
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t INF_BITS = 0x7F800000u;

// a of [2^-6, 448] on the 8-bit values, up or down by the chance (u << 4) + 8 of 2^20: an integer addition
// to the 20 mantissa bits that are cut off, which is floor(a / step + (u + 1/2) / 2^16) step (the sum has
// no more than 24 bits).  So is zero, at zero.  An a that rounding has left a few units above 448 stays there:
// the chance is at most 2^20 - 8.
__device__ __forceinline__ float eighth(float a, uint32_t chance) {
  return __uint_as_float((__float_as_uint(a) + chance) & 0xFFF00000u);
}
// The same of any a: below 2^-6 the steps stay 2^-9, a may have bits below the chance's, and the sum is
// rounded to fp32 before its floor.
__device__ __forceinline__ float eighth_or_less(float a, uint32_t chance) {
  const float low = floorf(__fmaf_rn(a, 0x1p29f, static_cast<float>(chance)) * 0x1p-20f) * 0x1p-9f;
  return a < 0x1p-6f ? low : eighth(a, chance);
}
// The root of x, correctly rounded, for x of [2^-96, 2^96): from the hardware's inverse root, and what its
// product with x leaves of x.  (Every such x was compared with a float64 root's rounding.)
__device__ __forceinline__ float root_of(float x) {
  const float y = __builtin_amdgcn_rsqf(x), s = x * y;
  return __fmaf_rn(__fmaf_rn(-s, s, x), 0.5f * y, s);
}
constexpr uint32_t ROOT_FROM = 0x0F800000u, ROOT_TO = 0x6F7FFFFFu;   // 2^-96, the last below 2^96
// Four 8-bit values from their floats, which they hold exactly, and back.
__device__ __forceinline__ uint32_t pack8(const float* v) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true));
}
__device__ __forceinline__ void unpack8(uint32_t w, float* v) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 0);
  v[1] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 1);
  v[2] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 2);
  v[3] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(w), 3);
}
__device__ __forceinline__ void load8(const uint8_t* p, bool vec, int64_t left, float (&v)[VE]) {
  uint32_t w[2] = {0, 0};
  if (vec && left >= VE) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < left) w[i / 4] |= static_cast<uint32_t>(p[i]) << (8 * (i % 4));
  }
  unpack8(w[0], v);
  unpack8(w[1], v + 4);
}
__device__ __forceinline__ void store8(uint8_t* p, bool vec, int64_t left, const float (&v)[VE]) {
  const uint32_t w[2] = {pack8(v), pack8(v + 4)};
  if (vec && left >= VE) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (i < left) p[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
  }
}

template <class E>
__global__ void __launch_bounds__(NT) adamw8_kernel(Tensors a, Factors f) {
  // each product and sum rounded by itself, in the order written
#pragma clang fp contract(off)
  const int k = tensor_of(a, blockIdx.x);
  const gs_adamw_tensor& t = a.t[k];
  const int64_t first = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.first[k]) * CHUNK;
  const bool vec = ((reinterpret_cast<uintptr_t>(t.p) | reinterpret_cast<uintptr_t>(t.g)) & 15) == 0;
  uint8_t* tm = static_cast<uint8_t*>(t.m);
  uint8_t* tv = static_cast<uint8_t*>(t.v);
  const bool vec8 = ((reinterpret_cast<uintptr_t>(tm) | reinterpret_cast<uintptr_t>(tv)) & 7) == 0;
  const int64_t i = first + threadIdx.x * VE, left = t.n - i;
  const int64_t b = i / BLOCK;
  const bool live = b * BLOCK < t.n;   // the same for the 32 lanes of a block
  float sm = 0.f, sr = 0.f;
  if (live) sm = t.m_scale[b], sr = t.v_scale[b];
  Eight<E> p, g;
  float m[VE], r[VE];
  p.load(static_cast<const E*>(t.p) + i, vec, left);
  g.load(static_cast<const E*>(t.g) + i, vec, left);
  load8(tm + i, vec8, left, m);
  load8(tv + i, vec8, left, r);
  uint32_t beyond = 0, most = 0;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    m[e] = f.b1 * (m[e] * sm) + f.rest1 * g.v[e];
    const float old = r[e] * sr;
    r[e] = f.b2 * (old * old) + f.rest2 * (g.v[e] * g.v[e]);
    beyond = max(beyond, __float_as_uint(r[e]) - ROOT_FROM);
    most = max(most, __float_as_uint(r[e]));
  }
  if (beyond <= ROOT_TO - ROOT_FROM) {
#pragma unroll
    for (int e = 0; e < VE; ++e) r[e] = root_of(r[e]);
  } else if (most > 0) {   // zeros stay: rows of an embedding that no batch has had
#pragma unroll
    for (int e = 0; e < VE; ++e) r[e] = sqrtf(r[e]);
  }
  uint32_t top_m = 0, top_r = 0;   // magnitudes by their bits: larger than infinity's, a NaN
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    float by = r[e] * f.root + f.eps;   // NaN with the root
    if (f.eps == 0.f && by == 0.f) by = INFINITY;
    p.v[e] = f.keep * p.v[e] - f.step * m[e] / by;
    top_m = max(top_m, magnitude(m[e]));
    top_r = max(top_r, __float_as_uint(r[e]));   // not below zero
  }
  p.store(static_cast<E*>(t.p) + i, vec, left);
  const bool whole = max(top_m, top_r) < INF_BITS;   // all of them finite
  if (!whole) {
    top_m = top_r = 0;
    for (int e = 0; e < VE; ++e) {
      top_m = max(top_m, magnitude(m[e]) < INF_BITS ? magnitude(m[e]) : 0u);
      top_r = max(top_r, magnitude(r[e]) < INF_BITS ? magnitude(r[e]) : 0u);
    }
  }
  const float most_m = __uint_as_float(half_max(top_m)), most_r = __uint_as_float(half_max(top_r));
  const bool some_m = most_m >= LEAST, some_r = most_r >= LEAST;
  const float im = some_m ? 1.f / most_m * TOP : 0.f, ir = some_r ? 1.f / most_r * TOP : 0.f;
  float least_m = INFINITY, least_r = INFINITY;
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    least_m = fminf(least_m, fabsf(m[e]) * im);
    least_r = fminf(least_r, r[e] * ir);
  }
  const auto hold = [&](auto any_size, auto any_value) {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      uint32_t x = (static_cast<uint32_t>(i + e) + f.key) * 0x9E3779B9u;
      x = (x ^ (x >> 15)) * 0xBB67AE85u;
      x ^= x >> 13;
      const uint32_t um = ((x & 0xFFFFu) << 4) + 8u, ur = ((x >> 16) << 4) + 8u;
      const float am = fabsf(m[e]) * im, ar = r[e] * ir;
      float hm, hr;
      if constexpr (!decltype(any_size)::value) {
        hm = eighth(am, um), hr = eighth(ar, ur);
      } else {
        hm = eighth_or_less(am, um);
        hr = fmaxf(eighth_or_less(ar, ur), r[e] > 0.f && some_r ? 0x1p-9f : 0.f);
      }
      if constexpr (decltype(any_value)::value) {
        m[e] = magnitude(m[e]) < INF_BITS ? copysignf(hm, m[e]) : NAN;
        r[e] = magnitude(r[e]) < INF_BITS ? hr : NAN;
      } else {
        m[e] = copysignf(hm, m[e]), r[e] = hr;
      }
    }
  };
  if (!whole)
    hold(std::true_type{}, std::true_type{});
  else if ((some_m && least_m < 0x1p-6f) || (some_r && least_r < 0x1p-6f))
    hold(std::true_type{}, std::false_type{});
  else   // a block of zeros is one of these: a is zero all over
    hold(std::false_type{}, std::false_type{});
  store8(tm + i, vec8, left, m);
  store8(tv + i, vec8, left, r);
  if (live && (threadIdx.x & 31) == 0) {
    t.m_scale[b] = some_m ? most_m * (1.f / TOP) : 0.f;
    t.v_scale[b] = some_r ? most_r * (1.f / TOP) : 0.f;
  }
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_adamw(const gs_adamw_tensor* tensors, int64_t count, int dtype, int state_bits,
                        double lr, double beta1, double beta2, double eps, double weight_decay,
                        int64_t step, uint32_t seed, void* stream) {
  if (dtype != GS_DTYPE_BF16 && dtype != GS_DTYPE_F32)
    return fail(GS_ERR_DTYPE, "gs_adamw: dtype must be bf16 or fp32");
  if (count < 0 || (count > 0 && tensors == nullptr) || (state_bits != 8 && state_bits != 32) ||
      step < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
    return fail(GS_ERR_INVALID, "gs_adamw: invalid arguments");
  for (int64_t i = 0; i < count; ++i) {
    const gs_adamw_tensor& t = tensors[i];
    if (t.n < 0 || (t.n > 0 && (t.p == nullptr || t.g == nullptr || t.m == nullptr || t.v == nullptr ||
                                (state_bits == 8 && (t.m_scale == nullptr || t.v_scale == nullptr)))))
      return fail(GS_ERR_INVALID, "gs_adamw: invalid tensor");
    if (t.n > MOST_RUNS * CHUNK)
      return fail(GS_ERR_UNSUPPORTED, "gs_adamw: a tensor of more than 2^34 elements");
  }
  Factors f{};
  f.keep = static_cast<float>(1.0 - lr * weight_decay);
  f.b1 = static_cast<float>(beta1), f.b2 = static_cast<float>(beta2);
  f.rest1 = static_cast<float>(1.0 - beta1), f.rest2 = static_cast<float>(1.0 - beta2);
  f.step = static_cast<float>(lr / (1.0 - std::pow(beta1, static_cast<double>(step))));
  f.root = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step))));
  f.eps = static_cast<float>(eps);
  f.key = static_cast<uint32_t>(step) * 0x9E3779B9u + seed * 0x6A09E667u;
  hipStream_t s = static_cast<hipStream_t>(stream);
  Tensors a;
  bool launched = false;
  for (int64_t i = 0; i < count;) {
    a.count = 0;
    int64_t runs = 0;
    for (; i < count && a.count < MOST; ++i) {
      if (tensors[i].n == 0) continue;
      const int64_t more = cdiv(tensors[i].n, CHUNK);
      if (runs + more > MOST_RUNS && a.count > 0) break;
      a.t[a.count] = tensors[i];
      a.first[a.count++] = static_cast<int32_t>(runs);
      runs += more;
    }
    if (a.count == 0) break;
    launched = true;
    a.first[a.count] = static_cast<int32_t>(runs);
    const dim3 grid(static_cast<unsigned>(runs));
    if (state_bits == 32) {
      if (dtype == GS_DTYPE_BF16)
        hipLaunchKernelGGL(adamw_kernel<uint16_t>, grid, dim3(NT), 0, s, a, f);
      else
        hipLaunchKernelGGL(adamw_kernel<float>, grid, dim3(NT), 0, s, a, f);
    } else {
      if (dtype == GS_DTYPE_BF16)
        hipLaunchKernelGGL(adamw8_kernel<uint16_t>, grid, dim3(NT), 0, s, a, f);
      else
        hipLaunchKernelGGL(adamw8_kernel<float>, grid, dim3(NT), 0, s, a, f);
    }
  }
  return launched ? check_launch("gs_adamw") : GS_OK;
}
