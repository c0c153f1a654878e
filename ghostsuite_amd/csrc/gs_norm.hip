// Root-mean-square norm of a residual stream, with the residual's addition.
//
// Per row of F features, w the weight:
//   h = x + residual, rounded to the rows' type (h = x without a residual)
//   y = w h r,  r = (mean h^2 + eps)^(-1/2)
// and backward, from the gradients g of y and gh of h:
//   dh = r (w g - h r mean(w g h r)) + gh,  dx = dresidual = dh,  dw = sum over rows of g h r
// Bound by memory: forward reads x and the residual once and writes y and h; backward reads h, g
// and gh once and writes dh.  A group of lanes holds its row in registers from the first read to
// the last write, so each row is read once; the weight's gradient stays in the lanes' registers
// over all rows of a workgroup, then adds up across its groups in LDS, and a second launch adds the
// workgroups' rows in a fixed order.  Sums and products are fp32, one rounding at each output.
// 16384 rows of 2048 bf16 features: forward 46 us, backward 44 and the weight gradient's sums 4, at 5.8 and
// 6.2 TB/s (a part of what backward reads is still in the last-level cache); eight rows of 768 2.6 us.

#include <algorithm>

#include "gs_common.h"

namespace gs {
namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int NT = 256;    // threads of a workgroup, forward
constexpr int NTB = 512;   // and backward: twice the rows in flight for as many rows of dw's parts

struct NormArgs {
  const void *x, *res, *w;   // res null: no residual
  void *y, *h;               // h null without a residual
  const void *g, *gh;        // backward: gradients of y and h (null: zeros)
  void* dx;                  // null: not wanted
  float* dw;                 // [workgroups][F], null: not wanted
  int64_t rows, F;
  float eps;
};

// VE elements as they lie in memory (16 bytes, or one), taken out where they are used: bf16 ones held
// apart take twice the registers, and half of the rows in flight.
template <class E, int VE>
struct Piece {
  static constexpr int WORDS = VE == 1 ? 1 : 4;
  uint32_t u[WORDS];
  __device__ __forceinline__ void load(const E* p, bool in) {
    if constexpr (VE == 1) {
      if constexpr (sizeof(E) == 2)
        u[0] = in ? static_cast<uint32_t>(*p) << 16 : 0u;
      else
        u[0] = in ? __float_as_uint(*p) : 0u;
    } else {
      static_assert(sizeof(E) * VE == 16, "16 bytes");
      const uint4 w = in ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
      u[0] = w.x, u[1] = w.y, u[2] = w.z, u[3] = w.w;
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (VE == 8) return __uint_as_float(i & 1 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16);
    return __uint_as_float(u[i]);
  }
  // The piece of these values, each rounded.
  __device__ __forceinline__ void set(const float (&v)[VE]) {
    if constexpr (VE == 8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        u[i] = __float_as_uint(sizeof(E) == 2 ? round_bf16(v[i]) : v[i]);
    }
  }
  __device__ __forceinline__ void store(E* p, bool in) const {
    if (!in) return;
    if constexpr (VE != 1)
      *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    else if constexpr (sizeof(E) == 2)
      *p = static_cast<E>(u[0] >> 16);
    else
      *p = __uint_as_float(u[0]);
  }
};

// The sums of two values over a group of LANES lanes (32, 64, or 256 of the workgroup), in each of them.
template <int LANES>
__device__ __forceinline__ float2 group_sums(float a, float b, float2* red) {
  if constexpr (LANES == 32) return make_float2(half_sum_dpp(a), half_sum_dpp(b));
  a = wave_sum_dpp(a), b = wave_sum_dpp(b);
  if constexpr (LANES == 64) return make_float2(a, b);
  const int wid = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[wid] = make_float2(a, b);
  __syncthreads();
  const float2* g = red + wid / 4 * 4;
  return make_float2((g[0].x + g[1].x) + (g[2].x + g[3].x), (g[0].y + g[1].y) + (g[2].y + g[3].y));
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v, float2* red) {
  return group_sums<LANES>(v, 0.f, red).x;
}

// LANES lanes to a row, PC pieces of VE elements a lane.
template <class E, int VE, int PC, int LANES>
__global__ void __launch_bounds__(NT) norm_forward_kernel(NormArgs a) {
  __shared__ float2 red[4];
  constexpr int GROUPS = NT / LANES;
  const int li = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + grp;
  const bool live = row < a.rows;   // the same for the whole group
  const int64_t at = (live ? row : 0) * a.F;
  Piece<E, VE> h[PC];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < PC; ++k) {
    const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
    h[k].load(static_cast<const E*>(a.x) + at + f, live && f < a.F);
  }
  if (a.res != nullptr) {
    Piece<E, VE> q[PC];
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      q[k].load(static_cast<const E*>(a.res) + at + f, live && f < a.F);
    }
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      float v[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) v[i] = h[k].get(i) + q[k].get(i);
      h[k].set(v);
      h[k].store(static_cast<E*>(a.h) + at + f, live && f < a.F);
    }
  }
#pragma unroll
  for (int k = 0; k < PC; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) ss += h[k].get(i) * h[k].get(i);
  const float r = rsqrtf(group_sum<LANES>(ss, red) / static_cast<float>(a.F) + a.eps);
#pragma unroll
  for (int k = 0; k < PC; ++k) {
    const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
    const bool in = live && f < a.F;
    Piece<E, VE> w, y;
    w.load(static_cast<const E*>(a.w) + f, in);
    float v[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = w.get(i) * (h[k].get(i) * r);
    y.set(v);
    y.store(static_cast<E*>(a.y) + at + f, in);
  }
}

template <class E, int VE, int PC, int LANES>
__global__ void __launch_bounds__(NTB) norm_backward_kernel(NormArgs a) {
  __shared__ float2 red[NTB / 64];
  extern __shared__ float sums[];   // [groups - 1][F], with dw
  constexpr int GROUPS = NTB / LANES;
  const int li = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  float dw[PC][VE];
  Piece<E, VE> w[PC];
#pragma unroll
  for (int k = 0; k < PC; ++k) {
    const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
    w[k].load(static_cast<const E*>(a.w) + f, f < a.F);
#pragma unroll
    for (int i = 0; i < VE; ++i) dw[k][i] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(a.F);
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  // every group of the workgroup makes the same number of turns: group_sums may be a barrier
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * GROUPS; base < a.rows; base += step) {
    const bool live = base + grp < a.rows;
    const int64_t at = (live ? base + grp : 0) * a.F;
    Piece<E, VE> h[PC], g[PC], gh[PC];
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      const bool in = live && f < a.F;
      h[k].load(static_cast<const E*>(a.x) + at + f, in);
      g[k].load(static_cast<const E*>(a.g) + at + f, in && a.g != nullptr);
      gh[k].load(static_cast<const E*>(a.gh) + at + f, in && a.gh != nullptr);
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < PC; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float u = h[k].get(i);
        ss += u * u;
        dot += w[k].get(i) * g[k].get(i) * u;
      }
    const float2 s = group_sums<LANES>(ss, dot, red);
    const float r = rsqrtf(s.x * inv + a.eps);
    const float mean = s.y * r * inv;   // of w g h r
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      Piece<E, VE> o;
      float v[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float n = h[k].get(i) * r, gi = g[k].get(i);
        dw[k][i] += gi * n;
        v[i] = r * (w[k].get(i) * gi - n * mean) + gh[k].get(i);
      }
      o.set(v);
      if (a.dx != nullptr) o.store(static_cast<E*>(a.dx) + at + f, live && f < a.F);
    }
  }
  if (a.dw == nullptr) return;
  if (grp > 0) {
#pragma unroll
    for (int k = 0; k < PC; ++k)
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int64_t f = static_cast<int64_t>(li + k * LANES) * VE + i;
        if (f < a.F) sums[(grp - 1) * a.F + f] = dw[k][i];
      }
  }
  __syncthreads();
  if (grp > 0) return;
#pragma unroll
  for (int k = 0; k < PC; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE + i;
      if (f >= a.F) continue;
      float s = dw[k][i];
#pragma unroll
      for (int q = 0; q < GROUPS - 1; ++q) s += sums[q * a.F + f];
      a.dw[static_cast<int64_t>(blockIdx.x) * a.F + f] = s;
    }
}

// Rows of more features than a workgroup's registers hold: read again from the caches.
template <class E, bool BACKWARD>
__global__ void __launch_bounds__(NT) norm_wide_kernel(NormArgs a) {
  __shared__ float2 red[4];
  const float inv = 1.f / static_cast<float>(a.F);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * a.F;
    const E* x = static_cast<const E*>(a.x) + at;
    const E* w = static_cast<const E*>(a.w);
    const E* g = a.g != nullptr ? static_cast<const E*>(a.g) + at : nullptr;
    float ss = 0.f, dot = 0.f;
    for (int64_t f = threadIdx.x; f < a.F; f += NT) {
      float u = to_f32<E>(x[f]);
      if constexpr (!BACKWARD) {
        if (a.res != nullptr) {
          const E s = from_f32<E>(u + to_f32<E>(static_cast<const E*>(a.res)[at + f]));
          static_cast<E*>(a.h)[at + f] = s;
          u = to_f32<E>(s);
        }
      } else if (g != nullptr) {
        dot += to_f32<E>(w[f]) * to_f32<E>(g[f]) * u;
      }
      ss += u * u;
    }
    const float r = rsqrtf(group_sum<NT>(ss, red) * inv + a.eps);
    if constexpr (!BACKWARD) {
      const E* h = a.res != nullptr ? static_cast<const E*>(a.h) + at : x;   // a thread's own stores
      for (int64_t f = threadIdx.x; f < a.F; f += NT)
        static_cast<E*>(a.y)[at + f] = from_f32<E>(to_f32<E>(w[f]) * (to_f32<E>(h[f]) * r));
    } else {
      const float mean = group_sum<NT>(dot, red) * r * inv;
      if (a.dx != nullptr)
        for (int64_t f = threadIdx.x; f < a.F; f += NT) {
          const float gi = g != nullptr ? to_f32<E>(g[f]) : 0.f;
          const float gh = a.gh != nullptr ? to_f32<E>(static_cast<const E*>(a.gh)[at + f]) : 0.f;
          static_cast<E*>(a.dx)[at + f] =
              from_f32<E>(r * (to_f32<E>(w[f]) * gi - to_f32<E>(x[f]) * r * mean) + gh);
        }
      if (a.dw != nullptr && threadIdx.x == 0) a.dw[row] = r;   // for norm_wide_dw_kernel
    }
  }
}
// Its weight gradient, from the rows' r: workgroup (f, c) sums a share of the rows.
template <class E>
__global__ void __launch_bounds__(NT) norm_wide_dw_kernel(NormArgs a, const float* r, float* part,
                                                          int64_t per) {
  const int64_t f = static_cast<int64_t>(blockIdx.x) * NT + threadIdx.x, c = blockIdx.y;
  if (f >= a.F) return;
  const int64_t r1 = std::min<int64_t>(a.rows, (c + 1) * per);
  float s = 0.f;
#pragma unroll 4
  for (int64_t row = c * per; row < r1; ++row)
    s += to_f32<E>(static_cast<const E*>(a.g)[row * a.F + f]) *
         (to_f32<E>(static_cast<const E*>(a.x)[row * a.F + f]) * r[row]);
  part[c * a.F + f] = s;
}

// dw[f] = the sum of n rows, rounded once.  64 features a workgroup, sixteen waves to them: 512 rows of
// 2048 features, 4 MB, are 21 us with four.
constexpr int DW_WAVES = 16;
template <class E>
__global__ void __launch_bounds__(64 * DW_WAVES) norm_dw_kernel(const float* part, int64_t n, int64_t F,
                                                                E* dw) {
  __shared__ float red[DW_WAVES][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t f = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (f < F) {
    int64_t i = g;
    for (; i + 3 * DW_WAVES < n; i += 4 * DW_WAVES)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += part[(i + u * DW_WAVES) * F + f];
    for (; i < n; i += DW_WAVES) s[0] += part[i * F + f];
  }
  red[g][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (g != 0 || f >= F) return;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < DW_WAVES; ++k) t += red[k][lane];
  dw[f] = from_f32<E>(t);
}

// ------------------------------------------------------------------------------ host side

constexpr int64_t WIDE_F = 8192;          // features of a row from here on: norm_wide_kernel
constexpr int64_t BACKWARD_GROUPS = 512;  // workgroups of a backward pass, each a row of dw's parts
constexpr int64_t WIDE_SHARES = 64;

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
  return true;
}

template <class E, int VE, int PC, int LANES>
void launch(const NormArgs& a, bool backward, int64_t groups, hipStream_t s) {
  constexpr int G = NT / LANES;
  if (!backward) {
    // at most 2^30 threads to a launch
    constexpr int64_t MOST = int64_t{G} << 22;
    for (int64_t at = 0; at < a.rows; at += MOST) {
      NormArgs b = a;
      const int64_t by = at * a.F;
      b.rows = std::min(a.rows - at, MOST);
      b.x = static_cast<const E*>(a.x) + by, b.y = static_cast<E*>(a.y) + by;
      if (a.res != nullptr) b.res = static_cast<const E*>(a.res) + by, b.h = static_cast<E*>(a.h) + by;
      hipLaunchKernelGGL((norm_forward_kernel<E, VE, PC, LANES>),
                         dim3(static_cast<unsigned>(cdiv(b.rows, G))), dim3(NT), 0, s, b);
    }
  } else {
    const size_t lds = a.dw != nullptr ? (NTB / LANES - 1) * a.F * sizeof(float) : 0;
    hipLaunchKernelGGL((norm_backward_kernel<E, VE, PC, LANES>),
                       dim3(static_cast<unsigned>(groups)), dim3(NTB), lds, s, a);
  }
}

// Lanes to a row so that each holds few pieces: half a wave, a wave, or the workgroup.  `lanes`
// answers which.
template <class E, int VE>
int rows_kernel(const NormArgs* a, bool backward, int64_t groups, hipStream_t s, int64_t F) {
  const int64_t pieces = cdiv(F, VE);
#define GS_NORM(PC, LANES)                                  \
  do {                                                      \
    if (a != nullptr) launch<E, VE, PC, LANES>(*a, backward, groups, s); \
    return LANES;                                           \
  } while (0)
  if (pieces <= 32) GS_NORM(1, 32);
  if (pieces <= 64) GS_NORM(1, 64);
  if (pieces <= 128) GS_NORM(2, 64);
  if (pieces <= 256) GS_NORM(1, 256);
  if (pieces <= 512) GS_NORM(2, 256);
  if (pieces <= 1024) GS_NORM(4, 256);
  if constexpr (VE != 8) {
    if (pieces <= 2048) GS_NORM(8, 256);
  }
  if constexpr (VE == 1) {
    if (pieces <= 4096) GS_NORM(16, 256);
    GS_NORM(32, 256);
  }
#undef GS_NORM
  return 0;
}

template <class E>
int pick(const NormArgs* a, bool vec, bool backward, int64_t groups, hipStream_t s, int64_t F) {
  if (vec) return rows_kernel<E, 16 / sizeof(E)>(a, backward, groups, s, F);
  return rows_kernel<E, 1>(a, backward, groups, s, F);
}

int check_shape(int dtype, int64_t rows, int64_t F, const char* what) {
  if (dtype != GS_DTYPE_BF16 && dtype != GS_DTYPE_F32)
    return fail(GS_ERR_DTYPE, std::string(what) + ": dtype must be bf16 or fp32");
  if (rows <= 0 || F <= 0) return fail(GS_ERR_INVALID, std::string(what) + ": invalid arguments");
  if (rows > (int64_t{1} << 40) / F || rows > INT32_MAX)
    return fail(GS_ERR_UNSUPPORTED, std::string(what) + ": more than 2^31 rows or 2^40 elements");
  return GS_OK;
}

bool whole_pieces(int dtype, int64_t F) { return F * static_cast<int64_t>(elem_size(dtype)) % 16 == 0; }

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_rms_norm(const void* x, const void* residual, const void* weight, int dtype,
                           int64_t rows, int64_t F, float eps, void* y, void* h, void* stream) {
  if (const int rc = check_shape(dtype, rows, F, "gs_rms_norm")) return rc;
  if (x == nullptr || weight == nullptr || y == nullptr || (residual != nullptr) != (h != nullptr))
    return fail(GS_ERR_INVALID, "gs_rms_norm: invalid arguments");
  hipStream_t s = static_cast<hipStream_t>(stream);
  NormArgs a{};
  a.x = x, a.res = residual, a.w = weight, a.y = y, a.h = h, a.rows = rows, a.F = F, a.eps = eps;
  if (F > WIDE_F) {
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, 65536)));
    if (dtype == GS_DTYPE_BF16)
      hipLaunchKernelGGL((norm_wide_kernel<uint16_t, false>), grid, dim3(NT), 0, s, a);
    else
      hipLaunchKernelGGL((norm_wide_kernel<float, false>), grid, dim3(NT), 0, s, a);
    return check_launch("gs_rms_norm");
  }
  const bool vec = whole_pieces(dtype, F) && aligned16({x, residual, weight, y, h});
  if (dtype == GS_DTYPE_BF16)
    pick<uint16_t>(&a, vec, false, 0, s, F);
  else
    pick<float>(&a, vec, false, 0, s, F);
  return check_launch("gs_rms_norm");
}

extern "C" size_t gs_rms_norm_grad_workspace(int64_t rows, int64_t F) {
  if (rows <= 0 || F <= 0) return 0;
  Sizer z;
  if (F > WIDE_F) z.take<float>(rows);
  z.take<float>((F > WIDE_F ? WIDE_SHARES : BACKWARD_GROUPS) * F);
  return z.used + 256;
}

extern "C" int gs_rms_norm_grad(const void* h, const void* weight, const void* gy, const void* gh,
                                int dtype, int64_t rows, int64_t F, float eps, void* dx, void* dw,
                                void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_shape(dtype, rows, F, "gs_rms_norm_grad")) return rc;
  if (h == nullptr || weight == nullptr)
    return fail(GS_ERR_INVALID, "gs_rms_norm_grad: invalid arguments");
  if (dx == nullptr && dw == nullptr) return GS_OK;
  NormArgs a{};
  a.x = h, a.w = weight, a.g = gy, a.gh = gh, a.dx = dx, a.rows = rows, a.F = F, a.eps = eps;
  float *part = nullptr, *r = nullptr;
  if (dw != nullptr) {
    Carver c(workspace, workspace_bytes);
    if (F > WIDE_F) r = c.take<float>(rows);
    part = c.take<float>((F > WIDE_F ? WIDE_SHARES : BACKWARD_GROUPS) * F);
    if (workspace == nullptr || !c.ok())
      return fail(GS_ERR_WORKSPACE, "gs_rms_norm_grad: workspace too small");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == GS_DTYPE_BF16;
  int64_t parts;
  if (F > WIDE_F) {
    a.dw = gy != nullptr ? r : nullptr;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, 65536)));
    if (bf16)
      hipLaunchKernelGGL((norm_wide_kernel<uint16_t, true>), grid, dim3(NT), 0, s, a);
    else
      hipLaunchKernelGGL((norm_wide_kernel<float, true>), grid, dim3(NT), 0, s, a);
    parts = gy != nullptr ? std::min(rows, WIDE_SHARES) : 0;
    if (parts > 0 && dw != nullptr) {
      const int64_t per = cdiv(rows, parts);
      parts = cdiv(rows, per);
      const dim3 g2(static_cast<unsigned>(cdiv(F, NT)), static_cast<unsigned>(parts));
      if (bf16)
        hipLaunchKernelGGL(norm_wide_dw_kernel<uint16_t>, g2, dim3(NT), 0, s, a, r, part, per);
      else
        hipLaunchKernelGGL(norm_wide_dw_kernel<float>, g2, dim3(NT), 0, s, a, r, part, per);
    }
  } else {
    a.dw = part;
    const bool vec = whole_pieces(dtype, F) && aligned16({h, weight, gy, gh, dx});
    const int lanes = bf16 ? pick<uint16_t>(nullptr, vec, true, 0, s, F)
                           : pick<float>(nullptr, vec, true, 0, s, F);
    parts = std::min(cdiv(rows, NTB / lanes), BACKWARD_GROUPS);
    if (bf16)
      pick<uint16_t>(&a, vec, true, parts, s, F);
    else
      pick<float>(&a, vec, true, parts, s, F);
  }
  if (dw != nullptr) {
    const dim3 grid(static_cast<unsigned>(cdiv(F, 64)));
    if (bf16)
      hipLaunchKernelGGL(norm_dw_kernel<uint16_t>, grid, dim3(64 * DW_WAVES), 0, s, part, parts, F,
                         static_cast<uint16_t*>(dw));
    else
      hipLaunchKernelGGL(norm_dw_kernel<float>, grid, dim3(64 * DW_WAVES), 0, s, part, parts, F,
                         static_cast<float*>(dw));
  }
  return check_launch("gs_rms_norm_grad");
}
