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

#include <algorithm>

#include "gs_common.h"

namespace gs {
namespace {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int NT = 256;   // threads of a workgroup

struct NormArgs {
  const void *x, *res, *w;   // res null: no residual
  void *y, *h;               // h null without a residual
  const void *g, *gh;        // backward: gradients of y and h (null: zeros)
  void* dx;                  // null: not wanted
  float* dw;                 // [workgroups][F], null: not wanted
  int64_t rows, F;
  float eps;
};

// VE elements at row + f, zeros past F (only with VE = 1 can a piece be cut).
template <class E, int VE>
struct Piece {
  E e[VE];
  __device__ __forceinline__ void load(const E* p, bool in) {
    if constexpr (VE == 1) {
      e[0] = in ? *p : E(0);
    } else {
      static_assert(sizeof(E) * VE == 16, "16 bytes");
      const uint4 u = in ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
      __builtin_memcpy(e, &u, 16);
    }
  }
  __device__ __forceinline__ void store(E* p, bool in) const {
    if (!in) return;
    if constexpr (VE == 1) {
      *p = e[0];
    } else {
      uint4 u;
      __builtin_memcpy(&u, e, 16);
      *reinterpret_cast<uint4*>(p) = u;
    }
  }
};

// The sum over a group of LANES lanes (32, 64, or the workgroup's 256), in each of them.
template <int LANES>
__device__ __forceinline__ float group_sum(float v, float* red) {
  if constexpr (LANES == 32) return half_sum_dpp(v);
  if constexpr (LANES == 64) return wave_sum_dpp(v);
  const float s = wave_sum_dpp(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// LANES lanes to a row, PC pieces of VE elements a lane.
template <class E, int VE, int PC, int LANES>
__global__ void __launch_bounds__(NT) norm_forward_kernel(NormArgs a) {
  __shared__ float red[4];
  constexpr int GROUPS = NT / LANES;
  const int li = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + grp;
  const bool live = row < a.rows;   // the same for the whole group
  const int64_t at = (live ? row : 0) * a.F;
  float v[PC][VE];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < PC; ++k) {
    const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
    const bool in = live && f < a.F;
    Piece<E, VE> p, q;
    p.load(static_cast<const E*>(a.x) + at + f, in);
    if (a.res != nullptr) {
      q.load(static_cast<const E*>(a.res) + at + f, in);
#pragma unroll
      for (int i = 0; i < VE; ++i) p.e[i] = from_f32<E>(to_f32<E>(p.e[i]) + to_f32<E>(q.e[i]));
      p.store(static_cast<E*>(a.h) + at + f, in);
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      v[k][i] = to_f32<E>(p.e[i]);
      ss += v[k][i] * v[k][i];
    }
  }
  const float r = rsqrtf(group_sum<LANES>(ss, red) / static_cast<float>(a.F) + a.eps);
#pragma unroll
  for (int k = 0; k < PC; ++k) {
    const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
    const bool in = live && f < a.F;
    Piece<E, VE> w, y;
    w.load(static_cast<const E*>(a.w) + f, in);
#pragma unroll
    for (int i = 0; i < VE; ++i) y.e[i] = from_f32<E>(to_f32<E>(w.e[i]) * (v[k][i] * r));
    y.store(static_cast<E*>(a.y) + at + f, in);
  }
}

template <class E, int VE, int PC, int LANES>
__global__ void __launch_bounds__(NT) norm_backward_kernel(NormArgs a) {
  __shared__ float red[4];
  extern __shared__ float sums[];   // [groups - 1][F], with dw
  constexpr int GROUPS = NT / LANES;
  const int li = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  float dw[PC][VE];
#pragma unroll
  for (int k = 0; k < PC; ++k)
#pragma unroll
    for (int i = 0; i < VE; ++i) dw[k][i] = 0.f;
  const float inv = 1.f / static_cast<float>(a.F);
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  // every group of the workgroup makes the same number of turns: group_sum may be a barrier
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * GROUPS; base < a.rows; base += step) {
    const bool live = base + grp < a.rows;
    const int64_t at = (live ? base + grp : 0) * a.F;
    Piece<E, VE> h[PC], g[PC];
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      const bool in = live && f < a.F;
      h[k].load(static_cast<const E*>(a.x) + at + f, in);
      g[k].load(static_cast<const E*>(a.g) + at + f, in && a.g != nullptr);
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      Piece<E, VE> w;
      w.load(static_cast<const E*>(a.w) + f, f < a.F);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float u = to_f32<E>(h[k].e[i]);
        ss += u * u;
        dot += to_f32<E>(w.e[i]) * to_f32<E>(g[k].e[i]) * u;
      }
    }
    const float r = rsqrtf(group_sum<LANES>(ss, red) * inv + a.eps);
    const float mean = group_sum<LANES>(dot, red) * r * inv;   // of w g h r
#pragma unroll
    for (int k = 0; k < PC; ++k) {
      const int64_t f = static_cast<int64_t>(li + k * LANES) * VE;
      const bool in = live && f < a.F;
      Piece<E, VE> w, gh, o;
      w.load(static_cast<const E*>(a.w) + f, in);
      gh.load(static_cast<const E*>(a.gh) + at + f, in && a.gh != nullptr);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float n = to_f32<E>(h[k].e[i]) * r, gi = to_f32<E>(g[k].e[i]);
        dw[k][i] += gi * n;
        o.e[i] = from_f32<E>(r * (to_f32<E>(w.e[i]) * gi - n * mean) + to_f32<E>(gh.e[i]));
      }
      if (a.dx != nullptr) o.store(static_cast<E*>(a.dx) + at + f, in);
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
  __shared__ float red[4];
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

// dw[f] = the sum of n rows, rounded once.  64 features a workgroup, four threads to each.
template <class E>
__global__ void __launch_bounds__(NT) norm_dw_kernel(const float* part, int64_t n, int64_t F, E* dw) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t f = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float s0 = 0.f, s1 = 0.f;
  if (f < F) {
    int64_t i = g;
    for (; i + 4 < n; i += 8) {
      s0 += part[i * F + f];
      s1 += part[(i + 4) * F + f];
    }
    if (i < n) s0 += part[i * F + f];
  }
  red[g][lane] = s0 + s1;
  __syncthreads();
  if (g == 0 && f < F)
    dw[f] = from_f32<E>((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]));
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
    hipLaunchKernelGGL((norm_forward_kernel<E, VE, PC, LANES>),
                       dim3(static_cast<unsigned>(cdiv(a.rows, G))), dim3(NT), 0, s, a);
  } else {
    const size_t lds = a.dw != nullptr ? (G - 1) * a.F * sizeof(float) : 0;
    hipLaunchKernelGGL((norm_backward_kernel<E, VE, PC, LANES>),
                       dim3(static_cast<unsigned>(groups)), dim3(NT), lds, s, a);
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
  if (pieces <= 64) GS_NORM(2, 32);
  if (pieces <= 96) GS_NORM(3, 32);
  if (pieces <= 128) GS_NORM(2, 64);
  if (pieces <= 256) GS_NORM(4, 64);
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
    parts = std::min(cdiv(rows, NT / lanes), BACKWARD_GROUPS);
    if (bf16)
      pick<uint16_t>(&a, vec, true, parts, s, F);
    else
      pick<float>(&a, vec, true, parts, s, F);
  }
  if (dw != nullptr) {
    const dim3 grid(static_cast<unsigned>(cdiv(F, 64)));
    if (bf16)
      hipLaunchKernelGGL(norm_dw_kernel<uint16_t>, grid, dim3(NT), 0, s, part, parts, F,
                         static_cast<uint16_t*>(dw));
    else
      hipLaunchKernelGGL(norm_dw_kernel<float>, grid, dim3(NT), 0, s, part, parts, F,
                         static_cast<float*>(dw));
  }
  return check_launch("gs_rms_norm_grad");
}
