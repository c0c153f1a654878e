// Loss of a student's logits against a teacher's top logits and the labels, with its gradient,
// gfx950.  Per row z (V logits), teacher entries (id_k, t_k) and label y, with tau the temperature:
//
//   p = softmax(t / tau)   q = softmax(z / tau)   s = softmax(z)
//   loss = alpha tau^2 sum_k p_k (log p_k - log q[id_k]) + (1 - alpha) (log sum exp z - z_y)
//   dz   = w (alpha tau (q - P) + (1 - alpha) (s - 1_y)),   P the p_k at their ids
//
// A workgroup owns a row.  The row is read once, in 16-byte pieces that stay in registers as they
// came: the maximum, then both sums of exponentials, then the gradient are formed from them, so a
// training step's loss and gradient cost one read and one write of the logits, and the rate of a
// copy bounds them.  Rows too long for the registers are read again in the second sweep (running
// maximum and sums in the first).  The gradient is written for the whole row as if no entry stood
// there; after a barrier the K entries and the label are written again with their masses taken off,
// from the logits themselves, so each element is rounded once.
//
// Sums, maxima and exponentials are fp32; a thread adds its own pieces, a wave its threads and the
// workgroup its waves, in a fixed order (the same bits on every run).
#include <algorithm>
#include <cmath>

#include "gs_common.h"

namespace gs {
namespace {

constexpr int DS_MAX_K = 1024;
constexpr int DS_COUNT_THREADS = 1024;

struct DsArgs {
  const void* z;
  int64_t N, inner, s_outer, s_inner;
  int V, K;
  const int64_t* ids;
  const void* t;
  int t_bf16;
  const int64_t* labels;
  int64_t ignore;
  float tau, alpha, inv_tau;
  int mean;                // divide by the rows not ignored
  int per_row;             // upstream is [N]
  const float* count;      // the number of rows not ignored (labels, mean), or null: N
  float* rows;             // [N] row losses, or null
  void* grad;              // or null
  const float* upstream;   // or null
  int filled;
};

// 16 bytes of a row as they lie in memory; element i is unpacked where it is used.
template <class E>
__device__ __forceinline__ float ds_elem(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(E) == 4) return __uint_as_float(w[i]);
  return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}
template <class E, class F>
__device__ __forceinline__ uint4 ds_map(const uint4& v, F f) {
  if constexpr (sizeof(E) == 4)
    return make_uint4(__float_as_uint(f(ds_elem<E>(v, 0))), __float_as_uint(f(ds_elem<E>(v, 1))),
                      __float_as_uint(f(ds_elem<E>(v, 2))), __float_as_uint(f(ds_elem<E>(v, 3))));
  else
    return make_uint4(pack_bf16x2(f(ds_elem<E>(v, 0)), f(ds_elem<E>(v, 1))),
                      pack_bf16x2(f(ds_elem<E>(v, 2)), f(ds_elem<E>(v, 3))),
                      pack_bf16x2(f(ds_elem<E>(v, 4)), f(ds_elem<E>(v, 5))),
                      pack_bf16x2(f(ds_elem<E>(v, 6)), f(ds_elem<E>(v, 7))));
}
// Keeps the compiler from carrying the unpacked elements of one sweep to the next: twice the
// registers for bf16, and spills.
__device__ __forceinline__ void ds_packed(uint4& v) {
  asm("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
}

// Maximum / sums over the workgroup, for three values at once (max for the first two of `max3`,
// sum for all of `sum3`).
template <int WAVES>
__device__ __forceinline__ void block_max2(float& a, float& b, float (*red)[4]) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    a = fmaxf(a, __shfl_xor(a, k, 64));
    b = fmaxf(b, __shfl_xor(b, k, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = a;
    red[threadIdx.x >> 6][1] = b;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    a = fmaxf(a, red[w][0]);
    b = fmaxf(b, red[w][1]);
  }
}
template <int WAVES>
__device__ __forceinline__ void block_sum3(float& a, float& b, float& c, float (*red)[4]) {
  a = wave_sum(a);
  b = wave_sum(b);
  c = wave_sum(c);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = a;
    red[threadIdx.x >> 6][1] = b;
    red[threadIdx.x >> 6][2] = c;
  }
  __syncthreads();
  a = b = c = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    a += red[w][0];
    b += red[w][1];
    c += red[w][2];
  }
}

// exp(x / tau) for x <= 0, `k` = log2(e) / tau.
__device__ __forceinline__ float ds_exp(float x, float k) { return __builtin_amdgcn_exp2f(x * k); }

constexpr float DS_LOG2E = 1.44269504088896340736f;

// NP: pieces a thread keeps (0: none are kept, the row is read twice).  TWO: the two softmaxes
// differ and both count.
template <class E, int THREADS, int NP, bool TWO>
__global__ void __launch_bounds__(THREADS) distill_kernel(DsArgs a) {
  constexpr int VE = 16 / sizeof(E);
  constexpr int WAVES = THREADS / 64;
  __shared__ float red[WAVES][4];
  extern __shared__ char dyn[];
  // Per entry (the label last): its id (-1: none), and its mass in the gradient.
  int* const e_id = reinterpret_cast<int*>(dyn);
  float* const e_mass = reinterpret_cast<float*>(dyn) + a.K + 1;
  const float NEG_INF = -__builtin_inff();
  const int tid = threadIdx.x;
  const float kq = DS_LOG2E * a.inv_tau;

  if (a.filled && !a.per_row && a.upstream[0] == 1.f) return;   // nothing to change

  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    const int64_t at = a.inner == a.N ? n * a.s_inner
                                      : n / a.inner * a.s_outer + n % a.inner * a.s_inner;
    const E* z = static_cast<const E*>(a.z) + at;
    E* dz = static_cast<E*>(a.grad) + at;
    const int64_t y = a.labels != nullptr ? a.labels[n] : 0;
    const bool ignored = a.labels != nullptr && y == a.ignore;
    // The row from its first 16-byte boundary in whole pieces; `head` and `tail` single elements
    // around them belong to the first threads of the first two waves.
    const int head = min(a.V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) /
                                  static_cast<int>(sizeof(E)));
    const int pieces = (a.V - head) / VE, tail0 = head + pieces * VE;
    const int single = tid < head ? tid
                       : tid >= 64 && tid - 64 < a.V - tail0 ? tail0 + tid - 64 : -1;
    if (ignored) {
      if (a.rows != nullptr && tid == 0) a.rows[n] = 0.f;
      if (a.grad != nullptr) {
        for (int p = tid; p < pieces; p += THREADS)
          reinterpret_cast<uint4*>(dz + head)[p] = make_uint4(0u, 0u, 0u, 0u);
        if (single >= 0) dz[single] = from_f32<E>(0.f);
      }
      continue;
    }
    const uint4* zp = reinterpret_cast<const uint4*>(z + head);

    // ---- the row and the teacher's entries
    uint4 x[NP > 0 ? NP : 1];
    float m = NEG_INF, sq = 0.f, s1 = 0.f;
    if constexpr (NP > 0) {
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (k * THREADS + tid < pieces) x[k] = zp[k * THREADS + tid];
    }
    const float xs = single >= 0 ? to_f32<E>(z[single]) : NEG_INF;
    float tm = NEG_INF;
    for (int k = tid; k < a.K; k += THREADS) {
      const int64_t id = a.ids[n * a.K + k];
      const bool use = id >= 0 && id < a.V;
      const float t = !use ? NEG_INF
                      : a.t_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.t)[n * a.K + k])
                                 : static_cast<const float*>(a.t)[n * a.K + k];
      e_id[k] = use ? static_cast<int>(id) : -1;
      e_mass[k] = t;
      tm = t != t ? t : fmaxf(tm, t);
    }
    if constexpr (NP > 0) {
      m = xs;
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (k * THREADS + tid < pieces) {
#pragma unroll
          for (int e = 0; e < VE; ++e) m = fmaxf(m, ds_elem<E>(x[k], e));
        }
    } else {
      // running maximum and sums of this thread
      m = xs;
      sq = xs == NEG_INF ? 0.f : 1.f;
      s1 = sq;
      for (int p = tid; p < pieces; p += THREADS) {
        const uint4 v = zp[p];
        float pm = m;
#pragma unroll
        for (int e = 0; e < VE; ++e) pm = fmaxf(pm, ds_elem<E>(v, e));
        if (pm == NEG_INF) {   // nothing yet (a NaN among them is seen by the sums)
          pm = 0.f;
        }
        const float d = m == NEG_INF ? 0.f : m - pm;
        sq *= ds_exp(d, kq);
        if (TWO) s1 *= ds_exp(d, DS_LOG2E);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float w = ds_elem<E>(v, e) - pm;
          sq += ds_exp(w, kq);
          if (TWO) s1 += ds_exp(w, DS_LOG2E);
        }
        m = pm;
      }
    }
    const float m_own = m;
    if constexpr (NP > 0) {
#pragma unroll
      for (int k = 0; k < NP; ++k) ds_packed(x[k]);
    }
    block_max2<WAVES>(m, tm, red);

    // ---- sums of exponentials
    if constexpr (NP > 0) {
      if (single >= 0) {
        sq = ds_exp(xs - m, kq);
        if (TWO) s1 = ds_exp(xs - m, DS_LOG2E);
      }
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (k * THREADS + tid < pieces) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float w = ds_elem<E>(x[k], e) - m;
            sq += ds_exp(w, kq);
            if (TWO) s1 += ds_exp(w, DS_LOG2E);
          }
        }
    } else {
      const float d = m_own == NEG_INF ? 0.f : m_own - m;
      sq *= ds_exp(d, kq);
      if (TWO) s1 *= ds_exp(d, DS_LOG2E);
    }
    if constexpr (NP > 0) {
#pragma unroll
      for (int k = 0; k < NP; ++k) ds_packed(x[k]);
    }
    float ts = 0.f;
    for (int k = tid; k < a.K; k += THREADS)
      if (e_id[k] >= 0 && e_mass[k] != NEG_INF) ts += ds_exp(e_mass[k] - tm, kq);
    block_sum3<WAVES>(sq, s1, ts, red);
    if (!TWO) s1 = sq;   // temperature one, or only one of the two counts
    const bool teacher = a.alpha != 0.f && ts != 0.f;   // NaN counts

    // ---- the loss
    if (a.rows != nullptr) {
      float kl = 0.f;
      if (teacher) {
        const float ltq = logf(sq), lts = logf(ts);
        for (int k = tid; k < a.K; k += THREADS) {
          if (e_id[k] < 0) continue;
          const float u = (e_mass[k] - tm) * a.inv_tau - lts;
          const float p = ds_exp(e_mass[k] - tm, kq) / ts;
          const float lq = (to_f32<E>(z[e_id[k]]) - m) * a.inv_tau - ltq;
          if (p != 0.f) kl += p * (u - lq);
        }
      }
      float u1 = 0.f, u2 = 0.f;
      block_sum3<WAVES>(kl, u1, u2, red);
      if (tid == 0) {
        float loss = a.alpha * a.tau * a.tau * kl;
        if (a.alpha != 1.f) {
          const bool in = y >= 0 && y < a.V;
          const float ce = in ? logf(s1) - (to_f32<E>(z[y]) - m) : __builtin_nanf("");
          loss += (1.f - a.alpha) * ce;
        }
        a.rows[n] = loss;
      }
    }
    if (a.grad == nullptr) {
      __syncthreads();   // the entries' LDS is written again for the next row
      continue;
    }

    // ---- the gradient
    float w = a.upstream != nullptr ? a.upstream[a.per_row ? n : 0] : 1.f;
    if (a.mean) w /= a.count != nullptr ? a.count[0] : static_cast<float>(a.N);
    const float wq = teacher ? w * a.alpha * a.tau : 0.f, w1 = w * (1.f - a.alpha);
    const float cq = wq / sq;
    float c1 = a.alpha != 1.f ? w1 / s1 : 0.f;
    if (a.alpha != 1.f && (y < 0 || y >= a.V)) c1 = __builtin_nanf("");
    const auto value = [&](float v) {
      const float d = v - m;
      if (TWO) return cq * ds_exp(d, kq) + c1 * ds_exp(d, DS_LOG2E);
      return (cq + c1) * ds_exp(d, kq);
    };
    uint4* dzp = reinterpret_cast<uint4*>(dz + head);
    if constexpr (NP > 0) {
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (k * THREADS + tid < pieces) dzp[k * THREADS + tid] = ds_map<E>(x[k], value);
    } else {
      for (int p = tid; p < pieces; p += THREADS) dzp[p] = ds_map<E>(zp[p], value);
    }
    if (single >= 0) dz[single] = from_f32<E>(value(xs));
    // Masses of the entries; the label is entry K.
    for (int k = tid; k < a.K; k += THREADS)
      e_mass[k] = teacher && e_id[k] >= 0 ? wq * (ds_exp(e_mass[k] - tm, kq) / ts) : 0.f;
    if (tid == 0) {
      e_id[a.K] = a.alpha != 1.f && y >= 0 && y < a.V ? static_cast<int>(y) : -1;
      e_mass[a.K] = w1;
    }
    __syncthreads();
    for (int k = tid; k <= a.K; k += THREADS) {
      const int id = e_id[k];
      if (id < 0) continue;
      // every entry of this id, in order: the same sum whichever of them writes it
      float mass = 0.f;
      for (int j = 0; j <= a.K; ++j)
        if (e_id[j] == id) mass += e_mass[j];
      dz[id] = from_f32<E>(value(to_f32<E>(z[id])) - mass);
    }
    __syncthreads();
  }
}

// count[0] = the number of labels that are not `ignore`.
__global__ void __launch_bounds__(DS_COUNT_THREADS) distill_count_kernel(
    const int64_t* __restrict__ labels, int64_t N, int64_t ignore, float* __restrict__ count) {
  __shared__ int red[DS_COUNT_THREADS / 64];
  int c = 0;
  for (int64_t i = threadIdx.x; i < N; i += DS_COUNT_THREADS) c += labels[i] != ignore;
  for (int k = 32; k > 0; k >>= 1) c += __shfl_xor(c, k, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x != 0) return;
  int t = 0;
  for (int w = 0; w < DS_COUNT_THREADS / 64; ++w) t += red[w];
  count[0] = static_cast<float>(t);
}

// out[0] = the sum of the rows' losses, divided by the rows not ignored with `mean`.
__global__ void __launch_bounds__(DS_COUNT_THREADS) distill_total_kernel(
    const float* __restrict__ rows, int64_t N, int mean, const float* __restrict__ count,
    float* __restrict__ out) {
  __shared__ float red[DS_COUNT_THREADS / 64];
  float t = 0.f;
  for (int64_t i = threadIdx.x; i < N; i += DS_COUNT_THREADS) t += rows[i];
  t = block_sum(t, red);
  if (threadIdx.x == 0)
    out[0] = mean ? t / (count != nullptr ? count[0] : static_cast<float>(N)) : t;
}

struct DsScratch {
  float *rows, *count;
  template <class S>
  DsScratch(S& c, const gs_distill* d) {
    rows = c.template take<float>(d->reduction == GS_REDUCE_NONE ? 0 : d->N);
    count = c.template take<float>(1);
  }
};

template <class E, int THREADS, int NP>
void ds_launch(const DsArgs& a, bool two, int64_t grid, hipStream_t s) {
  const unsigned lds = static_cast<unsigned>((a.K + 1) * 8);
  if (two)
    hipLaunchKernelGGL((distill_kernel<E, THREADS, NP, true>), dim3(static_cast<unsigned>(grid)),
                       dim3(THREADS), lds, s, a);
  else
    hipLaunchKernelGGL((distill_kernel<E, THREADS, NP, false>), dim3(static_cast<unsigned>(grid)),
                       dim3(THREADS), lds, s, a);
}

// The smallest workgroup whose threads hold the row in 8 pieces each; 1024 threads of 16 for longer
// rows; beyond those the row is read twice.
template <class E>
int ds_run(const DsArgs& a, bool two, int64_t grid, hipStream_t s) {
  constexpr int VE = 16 / sizeof(E);
  const int pieces = a.V / VE + 1;
  if (pieces <= 256 * 8)
    ds_launch<E, 256, 8>(a, two, grid, s);
  else if (pieces <= 512 * 8)
    ds_launch<E, 512, 8>(a, two, grid, s);
  else if (pieces <= 1024 * 8)
    ds_launch<E, 1024, 8>(a, two, grid, s);
  else if (pieces <= 1024 * 16)
    ds_launch<E, 1024, 16>(a, two, grid, s);
  else
    ds_launch<E, 1024, 0>(a, two, grid, s);
  return check_launch("distill_kernel");
}

int ds_args(DsArgs& a, const char* name, const gs_distill* d) {
  const std::string n(name);
  if (d == nullptr) return fail(GS_ERR_INVALID, n + ": no arguments");
  if ((d->dtype != GS_DTYPE_BF16 && d->dtype != GS_DTYPE_F32) ||
      (d->teacher_dtype != GS_DTYPE_BF16 && d->teacher_dtype != GS_DTYPE_F32))
    return fail(GS_ERR_DTYPE, n + ": logits must be bf16 or fp32");
  if (d->Z == nullptr || d->teacher_ids == nullptr || d->teacher == nullptr || d->N <= 0 ||
      d->V <= 0 || d->K <= 0 || d->inner <= 0 || d->inner > d->N || d->N % d->inner != 0 ||
      (d->N > 1 && (d->stride_inner < d->V && d->inner > 1)) ||
      (d->N > d->inner && d->stride_outer < d->V) || !(d->temperature > 0.f) ||
      !std::isfinite(d->temperature) || !(d->alpha >= 0.f && d->alpha <= 1.f) ||
      (d->labels == nullptr && d->alpha != 1.f) || d->reduction < GS_REDUCE_NONE ||
      d->reduction > GS_REDUCE_MEAN ||
      reinterpret_cast<uintptr_t>(d->Z) % elem_size(d->dtype) != 0)
    return fail(GS_ERR_INVALID, n + ": invalid arguments");
  if (d->K > DS_MAX_K || d->V > INT32_MAX - 4096 || d->N > INT32_MAX)
    return fail(GS_ERR_UNSUPPORTED, n + ": more than 1024 teacher entries, 2^31 logits or rows");
  a = DsArgs{};
  a.z = d->Z, a.N = d->N, a.inner = d->inner, a.s_outer = d->stride_outer;
  a.s_inner = d->stride_inner, a.V = static_cast<int>(d->V), a.K = static_cast<int>(d->K);
  a.ids = d->teacher_ids, a.t = d->teacher, a.t_bf16 = d->teacher_dtype == GS_DTYPE_BF16;
  a.labels = d->labels, a.ignore = d->ignore_index;
  a.tau = d->temperature, a.alpha = d->alpha, a.inv_tau = 1.f / d->temperature;
  a.mean = d->reduction == GS_REDUCE_MEAN, a.per_row = d->reduction == GS_REDUCE_NONE;
  return GS_OK;
}

// One softmax serves where the temperature is one, or where only one of the two terms counts; a
// lone cross entropy (alpha 0) runs at temperature one.
bool ds_two(DsArgs& a) {
  if (a.alpha == 0.f) a.tau = a.inv_tau = 1.f;
  return a.tau != 1.f && a.alpha != 1.f;
}

int ds_check_grad(const char* name, const gs_distill* d, const void* grad) {
  if ((reinterpret_cast<uintptr_t>(grad) - reinterpret_cast<uintptr_t>(d->Z)) % 16 != 0)
    return fail(GS_ERR_INVALID,
                std::string(name) + ": grad at another offset from a 16-byte boundary than Z");
  return GS_OK;
}

int ds_count(DsArgs& a, float* count, hipStream_t s) {
  if (!a.mean || a.labels == nullptr) return GS_OK;
  hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(DS_COUNT_THREADS), 0, s, a.labels, a.N,
                     a.ignore, count);
  a.count = count;
  return check_launch("distill_count_kernel");
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_distill_workspace(const gs_distill* d) {
  DsArgs a;
  if (ds_args(a, "gs_distill", d) != GS_OK) return 0;
  Sizer sz;
  DsScratch unused(sz, d);
  return sz.used + 256;
}

extern "C" int gs_distill_loss(const gs_distill* d, float* out_loss, void* grad, void* workspace,
                               size_t workspace_bytes, void* stream) {
  DsArgs a;
  if (int rc = ds_args(a, "gs_distill_loss", d)) return rc;
  if (out_loss == nullptr) return fail(GS_ERR_INVALID, "gs_distill_loss: invalid arguments");
  if (grad != nullptr)
    if (int rc = ds_check_grad("gs_distill_loss", d, grad)) return rc;
  Sizer sz;
  DsScratch unused(sz, d);
  if (workspace == nullptr || workspace_bytes < sz.used)
    return fail(GS_ERR_WORKSPACE, "gs_distill_loss: workspace too small");
  Carver cv(workspace, workspace_bytes);
  const DsScratch w(cv, d);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = ds_count(a, w.count, s)) return rc;
  const bool two = ds_two(a);
  a.rows = a.per_row ? out_loss : w.rows;
  a.grad = grad;
  const int rc = d->dtype == GS_DTYPE_BF16 ? ds_run<uint16_t>(a, two, a.N, s)
                                           : ds_run<float>(a, two, a.N, s);
  if (rc || a.per_row) return rc;
  hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(DS_COUNT_THREADS), 0, s, w.rows, a.N,
                     a.mean, a.count, out_loss);
  return check_launch("distill_total_kernel");
}

extern "C" int gs_distill_grad(const gs_distill* d, const float* upstream, int filled, void* grad,
                               void* workspace, size_t workspace_bytes, void* stream) {
  DsArgs a;
  if (int rc = ds_args(a, "gs_distill_grad", d)) return rc;
  if (grad == nullptr || (filled && upstream == nullptr))
    return fail(GS_ERR_INVALID, "gs_distill_grad: invalid arguments");
  if (int rc = ds_check_grad("gs_distill_grad", d, grad)) return rc;
  Sizer sz;
  DsScratch unused(sz, d);
  if (workspace == nullptr || workspace_bytes < sz.used)
    return fail(GS_ERR_WORKSPACE, "gs_distill_grad: workspace too small");
  Carver cv(workspace, workspace_bytes);
  const DsScratch w(cv, d);
  hipStream_t s = static_cast<hipStream_t>(stream);
  a.filled = filled && !a.per_row;
  if (a.filled)   // the loss's call left the count
    a.count = a.mean && a.labels != nullptr ? w.count : nullptr;
  else if (int rc = ds_count(a, w.count, s))
    return rc;
  const bool two = ds_two(a);
  a.grad = grad;
  a.upstream = upstream;
  // A filled gradient is mostly left as it is: few workgroups then look at the upstream and end.
  const int64_t grid = a.filled ? std::min<int64_t>(a.N, 512) : a.N;
  return d->dtype == GS_DTYPE_BF16 ? ds_run<uint16_t>(a, two, grid, s)
                                   : ds_run<float>(a, two, grid, s);
}
