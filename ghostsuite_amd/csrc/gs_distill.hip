// Loss of a student's logits against a teacher's top logits and the labels, with its gradient,
// gfx950.  Per row z (V logits), teacher entries (id_k, t_k) and label y, with tau the temperature:
//
//   p = softmax(t / tau)   q = softmax(z / tau)   s = softmax(z)
//   loss = alpha tau^2 sum_k p_k (log p_k - log q[id_k]) + (1 - alpha) (log sum exp z - z_y)
//   dz   = w (alpha tau (q - P) + (1 - alpha) (s - 1_y)),   P the p_k at their ids
//
// A workgroup owns a row.  The row is read once, in 16-byte pieces that stay in registers as they
// came: the maximum, then both sums of exponentials, then the gradient are formed from them, so the
// loss and the gradient for an upstream of one cost one read and one write of the logits, and the rate
// of a copy bounds them (8192 rows of 50257 bf16: 390 us, 4.2 of a copy's 4.7 TB/s; with two softmaxes the
// exponentials, four to an element, come close behind).  Rows too long for the registers are read
// again in a second sweep, out of the caches (running maximum and sums in the first).  The gradient is
// written for the whole row as if no entry stood there; the elements of the K entries and the label are
// then written again with their masses taken off, by the threads that wrote them, from the logits
// themselves, so that each element is rounded once.  An id that stands several times gets its masses
// added up in the entries' order.
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
constexpr int DS_COUNT_HERE = 256;   // rows that every wave counts itself
constexpr int64_t DS_MAX_BLOCKS = int64_t{1} << 21;   // below 2^32 threads; more rows are looped over

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
  const float* count;      // the number of rows not ignored (labels, mean), or null
  int count_here;          // without it: every wave counts them itself (else N)
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
// Ends one sweep over a piece: its sums are formed (`a`, `b` are taken in) before the piece counts as
// a new value, so the compiler neither carries unpacked elements to the next sweep (twice the
// registers for bf16) nor keeps two copies of the piece for sums that it puts off.
__device__ __forceinline__ void ds_swept(uint4& v, float& a, float& b) {
  asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w), "+v"(a), "+v"(b));
}

// A value the compiler takes for a new one: what it made of the old one is formed again, not kept.
__device__ __forceinline__ uint32_t ds_fresh(uint32_t v) {
  asm("" : "+v"(v));
  return v;
}

// Piece p of a row: a scalar base and 32 bits of offset (rows are below 2^32 bytes where pieces are
// kept), so that no 64-bit address takes registers for each of them.
__device__ __forceinline__ uint4 ds_piece(const uint4* row, uint32_t p) {
  return *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(row) + p * 16u);
}

// The wave's maximum (wave-uniform), by DPP as wave_sum_dpp; lanes without a source keep their own.
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
  const int i = __builtin_bit_cast(int, v);
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_max_dpp(float v) {
  v = dpp_max<0x111>(v);   // row_shr:1, 2, 4, 8: lane 15 of each row holds the row's
  v = dpp_max<0x112>(v);
  v = dpp_max<0x114>(v);
  v = dpp_max<0x118>(v);
  v = dpp_max<0x142>(v);   // row_bcast:15, :31: lane 63 holds the wave's
  v = dpp_max<0x143>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// exp(x / tau) for x <= 0, `k` = log2(e) / tau.
__device__ __forceinline__ float ds_exp(float x, float k) { return __builtin_amdgcn_exp2f(x * k); }

constexpr float DS_LOG2E = 1.44269504088896340736f;

// One teacher entry (the label is entry K): its id (-1: none), the thread that writes the id's
// element, the entry's logit, then its mass in the gradient, the student's logit there, and the
// masses of all entries of its id.
struct DsEntries {
  int *id, *owner;
  float *t, *z, *mass;
  __device__ DsEntries(void* lds, int n) {
    id = static_cast<int*>(lds);
    owner = id + n;
    t = reinterpret_cast<float*>(owner + n);
    z = t + n;
    mass = z + n;
  }
};
__host__ __device__ inline int ds_entries(int K) { return (K + 1 + 3) & ~3; }   // whole int4s

// NP: pieces a thread keeps; below zero none are kept, the row is read twice with -NP pieces of a thread
// on their way at once.  TWO: the two softmaxes differ and both count.  WPE: waves on a SIMD the
// registers are held to.
template <class E, int THREADS, int NP, bool TWO, int WPE>
__global__ void __launch_bounds__(THREADS, WPE) distill_kernel(DsArgs a) {
  constexpr int VE = 16 / sizeof(E);
  constexpr int WAVES = THREADS / 64;
  constexpr bool KEEP = NP > 0;
  constexpr uint32_t AHEAD = KEEP ? 1 : -NP;
  __shared__ float red[3][WAVES][4];
  extern __shared__ int4 dyn[];
  const DsEntries ent(dyn, ds_entries(a.K));
  const float NEG_INF = -__builtin_inff();
  const uint32_t wid = threadIdx.x >> 6, K = a.K, V = a.V;
  const bool lead = (threadIdx.x & 63) == 0;
  const float kq = DS_LOG2E * a.inv_tau;

  if (a.filled && !a.per_row && a.upstream[0] == 1.f) return;   // nothing to change
  int counted = static_cast<int>(a.N);
  if (a.count_here) {
    counted = 0;
#pragma unroll
    for (int k = 0; k < DS_COUNT_HERE; k += 64) {
      const int64_t i = k + (threadIdx.x & 63);
      counted += __popcll(__ballot(i < a.N && a.labels[i] != a.ignore));
    }
  }

  for (uint32_t n = blockIdx.x; n < static_cast<uint32_t>(a.N); n += gridDim.x) {
    const uint32_t tid = ds_fresh(threadIdx.x);
    if (n != blockIdx.x) __syncthreads();   // the last row's LDS has been read
    const uint32_t outer = a.inner == a.N ? 0 : n / static_cast<uint32_t>(a.inner);
    const int64_t at = outer * a.s_outer + (n - outer * static_cast<uint32_t>(a.inner)) * a.s_inner;
    const E* z = static_cast<const E*>(a.z) + at;
    E* dz = static_cast<E*>(a.grad) + at;
    const int64_t y = a.labels != nullptr ? a.labels[n] : 0;
    const bool ignored = a.labels != nullptr && y == a.ignore;
    // The row from its first 16-byte boundary in whole pieces, piece p = k S + tid with thread tid
    // (S = the threads that NP pieces each need); the single elements around them belong to the
    // first threads of the first two waves.
    const uint32_t head = min(V, static_cast<uint32_t>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) /
                                     static_cast<uint32_t>(sizeof(E)));
    const uint32_t pieces = (V - head) / VE, tail0 = head + pieces * VE;
    const uint32_t S = KEEP ? (pieces + NP - 1) / (KEEP ? NP : 1) : THREADS;
    const int single = tid < head ? static_cast<int>(tid)
                       : tid >= 64 && tid - 64 < V - tail0 ? static_cast<int>(tail0 + tid - 64) : -1;
    const uint4* zp = reinterpret_cast<const uint4*>(z + head);
    uint4* dzp = reinterpret_cast<uint4*>(dz + head);
    if (ignored) {
      if (a.rows != nullptr && tid == 0) a.rows[n] = 0.f;
      if (a.grad != nullptr) {
        for (uint32_t p = tid; p < pieces; p += THREADS) dzp[p] = make_uint4(0u, 0u, 0u, 0u);
        if (single >= 0) dz[single] = from_f32<E>(0.f);
      }
      continue;
    }

    // ---- the row and the teacher's entries
    const auto entry_id = [&](uint32_t k) { return a.ids[static_cast<int64_t>(n) * a.K + k]; };
    const auto entry_t = [&](uint32_t k) {
      const int64_t i = static_cast<int64_t>(n) * a.K + k;
      return a.t_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.t)[i])
                      : static_cast<const float*>(a.t)[i];
    };
    const int64_t id0 = tid < K ? entry_id(tid) : -1;   // the loads ahead of the row's
    const float t0 = tid < K ? entry_t(tid) : NEG_INF;
    const float xs = single >= 0 ? to_f32<E>(z[single]) : NEG_INF;
    // A thread past S holds copies of another's pieces, and one whose last piece (only the last:
    // S >= NP) is past the row's end a copy of the row's: neither is added nor stored.
    const bool mine = !KEEP || tid < S, last = !KEEP || tid + (NP - 1) * S < pieces;
    uint4 x[KEEP ? NP : 1];
    if constexpr (KEEP) {
      uint32_t p = min(tid, S - 1);
#pragma unroll
      for (int k = 0; k < NP; ++k, p += S) x[k] = ds_piece(zp, k < NP - 1 ? p : min(p, pieces - 1));
    }
    float tm = NEG_INF;
    const auto take = [&](uint32_t k, int64_t id, float t) {
      const bool use = id >= 0 && id < V;
      t = use ? t : NEG_INF;
      ent.id[k] = use ? static_cast<int>(id) : -1;
      ent.t[k] = t;
      ent.z[k] = use ? to_f32<E>(z[id]) : 0.f;
      tm = t != t ? t : fmaxf(tm, t);
    };
    if (tid < K) take(tid, id0, t0);
    for (uint32_t k = tid + THREADS; k < K; k += THREADS) take(k, entry_id(k), entry_t(k));
    float m = xs, sq = 0.f, s1 = 0.f;
    if constexpr (KEEP) {
#pragma unroll
      for (int k = 0; k < NP; ++k) {
#pragma unroll
        for (int e = 0; e < VE; ++e) m = fmaxf(m, ds_elem<E>(x[k], e));
        ds_swept(x[k], m, tm);
      }
    } else {
      // running maximum and sums of this thread
      sq = xs == NEG_INF ? 0.f : 1.f;
      s1 = sq;
      for (uint32_t p = tid; p < pieces; p += AHEAD * THREADS) {
        uint4 v[AHEAD];
#pragma unroll
        for (uint32_t q = 0; q < AHEAD; ++q) v[q] = zp[min(p + q * THREADS, pieces - 1)];
        float pm = m;   // (a piece past the end is a copy of the last)
#pragma unroll
        for (uint32_t q = 0; q < AHEAD; ++q)
#pragma unroll
          for (int e = 0; e < VE; ++e) pm = fmaxf(pm, ds_elem<E>(v[q], e));
        // no maximum yet: any reference will do (a NaN among them is seen by the sums)
        const float ref = pm == NEG_INF ? 0.f : pm, d = m == NEG_INF ? 0.f : m - ref;
        sq *= ds_exp(d, kq);
        if (TWO) s1 *= ds_exp(d, DS_LOG2E);
#pragma unroll
        for (uint32_t q = 0; q < AHEAD; ++q) {
          float pq = 0.f, p1 = 0.f;
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float w = ds_elem<E>(v[q], e) - ref;
            pq += ds_exp(w, kq);
            if (TWO) p1 += ds_exp(w, DS_LOG2E);
          }
          if (p + q * THREADS < pieces) {
            sq += pq;
            s1 += p1;
          }
        }
        m = pm;
      }
    }
    const float m_own = m;
    m = wave_max_dpp(m);
    tm = wave_max_dpp(tm);
    if (lead) {
      red[0][wid][0] = m;
      red[0][wid][1] = tm;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      m = fmaxf(m, red[0][w][0]);
      tm = fmaxf(tm, red[0][w][1]);
    }

    // ---- sums of exponentials
    if constexpr (KEEP) {
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        float pq = 0.f, p1 = 0.f;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float w = ds_elem<E>(x[k], e) - m;
          pq += ds_exp(w, kq);
          if (TWO) p1 += ds_exp(w, DS_LOG2E);
        }
        if (k < NP - 1 || last) {
          sq += pq;
          s1 += p1;
        }
        ds_swept(x[k], sq, s1);
      }
      if (!mine) sq = s1 = 0.f;
      if (single >= 0) {
        sq += ds_exp(xs - m, kq);
        if (TWO) s1 += ds_exp(xs - m, DS_LOG2E);
      }
    } else {
      const float d = m_own == NEG_INF ? 0.f : m_own - m;
      sq *= ds_exp(d, kq);
      if (TWO) s1 *= ds_exp(d, DS_LOG2E);
    }
    float ts = 0.f;
    for (uint32_t k = tid; k < K; k += THREADS)
      if (ent.id[k] >= 0 && ent.t[k] != NEG_INF) ts += ds_exp(ent.t[k] - tm, kq);
    sq = wave_sum_dpp(sq);
    if (TWO) s1 = wave_sum_dpp(s1);
    ts = wave_sum_dpp(ts);
    if (lead) {
      red[1][wid][0] = sq;
      red[1][wid][1] = s1;
      red[1][wid][2] = ts;
    }
    __syncthreads();
    sq = s1 = ts = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      sq += red[1][w][0];
      s1 += red[1][w][1];
      ts += red[1][w][2];
    }
    if (!TWO) s1 = sq;   // temperature one, or only one of the two counts
    const bool teacher = a.alpha != 0.f && ts != 0.f;   // NaN counts

    // ---- the entries' part: the loss, and each id's mass in the gradient.  The loss adds up tau (log p -
    // log q), from differences of logits as they are: divided by a temperature below one, a student's
    // logit at its type's lowest value would be infinite.
    float w = a.upstream != nullptr ? a.upstream[a.per_row ? n : 0] : 1.f;
    if (a.mean) w /= a.count != nullptr ? a.count[0] : static_cast<float>(counted);
    const float nan_or_one = ts != ts ? ts : 1.f;   // a NaN entry leaves no element of the row as if valid
    const float wq = teacher ? w * a.alpha * a.tau * nan_or_one : 0.f, w1 = w * (1.f - a.alpha);
    const bool hard = a.alpha != 1.f, in = y >= 0 && y < V;
    float kl = 0.f;
    {
      const float ltq = logf(sq), lts = logf(ts), inv_ts = 1.f / ts;
      for (uint32_t k = tid; k <= K; k += THREADS) {
        const int id = k < K ? ent.id[k] : hard && in ? static_cast<int>(y) : -1;
        float mass = 0.f;
        if (k == K) {
          ent.z[K] = id >= 0 ? to_f32<E>(z[id]) : 0.f;
          ent.id[K] = id;
          mass = w1;
        } else if (teacher && id >= 0) {
          const float d = ent.t[k] - tm, p = ds_exp(d, kq) * inv_ts;
          if (p != 0.f) kl += a.alpha * a.tau * p * (d - (ent.z[k] - m) - a.tau * (lts - ltq));
          mass = wq * p;
        }
        ent.t[k] = mass;
        const uint32_t i = id - head, p = i / VE;
        ent.owner[k] = id < 0 ? -1
                       : static_cast<uint32_t>(id) < head ? id
                       : static_cast<uint32_t>(id) >= tail0 ? static_cast<int>(id - tail0 + 64)
                                                            : static_cast<int>(p % S);
      }
      if (a.rows != nullptr) {
        kl = wave_sum_dpp(kl);
        if (lead) red[2][wid][0] = kl;
      }
    }
    __syncthreads();
    if (a.rows != nullptr && tid == 0) {
      float loss = 0.f;
#pragma unroll
      for (int q = 0; q < WAVES; ++q) loss += red[2][q][0];
      if (hard) loss += (1.f - a.alpha) * (in ? logf(s1) - (ent.z[K] - m) : __builtin_nanf(""));
      a.rows[n] = loss;
    }
    if (a.grad == nullptr) continue;

    // ---- the gradient: the row as if no entry stood there, then each thread its entries' elements
    // again (its own stores stay in order)
    float c1 = hard ? w1 / s1 : 0.f;
    if (hard && !in) c1 = __builtin_nanf("");
    const float cq = TWO ? wq / sq : wq / sq + c1;
    const auto value = [&](float v) {
      const float d = v - m;
      const float g = cq * ds_exp(d, kq);
      return TWO ? g + c1 * ds_exp(d, DS_LOG2E) : g;
    };
    if constexpr (KEEP) {
      uint32_t p = ds_fresh(tid);
      if (mine) {
#pragma unroll
        for (int k = 0; k < NP; ++k, p += S) {
          const uint4 o = ds_map<E>(x[k], value);
          if (k < NP - 1 || last)
            *reinterpret_cast<uint4*>(reinterpret_cast<char*>(dzp) + p * 16u) = o;
          __builtin_amdgcn_sched_barrier(0);   // one piece after the other: few registers
        }
      }
    } else {
      for (uint32_t p = tid; p < pieces; p += AHEAD * THREADS) {
        uint4 v[AHEAD];
#pragma unroll
        for (uint32_t q = 0; q < AHEAD; ++q) v[q] = zp[min(p + q * THREADS, pieces - 1)];
#pragma unroll
        for (uint32_t q = 0; q < AHEAD; ++q)
          if (p + q * THREADS < pieces) dzp[p + q * THREADS] = ds_map<E>(v[q], value);
      }
    }
    if (single >= 0) dz[single] = from_f32<E>(value(xs));
    // while the stores drain: the masses of every id, added in the entries' order by each of them
    for (uint32_t k = tid; k <= K; k += THREADS) {
      const int id = ent.id[k];
      float mass = 0.f;
      for (uint32_t j = 0; j <= K; j += 4) {
        const int4 o = *reinterpret_cast<const int4*>(ent.id + j);
        if (o.x == id) mass += ent.t[j];
        if (o.y == id && j + 1 <= K) mass += ent.t[j + 1];
        if (o.z == id && j + 2 <= K) mass += ent.t[j + 2];
        if (o.w == id && j + 3 <= K) mass += ent.t[j + 3];
      }
      ent.mass[k] = mass;
    }
    __syncthreads();
    const int me = static_cast<int>(tid);
    for (uint32_t j = 0; j <= K; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(ent.owner + j);
      if (o.x != me && o.y != me && o.z != me && o.w != me) continue;
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q)
        if (j + q <= K && ent.owner[j + q] == me)
          dz[ent.id[j + q]] = from_f32<E>(value(ent.z[j + q]) - ent.mass[j + q]);
    }
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
__global__ void __launch_bounds__(DS_COUNT_THREADS) distill_total_kernel(DsArgs a,
                                                                         float* __restrict__ out) {
  __shared__ float red[2][DS_COUNT_THREADS / 64];
  float t = 0.f;
  for (int64_t i = threadIdx.x; i < a.N; i += DS_COUNT_THREADS) t += a.rows[i];
  float rows = a.count != nullptr ? a.count[0] : static_cast<float>(a.N);
  if (a.count_here)
    rows = block_sum(threadIdx.x < a.N && a.labels[threadIdx.x] != a.ignore ? 1.f : 0.f, red[1]);
  t = block_sum(t, red[0]);
  if (threadIdx.x == 0) out[0] = a.mean ? t / rows : t;
}

struct DsScratch {
  float *rows, *count;
  template <class S>
  DsScratch(S& c, const gs_distill* d) {
    rows = c.template take<float>(d->reduction == GS_REDUCE_NONE ? 0 : d->N);
    count = c.template take<float>(1);
  }
};

template <class E, int THREADS, int NP, int WPE>
void ds_launch(const DsArgs& a, bool two, int64_t grid, hipStream_t s) {
  const unsigned lds = static_cast<unsigned>(ds_entries(a.K) * 20);
  if (two)
    hipLaunchKernelGGL((distill_kernel<E, THREADS, NP, true, WPE>), dim3(static_cast<unsigned>(grid)),
                       dim3(THREADS), lds, s, a);
  else
    hipLaunchKernelGGL((distill_kernel<E, THREADS, NP, false, WPE>), dim3(static_cast<unsigned>(grid)),
                       dim3(THREADS), lds, s, a);
}

// Rows of up to 6656 pieces are kept by 256 threads, of up to 9216 by 512 (the fewest pieces a thread:
// all NP are gone through, so a row should fill them); others, and rows of a few pieces, are read
// twice, the second time from the caches: few rows are worked on at once.  Few threads with many
// pieces leave several rows on a CU at different stages, where reading, exponentials and writing
// overlap.  Registers: 4 NP and about 45 more.  Measured on MI355X (loss and gradient of 4e8 bf16 / 4e8
// fp32 logits, K = 64, two softmaxes, us), by vocabulary:
//     50257: kept by 256 threads 408 / -, by 512 441 / 821, read twice by 512 475 / 772
//     32003: kept by 256 418 / -, by 512 - / 703, read twice 546 / 785
//     65000: kept by 512 (18, 32 pieces) 444 / 773, read twice 425 / 807
//    128256: kept by 512 (32) 511 / -, read twice by 512 415 / 938, by 1024 456 / 822
//    262144: read twice by 512 448 / 924, by 1024 446 / 866
// (The tiers count pieces, not types: at 65000 ids both types get the slower of their two, by 4%.)
template <class E>
int ds_run(const DsArgs& a, bool two, int64_t grid, hipStream_t s) {
  constexpr int VE = 16 / sizeof(E);
  const int most = a.V / VE, least = (a.V - VE + 1) / VE;   // pieces of a row, whatever its offset
#define GS_DS_TRY(THREADS, NP, WPE)                                               \
  if (most <= THREADS * NP && least > NP * (NP - 1)) {                            \
    ds_launch<E, THREADS, NP, WPE>(a, two, grid, s);                              \
    return check_launch("distill_kernel");                                        \
  }
  GS_DS_TRY(256, 4, 4)
  GS_DS_TRY(256, 8, 4)
  GS_DS_TRY(256, 13, 4)
  GS_DS_TRY(256, 18, 4)
  GS_DS_TRY(256, 26, 3)
  GS_DS_TRY(512, 18, 4)
#undef GS_DS_TRY
  if (most < 512)
    ds_launch<E, 256, -4, 4>(a, two, grid, s);
  else if (most <= 20480)
    ds_launch<E, 512, -8, 4>(a, two, grid, s);
  else
    ds_launch<E, 1024, -4, 4>(a, two, grid, s);
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
      (d->inner > 1 && d->stride_inner < d->V) || (d->N > d->inner && d->stride_outer < d->V) ||
      !(d->temperature > 0.f) || !std::isfinite(d->temperature * d->temperature) ||
      !std::isfinite(DS_LOG2E / d->temperature) || !(d->alpha >= 0.f && d->alpha <= 1.f) ||
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

// The rows not ignored, where a mean needs their number: by a launch of its own, or where they are few
// by every wave (8 rows of 50257: 5 us less of launches; with 2031 rows, counted by every workgroup
// while its row arrives, 5 us more in all).
int ds_count(DsArgs& a, float* count, bool counted, hipStream_t s) {
  if (!a.mean || a.labels == nullptr) return GS_OK;
  if (a.N <= DS_COUNT_HERE) {
    a.count_here = 1;
    return GS_OK;
  }
  a.count = count;
  if (counted) return GS_OK;
  hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(DS_COUNT_THREADS), 0, s, a.labels, a.N,
                     a.ignore, count);
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
  if (int rc = ds_count(a, w.count, false, s)) return rc;
  const bool two = ds_two(a);
  a.rows = a.per_row ? out_loss : w.rows;
  a.grad = grad;
  const int64_t grid = std::min(a.N, DS_MAX_BLOCKS);
  const int rc = d->dtype == GS_DTYPE_BF16 ? ds_run<uint16_t>(a, two, grid, s)
                                           : ds_run<float>(a, two, grid, s);
  if (rc || a.per_row) return rc;
  hipLaunchKernelGGL(distill_total_kernel, dim3(1), dim3(DS_COUNT_THREADS), 0, s, a, out_loss);
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
  if (int rc = ds_count(a, w.count, a.filled != 0, s)) return rc;   // filled: the loss's call left it
  const bool two = ds_two(a);
  a.grad = grad;
  a.upstream = upstream;
  // A filled gradient is mostly left as it is: few workgroups then look at the upstream and end.  For
  // another upstream they form it again, in 520 us for 8192 rows of 50257 bf16 (as many as fit the card
  // would be 768 or 1024; not measured).
  const int64_t grid = a.filled ? std::min<int64_t>(a.N, 512) : std::min(a.N, DS_MAX_BLOCKS);
  return d->dtype == GS_DTYPE_BF16 ? ds_run<uint16_t>(a, two, grid, s)
                                   : ds_run<float>(a, two, grid, s);
}
