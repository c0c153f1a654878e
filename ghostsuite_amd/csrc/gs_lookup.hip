// Embedding lookup with a scale, gfx950:
//
//   out[i] = scale * W[id_i]        out: [n, d], W: [vocab, d]
//
// formed in fp32 and rounded once to W's dtype; ids outside [0, vocab) give rows of zeros.  For
// the gradient (for few tokens the second kernel below, else gs_embedding_train_grad over the same
// ids) the pass also writes the ids as the gradient takes them: 64-bit, the padding id replaced by -1.
//
// Nothing is computed twice and every byte moves once, so the rate of a copy bounds it.  Each thread
// owns pieces of 16 bytes of the output: they are numbered through the whole output, so all lanes work
// whatever d is, and a wave writes one contiguous range.  Rows that are not whole pieces on 16-byte
// boundaries take pieces at their elements' alignment, which the hardware's loads and stores allow
// (element by element 24432 rows of 515 fp32 features took 26.9 us for 18.0, bf16 25.7 for 12.1).
// 16384 rows of 768 bf16: 9.1 us, 5.5 TB/s read and written.
#include <algorithm>
#include <type_traits>

#include "gs_common.h"

namespace gs {
namespace {

constexpr int LK_THREADS = 256;
constexpr int LK_PIECES = 4;   // per thread, loads of all in flight together
constexpr int64_t LK_MAX_BLOCKS = int64_t{1} << 23;   // of a launch: below 2^32 threads

__device__ __forceinline__ int64_t lk_id(const void* __restrict__ ids, int ids32, int64_t i) {
  return ids32 ? static_cast<const int32_t*>(ids)[i] : static_cast<const int64_t*>(ids)[i];
}

// V: elements of a piece, which lies on a boundary of ALIGN bytes; ppr: pieces per row, the pieces of
// all rows numbered through.  A row's last piece ends with the row, and writes again what it shares
// with the one before.
template <class E, int V, int ALIGN>
__global__ void __launch_bounds__(LK_THREADS) lookup_kernel(
    const void* __restrict__ ids, int ids32, int64_t n, const E* __restrict__ W, int64_t vocab,
    int64_t d, int64_t ppr, float scale, int64_t padding, E* __restrict__ out,
    int64_t* __restrict__ grad_ids, int64_t block0) {
  struct alignas(ALIGN) Piece { E e[V]; };
  const int64_t p0 = (block0 + blockIdx.x) * (LK_THREADS * LK_PIECES);
  const int64_t pieces = n * ppr;
  // A workgroup's pieces are within few rows: one 64-bit division, then 32-bit ones.
  const int64_t row0 = p0 / ppr;
  const uint32_t col0 = static_cast<uint32_t>(p0 - row0 * ppr);
  const uint32_t w = static_cast<uint32_t>(ppr);
  Piece x[LK_PIECES];
  int64_t to[LK_PIECES];
#pragma unroll
  for (int k = 0; k < LK_PIECES; ++k) {
    const uint32_t off = static_cast<uint32_t>(k * LK_THREADS + threadIdx.x);
    if (p0 + off < pieces) {
      const uint32_t c = col0 + off, r = c / w;
      const int64_t i = row0 + r;
      const uint32_t col = c - r * w;
      const int64_t id = lk_id(ids, ids32, i), f = min(static_cast<int64_t>(col) * V, d - V);
      to[k] = i * d + f;
      if (id >= 0 && id < vocab) {
        x[k] = *reinterpret_cast<const Piece*>(W + id * d + f);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[k].e[e] = from_f32<E>(0.f);
      }
      if (grad_ids != nullptr && col == 0) grad_ids[i] = id == padding ? -1 : id;
    }
  }
#pragma unroll
  for (int k = 0; k < LK_PIECES; ++k) {
    if (p0 + k * LK_THREADS + threadIdx.x < pieces) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[k].e[e] = from_f32<E>(scale * to_f32<E>(x[k].e[e]));
      *reinterpret_cast<Piece*>(out + to[k]) = x[k];
    }
  }
}

template <class E, int V, int ALIGN>
int launch_lookup(const void* ids, int ids32, int64_t n, const void* W, int64_t vocab, int64_t d,
                  float scale, int64_t padding, void* out, int64_t* grad_ids, hipStream_t s) {
  const int64_t ppr = (d + V - 1) / V;
  const int64_t blocks = (n * ppr + LK_THREADS * LK_PIECES - 1) / (LK_THREADS * LK_PIECES);
  for (int64_t b0 = 0; b0 < blocks; b0 += LK_MAX_BLOCKS) {
    const int64_t grid = std::min(blocks - b0, LK_MAX_BLOCKS);
    hipLaunchKernelGGL((lookup_kernel<E, V, ALIGN>), dim3(static_cast<unsigned>(grid)),
                       dim3(LK_THREADS), 0, s, ids, ids32, n, static_cast<const E*>(W), vocab, d,
                       ppr, scale, padding, static_cast<E*>(out), grad_ids, b0);
    if (int rc = check_launch("lookup_kernel")) return rc;
  }
  return GS_OK;
}

template <class E>
int launch_lookup_any(const void* ids, int ids32, int64_t n, const void* W, int64_t vocab,
                      int64_t d, float scale, int64_t padding, void* out, int64_t* grad_ids,
                      hipStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const bool whole = d % V == 0 && reinterpret_cast<uintptr_t>(W) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(out) % 16 == 0;
  constexpr int A = sizeof(E);
  if (whole)
    return launch_lookup<E, V, 16>(ids, ids32, n, W, vocab, d, scale, padding, out, grad_ids, s);
  if (d >= V)
    return launch_lookup<E, V, A>(ids, ids32, n, W, vocab, d, scale, padding, out, grad_ids, s);
  return launch_lookup<E, 1, A>(ids, ids32, n, W, vocab, d, scale, padding, out, grad_ids, s);
}

// A piece as it came, unpacked where it is used.
template <class E, int V>
struct LkRaw {
  std::conditional_t<(V * sizeof(E) >= 4), uint32_t, uint16_t> w[V > 1 ? 4 : 1];
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(E) == 4) return __uint_as_float(w[e]);
    else if constexpr (V == 1) return bf16_to_f32(w[0]);
    else return __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
};

// The gradient of few tokens in one launch: a wave owns a piece for each lane of 4 rows of the table, looks
// at all the ids (kept, 4 to a lane), and sums each row's tokens in order in fp32; most rows are written as
// zeros, which bounds it.  Nothing is sorted, and no wave waits for another.  Lookup and gradient, 768
// features in bf16, of 64 / 256 tokens spread over 1000 ids, then 50257 (us; in brackets by the sorted
// list): 9 (24) / 14 (26), 18 (34) / 20 (36), and three launches less for the host, 30 -> 24 a pass; 256
// tokens of one id 29 (25), 42 (35), 512 would be twice that.  (16 rows to a wave, all their features in
// turn: 20 / 43, 20 / 34.)
constexpr int LK_FEW = 256, LK_SETS = LK_FEW / 64;   // tokens; of a lane
constexpr int LK_ROWS = 4, LK_BATCH = 8;             // rows of a wave; loads in flight
template <class E, int V, int ALIGN>
__global__ void __launch_bounds__(LK_THREADS) lookup_few_grad_kernel(
    const int64_t* __restrict__ ids, int n, const E* __restrict__ G, int64_t vocab, int64_t d,
    float scale, E* __restrict__ grad) {
  struct alignas(ALIGN) Piece { E e[V]; };
  const int lane = threadIdx.x & 63;
  const int64_t v0 =
      (static_cast<int64_t>(blockIdx.x) * (LK_THREADS / 64) + (threadIdx.x >> 6)) * LK_ROWS;
  // the rows of the lane's tokens among the wave's (any other number: not among them)
  uint64_t row[LK_SETS];
#pragma unroll
  for (int k = 0; k < LK_SETS; ++k) {
    const int i = 64 * k + lane;
    row[k] = i < n ? static_cast<uint64_t>(ids[i]) - static_cast<uint64_t>(v0) : ~uint64_t{0};
  }
  const int64_t f0 = (static_cast<int64_t>(blockIdx.y) * 64 + lane) * V;
  const int64_t f = min(f0, d - V);   // a row's last piece ends with the row
  for (int r = 0; r < LK_ROWS && v0 + r < vocab; ++r) {
    unsigned long long mine[LK_SETS];
#pragma unroll
    for (int k = 0; k < LK_SETS; ++k) mine[k] = __ballot(row[k] == static_cast<uint64_t>(r));
    if (f0 >= d) continue;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.f;
#pragma unroll
    for (int k = 0; k < LK_SETS; ++k)
      for (unsigned long long left = mine[k]; left != 0;) {   // the same for the whole wave
        // all loads are made (past the last token its row again), so that none waits for another
        LkRaw<E, V> x[LK_BATCH];
        const int count = min(LK_BATCH, __popcll(left));
        int token = 0;
#pragma unroll
        for (int q = 0; q < LK_BATCH; ++q) {
          token = left != 0 ? __builtin_ctzll(left) : token;
          left &= left - 1;
          __builtin_memcpy(&x[q], reinterpret_cast<const Piece*>(G + (64 * k + token) * d + f),
                           sizeof(Piece));
        }
#pragma unroll
        for (int q = 0; q < LK_BATCH; ++q)
          if (q < count) {
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += x[q].get(e);
          }
      }
    Piece o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.e[e] = from_f32<E>(scale * acc[e]);
    *reinterpret_cast<Piece*>(grad + (v0 + r) * d + f) = o;
  }
}

template <class E>
int launch_few_grad(const int64_t* ids, int64_t n, const void* G, int64_t vocab, int64_t d,
                    float scale, void* grad, hipStream_t s) {
  constexpr int V = 16 / sizeof(E), A = sizeof(E);
  constexpr int64_t rows = LK_ROWS * (LK_THREADS / 64);
  const int64_t width = d >= V ? 64 * V : 64;   // a wave's features
  const dim3 grid(static_cast<unsigned>((vocab + rows - 1) / rows),
                  static_cast<unsigned>((d + width - 1) / width));
  const E* g = static_cast<const E*>(G);
  E* out = static_cast<E*>(grad);
  const int m = static_cast<int>(n);
  if (d % V == 0 && reinterpret_cast<uintptr_t>(G) % 16 == 0 &&
      reinterpret_cast<uintptr_t>(grad) % 16 == 0)
    hipLaunchKernelGGL((lookup_few_grad_kernel<E, V, 16>), grid, dim3(LK_THREADS), 0, s, ids, m, g,
                       vocab, d, scale, out);
  else if (d >= V)
    hipLaunchKernelGGL((lookup_few_grad_kernel<E, V, A>), grid, dim3(LK_THREADS), 0, s, ids, m, g,
                       vocab, d, scale, out);
  else
    hipLaunchKernelGGL((lookup_few_grad_kernel<E, 1, A>), grid, dim3(LK_THREADS), 0, s, ids, m, g,
                       vocab, d, scale, out);
  return check_launch("lookup_few_grad_kernel");
}

// Few tokens, and a grid's limits: 65535 pieces of a row, below 2^32 threads.
bool lookup_is_few(int64_t n, int64_t vocab, int64_t d) {
  const int64_t y = (d + 255) / 256;
  return n <= LK_FEW && y <= 65535 && vocab <= LK_MAX_BLOCKS * LK_ROWS / y;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_embedding_lookup_grad_workspace(int64_t n, int64_t vocab, int64_t d) {
  return n > 0 && lookup_is_few(n, vocab, d) ? 0
                                          : gs_embedding_train_grad_workspace(1, 0, n, d, vocab);
}

extern "C" int gs_embedding_lookup_grad(const int64_t* ids, const void* G, int dtype, int64_t n,
                                        int64_t vocab, int64_t d, float scale, void* grad,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != GS_DTYPE_BF16 && dtype != GS_DTYPE_F32)
    return fail(GS_ERR_DTYPE, "gs_embedding_lookup_grad: dtype must be bf16 or fp32");
  if (ids == nullptr || G == nullptr || grad == nullptr || n <= 0 || vocab <= 0 || d <= 0)
    return fail(GS_ERR_INVALID, "gs_embedding_lookup_grad: invalid arguments");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!lookup_is_few(n, vocab, d))   // one sample of all the tokens, none of them for validation
    return gs_embedding_train_grad(ids, G, dtype, 1, 0, 1, n, d, vocab, scale, grad, dtype, 0,
                                   workspace, workspace_bytes, stream);
  return dtype == GS_DTYPE_BF16 ? launch_few_grad<uint16_t>(ids, n, G, vocab, d, scale, grad, s)
                                : launch_few_grad<float>(ids, n, G, vocab, d, scale, grad, s);
}

extern "C" int gs_embedding_lookup(const void* ids, int ids_bits, int64_t n, const void* W,
                                   int dtype, int64_t vocab, int64_t d, float scale,
                                   int64_t padding_idx, void* out, int64_t* grad_ids,
                                   void* stream) {
  if (dtype != GS_DTYPE_BF16 && dtype != GS_DTYPE_F32)
    return fail(GS_ERR_DTYPE, "gs_embedding_lookup: dtype must be bf16 or fp32");
  if (ids == nullptr || W == nullptr || out == nullptr || n <= 0 || vocab <= 0 || d <= 0 ||
      (ids_bits != 32 && ids_bits != 64))
    return fail(GS_ERR_INVALID, "gs_embedding_lookup: invalid arguments");
  // 32-bit piece numbers within a workgroup; byte offsets well inside 64 bits.
  if (d >= (int64_t{1} << 30) || n > (int64_t{INT32_MAX} * LK_THREADS) / d)
    return fail(GS_ERR_UNSUPPORTED, "gs_embedding_lookup: 2^30 features or 2^39 elements or more");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int ids32 = ids_bits == 32;
  return dtype == GS_DTYPE_BF16
             ? launch_lookup_any<uint16_t>(ids, ids32, n, W, vocab, d, scale, padding_idx, out,
                                           grad_ids, s)
             : launch_lookup_any<float>(ids, ids32, n, W, vocab, d, scale, padding_idx, out,
                                        grad_ids, s);
}
