// Embedding lookup with a scale, gfx950:
//
//   out[i] = scale * W[id_i]        out: [n, d], W: [vocab, d]
//
// formed in fp32 and rounded once to W's dtype; ids outside [0, vocab) give rows of zeros.  For
// the gradient (gs_embedding_train_grad over the same ids) the pass also writes the ids as the
// gradient takes them: 64-bit, the padding id replaced by -1.
//
// Nothing is computed twice and every byte moves once, so the rate of a copy bounds it.  Each thread
// owns pieces of 16 bytes of the output: they are numbered through the whole output, so all lanes work
// whatever d is, and a wave writes one contiguous range.  Rows that are not whole pieces on 16-byte
// boundaries take pieces at their elements' alignment, which the hardware's loads and stores allow
// (element by element 24432 rows of 515 fp32 features took 26.9 us for 18.0, bf16 25.7 for 12.1).
// 16384 rows of 768 bf16: 9.1 us, 5.5 TB/s read and written.
#include <algorithm>

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

}  // namespace
}  // namespace gs

using namespace gs;

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
