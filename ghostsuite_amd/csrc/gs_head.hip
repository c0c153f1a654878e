// Output projection with its softmax cross entropy, in pieces of the vocabulary.
//
// Per hidden row x (d features) with label y, and W [V, d]:
//   z = W x,  loss = log sum_v e^(z_v) - z_y,  dz = w (softmax(z) - 1_y)
//   dx = W^T dz,  dW = sum over rows of dz x^T
// with w the row's upstream gradient (over the number of rows that count, for a mean).  The
// logits are never stored: the forward product's tiles leave only each row's maximum and sum
// of exponentials over the tile's 256 vocabulary entries and the label's logit; the backward
// pass forms a piece of the logits again, writes that piece of dz as bf16 and multiplies it
// into dx and into the piece's rows of dW.  Four products where keeping the logits takes three,
// for a workspace of one piece of dz.
//
// Rows that do not count (label ignore_index) take no part in any product: the rows that do are
// listed first, in order, and copied next to each other (with rows of a multiple of 8 features,
// which the 16-byte loads need).  Their number stays on the device; tiles past it end at once.
//
// fp32 operands are taken as three bf16 parts each, x = h + m + l with 8 bits apiece, and a
// product as the six products of parts above 2^-24 of it, accumulated in fp32 like the bf16
// one: the same kernels over six times the contraction, which at the bf16 matrix rate is still
// faster than fp32 matrix instructions (measured below).
//
// Tiles: BM x BN outputs, 64 of the contraction a stage, staged through LDS by wave-level
// 16-byte DMA, MFMA 32x32x16 (fp32 accumulators).  A side whose contraction index is contiguous
// in memory (KC) is read from LDS as 16-byte fragments, one whose contraction index is the row
// (KR) through the transpose read.  Result layout of the MFMA: lane l, element e is row
// 8 (e / 4) + 4 (l / 32) + e % 4 of the A side, column l % 32 of the B side.

#include <algorithm>

#include "gs_common.h"

namespace gs {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

constexpr int HK = 64;                 // contraction of a stage
constexpr unsigned OOB = 0x80000000u;  // past every buffer range: such lanes load zeros
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

__device__ __forceinline__ unsigned lds_addr(const void* p) {
  typedef const __attribute__((address_space(3))) unsigned char* lds_ptr;
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_ptr)p));
}
// 64 lanes' 16 bytes at base + voff to LDS address lds + 16 lane.  Nothing else here uses M0.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(r)
               : "memory");
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0,
                                           static_cast<int>(OOB - 1), 0x00020000);
}
// A value that is the same in every lane, in scalar registers (a division leaves it in vector ones,
// which a buffer's address cannot be in).
__device__ __forceinline__ int64_t scalar(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | 0x0F70);
  asm volatile("" ::: "memory");
}
// A barrier that leaves the DMA in flight; the caller waits for what it needs.
__device__ __forceinline__ void raw_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ s16x4_t lds_tr16(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4_t*)(p));
}

// WM x WN waves of MI x NI blocks of 32 x 32; NS stage slots.
template <int WM_, int WN_, int MI_, int NI_, int NS_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MI = MI_, NI = NI_, NS = NS_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int BM = WM * MI * 32, BN = WN * NI * 32;
  static constexpr int A_BYTES = BM * HK * 2, STAGE = (BM + BN) * HK * 2;
  static constexpr int LDS = NS * STAGE;
};

using Wide = Tile<2, 4, 4, 2, 2>;   // 256 x 256, eight waves of 128 x 64
using Few = Tile<4, 1, 1, 1, 4>;    // 128 x 32, four waves
using FewT = Tile<1, 4, 1, 1, 4>;   // 32 x 128

// The bf16 parts that dz is held in between the products: three for fp32; two of a few rows, whose
// products are bound by W's and dW's memory (rounded once, a label's p - 1 would be most of dW's error);
// one beyond.
template <class C>
__host__ __device__ constexpr int dz_parts(bool f32) {
  return f32 ? 3 : C::BN == Few::BN ? 2 : 1;
}

// One side of a product: the tile's first element, the stride between rows (of the side with
// KC, of the contraction with KR) and between the bf16 parts of an fp32 operand, in elements.
struct Side {
  const uint16_t* p;
  int64_t ld, part;
};

// The DMA of one side's stages.  KC: LDS row r (128 bytes) holds its 16-byte chunk c at slot
// c ^ (r / 2 % 8), so that the 16 rows of a fragment read lie in 16 different bank groups.
// KR: LDS row = contraction index, chunk c at slot c ^ swz(row): the 4 rows x 4 chunks of a
// transpose read in 16 different ones.
template <int B, int NW, bool KR>
struct Stream {
  static constexpr int Q = B * HK * 2 / 1024 / NW;   // loads of a wave
  static_assert(Q > 0 && B * HK * 2 % (1024 * NW) == 0, "stage bytes split over waves");
  static constexpr int RB = B * 2, CH = B / 8;
  __device__ static constexpr int swz(int r) {
    return CH >= 16 ? 4 * (r & 3) : CH == 8 ? 4 * ((r >> 1) & 1) : 0;
  }
  unsigned off[Q];
  int k[Q];
  // `extent`: how many of the side's rows (columns of memory with KR) there are from the tile's
  // first on.
  __device__ __forceinline__ void init(int64_t ld, int64_t extent) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if constexpr (KR) {
        const int byte = (wid + NW * q) * 1024 + lane * 16;
        const int r = byte / RB, c = (byte % RB) / 16 ^ swz(r);
        k[q] = r;
        off[q] = c * 8 < extent ? static_cast<unsigned>(r * ld * 2 + c * 16) : OOB;
      } else {
        const int r = 8 * (wid + NW * q) + lane / 8, c = lane % 8 ^ ((r >> 1) & 7);
        k[q] = c * 8;
        off[q] = r < extent ? static_cast<unsigned>(r * ld * 2 + c * 16) : OOB;
      }
    }
  }
  // The stage whose first element is at `base`; contraction indices at or past `lim` as zeros.
  __device__ __forceinline__ void issue(const uint16_t* base, int lim, unsigned lds) const {
    const __amdgpu_buffer_rsrc_t r = rsrc(base);
    const unsigned w = static_cast<unsigned>(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
#pragma unroll
    for (int q = 0; q < Q; ++q)
      dma16(r, k[q] < lim ? off[q] : OOB, lds + (w + NW * q) * 1024);
  }
};

template <int RD, int M, int G = 0>
__device__ __forceinline__ void sched_kstep() {
  __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
  constexpr int n = (RD * (G + 1)) / M - (RD * G) / M;
  if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x100, n, 0);
  if constexpr (G + 1 < M) sched_kstep<RD, M, G + 1>();
}

// The fragments of one side: F blocks of 32 rows from row `first` on, k-step ks of the stage.
template <int B, int F, bool KR>
struct Fragments {
  int at[KR ? F : 1];
  int lo, hi;
  __device__ __forceinline__ void init(int first) {
    const int lane = threadIdx.x & 63;
    if constexpr (KR) {
      using S = Stream<B, 1, true>;
      const int g = lane >> 4, row = 8 * (g >> 1) + ((lane >> 2) & 3);
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int col = first + i * 32 + 16 * (g & 1) + 4 * (lane & 3);
        at[i] = row * S::RB + ((col >> 3) ^ S::swz(row)) * 16 + (col & 7) * 2;
      }
      lo = hi = 0;
    } else {
      at[0] = (first + (lane & 31)) * 128;
      lo = ((lane & 31) >> 1) & 7, hi = lane >> 5;
    }
  }
  __device__ __forceinline__ void load(const unsigned char* side, int ks, bf16x8_t (&f)[F]) const {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if constexpr (KR) {
        const unsigned char* p = side + at[i] + ks * 16 * B * 2;
        f[i] = __builtin_bit_cast(
            bf16x8_t, __builtin_shufflevector(lds_tr16(p), lds_tr16(p + 4 * B * 2), 0, 1, 2, 3, 4,
                                              5, 6, 7));
      } else {
        f[i] = *reinterpret_cast<const bf16x8_t*>(side + at[0] + i * 32 * 128 +
                                                  ((2 * ks + hi) ^ lo) * 16);
      }
    }
  }
};

// acc = sum over the contraction [k0, k1) of A B^T, with six products of parts for fp32 (TERMS 6, the
// small ones first), two where A alone has two parts (TERMS 2).
template <class C, bool AKR, bool BKR, int TERMS>
__device__ __forceinline__ void product(Side a, int64_t a_extent, Side b, int64_t b_extent,
                                        int64_t k0, int64_t k1, unsigned char* lds,
                                        f32x16_t (&acc)[C::MI][C::NI]) {
  a.p = reinterpret_cast<const uint16_t*>(scalar(reinterpret_cast<int64_t>(a.p)));
  b.p = reinterpret_cast<const uint16_t*>(scalar(reinterpret_cast<int64_t>(b.p)));
  k0 = scalar(k0), k1 = scalar(k1);
  constexpr int AHEAD = C::NS - 1;
  Stream<C::BM, C::NW, AKR> sa;
  Stream<C::BN, C::NW, BKR> sb;
  sa.init(a.ld, a_extent);
  sb.init(b.ld, b_extent);
  constexpr int NQ = sa.Q + sb.Q;
  static_assert(NQ * (AHEAD - 1) < 64, "vmcnt range");
  const int wid = threadIdx.x >> 6, wm = wid / C::WN, wn = wid % C::WN;
  Fragments<C::BM, C::MI, AKR> fa;
  Fragments<C::BN, C::NI, BKR> fb;
  fa.init(wm * C::MI * 32);
  fb.init(wn * C::NI * 32);
#pragma unroll
  for (int i = 0; i < C::MI; ++i)
#pragma unroll
    for (int j = 0; j < C::NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  const unsigned lds0 = lds_addr(lds);
  const int nk = k1 > k0 ? static_cast<int>((k1 - k0 + HK - 1) / HK) : 0, total = nk * TERMS;
  // the next stage to load: its slot, its place in the contraction, and its term
  int slot_in = 0, kt = 0, term = 0;
  auto issue = [&] {
    const int64_t k = k0 + static_cast<int64_t>(kt) * HK;
    const int lim = k1 - k < HK ? static_cast<int>(k1 - k) : HK;
    int64_t pa = 0, pb = 0;
    if constexpr (TERMS == 6) {   // (l h) (h l) (m m) (m h) (h m) (h h)
      pa = (term == 0 ? 2 : term == 2 || term == 3 ? 1 : 0) * a.part;
      pb = (term == 1 ? 2 : term == 2 || term == 4 ? 1 : 0) * b.part;
    } else if constexpr (TERMS == 2) {   // (m h) (h h)
      pa = (term == 0 ? 1 : 0) * a.part;
    }
    const unsigned at = lds0 + slot_in * C::STAGE;
    sa.issue(a.p + pa + (AKR ? k * a.ld : k), lim, at);
    sb.issue(b.p + pb + (BKR ? k * b.ld : k), lim, at + C::A_BYTES);
    slot_in = slot_in + 1 == C::NS ? 0 : slot_in + 1;
    if (++kt == nk) kt = 0, ++term;
  };
  auto compute = [&](const unsigned char* stage) {
    bf16x8_t af[2][C::MI], bf[2][C::NI];
    fa.load(stage, 0, af[0]);
    fb.load(stage + C::A_BYTES, 0, bf[0]);
#pragma unroll
    for (int ks = 0; ks < HK / 16; ++ks) {
      if (ks + 1 < HK / 16) {
        fa.load(stage, ks + 1, af[(ks + 1) & 1]);
        fb.load(stage + C::A_BYTES, ks + 1, bf[(ks + 1) & 1]);
      }
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int j = 0; j < C::NI; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[ks & 1][i], bf[ks & 1][j],
                                                              acc[i][j], 0, 0, 0);
    }
    // order: the first k-step's reads, then each k-step's MFMAs with the next one's reads between
    constexpr int RD = (AKR ? 2 : 1) * C::MI + (BKR ? 2 : 1) * C::NI, M = C::MI * C::NI;
    __builtin_amdgcn_sched_group_barrier(0x100, RD, 0);
#pragma unroll
    for (int ks = 0; ks + 1 < HK / 16; ++ks) sched_kstep<RD, M>();
    __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
  };
#pragma unroll
  for (int s = 0; s < AHEAD; ++s)
    if (s < total) issue();
  int slot = 0;
  for (int s = 0; s < total; ++s) {
    // in flight behind stage s: the loads of the AHEAD - 1 stages after it, where there are any
    if (AHEAD == 1 || s + AHEAD > total)
      wait_vmcnt<0>();
    else
      wait_vmcnt<(AHEAD - 1) * NQ>();
    raw_barrier();
    if (s + AHEAD < total) issue();
    compute(lds + slot * C::STAGE);
    slot = slot + 1 == C::NS ? 0 : slot + 1;
  }
  raw_barrier();   // every wave is done reading: LDS is the caller's
}

// Workgroup w of `total` to its place in an order of which each XCD takes a contiguous run
// (workgroup w runs on XCD w mod 8).
__device__ __forceinline__ int64_t xcd_order(int64_t w, int64_t total) {
  const int64_t q = total / 8, r = total % 8, x = w % 8;
  return x * q + (x < r ? x : r) + w / 8;
}

// ------------------------------------------------------------------------------ rows that count

constexpr int CHUNK = 1024;   // labels counted by one workgroup
constexpr int GROUP = 16;     // rows copied by one workgroup

struct RowsArgs {
  const void* X;
  int64_t x_stride;
  const int64_t* labels;
  int64_t ignore_index, N, V, d, dp;
  uint16_t* Xc;        // [parts][N][dp]
  int32_t* at;         // [N]: the row's place among those that count, or -1
  int32_t* rows;       // [N]: the rows that count
  int32_t* label;      // [N]: their labels, -1 outside the vocabulary
  int32_t* count;      // how many
  const int32_t* chunk;  // [chunks]: how many count in each chunk of labels
  float* loss;         // null, or [N]: zero for the rows that do not count
};

__global__ void __launch_bounds__(256) head_count_kernel(RowsArgs a, int32_t* chunk) {
  __shared__ int red[4];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * CHUNK;
  int n = 0;
#pragma unroll
  for (int i = 0; i < CHUNK / 256; ++i) {
    const int64_t r = first + i * 256 + threadIdx.x;
    n += __popcll(__ballot(r < a.N && a.labels[r < a.N ? r : 0] != a.ignore_index));
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) chunk[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// The three bf16 parts of an fp32 value (the rounding of the last one is 2^-24 of it at most).
__device__ __forceinline__ void split3(float x, uint16_t (&p)[3]) {
  p[0] = f32_to_bf16(x);
  const float r = x - bf16_to_f32(p[0]);
  p[1] = f32_to_bf16(r);
  p[2] = f32_to_bf16(r - bf16_to_f32(p[1]));
}

// One row of `n` elements to a row of np (a multiple of 8) bf16 ones, zeros behind; fp32 into three
// parts `part` elements apart.  `t` of `nt` threads.
template <class E>
__device__ __forceinline__ void copy_row(const E* src, int64_t n, uint16_t* dst, int64_t np,
                                         int64_t part, int t, int nt) {
  constexpr bool F32 = sizeof(E) == 4;
  const bool vec = n % 8 == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0;
  for (int64_t f = static_cast<int64_t>(t) * 8; f < np; f += nt * 8) {
    union { uint4 u[sizeof(E) / 2]; E e[8]; } w;
    if (vec) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(E) / 2); ++i)
        w.u[i] = reinterpret_cast<const uint4*>(src + f)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w.e[i] = f + i < n ? src[f + i] : E(0);
    }
    if constexpr (!F32) {
      *reinterpret_cast<uint4*>(dst + f) = w.u[0];
    } else {
      union { uint4 u; uint16_t e[8]; } o[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint16_t p[3];
        split3(w.e[i], p);
#pragma unroll
        for (int k = 0; k < 3; ++k) o[k].e[i] = p[k];
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(dst + k * part + f) = o[k].u;
    }
  }
}

template <class E>
__global__ void __launch_bounds__(256) head_rows_kernel(RowsArgs a) {
  __shared__ int red[4];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * GROUP;
  const int64_t c = first / CHUNK;
  int n = 0;
  if (a.chunk != nullptr)
    for (int64_t i = threadIdx.x; i < c; i += 256) n += a.chunk[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  for (int64_t i = c * CHUNK + (threadIdx.x >> 6) * 64; i < first; i += 256) {
    const int64_t r = i + (threadIdx.x & 63);
    n += __popcll(__ballot(r < first && a.labels[r < first ? r : 0] != a.ignore_index));
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  int place = red[0] + red[1] + red[2] + red[3];
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int g = 0; g < GROUP && first + g < a.N; ++g) {
    const int64_t r = first + g, y = a.labels[r];
    const bool keep = y != a.ignore_index;
    if (g % 4 == wid) {
      if (lane == 0) {
        a.at[r] = keep ? place : -1;
        if (keep) {
          a.rows[place] = static_cast<int32_t>(r);
          a.label[place] = y >= 0 && y < a.V ? static_cast<int32_t>(y) : -1;
        } else if (a.loss != nullptr) {
          a.loss[r] = 0.f;
        }
      }
      if (keep)
        copy_row(static_cast<const E*>(a.X) + r * a.x_stride, a.d, a.Xc + place * a.dp, a.dp,
                 a.N * a.dp, lane, 64);
    }
    place += keep;
  }
  if (first + GROUP >= a.N && threadIdx.x == 0) *a.count = place;
}

// A piece of W as the products take it: rows of dp elements, in three parts for fp32.
template <class E>
__global__ void __launch_bounds__(256) head_weight_kernel(const E* W, int64_t rows, int64_t d,
                                                          uint16_t* out, int64_t dp) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r < rows) copy_row(W + r * d, d, out + r * dp, dp, rows * dp, threadIdx.x & 63, 64);
}

// ------------------------------------------------------------------------------ logits

struct LogitsArgs {
  Side w, x;                 // [V of the piece][dp], [count][dp]
  const int32_t* count;
  const int32_t* label;
  int64_t N, V, v0, dp;      // v0: the piece's first entry; V: the piece's entries
  int64_t v_tiles;
  // forward: per vocabulary tile (of all pieces) and row
  float2* part;              // [tiles][N]: maximum of z log2(e), sum of 2^(z log2(e) - maximum)
  int64_t tile0;
  float* label_z;            // [N]: the label's z log2(e)
  // backward
  const float* lse;          // [N]: log2 of the row's sum of exponentials
  const float* up;           // null, or the rows' upstream gradients
  const int32_t* rows;
  uint16_t* dz;              // [parts][N][vp]
  int64_t vp;
  // dz as the caller's tensor: rows where they were, every factor applied
  const float* up_all;       // null, or the upstream gradient of all rows
  int mean;
  void* out;                 // [N of the rows that came][vp]
};

// What the gradients are multiplied with before their rounding: the upstream gradient of a mean or a
// sum (rows with upstream gradients of their own have those in dz).
__device__ __forceinline__ float gradient_scale(const float* up, int mean, int64_t count) {
  if (count == 0) return 0.f;
  const float u = up != nullptr ? *up : 1.f;
  return mean ? u / static_cast<float>(count) : u;
}

// Work item to (vocabulary tile, token tile): groups of 8 token tiles, whose rows stay in an XCD's
// L2 while the vocabulary goes by.
__device__ __forceinline__ bool logits_item(int64_t v_tiles, int64_t t_tiles, int64_t& vt,
                                            int64_t& tt) {
  const int64_t total = v_tiles * t_tiles, w = blockIdx.x;
  if (w >= total) return false;
  const int64_t i = xcd_order(w, total), per = 8 * v_tiles, g = i / per, r = i - g * per;
  const int64_t size = t_tiles - 8 * g < 8 ? t_tiles - 8 * g : 8;
  tt = 8 * g + r % size, vt = r / size;
  return true;
}

// The tile's entries behind the vocabulary: those at or past `left` rows from the lane's first.
template <class C>
__device__ __forceinline__ void behind(f32x16_t (&acc)[C::MI][C::NI], int left, float value) {
#pragma unroll
  for (int i = 0; i < C::MI; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool past = 32 * i + 8 * (e / 4) + e % 4 >= left;
#pragma unroll
      for (int j = 0; j < C::NI; ++j) acc[i][j][e] = past ? value : acc[i][j][e];
    }
}

// What becomes of a tile of logits: the forward pass's parts, dz for the products, or dz for the caller.
enum { FORWARD, GRADIENT, ROWS };

template <class C, int TERMS, int MODE>
__global__ void __launch_bounds__(C::NT, C::NT / 256) head_logits_kernel(LogitsArgs p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  const int64_t count = *p.count;
  int64_t vt, tt;
  if (!logits_item(p.v_tiles, (count + C::BN - 1) / C::BN, vt, tt)) return;
  const int64_t m0 = vt * C::BM, n0 = tt * C::BN;
  f32x16_t acc[C::MI][C::NI];
  Side a = p.w, b = p.x;
  a.p += m0 * a.ld, b.p += n0 * b.ld;
  product<C, false, false, TERMS>(a, p.V - m0, b, count - n0, 0, p.dp, lds, acc);

  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid % C::WN, half = lane >> 5;
  const int row0 = wm * C::MI * 32 + 4 * half;     // this lane's first row of the tile
  const bool ragged = m0 + C::BM > p.V;
#pragma unroll
  for (int j = 0; j < C::NI; ++j)
#pragma unroll
    for (int i = 0; i < C::MI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] *= LOG2E;
  if (ragged) behind<C>(acc, static_cast<int>(p.V - m0) - row0, -INFINITY);

  if constexpr (MODE == FORWARD) {
    float2* red = reinterpret_cast<float2*>(lds);   // [WM][BN]
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int col = (wn * C::NI + j) * 32 + (lane & 31);
      float m = acc[0][j][0];
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float ref = fmaxf(m, -3e38f);   // rows of -inf: exponentials of zero, no NaN
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(acc[i][j][e] - ref);
      s += __shfl_xor(s, 32, 64);
      if (half == 0) red[wm * C::BN + col] = make_float2(ref, s);
      const int64_t n = n0 + col;
      const int64_t rel = n < count ? p.label[n] - p.v0 - m0 - row0 : -1;
      const bool mine = rel >= 0 && rel < C::MI * 32 && (rel & 4) == 0;
      if (__ballot(mine)) {
#pragma unroll
        for (int i = 0; i < C::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (mine && rel == 32 * i + 8 * (e / 4) + e % 4) p.label_z[n] = acc[i][j][e];
      }
    }
    __syncthreads();
    for (int col = threadIdx.x; col < C::BN; col += C::NT) {
      if (n0 + col >= count) continue;
      float2 t = red[col];
#pragma unroll
      for (int w = 1; w < C::WM; ++w) {
        const float2 u = red[w * C::BN + col];
        const float m = fmaxf(t.x, u.x);
        t.y = t.y * __builtin_amdgcn_exp2f(t.x - m) + u.y * __builtin_amdgcn_exp2f(u.x - m);
        t.x = m;
      }
      p.part[(p.tile0 + vt) * p.N + n0 + col] = t;
    }
  } else {
    // dz in place of the logits, then through LDS to rows of BM entries; chunk c (8 entries) of
    // row r at slot c ^ r % CH, so that neither side of the turn meets in a bank
    constexpr int CH = C::BM / 8, PARTS = MODE == ROWS ? 1 : dz_parts<C>(TERMS > 1);
    static_assert(C::BN * C::BM * 2 <= C::LDS, "the tile of dz fits the stages");
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int64_t n = n0 + (wn * C::NI + j) * 32 + (lane & 31);
      const bool live = n < count;
      const int32_t y = live ? p.label[n] : 0;
      const float lse = live && y >= 0 ? p.lse[n] : NAN;
      float w = live && p.up != nullptr ? p.up[p.rows[n]] : 1.f;
      if constexpr (MODE == ROWS) w *= gradient_scale(p.up_all, p.mean, count);
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = w * __builtin_amdgcn_exp2f(acc[i][j][e] - lse);
      const int64_t rel = live ? y - p.v0 - m0 - row0 : -1;
      const bool mine = rel >= 0 && rel < C::MI * 32 && (rel & 4) == 0;
      if (__ballot(mine)) {
#pragma unroll
        for (int i = 0; i < C::MI; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (mine && rel == 32 * i + 8 * (e / 4) + e % 4) acc[i][j][e] -= w;
      }
    }
    if (ragged) behind<C>(acc, static_cast<int>(p.V - m0) - row0, 0.f);   // also where the row is NaN
    if constexpr (MODE == ROWS && TERMS > 1) {   // fp32, straight from the lanes
#pragma unroll
      for (int j = 0; j < C::NI; ++j) {
        const int64_t n = n0 + (wn * C::NI + j) * 32 + (lane & 31);
        if (n >= count) continue;
        float* out = static_cast<float*>(p.out) + p.rows[n] * p.vp + m0 + row0;
#pragma unroll
        for (int i = 0; i < C::MI; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (m0 + row0 + 32 * i + 8 * g < p.vp)
              *reinterpret_cast<float4*>(out + 32 * i + 8 * g) =
                  make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2],
                              acc[i][j][4 * g + 3]);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      if (k > 0) __syncthreads();
#pragma unroll
      for (int j = 0; j < C::NI; ++j) {
        const int r = (wn * C::NI + j) * 32 + (lane & 31);
#pragma unroll
        for (int i = 0; i < C::MI; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint2 u;
            u.x = pack_bf16x2(acc[i][j][4 * g], acc[i][j][4 * g + 1]);
            u.y = pack_bf16x2(acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
            const int c = (wm * C::MI + i) * 4 + g;
            *reinterpret_cast<uint2*>(lds + r * C::BM * 2 + ((c ^ (r & (CH - 1))) * 16) + half * 8) =
                u;
            if constexpr (PARTS > 1) {   // what the parts so far leave
              acc[i][j][4 * g] -= __uint_as_float(u.x << 16);
              acc[i][j][4 * g + 1] -= __uint_as_float(u.x & 0xFFFF0000u);
              acc[i][j][4 * g + 2] -= __uint_as_float(u.y << 16);
              acc[i][j][4 * g + 3] -= __uint_as_float(u.y & 0xFFFF0000u);
            }
          }
      }
      __syncthreads();
      uint16_t* out = MODE == ROWS ? static_cast<uint16_t*>(p.out) : p.dz + k * p.N * p.vp;
      for (int i = threadIdx.x; i < C::BN * CH; i += C::NT) {
        const int r = i / CH, c = i % CH;
        if (n0 + r >= count || (MODE == ROWS && m0 + c * 8 >= p.vp)) continue;
        const int64_t row = MODE == ROWS ? p.rows[n0 + r] : n0 + r;
        *reinterpret_cast<uint4*>(out + row * p.vp + m0 + c * 8) =
            *reinterpret_cast<const uint4*>(lds + r * C::BM * 2 + ((c ^ (r & (CH - 1))) * 16));
      }
    }
  }
}

// Each row's log2 of the sum of exponentials from the tiles' parts, and its loss; the losses' sum of
// 64 rows.  Four threads to a row, each over every fourth tile.
struct FinishArgs {
  const float2* part;
  const float* label_z;
  const int32_t* count;
  const int32_t* rows;
  const int32_t* label;
  int64_t N, tiles;
  float* lse;
  float* loss;       // null, or [N]
  float* sums;       // null, or [blocks]
};
__global__ void __launch_bounds__(256) head_finish_kernel(FinishArgs p) {
  __shared__ float2 red[4][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 64 + lane, count = *p.count;
  float2 t = make_float2(-3e38f, 0.f);
  if (n < count) {
#pragma unroll 4
    for (int64_t k = g; k < p.tiles; k += 4) {
      const float2 u = p.part[k * p.N + n];
      const float m = fmaxf(t.x, u.x);
      t.y = t.y * __builtin_amdgcn_exp2f(t.x - m) + u.y * __builtin_amdgcn_exp2f(u.x - m);
      t.x = m;
    }
  }
  red[g][lane] = t;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int k = 1; k < 4; ++k) {
    const float2 u = red[k][lane];
    const float m = fmaxf(t.x, u.x);
    t.y = t.y * __builtin_amdgcn_exp2f(t.x - m) + u.y * __builtin_amdgcn_exp2f(u.x - m);
    t.x = m;
  }
  float loss = 0.f;
  if (n < count) {
    const float lse = t.x + __log2f(t.y);
    loss = p.label[n] >= 0 ? LN2 * (lse - p.label_z[n]) : NAN;
    p.lse[n] = lse;
    if (p.loss != nullptr) p.loss[p.rows[n]] = loss;
  }
  if (p.sums != nullptr) {
    loss = wave_sum(loss);
    if (lane == 0) p.sums[blockIdx.x] = loss;
  }
}
__global__ void __launch_bounds__(256) head_total_kernel(const float* sums, int64_t n,
                                                         const int32_t* count, int mean,
                                                         float* out) {
  __shared__ float red[4];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 256) s += sums[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *out = mean ? s / static_cast<float>(*count) : s;
}

// Zeros in the rows that do not count: `row` 16-byte pieces each.
__global__ void __launch_bounds__(256) head_zero_rows_kernel(const int32_t* at, int64_t N, uint4* out,
                                                             int64_t row) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= N || at[r] >= 0) return;
  for (int64_t i = threadIdx.x & 63; i < row; i += 64) out[r * row + i] = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------------------ gradients

struct DxArgs {
  Side dz, w;              // [count][vp], [V of the piece][dp]
  const int32_t* count;
  int64_t N, V, dp;        // V: the piece's entries
  int64_t f_tiles, splits, kper;
  float* out;              // [splits][N][dp]
  int add;                 // to what is there
};
template <class C, int TERMS>
__global__ void __launch_bounds__(C::NT, C::NT / 256) head_dx_kernel(DxArgs p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  const int64_t count = *p.count, t_tiles = (count + C::BM - 1) / C::BM;
  const int64_t tiles = p.f_tiles * t_tiles, total = tiles * p.splits;
  if (blockIdx.x >= total) return;
  const int64_t i0 = xcd_order(blockIdx.x, total), split = i0 / tiles, r0 = i0 - split * tiles;
  const int64_t m0 = r0 / p.f_tiles * C::BM, n0 = r0 % p.f_tiles * C::BN;
  const int64_t k0 = split * p.kper, k1 = k0 + p.kper < p.V ? k0 + p.kper : p.V;
  f32x16_t acc[C::MI][C::NI];
  Side a = p.dz, b = p.w;
  a.p += m0 * a.ld, b.p += n0;
  product<C, false, true, TERMS>(a, count - m0, b, p.dp - n0, k0, k1, lds, acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid % C::WN;
  float* out = p.out + split * p.N * p.dp;
#pragma unroll
  for (int j = 0; j < C::NI; ++j) {
    const int64_t f = n0 + (wn * C::NI + j) * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < C::MI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t r = m0 + (wm * C::MI + i) * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        if (r < count && f < p.dp) {
          float* o = out + r * p.dp + f;
          *o = p.add ? *o + acc[i][j][e] : acc[i][j][e];
        }
      }
  }
}

// dx of every row: its sums over the splits, scaled and rounded once; zeros where it does not count.
template <class E>
__global__ void __launch_bounds__(256) head_dx_finish_kernel(
    const float* sums, int64_t splits, const int32_t* at, const int32_t* count, int64_t N, int64_t d,
    int64_t dp, const float* up, int mean, E* dx) {
  const float scale = gradient_scale(up, mean, *count);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= N) return;
  const int64_t j = at[r];
  for (int64_t f = threadIdx.x & 63; f < d; f += 64) {
    float s = 0.f;
    if (j >= 0)
      for (int64_t k = 0; k < splits; ++k) s += sums[(k * N + j) * dp + f];
    dx[r * d + f] = from_f32<E>(j >= 0 ? s * scale : 0.f);
  }
}

struct DwArgs {
  Side dz, x;              // [count][vp], [count][dp]: the contraction is their rows
  const int32_t* count;
  int64_t V, d, dp;        // V: the piece's entries
  int64_t v_tiles, f_tiles, splits, kper;
  const float* up;
  int mean;
  void* out;               // the piece's rows of dW; or with several splits [splits][V][d] fp32 sums
};
template <class C, int TERMS, class E>
__global__ void __launch_bounds__(C::NT, C::NT / 256) head_dw_kernel(DwArgs p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  const int64_t count = *p.count, tiles = p.v_tiles * p.f_tiles;
  const int64_t i0 = xcd_order(blockIdx.x, tiles * p.splits), split = i0 / tiles;
  const int64_t r0 = i0 - split * tiles;
  const int64_t m0 = r0 / p.f_tiles * C::BM, n0 = r0 % p.f_tiles * C::BN;
  const int64_t k0 = split * p.kper, k1 = k0 + p.kper < count ? k0 + p.kper : count;
  f32x16_t acc[C::MI][C::NI];
  Side a = p.dz, b = p.x;
  a.p += m0, b.p += n0;
  product<C, true, true, TERMS>(a, C::BM, b, p.dp - n0, k0, k1, lds, acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid % C::WN;
  const bool sums = p.splits > 1;
  const float scale = sums ? 1.f : gradient_scale(p.up, p.mean, count);
#pragma unroll
  for (int j = 0; j < C::NI; ++j) {
    const int64_t f = n0 + (wn * C::NI + j) * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < C::MI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t v = m0 + (wm * C::MI + i) * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        if (v >= p.V || f >= p.d) continue;
        if (sums)
          static_cast<float*>(p.out)[(split * p.V + v) * p.d + f] = acc[i][j][e];
        else
          static_cast<E*>(p.out)[v * p.d + f] = from_f32<E>(acc[i][j][e] * scale);
      }
  }
}
template <class E>
__global__ void __launch_bounds__(256) head_dw_finish_kernel(const float* sums, int64_t splits,
                                                             int64_t n, const int32_t* count,
                                                             const float* up, int mean, E* out) {
  const float scale = gradient_scale(up, mean, *count);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int64_t k = 0; k < splits; ++k) s += sums[k * n + i];
  out[i] = from_f32<E>(s * scale);
}

// ------------------------------------------------------------------------------ host side

constexpr int64_t PIECE_BYTES = int64_t{512} << 20;   // of dz
constexpr int64_t FEW_ROWS = 32;
constexpr int64_t SLOTS = 512;      // workgroups that a product is split into at least

struct Plan {
  bool f32, few, copy_w;
  int64_t parts, dz_parts;   // bf16 parts of the operands, and of dz
  int64_t dp, cols, pieces, v_tiles_all;   // cols: vocabulary entries of a piece
  int64_t chunks, blocks;
  int64_t dx_splits, dx_kper, dw_splits, dw_kper;
};

int check_head(const gs_head* h, const char* what) {
  if (h == nullptr) return fail(GS_ERR_INVALID, std::string(what) + ": no arguments");
  if (h->dtype != GS_DTYPE_BF16 && h->dtype != GS_DTYPE_F32)
    return fail(GS_ERR_DTYPE, std::string(what) + ": dtype must be bf16 or fp32");
  if (h->N <= 0 || h->V <= 0 || h->d <= 0 || h->X == nullptr || h->W == nullptr ||
      h->labels == nullptr || h->x_stride < h->d || h->reduction < GS_REDUCE_NONE ||
      h->reduction > GS_REDUCE_MEAN)
    return fail(GS_ERR_INVALID, std::string(what) + ": invalid arguments");
  if (h->N > (int64_t{1} << 30) || h->V > (int64_t{1} << 30) || h->d > (int64_t{1} << 20))
    return fail(GS_ERR_UNSUPPORTED,
                std::string(what) + ": more than 2^30 rows or vocabulary entries, or 2^20 features");
  return GS_OK;
}

// The plan of a call.  `h` with null pointers is fine.
Plan plan_of(const gs_head& h, bool w_aligned) {
  Plan p{};
  p.f32 = h.dtype == GS_DTYPE_F32;
  p.parts = p.f32 ? 3 : 1;
  p.dp = round_up(h.d, 8);
  p.copy_w = p.f32 || h.d % 8 != 0 || !w_aligned;
  p.few = h.N <= FEW_ROWS;
  p.dz_parts = p.few ? dz_parts<Few>(p.f32) : dz_parts<Wide>(p.f32);
  const int64_t tile = p.few ? Few::BM : Wide::BM;
  const int64_t all = cdiv(h.V, tile);
  const int64_t per = std::max<int64_t>(1, PIECE_BYTES / (h.N * 2 * p.dz_parts * tile));
  p.pieces = cdiv(all, per);
  p.cols = cdiv(all, p.pieces) * tile;
  p.pieces = cdiv(h.V, p.cols);
  p.v_tiles_all = 0;
  for (int64_t i = 0; i < p.pieces; ++i)
    p.v_tiles_all += cdiv(std::min(p.cols, h.V - i * p.cols), tile);
  p.chunks = h.N > CHUNK ? cdiv(h.N, CHUNK) : 0;
  p.blocks = cdiv(h.N, 64);
  // dx: the piece split until every workgroup slot has a share of at least 256 entries
  const int64_t xt = p.few ? cdiv(h.N, FewT::BM) * cdiv(p.dp, FewT::BN)
                           : cdiv(h.N, Wide::BM) * cdiv(p.dp, Wide::BN);
  const int64_t most = std::min(p.cols, h.V);
  p.dx_splits = std::max<int64_t>(1, std::min(SLOTS / 2 / xt, cdiv(most, 256)));
  p.dx_kper = round_up(cdiv(most, p.dx_splits), HK);
  p.dx_splits = cdiv(most, p.dx_kper);
  const int64_t wt = cdiv(most, tile) * cdiv(h.d, p.few ? Few::BN : Wide::BN);
  p.dw_splits = std::max<int64_t>(1, std::min(SLOTS / 2 / wt, cdiv(h.N, 256)));
  p.dw_kper = round_up(cdiv(h.N, p.dw_splits), HK);
  p.dw_splits = cdiv(h.N, p.dw_kper);
  return p;
}

struct Buffers {
  uint16_t *xc, *wc, *dz;
  int32_t *at, *rows, *label, *count, *chunk;
  float2* part;
  float *label_z, *sums, *dx, *dw;
};
template <class S>
Buffers carve(S& s, const gs_head& h, const Plan& p, bool grad) {
  Buffers b{};
  b.xc = s.template take<uint16_t>(p.parts * h.N * p.dp);
  b.at = s.template take<int32_t>(h.N);
  b.rows = s.template take<int32_t>(h.N);
  b.label = s.template take<int32_t>(h.N);
  b.count = s.template take<int32_t>(1);
  b.chunk = s.template take<int32_t>(std::max<int64_t>(1, p.chunks));
  if (p.copy_w) b.wc = s.template take<uint16_t>(p.parts * std::min(p.cols, h.V) * p.dp);
  if (!grad) {
    b.part = s.template take<float2>(p.v_tiles_all * h.N);
    b.label_z = s.template take<float>(h.N);
    b.sums = s.template take<float>(p.blocks);
  } else {
    b.dz = s.template take<uint16_t>(p.dz_parts * h.N * p.cols);
    b.dx = s.template take<float>(p.dx_splits * h.N * p.dp);
    if (p.dw_splits > 1) b.dw = s.template take<float>(p.dw_splits * std::min(p.cols, h.V) * h.d);
  }
  return b;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

unsigned grid_of(int64_t n) { return static_cast<unsigned>(n); }

void launch_rows(const gs_head& h, const Plan& p, const Buffers& b, float* loss, hipStream_t s) {
  RowsArgs a{};
  a.X = h.X, a.x_stride = h.x_stride, a.labels = h.labels, a.ignore_index = h.ignore_index;
  a.N = h.N, a.V = h.V, a.d = h.d, a.dp = p.dp;
  a.Xc = b.xc, a.at = b.at, a.rows = b.rows, a.label = b.label, a.count = b.count;
  a.chunk = p.chunks > 0 ? b.chunk : nullptr;
  a.loss = loss;
  if (p.chunks > 0)
    hipLaunchKernelGGL(head_count_kernel, dim3(grid_of(p.chunks)), dim3(256), 0, s, a, b.chunk);
  const dim3 grid(grid_of(cdiv(h.N, GROUP)));
  if (p.f32)
    hipLaunchKernelGGL(head_rows_kernel<float>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(head_rows_kernel<uint16_t>, grid, dim3(256), 0, s, a);
}

// W's rows [v0, v0 + n) as the products take them.
Side weight_side(const gs_head& h, const Plan& p, const Buffers& b, int64_t v0, int64_t n,
                 hipStream_t s) {
  if (!p.copy_w) return Side{static_cast<const uint16_t*>(h.W) + v0 * h.d, h.d, 0};
  const dim3 grid(grid_of(cdiv(n, 4)));
  if (p.f32)
    hipLaunchKernelGGL(head_weight_kernel<float>, grid, dim3(256), 0, s,
                       static_cast<const float*>(h.W) + v0 * h.d, n, h.d, b.wc, p.dp);
  else
    hipLaunchKernelGGL(head_weight_kernel<uint16_t>, grid, dim3(256), 0, s,
                       static_cast<const uint16_t*>(h.W) + v0 * h.d, n, h.d, b.wc, p.dp);
  return Side{b.wc, p.dp, n * p.dp};
}

template <class C, int MODE>
void launch_logits(const LogitsArgs& a, bool f32, hipStream_t s) {
  const dim3 grid(grid_of(a.v_tiles * cdiv(a.N, C::BN)));
  if (f32)
    hipLaunchKernelGGL((head_logits_kernel<C, 6, MODE>), grid, dim3(C::NT), 0, s, a);
  else
    hipLaunchKernelGGL((head_logits_kernel<C, 1, MODE>), grid, dim3(C::NT), 0, s, a);
}
template <class C>
void launch_dx(const DxArgs& a, bool f32, hipStream_t s) {
  const dim3 grid(grid_of(a.f_tiles * cdiv(a.N, C::BM) * a.splits));
  if (f32)
    hipLaunchKernelGGL((head_dx_kernel<C, 6>), grid, dim3(C::NT), 0, s, a);
  else
    hipLaunchKernelGGL((head_dx_kernel<C, C::BM == FewT::BM ? 2 : 1>), grid, dim3(C::NT), 0, s, a);
}
template <class C>
void launch_dw(const DwArgs& a, bool f32, hipStream_t s) {
  const dim3 grid(grid_of(a.v_tiles * a.f_tiles * a.splits));
  if (f32)
    hipLaunchKernelGGL((head_dw_kernel<C, 6, float>), grid, dim3(C::NT), 0, s, a);
  else
    hipLaunchKernelGGL((head_dw_kernel<C, dz_parts<C>(false), uint16_t>), grid, dim3(C::NT), 0, s, a);
}

// The larger of the grids of a call (workgroups).
bool grids_fit(const gs_head& h, const Plan& p) {
  const int64_t t = cdiv(h.N, p.few ? Few::BN : Wide::BN);
  const int64_t v = cdiv(p.cols, p.few ? Few::BM : Wide::BM);
  return v * t < INT32_MAX && v * cdiv(h.d, 32) * p.dw_splits < INT32_MAX;
}

LogitsArgs logits_args(const gs_head& h, const Plan& p, const Buffers& b) {
  LogitsArgs a{};
  a.x = Side{b.xc, p.dp, h.N * p.dp};
  a.count = b.count, a.label = b.label, a.rows = b.rows;
  a.N = h.N, a.dp = p.dp;
  return a;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_head_loss_workspace(const gs_head* h) {
  if (check_head(h, "gs_head_loss") != GS_OK) return 0;
  Sizer s;
  carve(s, *h, plan_of(*h, aligned16(h->W)), false);
  return s.used + 256;
}

extern "C" int gs_head_loss(const gs_head* h, float* out_loss, float* lse, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int rc = check_head(h, "gs_head_loss")) return rc;
  if (out_loss == nullptr || lse == nullptr)
    return fail(GS_ERR_INVALID, "gs_head_loss: no place for the loss");
  const Plan p = plan_of(*h, aligned16(h->W));
  if (!grids_fit(*h, p)) return fail(GS_ERR_UNSUPPORTED, "gs_head_loss: grid too large");
  Carver c(workspace, workspace_bytes);
  const Buffers b = carve(c, *h, p, false);
  if (workspace == nullptr || !c.ok())
    return fail(GS_ERR_WORKSPACE, "gs_head_loss: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool rows = h->reduction == GS_REDUCE_NONE;
  launch_rows(*h, p, b, rows ? out_loss : nullptr, s);
  LogitsArgs a = logits_args(*h, p, b);
  a.part = b.part, a.label_z = b.label_z;
  for (int64_t v0 = 0; v0 < h->V; v0 += p.cols) {
    a.v0 = v0, a.V = std::min(p.cols, h->V - v0);
    a.w = weight_side(*h, p, b, v0, a.V, s);
    a.v_tiles = cdiv(a.V, p.few ? Few::BM : Wide::BM);
    if (p.few)
      launch_logits<Few, FORWARD>(a, p.f32, s);
    else
      launch_logits<Wide, FORWARD>(a, p.f32, s);
    a.tile0 += a.v_tiles;
  }
  FinishArgs f{};
  f.part = b.part, f.label_z = b.label_z, f.count = b.count, f.rows = b.rows, f.label = b.label;
  f.N = h->N, f.tiles = a.tile0, f.lse = lse;
  f.loss = rows ? out_loss : nullptr;
  f.sums = rows ? nullptr : b.sums;
  hipLaunchKernelGGL(head_finish_kernel, dim3(grid_of(p.blocks)), dim3(256), 0, s, f);
  if (!rows)
    hipLaunchKernelGGL(head_total_kernel, dim3(1), dim3(256), 0, s, b.sums, p.blocks, b.count,
                       h->reduction == GS_REDUCE_MEAN, out_loss);
  return check_launch("gs_head_loss");
}

extern "C" size_t gs_head_grad_workspace(const gs_head* h) {
  if (check_head(h, "gs_head_grad") != GS_OK) return 0;
  Sizer s;
  carve(s, *h, plan_of(*h, aligned16(h->W)), true);
  return s.used + 256;
}

extern "C" int gs_head_grad(const gs_head* h, const float* lse, const float* upstream, void* dx,
                            void* dw, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_head(h, "gs_head_grad")) return rc;
  if (lse == nullptr) return fail(GS_ERR_INVALID, "gs_head_grad: the forward pass's sums are missing");
  const Plan p = plan_of(*h, aligned16(h->W));
  if (!grids_fit(*h, p)) return fail(GS_ERR_UNSUPPORTED, "gs_head_grad: grid too large");
  Carver c(workspace, workspace_bytes);
  const Buffers b = carve(c, *h, p, true);
  if (workspace == nullptr || !c.ok())
    return fail(GS_ERR_WORKSPACE, "gs_head_grad: workspace too small");
  if (dx == nullptr && dw == nullptr) return GS_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int mean = h->reduction == GS_REDUCE_MEAN;
  const bool own = h->reduction == GS_REDUCE_NONE;   // upstream gradients of the rows' own
  const float* up = own ? nullptr : upstream;
  launch_rows(*h, p, b, nullptr, s);
  LogitsArgs a = logits_args(*h, p, b);
  a.lse = lse, a.up = own ? upstream : nullptr, a.dz = b.dz;
  for (int64_t v0 = 0; v0 < h->V; v0 += p.cols) {
    a.v0 = v0, a.V = std::min(p.cols, h->V - v0);
    a.w = weight_side(*h, p, b, v0, a.V, s);
    a.v_tiles = cdiv(a.V, p.few ? Few::BM : Wide::BM);
    a.vp = p.cols;
    if (p.few)
      launch_logits<Few, GRADIENT>(a, p.f32, s);
    else
      launch_logits<Wide, GRADIENT>(a, p.f32, s);
    const Side dz{b.dz, p.cols, h->N * p.cols};
    if (dx != nullptr) {
      DxArgs x{};
      x.dz = dz, x.w = a.w, x.count = b.count, x.N = h->N, x.V = a.V, x.dp = p.dp;
      x.f_tiles = cdiv(p.dp, p.few ? FewT::BN : Wide::BN);
      x.splits = p.dx_splits, x.kper = p.dx_kper, x.out = b.dx, x.add = v0 > 0;
      if (p.few)
        launch_dx<FewT>(x, p.f32, s);
      else
        launch_dx<Wide>(x, p.f32, s);
    }
    if (dw != nullptr) {
      DwArgs w{};
      w.dz = dz, w.x = a.x, w.count = b.count, w.V = a.V, w.d = h->d, w.dp = p.dp;
      w.v_tiles = a.v_tiles, w.f_tiles = cdiv(h->d, p.few ? Few::BN : Wide::BN);
      w.splits = p.dw_splits, w.kper = p.dw_kper, w.up = up, w.mean = mean;
      void* out = static_cast<char*>(dw) + v0 * h->d * static_cast<int64_t>(elem_size(h->dtype));
      w.out = p.dw_splits > 1 ? b.dw : out;
      if (p.few)
        launch_dw<Few>(w, p.f32, s);
      else
        launch_dw<Wide>(w, p.f32, s);
      if (p.dw_splits > 1) {
        const int64_t n = a.V * h->d;
        const dim3 grid(grid_of(cdiv(n, 256)));
        if (p.f32)
          hipLaunchKernelGGL(head_dw_finish_kernel<float>, grid, dim3(256), 0, s, b.dw, p.dw_splits,
                             n, b.count, up, mean, static_cast<float*>(out));
        else
          hipLaunchKernelGGL(head_dw_finish_kernel<uint16_t>, grid, dim3(256), 0, s, b.dw,
                             p.dw_splits, n, b.count, up, mean, static_cast<uint16_t*>(out));
      }
    }
  }
  if (dx != nullptr) {
    const dim3 grid(grid_of(cdiv(h->N, 4)));
    if (p.f32)
      hipLaunchKernelGGL(head_dx_finish_kernel<float>, grid, dim3(256), 0, s, b.dx, p.dx_splits, b.at,
                         b.count, h->N, h->d, p.dp, up, mean, static_cast<float*>(dx));
    else
      hipLaunchKernelGGL(head_dx_finish_kernel<uint16_t>, grid, dim3(256), 0, s, b.dx, p.dx_splits,
                         b.at, b.count, h->N, h->d, p.dp, up, mean, static_cast<uint16_t*>(dx));
  }
  return check_launch("gs_head_grad");
}

// A call for one piece of dz has a plan of its own: the piece is the vocabulary.
static Plan piece_plan(const gs_head& h, int64_t n, bool w_aligned) {
  gs_head piece = h;
  piece.V = n;
  Plan p = plan_of(piece, w_aligned);
  p.cols = round_up(n, p.few ? Few::BM : Wide::BM);
  return p;
}
static bool piece_aligned(const gs_head& h, int64_t v0) {
  return h.W != nullptr &&
         aligned16(static_cast<const char*>(h.W) + v0 * h.d * static_cast<int64_t>(elem_size(h.dtype)));
}
template <class S>
static Buffers carve_piece(S& s, const gs_head& h, int64_t n, const Plan& p) {
  gs_head piece = h;
  piece.V = n;
  Buffers b{};
  b.xc = s.template take<uint16_t>(p.parts * h.N * p.dp);
  b.at = s.template take<int32_t>(h.N);
  b.rows = s.template take<int32_t>(h.N);
  b.label = s.template take<int32_t>(h.N);
  b.count = s.template take<int32_t>(1);
  b.chunk = s.template take<int32_t>(std::max<int64_t>(1, p.chunks));
  if (p.copy_w) b.wc = s.template take<uint16_t>(p.parts * n * p.dp);
  return b;
}

extern "C" size_t gs_head_logit_grad_workspace(const gs_head* h, int64_t v0, int64_t n) {
  if (check_head(h, "gs_head_logit_grad") != GS_OK || v0 < 0 || n <= 0 || n > h->V - v0) return 0;
  Sizer s;
  carve_piece(s, *h, n, piece_plan(*h, n, piece_aligned(*h, v0)));
  return s.used + 256;
}

extern "C" int gs_head_logit_grad(const gs_head* h, const float* lse, const float* upstream, int64_t v0,
                                  int64_t n, void* out, int64_t out_stride, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (const int rc = check_head(h, "gs_head_logit_grad")) return rc;
  if (lse == nullptr || out == nullptr || !aligned16(out) || v0 < 0 || n <= 0 || n > h->V - v0 ||
      out_stride != round_up(n, 8))
    return fail(GS_ERR_INVALID, "gs_head_logit_grad: invalid arguments");
  const Plan p = piece_plan(*h, n, piece_aligned(*h, v0));
  if (!grids_fit(*h, p))
    return fail(GS_ERR_UNSUPPORTED, "gs_head_logit_grad: grid too large");
  Carver c(workspace, workspace_bytes);
  const Buffers b = carve_piece(c, *h, n, p);
  if (workspace == nullptr || !c.ok())
    return fail(GS_ERR_WORKSPACE, "gs_head_logit_grad: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  launch_rows(*h, p, b, nullptr, s);
  const bool own = h->reduction == GS_REDUCE_NONE;
  LogitsArgs a = logits_args(*h, p, b);
  a.lse = lse, a.up = own ? upstream : nullptr, a.up_all = own ? nullptr : upstream;
  a.mean = h->reduction == GS_REDUCE_MEAN;
  a.v0 = v0, a.V = n, a.vp = out_stride, a.out = out;
  a.w = weight_side(*h, p, b, v0, n, s);
  a.v_tiles = cdiv(n, p.few ? Few::BM : Wide::BM);
  if (p.few)
    launch_logits<Few, ROWS>(a, p.f32, s);
  else
    launch_logits<Wide, ROWS>(a, p.f32, s);
  hipLaunchKernelGGL(head_zero_rows_kernel, dim3(grid_of(cdiv(h->N, 4))), dim3(256), 0, s, b.at, h->N,
                     static_cast<uint4*>(out), out_stride * static_cast<int64_t>(elem_size(h->dtype)) / 16);
  return check_launch("gs_head_logit_grad");
}
