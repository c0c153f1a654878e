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
// Bound by the matrix cores but for a few rows, which are bound by W's memory.  18432 of 20480 rows of
// GPT-2's output projection (768 features, 50257 entries, bf16) 5.25 to 5.6 ms for 5.69 TFLOP, a stage of
// 256 x 256 x 64 in 1.48 us on every compute unit (1.45 PFLOP/s); the rest is the tiles' ends, 6 us with
// their exponentials and 11 with those and dz's writing, and the units that the last round of tiles leaves
// (dx's 72 x 3).  Matrix cores busy 56% of the forward product's cycles, 49% of dz's, 49% of dx's, 69% of
// dW's, at 1.7 to 1.9 GHz.  Eight rows 90 us: W read in 14 to 15 us three times, dW written in 19.
//
// Rows that do not count (label ignore_index) take no part in any product: the rows that do are
// listed first, in order, and copied next to each other (with rows of a multiple of 8 features,
// which the 16-byte loads need).  Their number stays on the device; tiles past it end at once.
//
// fp32 operands of many rows are taken as three bf16 parts each, x = h + m + l with 8 bits apiece, and a
// product as the six products of parts above 2^-24 of it, accumulated in fp32 like the bf16 one: the
// same kernels over six times the contraction, which at the bf16 matrix rate is still faster than fp32
// matrix instructions.  A few rows are bound by W's memory, and take it as it is, on those.
//
// Tiles: BM x BN outputs, 64 of the contraction a stage, staged through LDS by wave-level DMA
// of 16 bytes a lane (4 where a weight's rows are off 16-byte boundaries), MFMA 32x32x16 (fp32 accumulators).  A side whose contraction index is contiguous
// in memory (KC) is read from LDS as 16-byte fragments, one whose contraction index is the row
// (KR) through the transpose read.  Result layout of the MFMA: lane l, element e is row
// 8 (e / 4) + 4 (l / 32) + e % 4 of the A side, column l % 32 of the B side.

#include <algorithm>
#include <type_traits>

#include "gs_common.h"

namespace gs {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

constexpr unsigned OOB = 0x80000000u;  // past every buffer range: such lanes load zeros
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

__device__ __forceinline__ unsigned lds_addr(const void* p) {
  typedef const __attribute__((address_space(3))) unsigned char* lds_ptr;
  return static_cast<unsigned>(reinterpret_cast<uintptr_t>((lds_ptr)p));
}
// 64 lanes' G (16 or 4) bytes at base + voff to LDS address lds + G lane.  Nothing else here uses M0.
template <int G>
__device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t r, unsigned voff, unsigned lds) {
  if constexpr (G == 16)
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(voff), "s"(r)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dword %1, %2, 0 offen lds"
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
// The builtin, not assembly: the compiler has to know that the fragments are there, or it waits for later
// reads with them.
__device__ __forceinline__ void wait_lgkmcnt0() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
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

// WM x WN waves of MI x NI blocks of 32 x 32; NS slots for stages of K of the contraction.
template <int WM_, int WN_, int MI_, int NI_, int NS_, int K_ = 64>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MI = MI_, NI = NI_, NS = NS_, K = K_;
  static constexpr int NW = WM * WN, NT = 64 * NW;
  static constexpr int BM = WM * MI * 32, BN = WN * NI * 32;
  static constexpr int A_BYTES = BM * K * 2, STAGE = (BM + BN) * K * 2;
  // Two slots of equal sides are five halves: see product.
  static constexpr bool HALVES = NS == 2 && BM == BN;
  static constexpr int LDS = HALVES ? 5 * A_BYTES : NS * STAGE;
};
constexpr int FEW_K = 32;
using Wide = Tile<2, 4, 4, 2, 2>;    // 256 x 256, eight waves of 128 x 64
using Mid = Tile<2, 2, 2, 2, 2>;     // 128 x 128, four waves of 64 x 64, two workgroups to a unit
using Small = Tile<2, 2, 1, 1, 4>;   // 64 x 64, four waves of 32 x 32
using Few = Tile<4, 1, 1, 1, 4>;     // 128 x 32
using FewT = Tile<1, 4, 1, 1, 4>;    // 32 x 128
using FewT2 = Tile<1, 4, 2, 1, 4>;   // 64 x 128
using FewW = Tile<4, 1, 2, 2, 2, FEW_K>;   // 256 x 64: whole rows of dW leave at a time
constexpr int FEW_ROWS = 32;

// The bf16 parts that dz is held in between the products: three for fp32 (of a few rows fp32 itself); two
// of a few rows, whose products are bound by W's and dW's memory (rounded once, a label's p - 1 would be
// most of dW's error); one beyond.
template <class C>
__host__ __device__ constexpr int dz_parts(bool f32) {
  return f32 ? 3 : C::BN == Few::BN ? 2 : 1;
}

// One side of a product: the tile's first element, the stride between rows (of the side with
// KC, of the contraction with KR) and between the bf16 parts of an fp32 operand, in elements.
struct Side {
  const unsigned char* p;
  int64_t ld, part;
  // `i` elements of ES bytes further on.
  template <int ES>
  __device__ __forceinline__ void move(int64_t i) { p += i * ES; }
};
Side side_of(const void* p, int64_t ld, int64_t part) {
  return Side{static_cast<const unsigned char*>(p), ld, part};
}

// The DMA of one side's stages.  KC: LDS row r (K elements) holds its 16-byte chunk c at slot c ^ swz(r),
// so that the 16 rows of a fragment read lie in 16 different bank groups.  KR: LDS row = contraction
// index, chunk c at slot c ^ swz(row): the 4 rows x 4 chunks of a transpose read in 16 different ones.
// A stage is as many bytes with elements of 4 (ES) as with those of 2: half the contraction.
// G: the bytes of a lane's load; rows that do not begin at multiples of 16 bytes are loaded by 4.
template <int B, int NW, bool KR, int K, int ES, int G>
struct Stream {
  static constexpr int P = 16 / G, Q = B * K * 2 / 1024 / NW * P;   // loads of a wave
  static_assert(Q > 0 && B * K * 2 % (1024 * NW) == 0, "stage bytes split over waves");
  static constexpr int RB = KR ? B * ES : K * 2, CH = RB / 16;   // bytes and chunks of an LDS row
  static constexpr int VE = 16 / ES;                             // elements of a chunk
  __device__ static constexpr int swz(int r) {
    if (KR) return ES == 4 ? 0 : CH >= 16 ? 4 * (r & 3) : CH == 8 ? 4 * ((r >> 1) & 1) : 0;
    return CH == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
  }
  // Where load q of a wave begins, from the wave's first.
  __device__ static constexpr int at(int q) { return NW * (q / P) * 1024 + q % P * 64 * G; }
  unsigned off[Q];
  int k[Q];
  // `extent`: how many of the side's rows (columns of memory with KR) there are from the tile's
  // first on.
  __device__ __forceinline__ void init(int64_t ld, int64_t extent) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int byte = wid * 1024 + at(q) + lane * G;
      const int r = byte / RB, c = (byte % RB) / 16 ^ swz(r), e = c * VE + byte % 16 / ES;
      k[q] = KR ? r : e;
      off[q] = (KR ? e : r) < extent ? static_cast<unsigned>((r * ld + e) * ES) : OOB;
    }
  }
  // The stage whose first element is at `base` to the LDS address `lds` (of this wave's first load);
  // contraction indices at or past `lim` as zeros.
  __device__ __forceinline__ void issue(const unsigned char* base, unsigned lds) const {
    const __amdgpu_buffer_rsrc_t r = rsrc(base);
#pragma unroll
    for (int q = 0; q < Q; ++q) dma<G>(r, off[q], lds + at(q));
  }
  __device__ __forceinline__ void issue_cut(const unsigned char* base, unsigned lds, int lim) const {
    const __amdgpu_buffer_rsrc_t r = rsrc(base);
#pragma unroll
    for (int q = 0; q < Q; ++q) dma<G>(r, k[q] < lim ? off[q] : OOB, lds + at(q));
  }
};

// Order of a k-step: its M MFMAs, with the next k-step's RD reads spread between them.
template <int RD, int M, int G = 0>
__device__ __forceinline__ void sched_kstep() {
  __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
  constexpr int n = (RD * (G + 1)) / M - (RD * G) / M;
  if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x100, n, 0);
  if constexpr (G + 1 < M) sched_kstep<RD, M, G + 1>();
}

// The fragments of one side: F blocks of 32 rows from row `first` on, k-step ks (32 bytes of every row) of
// the stage.  bf16: a lane holds 8 of a k-step's 16 elements; fp32: 4 of its 8, those from 4 (lane / 32) on,
// whichever way they lie, one for each of four MFMAs.
template <int B, int F, bool KR, int K, int ES>
struct Fragments {
  using S = Stream<B, 1, KR, K, ES, 16>;
  int at[KR ? F : 1];
  int lo, hi;
  __device__ __forceinline__ void init(int first) {
    const int lane = threadIdx.x & 63;
    lo = hi = 0;
    if constexpr (KR && ES == 4) {
#pragma unroll
      for (int i = 0; i < F; ++i) at[i] = 4 * (lane >> 5) * S::RB + (first + i * 32 + (lane & 31)) * 4;
    } else if constexpr (KR) {
      const int g = lane >> 4, row = 8 * (g >> 1) + ((lane >> 2) & 3);
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int col = first + i * 32 + 16 * (g & 1) + 4 * (lane & 3);
        at[i] = row * S::RB + ((col >> 3) ^ S::swz(row)) * 16 + (col & 7) * 2;
      }
    } else {
      at[0] = (first + (lane & 31)) * S::RB;
      lo = S::swz(lane & 31), hi = lane >> 5;   // blocks start at multiples of 32 rows
    }
  }
  __device__ __forceinline__ void load(const unsigned char* side, int ks, f32x4_t (&f)[F]) const {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if constexpr (KR && ES == 4) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          f[i][q] = *reinterpret_cast<const float*>(side + at[i] + (8 * ks + q) * S::RB);
      } else if constexpr (KR) {
        const unsigned char* p = side + at[i] + ks * 16 * S::RB;
        f[i] = __builtin_bit_cast(
            f32x4_t, __builtin_shufflevector(lds_tr16(p), lds_tr16(p + 4 * S::RB), 0, 1, 2, 3, 4, 5, 6,
                                             7));
      } else {
        f[i] = *reinterpret_cast<const f32x4_t*>(side + at[0] + i * 32 * S::RB +
                                                 ((2 * ks + hi) ^ lo) * 16);
      }
    }
  }
};

// Which products a product is made of: the operands as they are; of dz in two parts on one side; of three
// parts on both, of which six count, the small ones first; of fp32 operands as they are, on fp32 MFMAs.
enum Terms { ONE = 1, TWO_B = 2, SIX = 6, FULL = 7 };
constexpr int size_of(int terms) { return terms == FULL ? 4 : 2; }   // of an operand's element
constexpr int terms_in(int terms) { return terms == FULL ? 1 : terms; }

// acc = sum over the contraction [k0, k1) of A B^T.
//
// The waves meet once a stage, before its last k-step's MFMAs: by then every wave holds that step's
// fragments, so the stage's slot can be loaded again, and the next stage has arrived, so its first
// fragments are read while those MFMAs run.  (Meeting between the stages left the matrix cores idle
// for the loads' issue and the first reads' latency.)
template <class C, bool AKR, bool BKR, int TERMS, int GA = 16, int GB = 16>
__device__ __forceinline__ void product(Side a, int64_t a_extent, Side b, int64_t b_extent,
                                        int64_t k0, int64_t k1, unsigned char* lds,
                                        f32x16_t (&acc)[C::MI][C::NI]) {
  a.p = reinterpret_cast<const unsigned char*>(scalar(reinterpret_cast<int64_t>(a.p)));
  b.p = reinterpret_cast<const unsigned char*>(scalar(reinterpret_cast<int64_t>(b.p)));
  k0 = scalar(k0), k1 = scalar(k1);
  constexpr int ES = size_of(TERMS), KE = C::K * 2 / ES;   // contraction of a stage
  constexpr int KS = C::K / 16;                            // k-steps of a stage
  static_assert(KS % 2 == 0, "the fragments' two buffers take turns");
  Stream<C::BM, C::NW, AKR, C::K, ES, GA> sa;
  Stream<C::BN, C::NW, BKR, C::K, ES, GB> sb;
  sa.init(a.ld, a_extent);
  sb.init(b.ld, b_extent);
  constexpr int NQ = sa.Q + sb.Q;
  static_assert(NQ * (C::NS - 2) < 64, "vmcnt range");
  const int wid = threadIdx.x >> 6, wm = wid / C::WN, wn = wid % C::WN;
  Fragments<C::BM, C::MI, AKR, C::K, ES> fa;
  Fragments<C::BN, C::NI, BKR, C::K, ES> fb;
  fa.init(wm * C::MI * 32);
  fb.init(wn * C::NI * 32);
#pragma unroll
  for (int i = 0; i < C::MI; ++i)
#pragma unroll
    for (int j = 0; j < C::NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  const unsigned lds0 =
      lds_addr(lds) + static_cast<unsigned>(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 1024u;
  const int nk = k1 > k0 ? static_cast<int>((k1 - k0 + KE - 1) / KE) : 0;
  const int total = nk * terms_in(TERMS);
  // The next stage of a side to load: its first elements, its term, and how many stages the term has left.
  // Only these change from stage to stage, in scalar registers.
  const int last = static_cast<int>((k1 - k0) % KE);   // contraction of a term's last stage, 0: a whole one
  struct Next {
    const unsigned char* p;
    int term, left;
  };
  Next na{nullptr, 0, nk}, nb{nullptr, 0, nk};
  const int64_t step_a = (AKR ? KE * a.ld : KE) * ES, step_b = (BKR ? KE * b.ld : KE) * ES;
  auto begin_a = [&] {   // SIX: (l h) (h l) (m m) (m h) (h m) (h h)
    na.p = a.p + (AKR ? k0 * a.ld : k0) * ES;
    if constexpr (TERMS == SIX)
      na.p += (na.term == 0 ? 2 : na.term == 2 || na.term == 3 ? 1 : 0) * a.part * ES;
  };
  auto begin_b = [&] {
    nb.p = b.p + (BKR ? k0 * b.ld : k0) * ES;
    if constexpr (TERMS == SIX)
      nb.p += (nb.term == 1 ? 2 : nb.term == 2 || nb.term == 4 ? 1 : 0) * b.part * ES;
    else if constexpr (TERMS == TWO_B)
      nb.p += nb.term == 0 ? b.part * ES : 0;
  };
  begin_a();
  begin_b();
  auto issue_a = [&](unsigned to) {
    if (na.left > 1 || last == 0)
      sa.issue(na.p, to);
    else
      sa.issue_cut(na.p, to, last);
    na.p += step_a;
    if (--na.left == 0) {
      na.left = nk;
      if constexpr (terms_in(TERMS) > 1) ++na.term, begin_a();
    }
  };
  auto issue_b = [&](unsigned to) {
    if (nb.left > 1 || last == 0)
      sb.issue(nb.p, to);
    else
      sb.issue_cut(nb.p, to, last);
    nb.p += step_b;
    if (--nb.left == 0) {
      nb.left = nk;
      if constexpr (terms_in(TERMS) > 1) ++nb.term, begin_b();
    }
  };
  f32x4_t af[2][C::MI], bf[2][C::NI];
  auto load = [&](int buf, const unsigned char* la, const unsigned char* lb, int ks) {
    fb.load(lb, ks, bf[buf]);   // the first MFMAs take all of B and one of A
    fa.load(la, ks, af[buf]);
  };
  auto mma = [&](int buf) {
#pragma unroll
    for (int i = 0; i < C::MI; ++i)
#pragma unroll
      for (int j = 0; j < C::NI; ++j) {
        if constexpr (ES == 4) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(af[buf][i][q], bf[buf][j][q], acc[i][j], 0, 0, 0);
        } else {
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, af[buf][i]),
                                                              __builtin_bit_cast(bf16x8_t, bf[buf][j]),
                                                              acc[i][j], 0, 0, 0);
        }
      }
  };
  constexpr int KRD = ES == 4 ? 4 : 2;   // reads of a fragment whose contraction index is the row
  constexpr int RD = (AKR ? KRD : 1) * C::MI + (BKR ? KRD : 1) * C::NI;
  constexpr int M = C::MI * C::NI * (ES == 4 ? 4 : 1);
  // The k-steps of the stage whose sides are at la and lb; the next stage's are at ma and mb.  PENDING:
  // loads that may be in flight when that one is read.  (Past the last stage the fragments are read and
  // not used.)
  auto steps = [&](const unsigned char* la, const unsigned char* lb, const unsigned char* ma,
                   const unsigned char* mb, auto pending) {
#pragma unroll
    for (int ks = 0; ks + 1 < KS; ++ks) {
      load((ks + 1) & 1, la, lb, ks + 1);
      mma(ks & 1);
      sched_kstep<RD, M>();
    }
    wait_lgkmcnt0();
    wait_vmcnt<decltype(pending)::value>();
    raw_barrier();
    load(0, ma, mb, 0);
    mma((KS - 1) & 1);
    sched_kstep<RD, M>();
  };
  using None = std::integral_constant<int, 0>;
  if constexpr (C::HALVES) {
    // Five halves of a stage: A of stage s in half 2s mod 5, B in the next.  While stage s is read, B of
    // stage s + 1 and A of s + 2 are loaded into the two that the stage before left, and only the former
    // has to be there at the end.  (With two slots all of the next stage has three k-steps' time to
    // arrive: 1.59 us a stage of 256 x 256 x 64.)
    constexpr unsigned H = C::A_BYTES;
    const auto two_on = [](unsigned at) { return at >= 3 * H ? at - 3 * H : at + 2 * H; };
    const auto one_on = [](unsigned at) { return at == 4 * H ? 0 : at + H; };
    if (total > 0) {
      issue_a(lds0);
      issue_b(lds0 + H);
      if (total > 1) {
        issue_a(lds0 + 2 * H);
        wait_vmcnt<sa.Q>();
      } else {
        wait_vmcnt<0>();
      }
      raw_barrier();
      load(0, lds, lds + H, 0);
      unsigned at = 0;   // A of the stage that is read
      auto run = [&](auto b_more, auto a_more, auto pending) {
        const unsigned next = two_on(at);
        if constexpr (decltype(b_more)::value) issue_b(lds0 + one_on(next));
        if constexpr (decltype(a_more)::value) issue_a(lds0 + two_on(next));
        steps(lds + at, lds + one_on(at), lds + next, lds + one_on(next), pending);
        at = next;
      };
      using Half = std::integral_constant<int, sa.Q>;
      int s = 0;
      for (; s + 2 < total; ++s) run(std::true_type{}, std::true_type{}, Half{});
      if (s + 1 < total) run(std::true_type{}, std::false_type{}, None{});
      run(std::false_type{}, std::false_type{}, None{});
    }
  } else if (total > 0) {
    unsigned slot_in = lds0;
    auto issue = [&] {
      issue_a(slot_in);
      issue_b(slot_in + C::A_BYTES);
      slot_in = slot_in + C::STAGE == lds0 + C::LDS ? lds0 : slot_in + C::STAGE;
    };
#pragma unroll
    for (int s = 0; s < C::NS - 1; ++s)
      if (s < total) issue();
    if (C::NS - 1 <= total)
      wait_vmcnt<(C::NS - 2) * NQ>();
    else
      wait_vmcnt<0>();
    raw_barrier();
    load(0, lds, lds + C::A_BYTES, 0);
    const unsigned char* stage = lds;
    auto run = [&](auto more, auto pending) {
      const unsigned char* next = stage + C::STAGE == lds + C::LDS ? lds : stage + C::STAGE;
      if constexpr (decltype(more)::value) issue();   // into the slot before, which every wave has read
      steps(stage, stage + C::A_BYTES, next, next + C::A_BYTES, pending);
      stage = next;
    };
    using Steady = std::integral_constant<int, (C::NS - 2) * NQ>;
    int s = 0;
    for (; s + C::NS - 1 < total; ++s) run(std::true_type{}, Steady{});
    for (; s < total; ++s) run(std::false_type{}, None{});
  }
  raw_barrier();   // every wave is done reading: LDS is the caller's
}

// Workgroup w of `total` to its place in an order of which each XCD takes a contiguous run
// (workgroup w runs on XCD w mod 8).  Places are 32-bit, as grids are: divisions of 64 bits cost the kernels
// of eight rows up to half a microsecond each.
__device__ __forceinline__ uint32_t xcd_order(uint32_t w, uint32_t total) {
  const uint32_t q = total / 8, r = total % 8, x = w % 8;
  return x * q + (x < r ? x : r) + w / 8;
}

// ------------------------------------------------------------------------------ rows that count

constexpr int CHUNK = 1024;   // labels counted by one workgroup

struct RowsArgs {
  const void* X;
  int64_t x_stride;
  const int64_t* labels;
  int64_t ignore_index, N, V, d, dp;
  void* Xc;            // [N][dp], for fp32 of many rows [parts][N][dp] bf16
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

// One row of `n` elements to a row of np (a multiple of 8), zeros behind; with SPLIT fp32 ones into three
// bf16 parts `part` elements apart.  `t` of `nt` threads.
template <class E, bool SPLIT>
__device__ __forceinline__ void copy_row(const E* src, int64_t n, void* to, int64_t np, int64_t part, int t,
                                         int nt) {
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
    if constexpr (!SPLIT) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(E) / 2); ++i)
        reinterpret_cast<uint4*>(static_cast<E*>(to) + f)[i] = w.u[i];
    } else {
      uint16_t* dst = static_cast<uint16_t*>(to);
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

// GROUP rows to a workgroup: a row to a wave while those are few (138 rows of 629 fp32 features by sixteens:
// 13 us), more where each workgroup's own count of the labels before it would be most of the work.
template <class E, bool SPLIT, int GROUP>
__global__ void __launch_bounds__(256) head_rows_kernel(RowsArgs a) {
  using O = std::conditional_t<SPLIT, uint16_t, E>;
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
#pragma unroll
  for (int g = 0; g < GROUP; ++g) {
    const int64_t r = first + g;
    if (r >= a.N) break;
    const int64_t y = a.labels[r];
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
        copy_row<E, SPLIT>(static_cast<const E*>(a.X) + r * a.x_stride, a.d,
                           static_cast<O*>(a.Xc) + place * a.dp, a.dp, a.N * a.dp, lane, 64);
    }
    place += keep;
  }
  if (first + GROUP >= a.N && threadIdx.x == 0) *a.count = place;
}

// A piece of W as the products take it: rows of dp elements, in three parts for fp32 of many rows.
template <class E, bool SPLIT>
__global__ void __launch_bounds__(256) head_weight_kernel(const E* W, int64_t rows, int64_t d, void* out,
                                                          int64_t dp) {
  using O = std::conditional_t<SPLIT, uint16_t, E>;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r < rows)
    copy_row<E, SPLIT>(W + r * d, d, static_cast<O*>(out) + r * dp, dp, rows * dp, threadIdx.x & 63, 64);
}

// ------------------------------------------------------------------------------ logits

struct LogitsArgs {
  Side w, x;                 // [V of the piece][dp or d], [count][dp]
  const int32_t* count;
  const int32_t* label;
  int64_t N, V, v0, k;       // v0: the piece's first entry; V: the piece's entries; k: W's features
  int64_t v_tiles;
  // forward: per vocabulary tile (of all pieces) and row
  float2* part;              // [tiles][N]: maximum of z log2(e), sum of 2^(z log2(e) - maximum)
  int64_t tile0;
  float* label_z;            // [N]: the label's z
  // backward
  const float* lse;          // [N][2]: as FinishArgs::lse
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
  const uint32_t vts = static_cast<uint32_t>(v_tiles), tts = static_cast<uint32_t>(t_tiles);
  const uint32_t total = vts * tts;
  if (blockIdx.x >= total) return false;
  const uint32_t i = xcd_order(blockIdx.x, total), per = 8 * vts, g = i / per, r = i - g * per;
  const uint32_t size = tts - 8 * g < 8 ? tts - 8 * g : 8, v = r / size;
  tt = 8 * g + (r - v * size), vt = v;
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

template <class C, int TERMS, int MODE, int GW>
__global__ void __launch_bounds__(C::NT, 2) head_logits_kernel(LogitsArgs p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  const int64_t count = *p.count;
  int64_t vt, tt;
  if (!logits_item(p.v_tiles, (count + C::BN - 1) / C::BN, vt, tt)) return;
  const int64_t m0 = vt * C::BM, n0 = tt * C::BN;
  f32x16_t acc[C::MI][C::NI];
  Side a = p.w, b = p.x;
  a.move<size_of(TERMS)>(m0 * a.ld), b.move<size_of(TERMS)>(n0 * b.ld);
  product<C, false, false, TERMS, GW>(a, p.V - m0, b, count - n0, 0, p.k, lds, acc);

  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid % C::WN, half = lane >> 5;
  const int row0 = wm * C::MI * 32 + 4 * half;     // this lane's first row of the tile
  const bool ragged = m0 + C::BM > p.V;
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
      const float ref = fmaxf(m * LOG2E, -3e38f);   // rows of -inf: exponentials of zero, no NaN
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], LOG2E, -ref));
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
    constexpr int CH = C::BM / 8, PARTS = MODE == ROWS || TERMS == FULL ? 1 : dz_parts<C>(TERMS == SIX);
    static_assert(C::BN * C::BM * 2 <= C::LDS, "the tile of dz fits the stages");
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int64_t n = n0 + (wn * C::NI + j) * 32 + (lane & 31);
      const bool live = n < count;
      const int32_t y = live ? p.label[n] : 0;
      const float ref = live && y >= 0 ? p.lse[2 * n] : NAN;
      float w = live && p.up != nullptr ? p.up[p.rows[n]] : 1.f;
      if constexpr (MODE == ROWS) w *= gradient_scale(p.up_all, p.mean, count);
      const float share = live ? w / p.lse[2 * n + 1] : 0.f;
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = share * __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], LOG2E, -ref));
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
    if constexpr (TERMS == FULL || (MODE == ROWS && TERMS == SIX)) {   // fp32, straight from the lanes
#pragma unroll
      for (int j = 0; j < C::NI; ++j) {
        const int64_t n = n0 + (wn * C::NI + j) * 32 + (lane & 31);
        if (n >= count) continue;
        float* out = MODE == ROWS ? static_cast<float*>(p.out) + p.rows[n] * p.vp
                                  : reinterpret_cast<float*>(p.dz) + n * p.vp;
        out += m0 + row0;
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

// Each row's log2 of the sum of exponentials from the tiles' parts, and its loss; the losses' sum of a
// workgroup's rows, or of all of them where there is one workgroup.
struct FinishArgs {
  const float2* part;
  const float* label_z;
  const int32_t* count;
  const int32_t* rows;
  const int32_t* label;
  int64_t N, tiles;
  // [N][2]: the row's reference, its largest z log2(e), and its sum of 2^(z log2(e) - reference).  Apart,
  // because in one number they would cost a row whose label has most of the mass its digits: the loss and
  // p - 1 would be what is left of numbers of the logits' size.
  float* lse;
  float* loss;       // null, or [N]
  float* sums;       // null, or [blocks]
  float* total;      // null, or where the sum or mean of one workgroup's rows goes
  int mean;
};
// The two parts as one.
__device__ __forceinline__ float2 joined(float2 t, float2 u) {
  const float m = fmaxf(t.x, u.x);
  return make_float2(m, t.y * __builtin_amdgcn_exp2f(t.x - m) + u.y * __builtin_amdgcn_exp2f(u.x - m));
}
// ROWS rows to a workgroup of 1024 threads: 64 where there are many, 32 of at most as many.  Its other
// threads share the tiles (four threads to a row and its 393 tiles are 11 us for eight rows).
template <int ROWS>
__global__ void __launch_bounds__(1024) head_finish_kernel(FinishArgs p) {
  constexpr int G = 1024 / ROWS;
  __shared__ float2 red[G][ROWS];
  const int r = threadIdx.x % ROWS, g = threadIdx.x / ROWS;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * ROWS + r, count = *p.count;
  float2 t = make_float2(-3e38f, 0.f);
  if (n < count) {
#pragma unroll 4
    for (int64_t k = g; k < p.tiles; k += G) t = joined(t, p.part[k * p.N + n]);
  }
  red[g][r] = t;
#pragma unroll
  for (int w = G / 2; w > 0; w /= 2) {
    __syncthreads();
    if (g < w) red[g][r] = joined(red[g][r], red[g + w][r]);
  }
  if (threadIdx.x >= 64) return;
  float loss = 0.f;
  if (g == 0 && n < count) {
    t = red[0][r];
    loss = p.label[n] >= 0 ? LN2 * (log2f(t.y) - fmaf(p.label_z[n], LOG2E, -t.x)) : NAN;
    p.lse[2 * n] = t.x, p.lse[2 * n + 1] = t.y;
    if (p.loss != nullptr) p.loss[p.rows[n]] = loss;
  }
  loss = wave_sum(loss);
  if (threadIdx.x != 0) return;
  if (p.total != nullptr) *p.total = p.mean ? loss / static_cast<float>(count) : loss;
  else if (p.sums != nullptr) p.sums[blockIdx.x] = loss;
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

// How often a piece's vocabulary is split among the workgroups for dx, by the rows that count, whose number
// only the device knows: `slots` workgroups for the tiles there are, in up to `most` shares.  (By the
// rows that came, a batch half of which is padding has every second unit without work.)
struct DxSplit {
  int64_t tile, f_tiles, slots, most;   // tile: rows of one
  __host__ __device__ int64_t operator()(int64_t count) const {
    const uint32_t b = static_cast<uint32_t>(tile);
    const uint32_t tiles = static_cast<uint32_t>(f_tiles) * ((static_cast<uint32_t>(count) + b - 1) / b);
    const int64_t s = tiles > 0 ? static_cast<uint32_t>(slots) / tiles : 1;
    return s < 1 ? 1 : s < most ? s : most;
  }
};
struct DxArgs {
  Side dz, w;              // [count][vp], [V of the piece][k]
  const int32_t* count;
  int64_t N, V, dp, k;     // V: the piece's entries; k: W's features
  DxSplit split;
  int64_t low;             // 0, or N: dz's rows from there on are its low part, two shares to a split
  float* out;              // [shares][count][dp]
  int add;                 // to what is there
};
template <class C, int TERMS, int GW>
__global__ void __launch_bounds__(C::NT, 2) head_dx_kernel(DxArgs p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  const int64_t count = *p.count, t_tiles = (count + C::BM - 1) / C::BM, f_tiles = p.split.f_tiles;
  const uint32_t fs = static_cast<uint32_t>(f_tiles), tiles = fs * static_cast<uint32_t>(t_tiles);
  const uint32_t splits = static_cast<uint32_t>(p.split(count)), total = tiles * splits;
  if (blockIdx.x >= total) return;
  const uint32_t i0 = xcd_order(blockIdx.x, total), part = i0 / tiles, r0 = i0 - part * tiles, tr = r0 / fs;
  const int64_t split = part, m0 = static_cast<int64_t>(tr) * C::BM, n0 = static_cast<int64_t>(r0 - tr * fs) * C::BN;
  const int64_t per = ((static_cast<uint32_t>(p.V) + splits - 1) / splits + 63) / 64 * 64;
  const int64_t k0 = split * per, k1 = k0 + per < p.V ? k0 + per : p.V;
  f32x16_t acc[C::MI][C::NI];
  Side a = p.dz, b = p.w;
  a.move<size_of(TERMS)>(m0 * a.ld), b.move<size_of(TERMS)>(n0);
  product<C, false, true, TERMS, 16, GW>(a, p.low + count - m0, b, p.k - n0, k0, k1, lds, acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid % C::WN;
  float* out = p.out + (p.low > 0 ? 2 * split : split) * count * p.dp;
#pragma unroll
  for (int j = 0; j < C::NI; ++j) {
    const int64_t f = n0 + (wn * C::NI + j) * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < C::MI; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        int64_t r = m0 + (wm * C::MI + i) * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4;
        float* o = out;
        if (p.low > 0 && r >= p.low) r -= p.low, o += count * p.dp;
        if (r < count && f < p.dp) {
          o += r * p.dp + f;
          *o = p.add ? *o + acc[i][j][e] : acc[i][j][e];
        }
      }
  }
}

// dx of every row: its sums over the splits, scaled and rounded once; zeros where it does not count.
struct DxFinishArgs {
  const float* sums;
  DxSplit split;
  int shares;              // of a split
  const int32_t *at, *count;
  int64_t N, d, dp, f_blocks;
  const float* up;
  int mean;
  void* dx;
};
// A workgroup takes 64 features of a row, its four waves every fourth split (a row's 42 splits of 768
// features by one wave: 119 us for eight rows).
template <class E>
__global__ void __launch_bounds__(256) head_dx_finish_kernel(DxFinishArgs p) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t r = blockIdx.x / static_cast<uint32_t>(p.f_blocks);
  const int64_t f = (blockIdx.x - r * p.f_blocks) * 64 + lane;
  const int64_t j = p.at[r], count = *p.count;
  float s = 0.f;
  if (j >= 0 && f < p.d) {
    const int splits = static_cast<int>(p.split(count)) * p.shares;
#pragma unroll 4
    for (int k = g; k < splits; k += 4) s += p.sums[(k * count + j) * p.dp + f];
  }
  red[g][lane] = s;
  __syncthreads();
  if (g != 0 || f >= p.d) return;
  s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
  static_cast<E*>(p.dx)[r * p.d + f] =
      from_f32<E>(j >= 0 ? s * gradient_scale(p.up, p.mean, count) : 0.f);
}
// The same of many rows and few splits: a thread to four features, whichever row they are in.  (4096 rows
// of 768 features in five splits 50 us by the kernel above.)
template <class E>
__global__ void __launch_bounds__(256) head_dx_rows_kernel(DxFinishArgs p) {
  const int64_t fours = p.dp / 4, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.N * fours) return;
  const int64_t r = i >> 32 ? i / fours : static_cast<uint32_t>(i) / static_cast<uint32_t>(fours);
  const int64_t f = (i - r * fours) * 4;
  const int64_t j = p.at[r], count = *p.count;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (j >= 0) {
    const int splits = static_cast<int>(p.split(count)) * p.shares;
    const float scale = gradient_scale(p.up, p.mean, count);
    const float* sums = p.sums + j * p.dp + f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 u = *reinterpret_cast<const float4*>(sums + k * count * p.dp);
      v[0] += u.x, v[1] += u.y, v[2] += u.z, v[3] += u.w;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] *= scale;
  }
  union { uint2 u[sizeof(E) / 2]; E e[4]; } o;
#pragma unroll
  for (int q = 0; q < 4; ++q) o.e[q] = from_f32<E>(v[q]);
  E* out = static_cast<E*>(p.dx) + r * p.d + f;
  if (p.d % 4 == 0 && reinterpret_cast<uintptr_t>(p.dx) % 16 == 0) {
    if (f >= p.d) return;
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(E) / 2); ++q) reinterpret_cast<uint2*>(out)[q] = o.u[q];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (f + q < p.d) out[q] = o.e[q];
  }
}

struct DwArgs {
  Side dz, x;              // [count][vp], [count][dp]: the contraction is their rows
  const int32_t* count;
  int64_t V, d, dp, cols;  // V: the entries; cols: dz's columns from the first of them on
  int64_t v_tiles, f_tiles, splits;
  const float* up;
  int mean;
  void* out;               // their rows of dW; or with several splits [splits][V][d] fp32 sums
};
// Features on the A side, so that a lane holds fours of neighbours of an entry's row.  bf16 rows leave
// through LDS, whole rows of the tile at a time (straight from the lanes, two bytes each: 83 us for the
// 77 MB of GPT-2's dW, eight rows).
template <class C, int TERMS, class E>
__global__ void __launch_bounds__(C::NT, 2) head_dw_kernel(DwArgs p) {
  __shared__ __attribute__((aligned(16))) unsigned char lds[C::LDS];
  const int64_t count = *p.count;
  const uint32_t fs = static_cast<uint32_t>(p.f_tiles), tiles = static_cast<uint32_t>(p.v_tiles) * fs;
  const uint32_t i0 = xcd_order(blockIdx.x, tiles * static_cast<uint32_t>(p.splits)), split = i0 / tiles;
  const uint32_t r0 = i0 - split * tiles, tv = r0 / fs;
  const int64_t m0 = static_cast<int64_t>(r0 - tv * fs) * C::BM, n0 = static_cast<int64_t>(tv) * C::BN;
  // shares of the rows that count, not of those that came
  const uint32_t shares = static_cast<uint32_t>(p.splits);
  const int64_t per = ((static_cast<uint32_t>(count) + shares - 1) / shares + 63) / 64 * 64;
  const int64_t k0 = split * per, k1 = k0 + per < count ? k0 + per : count;
  f32x16_t acc[C::MI][C::NI];
  Side a = p.x, b = p.dz;
  a.move<size_of(TERMS)>(m0), b.move<size_of(TERMS)>(n0);
  product<C, true, true, TERMS>(a, p.dp - m0, b, p.cols - n0, k0, k1, lds, acc);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int wm = wid / C::WN, wn = wid % C::WN, half = lane >> 5;
  const int64_t f0 = m0 + wm * C::MI * 32 + 4 * half;   // this lane's first feature
  const bool sums = p.splits > 1;
  const bool fours = p.d % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  const float scale = sums ? 1.f : gradient_scale(p.up, p.mean, count);
#pragma unroll
  for (int i = 0; i < C::MI; ++i)
#pragma unroll
    for (int j = 0; j < C::NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] *= scale;
  if (sums || sizeof(E) == 4) {
    float* out = sums ? static_cast<float*>(p.out) + split * p.V * p.d : static_cast<float*>(p.out);
#pragma unroll
    for (int j = 0; j < C::NI; ++j) {
      const int64_t v = n0 + (wn * C::NI + j) * 32 + (lane & 31);
      if (v >= p.V) continue;
#pragma unroll
      for (int i = 0; i < C::MI; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int64_t f = f0 + 32 * i + 8 * g;
          float* o = out + v * p.d + f;
          if (fours && f < p.d) {
            *reinterpret_cast<float4*>(o) = make_float4(acc[i][j][4 * g], acc[i][j][4 * g + 1],
                                                        acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (f + q < p.d) o[q] = acc[i][j][4 * g + q];
          }
        }
    }
    return;
  }
  if constexpr (sizeof(E) == 2) {
    constexpr int CH = C::BM / 8;
    static_assert(C::BN * C::BM * 2 <= C::LDS, "the tile of dW fits the stages");
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
          *reinterpret_cast<uint2*>(lds + r * C::BM * 2 + ((c ^ (r & (CH - 1))) * 16) + half * 8) = u;
        }
    }
    __syncthreads();
    uint16_t* out = static_cast<uint16_t*>(p.out);
    if (p.d % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0) {
      for (int i = threadIdx.x; i < C::BN * CH; i += C::NT) {
        const int r = i / CH, c = i % CH;
        if (n0 + r < p.V && m0 + c * 8 < p.d)
          *reinterpret_cast<uint4*>(out + (n0 + r) * p.d + m0 + c * 8) =
              *reinterpret_cast<const uint4*>(lds + r * C::BM * 2 + ((c ^ (r & (CH - 1))) * 16));
      }
    } else {
      for (int i = threadIdx.x; i < C::BN * C::BM; i += C::NT) {
        const int r = i / C::BM, f = i % C::BM;
        if (n0 + r < p.V && m0 + f < p.d)
          out[(n0 + r) * p.d + m0 + f] = *reinterpret_cast<const uint16_t*>(
              lds + r * C::BM * 2 + (((f / 8) ^ (r & (CH - 1))) * 16) + f % 8 * 2);
      }
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

constexpr int64_t PIECE_BYTES = int64_t{1} << 30;   // of dz at most, but for a piece of 256 entries
constexpr int64_t PIECE_ENTRIES = int64_t{1} << 25;
constexpr int64_t CUS = 256;

enum Size { WIDE, MID, SMALL, FEW };

// How a product is made: its tiles, and how often its contraction is split.
struct Shape {
  Size size;
  int64_t splits;
  int64_t slots;         // workgroups that the splits fill
  double us;
};

struct Plan {
  bool f32, few, copy_w;
  bool full;                 // fp32 operands as they are: a few rows, bound by W's memory
  bool by4;                  // W's rows as they are, loaded by 4 bytes
  int64_t row_bytes, dz_bytes;   // of the operands' elements, all parts, and of dz's
  int64_t dp, k, cols, pieces;   // k: features of W's rows as the products take them; cols: vocabulary entries of a piece
  int64_t tiles_all;         // vocabulary tiles of all pieces of the forward pass
  int64_t chunks, blocks;
  Size dx_size;
  DxSplit dx;
  int dx_shares;             // of a split: dz's parts in one product's rows
  int64_t dw_sums;           // fp32 elements that a split piece of dW needs
};

// The tiles of an m x n product over k (in `terms` products of parts), by what they were measured to take:
// a stage of 64 of the contraction 1.45 us with 256 x 256 tiles, one workgroup to a unit; 0.93 with 128 x
// 128 and 0.36 with 64 x 64 tiles, two to a unit (fp32's parts, of which there is more to read, 1.85,
// 1.15 and 0.5); 8, 3 and 1.5 us to begin and end a tile.  Splits cost
// writing and reading the shares' sums at 4 TB/s.  (43 rows of 791 fp32 features, 3655 entries: 314 us in
// 256 x 256 tiles, of which there are 15.)
Shape shape_of(int64_t m, int64_t n, int64_t k, int64_t terms, bool split) {
  static const struct { Size size; int64_t b, slots; double stage, parts, ends; } T[] = {
      {WIDE, 256, 256, 1.45, 1.85, 8.0}, {MID, 128, 512, 0.93, 1.15, 3.0}, {SMALL, 64, 512, 0.36, 0.5, 1.5}};
  Shape best{WIDE, 1, 256, 1e300};
  for (const auto& t : T) {
    const int64_t tiles = cdiv(m, t.b) * cdiv(n, t.b), stages = cdiv(k, 64);
    // shares that fill the units once or twice
    const int64_t fill[3] = {1, t.slots / tiles, 2 * t.slots / tiles};
    for (int i = 0; i < (split ? 3 : 1); ++i) {
      const int64_t want = std::max<int64_t>(1, std::min(fill[i], cdiv(stages, 4)));
      const int64_t per = cdiv(stages, want), splits = cdiv(stages, per);
      const double us = cdiv(tiles * splits, t.slots) * (per * terms * (terms > 1 ? t.parts : t.stage) + t.ends) +
                        (splits > 1 ? 4.0 + splits * m * n * 8 / 4e6 : 0.0);
      if (us < best.us) best = Shape{t.size, splits, i == 2 ? 2 * t.slots : t.slots, us};
    }
  }
  return best;
}

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

int64_t rows_of(Size s) { return s == WIDE ? 256 : s == MID ? 128 : s == SMALL ? 64 : Few::BM; }
int64_t terms_of(const Plan& p) { return p.f32 ? 6 : 1; }

Shape logits_shape(const gs_head& h, const Plan& p, int64_t n) {
  if (p.few) return Shape{FEW, 1, 0, 0.0};
  return shape_of(n, h.N, h.d, terms_of(p), false);
}
// dx of a piece of `most` entries.
Size dx_shape(const gs_head& h, const Plan& p, int64_t most, DxSplit& split) {
  if (p.few) {   // a share of at least 256 entries for every unit
    split = DxSplit{FewT::BM, cdiv(p.dp, FewT::BN), CUS, cdiv(most, 256)};
    return FEW;
  }
  const Shape s = shape_of(h.N, p.dp, most, terms_of(p), true);
  const int64_t tile = rows_of(s.size);
  split = DxSplit{tile, cdiv(p.dp, tile), s.slots, cdiv(most, 256)};
  return s.size;
}
// The fp32 sums that dx's shares take, for any number of rows that count.
int64_t dx_sums(const gs_head& h, const Plan& p) {
  int64_t most = h.N;
  for (int64_t n = p.dx.tile; n < h.N + p.dx.tile && p.dx(n) > 1; n += p.dx.tile)
    most = std::max(most, p.dx(n) * std::min(n, h.N));
  return most * p.dx_shares * p.dp;
}
// dW of n entries of the vocabulary, in one product or in two: as many entries as fill whole rounds over
// the compute units, and the rest, which is split over its rows.  (197 x 3 tiles of 8192 rows take three
// rounds in one product, 606 us.)
struct DwParts {
  int64_t n[2];
  Shape shape[2];
};
DwParts dw_parts(const gs_head& h, const Plan& p, int64_t n) {
  if (p.few) return DwParts{{n, 0}, {Shape{FEW, 1, 0, 0.0}, {}}};
  const auto shape = [&](int64_t n) { return shape_of(n, h.d, h.N, terms_of(p), true); };
  const Shape all = shape(n);
  const int64_t f = cdiv(h.d, 256), whole = cdiv(n, 256) * f / CUS * CUS / f * 256;
  if (whole > 0 && whole < n) {
    const Shape a = shape(whole), b = shape(n - whole);
    // a seventh to gain: where half of the rows count, a tenth has been lost
    if (a.us + b.us < 0.85 * all.us) return DwParts{{whole, n - whole}, {a, b}};
  }
  return DwParts{{n, 0}, {all, {}}};
}

// The plan of a call.
Plan plan_of(const gs_head& h, int w_align) {
  Plan p{};
  p.f32 = h.dtype == GS_DTYPE_F32;
  p.few = h.N <= FEW_ROWS;
  p.full = p.f32 && p.few;
  p.dp = round_up(h.d, 8);
  // A few rows are bound by W's memory: rows of it at multiples of 4 bytes are loaded by 4, without a copy.
  const int64_t row = h.d * static_cast<int64_t>(elem_size(h.dtype));
  const bool whole = h.d % 8 == 0 && w_align >= 16;
  p.by4 = p.few && !whole && row % 4 == 0 && w_align >= 4;
  p.copy_w = !p.by4 && ((p.f32 && !p.full) || !whole);
  p.k = p.by4 ? h.d : p.dp;
  p.row_bytes = p.full ? 4 : p.f32 ? 6 : 2;
  p.dz_bytes = p.full ? 4 : 2 * (p.few ? dz_parts<Few>(p.f32) : dz_parts<Wide>(p.f32));
  const int64_t all = cdiv(h.V, 256);
  const int64_t most = std::min(std::max<int64_t>(1, PIECE_BYTES / (h.N * p.dz_bytes * 256)), PIECE_ENTRIES / 256);
  if (all <= most) {
    p.cols = all * 256;
  } else {
    // Pieces whose tiles of dW are just below a whole number of rounds over the compute units, and a rest
    // that is split over its rows: GPT-2's 197 x 3 tiles in pieces of 85 x 3, 85 x 3 and 27 x 3 in shares of
    // a third each; in four pieces of 50 x 3 two fifths of the units had nothing to do.
    const int64_t f_tiles = cdiv(h.d, 256), rounds = std::max<int64_t>(1, most * f_tiles / CUS);
    p.cols = std::max<int64_t>(1, std::min(most, rounds * CUS / f_tiles)) * 256;
  }
  p.pieces = cdiv(h.V, p.cols);
  p.tiles_all = 0;
  p.dw_sums = 0;
  for (int64_t v0 = 0; v0 < h.V; v0 += p.cols) {
    const int64_t n = std::min(p.cols, h.V - v0);
    p.tiles_all += cdiv(n, rows_of(logits_shape(h, p, n).size));
    const DwParts w = dw_parts(h, p, n);
    for (int i = 0; i < 2; ++i)
      if (w.shape[i].splits > 1) p.dw_sums = std::max(p.dw_sums, w.shape[i].splits * w.n[i] * h.d);
  }
  p.dx_shares = p.few && !p.f32 ? dz_parts<Few>(false) : 1;
  p.dx_size = dx_shape(h, p, std::min(p.cols, h.V), p.dx);
  p.chunks = h.N > CHUNK ? cdiv(h.N, CHUNK) : 0;
  p.blocks = cdiv(h.N, 64);
  return p;
}

struct Buffers {
  unsigned char *xc, *wc, *dz;
  int32_t *at, *rows, *label, *count, *chunk;
  float2* part;
  float *label_z, *sums, *dx, *dw;
};
template <class S>
Buffers carve(S& s, const gs_head& h, const Plan& p, bool grad) {
  Buffers b{};
  b.xc = s.template take<unsigned char>(p.row_bytes * h.N * p.dp);
  b.at = s.template take<int32_t>(h.N);
  b.rows = s.template take<int32_t>(h.N);
  b.label = s.template take<int32_t>(h.N);
  b.count = s.template take<int32_t>(1);
  b.chunk = s.template take<int32_t>(std::max<int64_t>(1, p.chunks));
  if (p.copy_w) b.wc = s.template take<unsigned char>(p.row_bytes * std::min(p.cols, h.V) * p.dp);
  if (!grad) {
    b.part = s.template take<float2>(p.tiles_all * h.N);
    b.label_z = s.template take<float>(h.N);
    b.sums = s.template take<float>(p.blocks);
  } else {
    b.dz = s.template take<unsigned char>(p.dz_bytes * h.N * p.cols);
    b.dx = s.template take<float>(dx_sums(h, p));
    if (p.dw_sums > 0) b.dw = s.template take<float>(p.dw_sums);
  }
  return b;
}

int align_of(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 ? 16 : reinterpret_cast<uintptr_t>(p) % 4 == 0 ? 4 : 1; }
bool aligned16(const void* p) { return align_of(p) == 16; }

unsigned grid_of(int64_t n) { return static_cast<unsigned>(n); }

template <class E, bool SPLIT>
void launch_rows_of(const RowsArgs& a, hipStream_t s) {
  if (a.N <= 8192)
    hipLaunchKernelGGL((head_rows_kernel<E, SPLIT, 4>), dim3(grid_of(cdiv(a.N, 4))), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((head_rows_kernel<E, SPLIT, 16>), dim3(grid_of(cdiv(a.N, 16))), dim3(256), 0, s, a);
}
void launch_rows(const gs_head& h, const Plan& p, const Buffers& b, float* loss, hipStream_t s) {
  RowsArgs a{};
  a.X = h.X, a.x_stride = h.x_stride, a.labels = h.labels, a.ignore_index = h.ignore_index;
  a.N = h.N, a.V = h.V, a.d = h.d, a.dp = p.dp;
  a.Xc = b.xc, a.at = b.at, a.rows = b.rows, a.label = b.label, a.count = b.count;
  a.chunk = p.chunks > 0 ? b.chunk : nullptr;
  a.loss = loss;
  if (p.chunks > 0)
    hipLaunchKernelGGL(head_count_kernel, dim3(grid_of(p.chunks)), dim3(256), 0, s, a, b.chunk);
  if (p.full)
    launch_rows_of<float, false>(a, s);
  else if (p.f32)
    launch_rows_of<float, true>(a, s);
  else
    launch_rows_of<uint16_t, false>(a, s);
}

// W's rows [v0, v0 + n) as the products take them.
Side weight_side(const gs_head& h, const Plan& p, const Buffers& b, int64_t v0, int64_t n,
                 hipStream_t s) {
  const void* w = static_cast<const char*>(h.W) + v0 * h.d * static_cast<int64_t>(elem_size(h.dtype));
  if (!p.copy_w) return side_of(w, h.d, 0);
  const dim3 grid(grid_of(cdiv(n, 4)));
  if (p.full)
    hipLaunchKernelGGL((head_weight_kernel<float, false>), grid, dim3(256), 0, s,
                       static_cast<const float*>(w), n, h.d, b.wc, p.dp);
  else if (p.f32)
    hipLaunchKernelGGL((head_weight_kernel<float, true>), grid, dim3(256), 0, s,
                       static_cast<const float*>(w), n, h.d, b.wc, p.dp);
  else
    hipLaunchKernelGGL((head_weight_kernel<uint16_t, false>), grid, dim3(256), 0, s,
                       static_cast<const uint16_t*>(w), n, h.d, b.wc, p.dp);
  return side_of(b.wc, p.dp, n * p.dp);
}

template <class C, int MODE, int GW = 16>
void launch_logits_as(LogitsArgs& a, bool f32, hipStream_t s) {
  a.v_tiles = cdiv(a.V, C::BM);
  const dim3 grid(grid_of(a.v_tiles * cdiv(a.N, C::BN)));
  constexpr int F32 = C::BN == Few::BN ? FULL : SIX;
  if (f32)
    hipLaunchKernelGGL((head_logits_kernel<C, F32, MODE, GW>), grid, dim3(C::NT), 0, s, a);
  else
    hipLaunchKernelGGL((head_logits_kernel<C, ONE, MODE, GW>), grid, dim3(C::NT), 0, s, a);
}
template <int MODE>
void launch_logits(LogitsArgs& a, Size size, const Plan& p, hipStream_t s) {
  if (size == WIDE) launch_logits_as<Wide, MODE>(a, p.f32, s);
  if (size == MID) launch_logits_as<Mid, MODE>(a, p.f32, s);
  if (size == SMALL) launch_logits_as<Small, MODE>(a, p.f32, s);
  if (size == FEW && !p.by4) launch_logits_as<Few, MODE>(a, p.f32, s);
  if (size == FEW && p.by4) launch_logits_as<Few, MODE, 4>(a, p.f32, s);
}
template <class C, int TERMS, int GW = 16>
void launch_dx_as(DxArgs& a, hipStream_t s) {
  const dim3 grid(grid_of(std::max(a.split.slots, a.split.f_tiles * cdiv(a.N, C::BM))));
  hipLaunchKernelGGL((head_dx_kernel<C, TERMS, GW>), grid, dim3(C::NT), 0, s, a);
}
// A few rows: both parts of bf16's dz are one product's rows, so W is read once.  (As two terms of the
// contraction: 24 us for eight rows of GPT-2's, the logits' product 15.)
template <int GW>
void launch_dx_few(DxArgs& a, bool f32, hipStream_t s) {
  if (f32)
    launch_dx_as<FewT, FULL, GW>(a, s);
  else if (2 * a.N <= FewT::BM)
    launch_dx_as<FewT, ONE, GW>(a, s);
  else
    launch_dx_as<FewT2, ONE, GW>(a, s);
}
void launch_dx(DxArgs& a, const Plan& p, hipStream_t s) {
  if (p.dx_size == WIDE) p.f32 ? launch_dx_as<Wide, SIX>(a, s) : launch_dx_as<Wide, ONE>(a, s);
  if (p.dx_size == MID) p.f32 ? launch_dx_as<Mid, SIX>(a, s) : launch_dx_as<Mid, ONE>(a, s);
  if (p.dx_size == SMALL) p.f32 ? launch_dx_as<Small, SIX>(a, s) : launch_dx_as<Small, ONE>(a, s);
  if (p.dx_size == FEW) p.by4 ? launch_dx_few<4>(a, p.f32, s) : launch_dx_few<16>(a, p.f32, s);
}
template <class C, int TERMS>
void launch_dw_as(DwArgs& a, bool f32, hipStream_t s) {
  a.v_tiles = cdiv(a.V, C::BN), a.f_tiles = cdiv(a.d, C::BM);
  const dim3 grid(grid_of(a.v_tiles * a.f_tiles * a.splits));
  if (f32)
    hipLaunchKernelGGL((head_dw_kernel<C, C::BM == FewW::BM && C::BN == FewW::BN ? FULL : SIX, float>), grid, dim3(C::NT), 0, s, a);
  else
    hipLaunchKernelGGL((head_dw_kernel<C, TERMS, uint16_t>), grid, dim3(C::NT), 0, s, a);
}
void launch_dw(DwArgs& a, Size size, bool f32, hipStream_t s) {
  if (size == WIDE) launch_dw_as<Wide, ONE>(a, f32, s);
  if (size == MID) launch_dw_as<Mid, ONE>(a, f32, s);
  if (size == SMALL) launch_dw_as<Small, ONE>(a, f32, s);
  if (size == FEW) launch_dw_as<FewW, TWO_B>(a, f32, s);
}

// dW of n entries from entry v of a piece on, to `out`.
void launch_dw_part(const gs_head& h, const Plan& p, const Buffers& b, const LogitsArgs& a, int64_t n,
                    const Shape& shape, int64_t v, const float* up, int mean, void* out, hipStream_t s) {
  DwArgs w{};
  w.dz = side_of(b.dz + v * (p.full ? 4 : 2), p.cols, h.N * p.cols);
  w.cols = p.cols - v, w.x = a.x, w.count = b.count, w.V = n, w.d = h.d, w.dp = p.dp;
  w.splits = shape.splits, w.up = up, w.mean = mean;
  w.out = shape.splits > 1 ? b.dw : out;
  launch_dw(w, shape.size, p.f32, s);
  if (shape.splits == 1) return;
  const int64_t all = n * h.d;
  const dim3 grid(grid_of(cdiv(all, 256)));
  if (p.f32)
    hipLaunchKernelGGL(head_dw_finish_kernel<float>, grid, dim3(256), 0, s, b.dw, shape.splits, all, b.count,
                       up, mean, static_cast<float*>(out));
  else
    hipLaunchKernelGGL(head_dw_finish_kernel<uint16_t>, grid, dim3(256), 0, s, b.dw, shape.splits, all,
                       b.count, up, mean, static_cast<uint16_t*>(out));
}

template <class E>
void launch_dx_finish(const gs_head& h, const Plan& p, const Buffers& b, const float* up, int mean, void* dx,
                      hipStream_t s) {
  const DxFinishArgs a{b.dx, p.dx, p.dx_shares, b.at, b.count, h.N, h.d, p.dp, cdiv(h.d, 64), up, mean, dx};
  if (h.N >= 1024)
    hipLaunchKernelGGL(head_dx_rows_kernel<E>, dim3(grid_of(cdiv(h.N * (p.dp / 4), 256))), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(head_dx_finish_kernel<E>, dim3(grid_of(h.N * a.f_blocks)), dim3(256), 0, s, a);
}

// Whether every grid of a call can be launched: at most 2^31 threads.  dx, dw, rows: whether the call forms dx,
// dW, or the logits' gradient as rows of the caller's.  `vocab`: the entries of the call.
bool grids_fit(const gs_head& h, const Plan& p, int64_t vocab, bool dx, bool dw, bool rows) {
  constexpr int64_t MOST = int64_t{1} << 31;
  // a workgroup of 256 to 16 rows, of 1024 to 64, of 256 to 4
  if (h.N > MOST / 16 || (rows && h.N > MOST / 64)) return false;
  const auto threads = [](Size s) { return int64_t{s == WIDE ? Wide::NT : s == MID ? Mid::NT : s == SMALL ? Small::NT : Few::NT}; };
  const auto fits = [](int64_t a, int64_t b, int64_t c) {   // the product of three, none negative
    return a == 0 || b == 0 || c == 0 || (a <= MOST / b && a * b <= MOST / c);
  };
  for (int64_t v0 = 0; v0 < vocab; v0 += p.cols) {
    const int64_t n = std::min(p.cols, vocab - v0);
    if (n < p.cols || v0 == 0) {   // the pieces are alike but for the last
      if (p.copy_w && !fits(n, 64, 1)) return false;   // a wave to an entry
      const Size s = logits_shape(h, p, n).size;
      if (!fits(cdiv(n, rows_of(s)), cdiv(h.N, s == FEW ? Few::BN : rows_of(s)), threads(s))) return false;
      const DwParts w = dw_parts(h, p, n);
      for (int i = 0; i < 2 && dw; ++i) {
        const Size z = w.shape[i].size;
        const int64_t bv = z == FEW ? FewW::BN : rows_of(z), bf = z == FEW ? FewW::BM : rows_of(z);
        if (!fits(cdiv(w.n[i], bv) * std::max<int64_t>(1, w.shape[i].splits), cdiv(h.d, bf), threads(z)) ||
            (w.shape[i].splits > 1 && !fits(w.n[i], h.d, 1)))
          return false;
      }
    }
  }
  if (!dx) return true;
  const int64_t tiles = cdiv(h.N, p.dx_size == FEW ? FewT::BM : rows_of(p.dx_size));
  return fits(p.dx.f_tiles, tiles, threads(p.dx_size)) && fits(p.dx.slots, threads(p.dx_size), 1) &&
         (h.N >= 1024 ? fits(h.N, p.dp / 4, 1) : fits(h.N, cdiv(h.d, 64), 256));
}

LogitsArgs logits_args(const gs_head& h, const Plan& p, const Buffers& b) {
  LogitsArgs a{};
  a.x = side_of(b.xc, p.dp, h.N * p.dp);
  a.count = b.count, a.label = b.label, a.rows = b.rows;
  a.N = h.N, a.k = p.k;
  return a;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" size_t gs_head_loss_workspace(const gs_head* h) {
  if (check_head(h, "gs_head_loss") != GS_OK) return 0;
  Sizer s;
  carve(s, *h, plan_of(*h, align_of(h->W)), false);
  return s.used + 256;
}

extern "C" int gs_head_loss(const gs_head* h, float* out_loss, float* lse, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (const int rc = check_head(h, "gs_head_loss")) return rc;
  if (out_loss == nullptr || lse == nullptr)
    return fail(GS_ERR_INVALID, "gs_head_loss: no place for the loss");
  const Plan p = plan_of(*h, align_of(h->W));
  if (!grids_fit(*h, p, h->V, false, false, false))
    return fail(GS_ERR_UNSUPPORTED, "gs_head_loss: grid too large");
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
    launch_logits<FORWARD>(a, logits_shape(*h, p, a.V).size, p, s);
    a.tile0 += a.v_tiles;
  }
  FinishArgs f{};
  f.part = b.part, f.label_z = b.label_z, f.count = b.count, f.rows = b.rows, f.label = b.label;
  f.N = h->N, f.tiles = a.tile0, f.lse = lse;
  f.loss = rows ? out_loss : nullptr;
  f.sums = rows ? nullptr : b.sums;
  f.total = rows || !p.few ? nullptr : out_loss;
  f.mean = h->reduction == GS_REDUCE_MEAN;
  if (p.few)
    hipLaunchKernelGGL(head_finish_kernel<FEW_ROWS>, dim3(1), dim3(1024), 0, s, f);
  else
    hipLaunchKernelGGL(head_finish_kernel<64>, dim3(grid_of(p.blocks)), dim3(1024), 0, s, f);
  if (!rows && !p.few)
    hipLaunchKernelGGL(head_total_kernel, dim3(1), dim3(256), 0, s, b.sums, p.blocks, b.count,
                       h->reduction == GS_REDUCE_MEAN, out_loss);
  return check_launch("gs_head_loss");
}

extern "C" size_t gs_head_grad_workspace(const gs_head* h) {
  if (check_head(h, "gs_head_grad") != GS_OK) return 0;
  Sizer s;
  carve(s, *h, plan_of(*h, align_of(h->W)), true);
  return s.used + 256;
}

extern "C" int gs_head_grad(const gs_head* h, const float* lse, const float* upstream, void* dx,
                            void* dw, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check_head(h, "gs_head_grad")) return rc;
  if (lse == nullptr) return fail(GS_ERR_INVALID, "gs_head_grad: the forward pass's sums are missing");
  const Plan p = plan_of(*h, align_of(h->W));
  if (!grids_fit(*h, p, h->V, dx != nullptr, dw != nullptr, false))
    return fail(GS_ERR_UNSUPPORTED, "gs_head_grad: grid too large");
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
  a.lse = lse, a.up = own ? upstream : nullptr, a.dz = reinterpret_cast<uint16_t*>(b.dz);
  for (int64_t v0 = 0; v0 < h->V; v0 += p.cols) {
    a.v0 = v0, a.V = std::min(p.cols, h->V - v0);
    a.w = weight_side(*h, p, b, v0, a.V, s);
    a.vp = p.cols;
    launch_logits<GRADIENT>(a, logits_shape(*h, p, a.V).size, p, s);
    const Side dz = side_of(b.dz, p.cols, h->N * p.cols);
    if (dx != nullptr) {
      DxArgs x{};
      x.dz = dz, x.w = a.w, x.count = b.count, x.N = h->N, x.V = a.V, x.dp = p.dp, x.k = p.k;
      x.split = p.dx, x.low = p.dx_shares > 1 ? h->N : 0, x.out = b.dx, x.add = v0 > 0;
      launch_dx(x, p, s);
    }
    if (dw != nullptr) {
      const DwParts parts = dw_parts(*h, p, a.V);
      int64_t v = 0;   // the part's first entry, in the piece
      for (int i = 0; i < 2 && parts.n[i] > 0; v += parts.n[i++])
        launch_dw_part(*h, p, b, a, parts.n[i], parts.shape[i], v, up, mean,
                       static_cast<char*>(dw) + (v0 + v) * h->d * static_cast<int64_t>(elem_size(h->dtype)), s);
    }
  }
  if (dx != nullptr) {
    if (p.f32)
      launch_dx_finish<float>(*h, p, b, up, mean, dx, s);
    else
      launch_dx_finish<uint16_t>(*h, p, b, up, mean, dx, s);
  }
  return check_launch("gs_head_grad");
}

// A call for one piece of dz has a plan of its own: the piece is the vocabulary.
static Plan piece_plan(const gs_head& h, int64_t n, int w_align) {
  gs_head piece = h;
  piece.V = n;
  Plan p = plan_of(piece, w_align);
  p.cols = round_up(n, 256);
  return p;
}
static int piece_align(const gs_head& h, int64_t v0) {
  return align_of(static_cast<const char*>(h.W) + v0 * h.d * static_cast<int64_t>(elem_size(h.dtype)));
}
template <class S>
static Buffers carve_piece(S& s, const gs_head& h, int64_t n, const Plan& p) {
  gs_head piece = h;
  piece.V = n;
  Buffers b{};
  b.xc = s.template take<unsigned char>(p.row_bytes * h.N * p.dp);
  b.at = s.template take<int32_t>(h.N);
  b.rows = s.template take<int32_t>(h.N);
  b.label = s.template take<int32_t>(h.N);
  b.count = s.template take<int32_t>(1);
  b.chunk = s.template take<int32_t>(std::max<int64_t>(1, p.chunks));
  if (p.copy_w) b.wc = s.template take<unsigned char>(p.row_bytes * n * p.dp);
  return b;
}

extern "C" size_t gs_head_logit_grad_workspace(const gs_head* h, int64_t v0, int64_t n) {
  if (check_head(h, "gs_head_logit_grad") != GS_OK || v0 < 0 || n <= 0 || n > h->V - v0) return 0;
  Sizer s;
  carve_piece(s, *h, n, piece_plan(*h, n, piece_align(*h, v0)));
  return s.used + 256;
}

extern "C" int gs_head_logit_grad(const gs_head* h, const float* lse, const float* upstream, int64_t v0,
                                  int64_t n, void* out, int64_t out_stride, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (const int rc = check_head(h, "gs_head_logit_grad")) return rc;
  if (lse == nullptr || out == nullptr || !aligned16(out) || v0 < 0 || n <= 0 || n > h->V - v0 ||
      out_stride != round_up(n, 8))
    return fail(GS_ERR_INVALID, "gs_head_logit_grad: invalid arguments");
  const Plan p = piece_plan(*h, n, piece_align(*h, v0));
  if (!grids_fit(*h, p, n, false, false, true))
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
  launch_logits<ROWS>(a, logits_shape(*h, p, n).size, p, s);
  hipLaunchKernelGGL(head_zero_rows_kernel, dim3(grid_of(cdiv(h->N, 4))), dim3(256), 0, s, b.at, h->N,
                     static_cast<uint4*>(out), out_stride * static_cast<int64_t>(elem_size(h->dtype)) / 16);
  return check_launch("gs_head_logit_grad");
}
