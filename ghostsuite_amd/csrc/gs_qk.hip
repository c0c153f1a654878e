// Per-head norms of queries and keys with their rotation by position, gfx950.  Per head row x of
// D features (queries and keys, each with a weight w):
//
//   r = (mean x^2 + eps)^(-1/2)    u = w x r                       (norm; else u = x)
//   (y_a, y_b) = (u_a c - u_b s, u_b c + u_a s)   for the n_rot / 2 pairs (a, b), c and s the
//                cosine and sine of the row's position; the features past n_rot stay as u
//
// and values are copied, all into heads-first layout [B, H, T, D].  Backward, with h = R^T g (the
// rotation by -angle):
//
//   dw = sum h x r      dx = r (w h - x r mean(w h x r))
//
// Everything in fp32 registers, rounded once at the end; a row is read once and written once, so
// the rate of a copy bounds both passes.  A row is cut into units of two chunks of V features: for
// pairs half the rotated width apart a unit holds chunk u of each half, and likewise of the halves of
// the features past them; for neighbouring pairs chunk u of each half of the row.  So a pair's two
// features are always in one lane, only the row sums cross lanes, and the lanes of a load or store lie
// side by side (both chunks in a row, 16 of every 32 bytes to a load, took 93 us for 89 in the forward
// pass of 8 x 2048 tokens of 24 heads of 256, 64 of them turned).  A group of 2^k lanes owns a row; it
// takes one token, keeps the token's angles and the lane's weights in registers, and walks that token's
// heads, so the angles are read once per token and the groups of a wave write neighbouring rows of one
// head.
//
// V is 16 bytes of features where the widths and strides allow it, else 2 or 1 features.
//
// Weight gradients: a lane adds up its features over its tokens and heads, a workgroup adds its
// groups through LDS in a fixed order and leaves one fp32 row; a second launch adds those per
// sample or in all, also in a fixed order (the same bits on every run).
#include <algorithm>
#include <type_traits>

#include "gs_common.h"

namespace gs {
namespace {

constexpr int QK_THREADS = 256;
constexpr int QK_BATCH = 4;   // heads whose loads are in flight together (forward)

// Rows of one of the three parts (queries, keys, values): element (b, t, h, f) at
// p[b sb + t st + h sh + f].
struct QkRows {
  char* p;
  int64_t sb, st, sh;
};

struct QkArgs {
  QkRows x[3];       // layer input rows (forward and backward)
  QkRows g[3];       // forward: the outputs; backward: the output gradients (p may be null)
  QkRows dx[3];      // backward: input gradients (p null: not formed)
  const void* w[3];  // query / key weights, or null: ones (the values': null)
  int w_bf16[3];
  int heads[3];
  int64_t B, T;      // samples and tokens of each
  int D, rot, lanes_log2;   // features, rotated features, log2 of the lanes of a row
  int norm;
  float eps;
  const float* table;       // [positions][2][rot / 2]: cosines, sines
  int64_t n_pos;
  int wide;                 // units' angles lie in whole vectors of V / 2
  const void* pos;          // null: a token's place in its sample
  int pos_bits;
  int64_t pos_sb, pos_st;
  // The work of a workgroup: heads [h0, h0 + per) of a part, and of its segment's tokens (the
  // segments: one of B T tokens, or B of T) every chunks-th piece of as many as it has lane groups.
  int64_t segments, seg_tokens, chunks;
  int groups[3], per[3];    // head groups of each part, heads of a group
  float* part[2];           // [segment][chunk][group][D] weight-gradient sums (backward)
};

// V features as they lie in memory, in whole 32-bit words where there are such.
template <class E, int V>
struct alignas(V * sizeof(E)) QkChunk {
  static constexpr int W = V * sizeof(E) >= 4 ? V * sizeof(E) / 4 : 1;
  std::conditional_t<V * sizeof(E) >= 4, uint32_t, uint16_t> w[W];
};
template <class E, int V>
__device__ __forceinline__ float qk_elem(const QkChunk<E, V>& c, int i) {
  if constexpr (sizeof(E) == 4) return __uint_as_float(c.w[i]);
  else if constexpr (V == 1) return bf16_to_f32(c.w[0]);
  else return __uint_as_float(i & 1 ? c.w[i >> 1] & 0xffff0000u : c.w[i >> 1] << 16);
}
template <class E, int V>
__device__ __forceinline__ QkChunk<E, V> qk_pack(const float (&x)[V]) {
  QkChunk<E, V> c;
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) c.w[i] = __float_as_uint(x[i]);
  } else if constexpr (V == 1) {
    c.w[0] = f32_to_bf16(x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) c.w[i >> 1] = pack_bf16x2(x[i], x[i + 1]);
  }
  return c;
}

// Unit u of a row: where its two chunks lie and which pairs' angles turn them.
template <int V, bool INTER>
struct QkPlace {
  int o0, o1;         // first features of the chunks (>= D: nothing there)
  int pair0, pair1;   // pairs of angles [0, V / 2) and [V / 2, V) of the unit
  __device__ QkPlace(int u, int D, int rot) {
    const int half = rot / 2, n = INTER ? 0 : half / V;   // V divides half
    const int m = (D - 2 * V * n + 2 * V - 1) / (2 * V);  // units past the turned halves
    if (INTER && V == 1) {
      o0 = 2 * u;
      o1 = o0 + 1;
      pair0 = pair1 = u;
    } else if (u < n) {
      o0 = V * u;
      o1 = half + o0;
      pair0 = o0;
      pair1 = pair0 + V / 2;
    } else {
      o0 = u < n + m ? 2 * V * n + V * (u - n) : D;
      o1 = o0 + V * m;
      pair0 = INTER ? o0 / 2 : half;
      pair1 = INTER ? o1 / 2 : half;
    }
    if (o0 >= D) o0 = D;
    if (o1 >= D) o1 = D;
  }
};

// A chunk as it lies in memory (whatever where the lane has nothing), and its features.
template <class E, int V>
__device__ __forceinline__ QkChunk<E, V> qk_load(const E* __restrict__ row, int o, int D) {
  QkChunk<E, V> c;
  if (o < D) c = *reinterpret_cast<const QkChunk<E, V>*>(row + o);
  return c;
}
template <class E, int V>
__device__ __forceinline__ void qk_unpack(const QkChunk<E, V>& c, int o, int D, float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = o < D ? qk_elem<E, V>(c, i) : 0.f;
}

template <class E, int V>
__device__ __forceinline__ void qk_store(E* __restrict__ row, int o, int D, const float (&x)[V]) {
  if (o < D) *reinterpret_cast<QkChunk<E, V>*>(row + o) = qk_pack<E, V>(x);
}

// One unit's values: the two chunks.
template <int V>
struct QkUnit {
  float a[V], b[V];
};

// Which pairs of a unit turn: all or none ([0]), or where neighbours turn each for itself.
template <int V, bool INTER>
struct QkTurns {
  bool pair[INTER ? V : 1];
  __device__ __forceinline__ void set(const QkPlace<V, INTER>& pl, int rot) {
#pragma unroll
    for (int i = 0; i < (INTER ? V : 1); ++i)
      pair[i] = (!INTER || i < V / 2 ? pl.pair0 + i : pl.pair1 + i - V / 2) < rot / 2;
  }
};

// The rotation of a unit's pairs that turn by their angles (sign +1) or back (-1).  Others stay as
// they are, not turned by an angle of zero: an infinity times its sine would reach the pair's other
// feature.
template <int V, bool INTER>
__device__ __forceinline__ void qk_rotate(QkUnit<V>& u, const QkTurns<V, INTER>& t,
                                          const float (&c)[V], const float (&s)[V], float sign) {
  if constexpr (!INTER) {
    if (!t.pair[0]) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = u.a[i], y = u.b[i], si = sign * s[i];
      u.a[i] = x * c[i] - y * si;
      u.b[i] = y * c[i] + x * si;
    }
  } else {
    // Pair i is features 2 i and 2 i + 1 of the unit's 2 V.
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float& x = 2 * i < V ? u.a[2 * i < V ? 2 * i : 0] : u.b[2 * i < V ? 0 : 2 * i - V];
      float& y = 2 * i + 1 < V ? u.a[2 * i + 1 < V ? 2 * i + 1 : 0]
                               : u.b[2 * i + 1 < V ? 0 : 2 * i + 1 - V];
      const float x0 = x, y0 = y, si = sign * s[i];
      x = t.pair[i] ? x0 * c[i] - y0 * si : x0;
      y = t.pair[i] ? y0 * c[i] + x0 * si : y0;
    }
  }
}

// The sum over the 2^k lanes of a row's group, in each of them: by DPP within 16 lanes (pairs, quads,
// then mirrored halves, which are even by then), by shuffles beyond.
__device__ __forceinline__ float qk_group_sum(float v, int lanes_log2) {
  if (lanes_log2 >= 1) v += dpp_f32<0xb1, 0xf, 0xf>(v);
  if (lanes_log2 >= 2) v += dpp_f32<0x4e, 0xf, 0xf>(v);
  if (lanes_log2 >= 3) v += dpp_f32<0x141, 0xf, 0xf>(v);
  if (lanes_log2 >= 4) v += dpp_f32<0x140, 0xf, 0xf>(v);
  if (lanes_log2 >= 5) v += __shfl_xor(v, 16, 64);
  if (lanes_log2 >= 6) v += __shfl_xor(v, 32, 64);
  return v;
}

__device__ __forceinline__ int64_t qk_position(const QkArgs& a, int64_t b, int64_t t) {
  if (a.pos == nullptr) return t;
  const int64_t i = b * a.pos_sb + t * a.pos_st;
  return a.pos_bits == 32 ? static_cast<const int32_t*>(a.pos)[i]
                          : static_cast<const int64_t*>(a.pos)[i];
}

// Cosines and sines of a unit's pairs at a position (past the rotated ones 1 and 0, not used); a
// position outside the table: NaN.  In whole vectors where the table's rows split there: 20 x 1024
// tokens of 12 + 12 + 12 heads of 64, bf16, 16 loads of one number take 46.6 us forward, 4 of four 43.4.
template <int V>
__device__ __forceinline__ void qk_angles(const QkArgs& a, int64_t pos, int pair0, int pair1,
                                          float (&c)[V], float (&s)[V]) {
  constexpr int H = V > 1 ? V / 2 : 1;
  struct alignas(H * sizeof(float)) Angles { float f[H]; };
  const int half = a.rot / 2;
  const bool in = pos >= 0 && pos < a.n_pos;
  const float* row = a.table + (in ? pos : 0) * a.rot;
  const float nan = __builtin_nanf("");
  if (H > 1 && a.wide) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int pair = k ? pair1 : pair0;
      const bool turns = pair < half;
      Angles x, y;
      if (turns) {
        x = *reinterpret_cast<const Angles*>(row + pair);
        y = *reinterpret_cast<const Angles*>(row + half + pair);
      }
#pragma unroll
      for (int i = 0; i < H; ++i) {
        c[k * H + i] = turns ? (in ? x.f[i] : nan) : 1.f;
        s[k * H + i] = turns ? (in ? y.f[i] : nan) : 0.f;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int pair = i < V / 2 ? pair0 + i : pair1 + i - V / 2;
    const bool turns = pair < half;
    c[i] = turns ? (in ? row[pair] : nan) : 1.f;
    s[i] = turns ? (in ? row[half + pair] : nan) : 0.f;
  }
}

// V weights of a part from feature f on (ones past the row, or without weights).
template <int V>
__device__ __forceinline__ void qk_weights(const QkArgs& a, int part, int f, float (&w)[V]) {
  const void* p = a.w[part];
  if (p == nullptr || f >= a.D) {
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = 1.f;
  } else if (a.w_bf16[part]) {
    const QkChunk<uint16_t, V> x = qk_load<uint16_t, V>(static_cast<const uint16_t*>(p), f, a.D);
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = qk_elem<uint16_t, V>(x, i);
  } else {
    constexpr int N = V > 4 ? 4 : V;   // 16 bytes at most
#pragma unroll
    for (int k = 0; k < V; k += N) {
      const QkChunk<float, N> x = qk_load<float, N>(static_cast<const float*>(p), f + k, a.D);
#pragma unroll
      for (int i = 0; i < N; ++i) w[k + i] = qk_elem<float, N>(x, i);
    }
  }
}

// The workgroup's part and heads, and the lane group's tokens.  Workgroups are numbered through the head
// groups of a piece of tokens first, so that those at work at one time read and write near each other.
struct QkBlock {
  int part, h0, h1, group;
  uint32_t seg, chunk;
  uint32_t m0, m1, step;   // tokens m0, m0 + step, ... below m1, numbered over all samples (below 2^31)
  __device__ explicit QkBlock(const QkArgs& a) {
    const uint32_t gy = a.groups[0] + a.groups[1] + a.groups[2], bx = blockIdx.x / gy;
    int y = blockIdx.x - bx * gy;
    part = 0;
    while (part < 2 && y >= a.groups[part]) y -= a.groups[part++];
    group = y;
    h0 = y * a.per[part];
    h1 = min(a.heads[part], h0 + a.per[part]);
    const uint32_t chunks = static_cast<uint32_t>(a.chunks), slots = QK_THREADS >> a.lanes_log2;
    seg = bx / chunks;
    chunk = bx - seg * chunks;
    m0 = seg * static_cast<uint32_t>(a.seg_tokens);
    m1 = m0 + static_cast<uint32_t>(a.seg_tokens);
    m0 += chunk * slots + (threadIdx.x >> a.lanes_log2);
    step = chunks * slots;
  }
};

template <class E, int V, int UPL, bool INTER>
__global__ void __launch_bounds__(QK_THREADS) qk_forward_kernel(QkArgs a) {
  const QkBlock blk(a);
  const int lanes = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const bool turn = blk.part < 2 && a.rot > 0, norm = blk.part < 2 && a.norm;
  QkUnit<V> w[UPL];
  QkTurns<V, INTER> turns[UPL];
#pragma unroll
  for (int j = 0; j < UPL; ++j)
    turns[j].set(QkPlace<V, INTER>(lane + j * lanes, a.D, a.rot), a.rot);
  if (norm) {
#pragma unroll
    for (int j = 0; j < UPL; ++j) {
      const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
      qk_weights<V>(a, blk.part, pl.o0, w[j].a);
      qk_weights<V>(a, blk.part, pl.o1, w[j].b);
    }
  }
  const QkRows in = a.x[blk.part], out = a.g[blk.part];
  const float inv_d = 1.f / static_cast<float>(a.D);
  for (uint32_t m = blk.m0; m < blk.m1; m += blk.step) {
    const uint32_t of = m / static_cast<uint32_t>(a.T);
    const int64_t b = of, t = m - of * static_cast<uint32_t>(a.T);
    float c[UPL][V], s[UPL][V];
    if (turn) {
      const int64_t pos = qk_position(a, b, t);
#pragma unroll
      for (int j = 0; j < UPL; ++j) {
        const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
        qk_angles<V>(a, pos, pl.pair0, pl.pair1, c[j], s[j]);
      }
    }
    const E* xr = reinterpret_cast<const E*>(in.p) + b * in.sb + t * in.st;
    E* yr = reinterpret_cast<E*>(out.p) + b * out.sb + t * out.st;
    for (int h = blk.h0; h < blk.h1; h += QK_BATCH) {
      QkChunk<E, V> raw[QK_BATCH][UPL][2];
#pragma unroll
      for (int q = 0; q < QK_BATCH; ++q) {
        if (h + q >= blk.h1) break;
#pragma unroll
        for (int j = 0; j < UPL; ++j) {
          const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
          raw[q][j][0] = qk_load<E, V>(xr + (h + q) * in.sh, pl.o0, a.D);
          raw[q][j][1] = qk_load<E, V>(xr + (h + q) * in.sh, pl.o1, a.D);
        }
      }
#pragma unroll
      for (int q = 0; q < QK_BATCH; ++q) {
        if (h + q >= blk.h1) break;
        QkUnit<V> u[UPL];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < UPL; ++j) {
          const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
          qk_unpack<E, V>(raw[q][j][0], pl.o0, a.D, u[j].a);
          qk_unpack<E, V>(raw[q][j][1], pl.o1, a.D, u[j].b);
#pragma unroll
          for (int i = 0; i < V; ++i) ss += u[j].a[i] * u[j].a[i] + u[j].b[i] * u[j].b[i];
        }
        const float r = norm ? rsqrtf(qk_group_sum(ss, a.lanes_log2) * inv_d + a.eps) : 1.f;
#pragma unroll
        for (int j = 0; j < UPL; ++j) {
          if (norm) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              u[j].a[i] *= r * w[j].a[i];
              u[j].b[i] *= r * w[j].b[i];
            }
          }
          if (turn) qk_rotate<V, INTER>(u[j], turns[j], c[j], s[j], 1.f);
          const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
          qk_store<E, V>(yr + (h + q) * out.sh, pl.o0, a.D, u[j].a);
          qk_store<E, V>(yr + (h + q) * out.sh, pl.o1, a.D, u[j].b);
        }
      }
    }
  }
}

template <class E, int V, int UPL, bool INTER>
__global__ void __launch_bounds__(QK_THREADS) qk_backward_kernel(QkArgs a) {
  const QkBlock blk(a);
  const int lanes = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const QkRows in = a.x[blk.part], go = a.g[blk.part], dx = a.dx[blk.part];
  const bool any_g = go.p != nullptr;   // else every gradient of the part is zero
  const bool turn = blk.part < 2 && a.rot > 0 && any_g, norm = blk.part < 2 && a.norm && any_g;
  const bool want_w = blk.part < 2 && a.part[blk.part] != nullptr;
  QkUnit<V> w[UPL], dw[UPL];
  QkTurns<V, INTER> turns[UPL];
#pragma unroll
  for (int j = 0; j < UPL; ++j) {
    const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
    turns[j].set(pl, a.rot);
    qk_weights<V>(a, norm ? blk.part : 2, pl.o0, w[j].a);
    qk_weights<V>(a, norm ? blk.part : 2, pl.o1, w[j].b);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[j].a[i] = dw[j].b[i] = 0.f;
  }
  const float inv_d = 1.f / static_cast<float>(a.D);
  for (uint32_t m = blk.m0; m < blk.m1; m += blk.step) {
    const uint32_t of = m / static_cast<uint32_t>(a.T);
    const int64_t b = of, t = m - of * static_cast<uint32_t>(a.T);
    float c[UPL][V], s[UPL][V];
    if (turn) {
      const int64_t pos = qk_position(a, b, t);
#pragma unroll
      for (int j = 0; j < UPL; ++j) {
        const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
        qk_angles<V>(a, pos, pl.pair0, pl.pair1, c[j], s[j]);
      }
    }
    const E* xr = reinterpret_cast<const E*>(in.p) + b * in.sb + t * in.st;
    const E* gr = reinterpret_cast<const E*>(go.p) + b * go.sb + t * go.st;
    E* dr = reinterpret_cast<E*>(dx.p) + b * dx.sb + t * dx.st;
    // the next head's rows are on their way while one is worked on
    QkChunk<E, V> graw[UPL][2], xraw[UPL][2];
    const auto fetch = [&](int h) {
#pragma unroll
      for (int j = 0; j < UPL; ++j) {
        const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
        if (any_g) {
          graw[j][0] = qk_load<E, V>(gr + h * go.sh, pl.o0, a.D);
          graw[j][1] = qk_load<E, V>(gr + h * go.sh, pl.o1, a.D);
        }
        if (norm) {
          xraw[j][0] = qk_load<E, V>(xr + h * in.sh, pl.o0, a.D);
          xraw[j][1] = qk_load<E, V>(xr + h * in.sh, pl.o1, a.D);
        }
      }
    };
    fetch(blk.h0);
    for (int h = blk.h0; h < blk.h1; ++h) {
      QkUnit<V> x[UPL], g[UPL];
#pragma unroll
      for (int j = 0; j < UPL; ++j) {
        const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
        qk_unpack<E, V>(graw[j][0], any_g ? pl.o0 : a.D, a.D, g[j].a);
        qk_unpack<E, V>(graw[j][1], any_g ? pl.o1 : a.D, a.D, g[j].b);
        if (norm) {
          qk_unpack<E, V>(xraw[j][0], pl.o0, a.D, x[j].a);
          qk_unpack<E, V>(xraw[j][1], pl.o1, a.D, x[j].b);
        }
      }
      if (h + 1 < blk.h1) fetch(h + 1);
      if (turn) {
#pragma unroll
        for (int j = 0; j < UPL; ++j) qk_rotate<V, INTER>(g[j], turns[j], c[j], s[j], -1.f);
      }
      if (norm) {
        float ss = 0.f, sd = 0.f;
#pragma unroll
        for (int j = 0; j < UPL; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            ss += x[j].a[i] * x[j].a[i] + x[j].b[i] * x[j].b[i];
            sd += w[j].a[i] * g[j].a[i] * x[j].a[i] + w[j].b[i] * g[j].b[i] * x[j].b[i];
          }
        ss = qk_group_sum(ss, a.lanes_log2);
        sd = qk_group_sum(sd, a.lanes_log2);
        const float r = rsqrtf(ss * inv_d + a.eps);
        const float k = sd * r * r * inv_d;   // mean(w h x r) r
#pragma unroll
        for (int j = 0; j < UPL; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            dw[j].a[i] += g[j].a[i] * (x[j].a[i] * r);
            dw[j].b[i] += g[j].b[i] * (x[j].b[i] * r);
            g[j].a[i] = r * (w[j].a[i] * g[j].a[i] - x[j].a[i] * k);
            g[j].b[i] = r * (w[j].b[i] * g[j].b[i] - x[j].b[i] * k);
          }
      }
      if (dx.p != nullptr) {
#pragma unroll
        for (int j = 0; j < UPL; ++j) {
          const QkPlace<V, INTER> pl(lane + j * lanes, a.D, a.rot);
          qk_store<E, V>(dr + h * dx.sh, pl.o0, a.D, g[j].a);
          qk_store<E, V>(dr + h * dx.sh, pl.o1, a.D, g[j].b);
        }
      }
    }
  }
  if (!want_w) return;   // the same for the whole workgroup
  // The workgroup's sum: groups of a wave by shuffles, waves through LDS, in wave order.
  __shared__ float red[QK_THREADS / 64][2 * V * UPL * 64];
  const int wid = threadIdx.x >> 6, wl = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < UPL; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float p = dw[j].a[i], q = dw[j].b[i];
      for (int k = lanes; k < 64; k <<= 1) {
        p += __shfl_xor(p, k, 64);
        q += __shfl_xor(q, k, 64);
      }
      if (wl < lanes) {
        red[wid][((j * 2 + 0) * V + i) * 64 + wl] = p;
        red[wid][((j * 2 + 1) * V + i) * 64 + wl] = q;
      }
    }
  __syncthreads();
  float* out = a.part[blk.part] +
               ((blk.seg * a.chunks + blk.chunk) * a.groups[blk.part] + blk.group) * a.D;
  for (int k = threadIdx.x; k < 2 * V * UPL * lanes; k += QK_THREADS) {
    const int l = k & (lanes - 1), v = k >> a.lanes_log2;   // v = (j * 2 + side) * V + i
    const int i = v % V, side = (v / V) & 1, j = v / (2 * V);
    const QkPlace<V, INTER> pl(l + j * lanes, a.D, a.rot);
    const int f = (side ? pl.o1 : pl.o0) + i;
    float t = 0.f;
#pragma unroll
    for (int q = 0; q < QK_THREADS / 64; ++q) t += red[q][v * 64 + l];
    if (f < a.D) out[f] = t;
  }
}

// Sums of the partial rows, one for each row y of the grid (from y0 on).  y below `samples`:
// out[part][y][f] = the sum of sample y's rows; y = samples: `val`, the val samples' rows; y = samples
// + 1: the train samples' rows times the scale, as a weight gradient (outputs that are null are left
// out).  Partial rows lie in sample order, so each is one range of rows or two.  A workgroup takes 16
// features; its 64 groups of 16 threads take every 64th row and are added in a fixed order.
constexpr int QR_COLS = 16, QR_GROUPS = 64;
struct QkSums {
  const float* part[2];
  int64_t rows[2];      // partial rows of a sample
  int64_t samples, n_val, val_start, y0;
  float* out[2];        // [samples][D] or null
  float* val[2];        // [D] or null
  void* grad[2];        // [D] or null
  int grad_bf16[2];
  float scale;
  int D;
};
__global__ void __launch_bounds__(QR_COLS * QR_GROUPS) qk_sums_kernel(QkSums q) {
  __shared__ float red[QR_GROUPS][QR_COLS];
  const int part = blockIdx.z;
  const int64_t y = q.y0 + blockIdx.y, n = q.samples;
  const int col = threadIdx.x % QR_COLS, grp = threadIdx.x / QR_COLS;
  const int f = blockIdx.x * QR_COLS + col;
  const int64_t rows = q.rows[part], v0 = q.val_start, v1 = v0 + q.n_val;
  const bool is_sample = y < n, is_val = y == n;
  const int64_t lo[2] = {is_sample ? y : is_val ? v0 : 0, is_sample || is_val ? 0 : v1};
  const int64_t hi[2] = {is_sample ? y + 1 : is_val ? v1 : v0, is_sample || is_val ? 0 : n};
  float t0 = 0.f, t1 = 0.f;
  if (f < q.D && q.part[part] != nullptr) {
    const float* p = q.part[part] + f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      int64_t r = lo[k] * rows + grp;
      const int64_t end = hi[k] * rows;
      for (; r + QR_GROUPS < end; r += 2 * QR_GROUPS) {
        t0 += p[r * q.D];
        t1 += p[(r + QR_GROUPS) * q.D];
      }
      if (r < end) t0 += p[r * q.D];
    }
  }
  red[grp][col] = t0 + t1;
  for (int k = QR_GROUPS / 2; k > 0; k >>= 1) {
    __syncthreads();
    if (grp < k) red[grp][col] += red[grp + k][col];
  }
  if (grp != 0 || f >= q.D) return;
  const float t = red[0][col];
  if (is_sample) {
    if (q.out[part] != nullptr) q.out[part][y * q.D + f] = t;
  } else if (is_val) {
    if (q.val[part] != nullptr) q.val[part][f] = t;
  } else if (q.grad[part] != nullptr) {
    if (q.grad_bf16[part])
      static_cast<uint16_t*>(q.grad[part])[f] = f32_to_bf16(q.scale * t);
    else
      static_cast<float*>(q.grad[part])[f] = q.scale * t;
  }
}

// dot[part][i] = <S[part][train sample i], val[part]>, a wave each.
struct QkDots {
  const float* S[2];
  const float* val[2];
  float* dot[2];
};
__global__ void __launch_bounds__(64) qk_dots_kernel(QkDots q, RowMap train, int D) {
  const int part = blockIdx.y;
  if (q.dot[part] == nullptr) return;
  const float* row = q.S[part] + train.phys_sample(blockIdx.x) * D;
  float t = 0.f;
  for (int f = threadIdx.x; f < D; f += 64) t += row[f] * q.val[part][f];
  t = wave_sum(t);
  if (threadIdx.x == 0) q.dot[part][blockIdx.x] = t;
}

// Dots and train gradients of few samples in one launch: workgroup x below the train samples adds the
// val samples' rows up for itself (they lie in the caches) and takes sample x's dot; those behind take
// 64 features each of the gradient, the train samples' rows in order.  (The host's part is what counts
// here: 14 us a call with two launches and their workspace, 10 with this.)
constexpr int64_t QK_FEW_SAMPLES = 128;
struct QkFew {
  const float* S[2];
  float* dot[2];
  void* grad[2];
  int grad_bf16[2];
  int n_train, n_val, val_start, D;
  float scale;
};
__global__ void __launch_bounds__(64) qk_few_dots_kernel(QkFew q) {
  const int part = blockIdx.y, x = blockIdx.x, lane = threadIdx.x;
  const float* S = q.S[part];
  const auto train = [&](int i) {
    return S + static_cast<int64_t>(i + (i >= q.val_start ? q.n_val : 0)) * q.D;
  };
  if (x < q.n_train) {
    if (q.dot[part] == nullptr) return;
    const float *row = train(x), *val = S + static_cast<int64_t>(q.val_start) * q.D;
    float t = 0.f;
    for (int f = lane; f < q.D; f += 64) {
      float v = 0.f;
#pragma unroll 8
      for (int j = 0; j < q.n_val; ++j) v += val[static_cast<int64_t>(j) * q.D + f];
      t += row[f] * v;
    }
    t = wave_sum(t);
    if (lane == 0) q.dot[part][x] = t;
    return;
  }
  const int f = (x - q.n_train) * 64 + lane;
  if (f >= q.D || q.grad[part] == nullptr) return;
  float t = 0.f;
#pragma unroll 8
  for (int i = 0; i < q.n_train; ++i) t += train(i)[f];
  t *= q.scale;
  if (q.grad_bf16[part])
    static_cast<uint16_t*>(q.grad[part])[f] = f32_to_bf16(t);
  else
    static_cast<float*>(q.grad[part])[f] = t;
}

constexpr int QK_MAX_D = 512;

// Features a lane takes at once: 16 bytes of them where every row starts and splits there.
int qk_vec(const QkArgs& a, size_t esz, bool inter, bool backward) {
  const int half = a.rot / 2;
  for (int v : {static_cast<int>(16 / esz), 2}) {
    bool ok = a.D % v == 0 && (inter || half % v == 0) && (inter || a.rot % v == 0);
    for (int k = 0; k < 2 && ok; ++k)   // weights are read in chunks of 16 bytes at most
      ok = a.w[k] == nullptr || a.heads[k] == 0 ||
           reinterpret_cast<uintptr_t>(a.w[k]) %
                   std::min<size_t>(16, v * (a.w_bf16[k] ? 2 : 4)) == 0;
    for (int k = 0; k < 3 && ok; ++k) {
      if (a.heads[k] == 0) continue;
      for (const QkRows* r : {&a.x[k], &a.g[k], &a.dx[k]}) {
        if (r == &a.dx[k] && !backward) continue;
        if (r->p == nullptr) continue;
        ok = ok && reinterpret_cast<uintptr_t>(r->p) % (v * esz) == 0 && r->sb % v == 0 &&
             r->st % v == 0 && r->sh % v == 0;
      }
    }
    if (ok) return v;
  }
  return 1;
}

int qk_units(int D, int rot, int V, bool inter) {
  if (inter) return (D + 2 * V - 1) / (2 * V);
  return rot / 2 / V + (D - rot + 2 * V - 1) / (2 * V);
}

int ceil_log2(int64_t x) {
  int k = 0;
  while ((int64_t{1} << k) < x) ++k;
  return k;
}

// How the work is shared out.  Backward into the waves whose registers fit at once (3 for each SIMD; a
// wave's end, its sum of weight gradients, costs more than its start), forward into 16 for each SIMD.
// Few heads to a workgroup give many workgroups to a token, which then read its row together; a few
// heads share the angles: 4 forward; backward, of 4, 6 and 3, the number that leaves the fewest turns, a
// turn costing its heads and half of one more for the angles; fewer where two workgroups to a CU would
// not be reached.  Measured on MI355X, two inputs in turn (forward / both passes, us), with tokens in
// ranges of their own, part after part, 3 waves a SIMD -> this: 20 x 1024 tokens of 12 + 12 + 12 heads
// of 64, bf16, 42.5 / 107 -> 37.5 / 104; 8 x 2048 of 8 + 8 + 8 of 256, 64 turned, 93 / 226 -> 79 / 190;
// 20 x 512 of 16 + 4 + 4 of 128, 23.5 / 71 -> 24 / 71, fp32 54 / 158 -> 44.5 / 125 (copies of the forward
// pass's bytes: 35, 76, 20 in bf16).
constexpr int64_t QK_FORWARD_GROUPS = 16 * 256, QK_BACKWARD_GROUPS = 3 * 256;   // workgroups of 4 waves
constexpr int64_t QK_FEW_GROUPS = 2 * 256;
constexpr int64_t QK_MAX_GROUPS = int64_t{1} << 22;   // of a launch: below 2^32 threads
void qk_share(QkArgs& a, int upl, int units, bool per_sample, bool backward) {
  a.lanes_log2 = std::min(6, ceil_log2((units + upl - 1) / upl));
  const int64_t slots = QK_THREADS >> a.lanes_log2;
  a.segments = per_sample ? a.B : 1;
  a.seg_tokens = per_sample ? a.T : a.B * a.T;
  const int64_t pieces = (a.seg_tokens + slots - 1) / slots;
  const int64_t want = backward ? QK_BACKWARD_GROUPS : QK_FORWARD_GROUPS;
  const auto groups = [&](int per) {
    int64_t y = 0;
    for (int k = 0; k < 3; ++k) y += (a.heads[k] + per - 1) / per;
    return y;
  };
  const auto chunks = [&](int per) {
    return std::max<int64_t>(1, std::min(pieces, want / (a.segments * groups(per))));
  };
  const auto turns = [&](int per) {
    const int64_t c = chunks(per), n = a.segments * c * groups(per);
    return (pieces + c - 1) / c * ((n + want - 1) / want);
  };
  int per = 4;
  for (int p : {6, 3})
    if (backward && turns(p) * (2 * p + 1) < turns(per) * (2 * per + 1)) per = p;
  while (per > 1 && a.segments * chunks(per) * groups(per) < QK_FEW_GROUPS) --per;
  if (a.segments * groups(per) > QK_MAX_GROUPS) per = std::max({a.heads[0], a.heads[1], a.heads[2]});
  for (int k = 0; k < 3; ++k) {
    a.groups[k] = (a.heads[k] + per - 1) / per;
    a.per[k] = a.groups[k] ? (a.heads[k] + a.groups[k] - 1) / a.groups[k] : 1;
  }
  a.chunks = chunks(per);
}

template <class E, bool BWD, bool INTER>
int qk_launch(const QkArgs& a, int v, hipStream_t s) {
  constexpr int V16 = 16 / sizeof(E);
  const dim3 grid(static_cast<unsigned>(a.segments * a.chunks *
                                        (a.groups[0] + a.groups[1] + a.groups[2])));
#define GS_QK_GO(V, UPL)                                                                       \
  do {                                                                                         \
    if constexpr (BWD)                                                                         \
      hipLaunchKernelGGL((qk_backward_kernel<E, V, UPL, INTER>), grid, dim3(QK_THREADS), 0, s, \
                         a);                                                                   \
    else                                                                                       \
      hipLaunchKernelGGL((qk_forward_kernel<E, V, UPL, INTER>), grid, dim3(QK_THREADS), 0, s,  \
                         a);                                                                   \
  } while (0)
  if (v == V16)
    GS_QK_GO(V16, 1);
  else if (v == 2)
    GS_QK_GO(2, 2);
  else
    GS_QK_GO(1, 4);
#undef GS_QK_GO
  return check_launch(BWD ? "qk_backward_kernel" : "qk_forward_kernel");
}

int qk_units_per_lane(int v, size_t esz) {
  return v == static_cast<int>(16 / esz) ? 1 : v == 2 ? 2 : 4;
}

template <bool BWD>
int qk_run(const QkArgs& a, int dtype, bool inter, int v, hipStream_t s) {
  if (dtype == GS_DTYPE_BF16)
    return inter ? qk_launch<uint16_t, BWD, true>(a, v, s)
                 : qk_launch<uint16_t, BWD, false>(a, v, s);
  return inter ? qk_launch<float, BWD, true>(a, v, s) : qk_launch<float, BWD, false>(a, v, s);
}

QkRows rows_of(const gs_qk_rows& r) {
  return QkRows{static_cast<char*>(r.data), r.stride_b, r.stride_t, r.stride_h};
}

// Fills the common arguments; a status other than GS_OK refuses the call.
int qk_args(QkArgs& a, const char* name, const gs_qk_shape* sh, const gs_qk_rows x[3],
            const gs_qk_rows g[3], const gs_qk_rows dx[3]) {
  const std::string n(name);
  if (sh == nullptr) return fail(GS_ERR_INVALID, n + ": no shape");
  if (sh->dtype != GS_DTYPE_BF16 && sh->dtype != GS_DTYPE_F32)
    return fail(GS_ERR_DTYPE, n + ": dtype must be bf16 or fp32");
  for (int k = 0; k < 2; ++k)
    if (sh->weight[k] != nullptr && sh->weight_dtype[k] != GS_DTYPE_BF16 &&
        sh->weight_dtype[k] != GS_DTYPE_F32)
      return fail(GS_ERR_DTYPE, n + ": weight dtypes must be bf16 or fp32");
  if (sh->B <= 0 || sh->T <= 0 || sh->D <= 0 || sh->n_rot < 0 || sh->n_rot > sh->D ||
      sh->n_rot % 2 != 0 || sh->heads[0] < 0 || sh->heads[1] < 0 || sh->heads[2] < 0 ||
      static_cast<int64_t>(sh->heads[0]) + sh->heads[1] + sh->heads[2] <= 0 || !(sh->eps >= 0.f) ||
      (sh->positions != nullptr && sh->position_bits != 32 && sh->position_bits != 64) ||
      (sh->n_rot > 0 && (sh->table == nullptr || sh->n_positions <= 0)))
    return fail(GS_ERR_INVALID, n + ": invalid arguments");
  if (sh->D > QK_MAX_D)
    return fail(GS_ERR_UNSUPPORTED, n + ": more than 512 features to a head");
  // tokens, and the workgroups of one sample's head groups, are numbered in 32 bits with room to spare
  if (static_cast<int64_t>(sh->heads[0]) + sh->heads[1] + sh->heads[2] > 65535 ||
      sh->B > INT32_MAX / sh->T)
    return fail(GS_ERR_UNSUPPORTED, n + ": more than 65535 heads or 2^31 tokens");
  if (sh->n_rot > 0 && sh->positions == nullptr && sh->T > sh->n_positions)
    return fail(GS_ERR_INVALID, n + ": more tokens to a sample than positions in the table");
  a = QkArgs{};
  for (int k = 0; k < 3; ++k) {
    a.heads[k] = sh->heads[k];
    if (a.heads[k] == 0) continue;
    if (x != nullptr) a.x[k] = rows_of(x[k]);
    if (g != nullptr) a.g[k] = rows_of(g[k]);
    if (dx != nullptr) a.dx[k] = rows_of(dx[k]);
  }
  for (int k = 0; k < 2; ++k) {
    a.w[k] = sh->weight[k];
    a.w_bf16[k] = sh->weight_dtype[k] == GS_DTYPE_BF16;
  }
  a.B = sh->B, a.T = sh->T, a.D = static_cast<int>(sh->D), a.rot = static_cast<int>(sh->n_rot);
  a.norm = sh->norm, a.eps = sh->eps;
  a.table = sh->table, a.n_pos = sh->n_positions;
  a.pos = sh->positions, a.pos_bits = sh->position_bits;
  a.pos_sb = sh->position_stride_b, a.pos_st = sh->position_stride_t;
  return GS_OK;
}

struct QkPlan {
  int v;
  int64_t rows[2];   // partial rows of a segment
};

QkPlan qk_plan(QkArgs& a, int dtype, bool inter, bool backward, bool per_sample, int force_v = 0) {
  QkPlan p;
  const size_t esz = elem_size(dtype);
  p.v = force_v ? force_v : qk_vec(a, esz, inter, backward);
  a.wide = p.v > 2 && a.rot / 2 % (p.v / 2) == 0 &&
           reinterpret_cast<uintptr_t>(a.table) % (p.v / 2 * sizeof(float)) == 0;
  qk_share(a, qk_units_per_lane(p.v, esz), qk_units(a.D, a.rot, p.v, inter), per_sample, backward);
  for (int k = 0; k < 2; ++k) p.rows[k] = a.chunks * a.groups[k];
  return p;
}

struct QkScratch {
  float *part[2], *sums[2], *val[2];
  template <class S>
  QkScratch(S& c, const QkArgs& a, const QkPlan& p) {
    for (int k = 0; k < 2; ++k) {
      part[k] = c.template take<float>(a.segments * p.rows[k] * a.D);
      sums[k] = c.template take<float>(a.segments * a.D);
      val[k] = c.template take<float>(a.D);
    }
  }
};

// The strides decide the vector width and so the plan; the query does not know them, so it takes
// the most any plan needs, with and without the values' heads.
size_t qk_workspace(const gs_qk_shape* sh, bool per_sample) {
  QkArgs a;
  if (qk_args(a, "gs_qk_rotary", sh, nullptr, nullptr, nullptr) != GS_OK) return 0;
  size_t most = 0;
  for (int values : {a.heads[2], 0}) {
    for (int v : {static_cast<int>(16 / elem_size(sh->dtype)), 2, 1}) {
      QkArgs t = a;
      t.heads[2] = values;
      if (t.heads[0] + t.heads[1] == 0 || (sh->interleaved == 0 && a.rot / 2 % v != 0)) continue;
      const QkPlan p = qk_plan(t, sh->dtype, sh->interleaved != 0, true, per_sample, v);
      Sizer sz;
      QkScratch unused(sz, t, p);
      most = std::max(most, sz.used);
    }
  }
  return most + 256;
}

int qk_check_rows(const char* name, const gs_qk_shape* sh, const gs_qk_rows* r, bool needed) {
  for (int k = 0; k < 3; ++k)
    if (needed && sh->heads[k] > 0 && r[k].data == nullptr)
      return fail(GS_ERR_INVALID, std::string(name) + ": invalid arguments");
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_qk_rotary(const gs_qk_shape* shape, const gs_qk_rows x[3],
                            const gs_qk_rows y[3], void* stream) {
  QkArgs a;
  if (int rc = qk_args(a, "gs_qk_rotary", shape, x, y, nullptr)) return rc;
  if (x == nullptr || y == nullptr || qk_check_rows("gs_qk_rotary", shape, x, true) != GS_OK ||
      qk_check_rows("gs_qk_rotary", shape, y, true) != GS_OK)
    return fail(GS_ERR_INVALID, "gs_qk_rotary: invalid arguments");
  const bool inter = shape->interleaved != 0;
  const QkPlan p = qk_plan(a, shape->dtype, inter, false, false);
  return qk_run<false>(a, shape->dtype, inter, p.v, static_cast<hipStream_t>(stream));
}

namespace gs {
namespace {

// The dots from the samples' and the val samples' sums; one launch.
int qk_launch_dots(const float* const S[2], float* const val[2], float* const dot[2], int64_t B,
                   int64_t n_val, int64_t val_start, int D, hipStream_t s) {
  QkDots o{};
  for (int k = 0; k < 2; ++k) o.S[k] = S[k], o.val[k] = val[k], o.dot[k] = dot[k];
  hipLaunchKernelGGL(qk_dots_kernel, dim3(static_cast<unsigned>(B - n_val), 2), dim3(64), 0, s, o,
                     train_rows(B, n_val, val_start, 1), D);
  return check_launch("qk_dots_kernel");
}

void qk_launch_sums(const QkSums& q, int64_t rows, hipStream_t s) {
  hipLaunchKernelGGL(qk_sums_kernel,
                     dim3((q.D + QR_COLS - 1) / QR_COLS, static_cast<unsigned>(rows), 2),
                     dim3(QR_COLS * QR_GROUPS), 0, s, q);
}

bool qk_split_ok(int64_t B, int64_t n_val, int64_t val_start) {
  return n_val > 0 && n_val < B && val_start >= 0 && val_start + n_val <= B;
}
constexpr int64_t QK_MAX_SAMPLES = 65533;   // the sums' grid

}  // namespace
}  // namespace gs

extern "C" size_t gs_qk_rotary_grad_workspace(const gs_qk_shape* shape, int per_sample) {
  return qk_workspace(shape, per_sample != 0);
}

extern "C" int gs_qk_rotary_grad(const gs_qk_shape* shape, const gs_qk_rows x[3],
                                 const gs_qk_rows dy[3], const gs_qk_rows dx[3], void* grad_qw,
                                 void* grad_kw, float* sample_grads, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  QkArgs a;
  if (int rc = qk_args(a, "gs_qk_rotary_grad", shape, x, dy, dx)) return rc;
  void* gw[2] = {grad_qw, grad_kw};
  const bool samples = sample_grads != nullptr;
  const bool want_w = grad_qw != nullptr || grad_kw != nullptr || samples;
  if (x == nullptr || dy == nullptr || (dx == nullptr && !want_w) ||
      qk_check_rows("gs_qk_rotary_grad", shape, x, shape->norm != 0) != GS_OK ||
      (dx != nullptr && qk_check_rows("gs_qk_rotary_grad", shape, dx, true) != GS_OK))
    return fail(GS_ERR_INVALID, "gs_qk_rotary_grad: invalid arguments");
  for (int k = 0; k < 2; ++k)
    if ((gw[k] != nullptr && shape->weight[k] == nullptr) || (want_w && shape->norm == 0))
      return fail(GS_ERR_INVALID, "gs_qk_rotary_grad: a weight's gradient without the weight");
  if (samples && a.B > QK_MAX_SAMPLES)
    return fail(GS_ERR_UNSUPPORTED, "gs_qk_rotary_grad: sums of more than 65533 samples");
  if (dx == nullptr) a.heads[2] = 0;   // values have no part in the weights' gradients
  if (a.heads[0] + a.heads[1] + a.heads[2] == 0)
    return fail(GS_ERR_INVALID, "gs_qk_rotary_grad: invalid arguments");
  const bool inter = shape->interleaved != 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const QkPlan p = qk_plan(a, shape->dtype, inter, true, samples);
  QkSums q{};
  if (want_w) {
    Sizer sz;
    QkScratch unused(sz, a, p);
    if (workspace == nullptr || workspace_bytes < sz.used)
      return fail(GS_ERR_WORKSPACE, "gs_qk_rotary_grad: workspace too small");
    Carver cv(workspace, workspace_bytes);
    const QkScratch w(cv, a, p);
    for (int k = 0; k < 2; ++k) {
      if ((gw[k] != nullptr || samples) && a.heads[k] > 0) q.part[k] = a.part[k] = w.part[k];
      q.rows[k] = p.rows[k];
      q.out[k] = samples ? sample_grads + k * a.B * a.D : nullptr;
      q.grad[k] = gw[k];
      q.grad_bf16[k] = shape->weight_dtype[k] == GS_DTYPE_BF16;
    }
  }
  if (int rc = qk_run<true>(a, shape->dtype, inter, p.v, s)) return rc;
  if (!want_w) return GS_OK;
  // every segment is a "train sample" here: the total is the sum over all of them
  q.samples = a.segments;
  q.y0 = samples ? 0 : a.segments + 1;
  q.scale = 1.f;
  q.D = a.D;
  qk_launch_sums(q, a.segments + 2 - q.y0, s);
  return check_launch("qk_sums_kernel");
}

extern "C" size_t gs_qk_sample_dots_workspace(int64_t B, int64_t D) {
  return D > 0 && B > QK_FEW_SAMPLES ? static_cast<size_t>(2 * D) * sizeof(float) + 512 : 0;
}

extern "C" int gs_qk_sample_dots(const float* sample_grads, int64_t B, int64_t D, int64_t n_val,
                                 int64_t val_start, float* out_dot_q, float* out_dot_k,
                                 void* out_grad_q, int grad_q_dtype, void* out_grad_k,
                                 int grad_k_dtype, float grad_scale, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  for (int dt : {grad_q_dtype, grad_k_dtype})
    if (dt != GS_DTYPE_BF16 && dt != GS_DTYPE_F32)
      return fail(GS_ERR_DTYPE, "gs_qk_sample_dots: gradients must be bf16 or fp32");
  if (sample_grads == nullptr || B <= 0 || D <= 0 || !qk_split_ok(B, n_val, val_start))
    return fail(GS_ERR_INVALID, "gs_qk_sample_dots: invalid arguments");
  if (B > QK_MAX_SAMPLES || D > QK_MAX_D)
    return fail(GS_ERR_UNSUPPORTED, "gs_qk_sample_dots: more than 65533 samples or 512 features");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (B <= QK_FEW_SAMPLES) {
    QkFew q{};
    q.n_train = static_cast<int>(B - n_val), q.n_val = static_cast<int>(n_val);
    q.val_start = static_cast<int>(val_start), q.D = static_cast<int>(D), q.scale = grad_scale;
    q.S[0] = sample_grads, q.S[1] = sample_grads + B * D;
    q.dot[0] = out_dot_q, q.dot[1] = out_dot_k;
    q.grad[0] = out_grad_q, q.grad[1] = out_grad_k;
    q.grad_bf16[0] = grad_q_dtype == GS_DTYPE_BF16, q.grad_bf16[1] = grad_k_dtype == GS_DTYPE_BF16;
    hipLaunchKernelGGL(qk_few_dots_kernel, dim3(static_cast<unsigned>(q.n_train + (D + 63) / 64), 2),
                       dim3(64), 0, s, q);
    return check_launch("qk_few_dots_kernel");
  }
  if (workspace == nullptr || workspace_bytes < gs_qk_sample_dots_workspace(B, D))
    return fail(GS_ERR_WORKSPACE, "gs_qk_sample_dots: workspace too small");
  Carver cv(workspace, workspace_bytes);
  const float* S[2] = {sample_grads, sample_grads + B * D};
  float* dot[2] = {out_dot_q, out_dot_k};
  float* val[2];
  void* gw[2] = {out_grad_q, out_grad_k};
  const int dt[2] = {grad_q_dtype, grad_k_dtype};
  QkSums q{};
  for (int k = 0; k < 2; ++k) {
    val[k] = cv.take<float>(D);
    q.part[k] = S[k], q.rows[k] = 1, q.val[k] = val[k];
    q.grad[k] = gw[k], q.grad_bf16[k] = dt[k] == GS_DTYPE_BF16;
  }
  q.samples = B, q.n_val = n_val, q.val_start = val_start, q.y0 = B;
  q.scale = grad_scale;
  q.D = static_cast<int>(D);
  qk_launch_sums(q, 2, s);
  return qk_launch_dots(S, val, dot, B, n_val, val_start, q.D, s);
}

extern "C" size_t gs_qk_rotary_dots_workspace(const gs_qk_shape* shape) {
  return qk_workspace(shape, true);
}

extern "C" int gs_qk_rotary_dots(const gs_qk_shape* shape, const gs_qk_rows x[3],
                                 const gs_qk_rows dy[3], int64_t n_val, int64_t val_start,
                                 float* out_dot_q, float* out_dot_k, void* out_grad_q,
                                 void* out_grad_k, float grad_scale, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  QkArgs a;
  if (int rc = qk_args(a, "gs_qk_rotary_dots", shape, x, dy, nullptr)) return rc;
  void* gw[2] = {out_grad_q, out_grad_k};
  float* dot[2] = {out_dot_q, out_dot_k};
  if (x == nullptr || dy == nullptr || shape->norm == 0 || !qk_split_ok(shape->B, n_val, val_start) ||
      qk_check_rows("gs_qk_rotary_dots", shape, x, true) != GS_OK)
    return fail(GS_ERR_INVALID, "gs_qk_rotary_dots: invalid arguments");
  if (a.B > QK_MAX_SAMPLES)
    return fail(GS_ERR_UNSUPPORTED, "gs_qk_rotary_dots: more than 65533 samples");
  a.heads[2] = 0;
  if (a.heads[0] + a.heads[1] == 0)
    return fail(GS_ERR_INVALID, "gs_qk_rotary_dots: invalid arguments");
  const bool inter = shape->interleaved != 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const QkPlan p = qk_plan(a, shape->dtype, inter, true, true);
  Sizer sz;
  QkScratch unused(sz, a, p);
  if (workspace == nullptr || workspace_bytes < sz.used)
    return fail(GS_ERR_WORKSPACE, "gs_qk_rotary_dots: workspace too small");
  Carver cv(workspace, workspace_bytes);
  const QkScratch w(cv, a, p);
  QkSums q{};
  for (int k = 0; k < 2; ++k) {
    if (a.heads[k] > 0) q.part[k] = a.part[k] = w.part[k];
    q.rows[k] = p.rows[k];
    q.out[k] = w.sums[k];
    q.val[k] = w.val[k];
    q.grad[k] = gw[k];
    q.grad_bf16[k] = shape->weight_dtype[k] == GS_DTYPE_BF16;
  }
  q.samples = a.B, q.n_val = n_val, q.val_start = val_start;
  q.scale = grad_scale;
  q.D = a.D;
  if (int rc = qk_run<true>(a, shape->dtype, inter, p.v, s)) return rc;
  qk_launch_sums(q, a.B + 2, s);
  const float* S[2] = {w.sums[0], w.sums[1]};
  return qk_launch_dots(S, w.val, dot, a.B, n_val, val_start, a.D, s);
}
