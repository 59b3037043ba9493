// Shared parts of the selective scan's kernels (bssm_select_fwd.hip,
// bssm_select_bwd.hip): 16 x 16 tile products with 32 values of the summed
// index, on bfloat16 or float32 operands, and the tiles' ways into LDS.
//
// Operand layout.  A lane l of a wave holds row (column) l % 16 of an operand
// and 8 values of the summed index k, group g = l / 16.  Two orders of k are
// used, each for both operands of a product:
//   plain:  element e is k = 8 g + e;
//   folded: element e is k = 4 g + e for e < 4, else 16 + 4 g + e - 4.
// A product's result has row 4 g + r (r = 0..3), column l % 16 in lane l, so
// that two results below each other are an operand in the folded order, with
// their rows as k, without any move between lanes.
// bfloat16: one v_mfma_f32_16x16x32_bf16; float32: 8 v_mfma_f32_16x16x4_f32.
#ifndef BSSM_SELECT_H_
#define BSSM_SELECT_H_

#include "bssm_lane.h"
#include "bssm_sequence.h"

namespace bssm {
namespace select_scan {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v4b __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

using lane::kWave;
using lane::Pack;

template <typename T>
struct Operand;
template <>
struct Operand<__bf16> {
  v8b v;
  __device__ __forceinline__ float get(int e) const { return static_cast<float>(v[e]); }
  __device__ __forceinline__ void set(int e, float x) { v[e] = static_cast<__bf16>(x); }
};
template <>
struct Operand<float> {
  float v[8];
  __device__ __forceinline__ float get(int e) const { return v[e]; }
  __device__ __forceinline__ void set(int e, float x) { v[e] = x; }
};

__device__ __forceinline__ void mma(v4f& acc, const Operand<__bf16>& a, const Operand<__bf16>& b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(v4f& acc, const Operand<float>& a, const Operand<float>& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], acc, 0, 0, 0);
}

// A computed float32 operand: in float32 itself; in bfloat16 as the nearest
// value (16 of the 24 bits are lost with PLANES = 1), or as a sum of three,
// each the nearest to what the ones before leave (PLANES = 3, all 24 bits),
// which is what feeds float32 results.
template <typename T, int PLANES>
struct Computed {
  static constexpr int kPlanes = sizeof(T) == 4 ? 1 : PLANES;
  Operand<T> part[kPlanes];
  __device__ __forceinline__ void set(int e, float x) {
#pragma unroll
    for (int i = 0; i < kPlanes; ++i) {
      part[i].set(e, x);
      x -= part[i].get(e);
    }
  }
};
template <typename T, int PLANES>
__device__ __forceinline__ void mma(v4f& acc, const Operand<T>& a, const Computed<T, PLANES>& b) {
#pragma unroll
  for (int i = 0; i < Computed<T, PLANES>::kPlanes; ++i) mma(acc, a, b.part[i]);
}

// Tiles in LDS: rows of W values, PITCH apart; 16 bytes more than W, so that
// 16 rows at one column lie in different banks.
template <typename T>
constexpr int pitch(int w) {
  return w + 16 / static_cast<int>(sizeof(T));
}

// The operand whose row is an LDS row and whose k is a column, plain order:
// p points at (row of lane l % 16, column k0).
template <typename T>
__device__ __forceinline__ Operand<T> along(const T* p, int g) {
  Operand<T> o;
  if constexpr (sizeof(T) == 2) {
    o.v = *reinterpret_cast<const v8b*>(p + g * 8);
  } else {
    const v4f a = *reinterpret_cast<const v4f*>(p + g * 8), b = *reinterpret_cast<const v4f*>(p + g * 8 + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o.v[e] = a[e];
      o.v[e + 4] = b[e];
    }
  }
  return o;
}

// The operand whose row is an LDS column and whose k is an LDS row: tile
// points at (row k0, first column) and has the pitch ld.  bfloat16 takes the
// transposing LDS read: 16 lanes give 4 rows of 16 columns by 8 bytes each
// and get a column's 4 rows.
template <bool FOLDED, typename T>
__device__ __forceinline__ Operand<T> across(const T* tile, int ld, int ln) {
  const int g = ln / 16;
  const int r0 = FOLDED ? 4 * g : 8 * g, r1 = FOLDED ? 16 + 4 * g : 8 * g + 4;
  Operand<T> o;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) v4s* Lds;
    const T* p = tile + (ln % 16) / 4 * ld + (ln % 4) * 4;
    const v4b a = __builtin_bit_cast(v4b, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + r0 * ld)));
    const v4b b = __builtin_bit_cast(v4b, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + r1 * ld)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o.v[e] = a[e];
      o.v[e + 4] = b[e];
    }
  } else {
    const T* p = tile + ln % 16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o.v[e] = p[(r0 + e) * ld];
      o.v[e + 4] = p[(r1 + e) * ld];
    }
  }
  return o;
}

// 8 values of a global row from column c on; zeros from column n on.
template <typename T>
__device__ __forceinline__ Pack<T, 8> row_piece(const T* row, int64_t c, int64_t n, bool vec) {
  Pack<T, 8> p;
  if (vec && c + 8 <= n) {
    const auto* q = reinterpret_cast<const v4f*>(row + c);
    auto* o = reinterpret_cast<v4f*>(&p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) o[i] = q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p.v[i] = c + i < n ? row[c + i] : static_cast<T>(0.f);
  }
  return p;
}
template <typename T>
__device__ __forceinline__ void put_piece(T* lds, const Pack<T, 8>& p) {
  const auto* q = reinterpret_cast<const v4f*>(&p);
  auto* o = reinterpret_cast<v4f*>(lds);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) o[i] = q[i];
}

// ROWS rows of a stream (stride st), columns [c0, c0 + W) of n, into LDS; rows from `rows` on and columns from n on are 0.
template <int ROWS, int W, int THREADS, typename T>
__device__ __forceinline__ void stage(T* lds, const T* src, int64_t st, int64_t rows, int64_t c0, int64_t n, bool vec) {
  constexpr int kPieces = W / 8;
  static_assert(ROWS * kPieces % THREADS == 0 || ROWS * kPieces < THREADS, "whole pieces a thread");
#pragma unroll
  for (int i = threadIdx.x; i < ROWS * kPieces; i += THREADS) {
    const int r = i / kPieces, c = i % kPieces * 8;
    Pack<T, 8> p{};
    if (r < rows) p = row_piece(src + r * st, c0 + c, n, vec);
    put_piece(lds + r * pitch<T>(W) + c, p);
  }
}

__device__ __forceinline__ int64_t row_length(const SelectArgs& a, int64_t b) {
  if (a.lengths == nullptr) return a.t;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n > a.t ? a.t : n;
}

// The time step of token t: (step, derivative of the step by dt).
__device__ __forceinline__ float time_step(const SelectArgs& a, int64_t b, int64_t t, int64_t h, float& slope) {
  const int64_t at = b * a.dt_batch + t * a.dt_row + h;
  float v = lane::param(a.dt, at, a.dt_bf16);
  if (a.dt_bias != nullptr) v += a.dt_bias[h];
  slope = 1.f;
  if (!a.softplus) return v;
  slope = lane::softplus_slope_(v);
  return lane::softplus_(v);
}

// Inclusive sum over the wave's lanes.
template <typename V>
__device__ __forceinline__ V lanes_prefix(V x) {
  const int ln = threadIdx.x % kWave;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const V up = __shfl_up(x, o, kWave);
    if (ln >= o) x += up;
  }
  return x;
}

// The running sums s of d A (to base 2) of L tokens, kept so that differences
// of near tokens are exact to float32: a sum of -100 has steps of 8e-6, which
// would be the relative error of every decay in a fast head.  near[t] is the
// sum from t's 16 tokens' start, base[i] (float64) the sum before those.
template <int L>
struct Sums {
  alignas(16) float near[L];
  double base[L / 16];
  // s_i - s_j for tokens of the 16-token blocks bi and bj is
  // (near[i] + between(bi, bj)) - near[j].
  __device__ __forceinline__ float between(int bi, int bj) const { return static_cast<float>(base[bi] - base[bj]); }
  __device__ __forceinline__ double at(int t) const { return base[t / 16] + near[t]; }
  // By one wave: a lane gives the steps' logarithms of PER tokens from PER * lane on.
  template <int PER>
  __device__ __forceinline__ void fill(const float (&log2_fade)[PER]) {
    const int ln = threadIdx.x % kWave;
    double own = 0.;
#pragma unroll
    for (int e = 0; e < PER; ++e) own += log2_fade[e];
    double s = lanes_prefix(own) - own;
    const int first = PER * ln / 16 * 16 / PER;  // the lane that the 16 tokens start in
    const double start = __shfl(s, first, kWave);
    if (PER * ln % 16 == 0) base[PER * ln / 16] = s;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      s += log2_fade[e];
      near[PER * ln + e] = static_cast<float>(s - start);
    }
  }
};

}  // namespace select_scan
}  // namespace bssm

#endif  // BSSM_SELECT_H_
