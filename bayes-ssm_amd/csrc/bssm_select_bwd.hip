// Selective state space scan, gradients, gfx950.  See bssm_select_fwd.hip for
// the scan and its chunk form.  The chunks here are the records: L = 128
// tokens (64 for float32, whose tiles take twice the LDS).  With h the state
// before a record (kept by the forward), gh the adjoint of the state behind it
// (from the reverse pass of the state, launch_adjoints), E_ij = exp(s_i - s_j)
// for i >= j, S = C B^T and G = gy x^T over the record's tokens:
//   gu_j = sum_i E_ij S_ij gy_i + exp(s_L - s_j) gh B_j          (u = d x)
//   gC_i = sum_j E_ij G_ij d_j B_j + exp(s_i) h^T gy_i
//   gB_j = d_j (sum_i E_ij G_ij C_i + exp(s_L - s_j) gh^T x_j)
//   gx_j = d_j gu_j + D gy_j,   gD = sum gy . x
// A decay's logarithm a = d A moves every later term of the sums s:
//   ga_j = sum_{k >= j} (row_k - d_k col_k + C_k . gC'_k) + sum_{k < j} B_k . gB'_k + exp(s_L) <gh, h>
// with row_i = sum_{j < i} W_ij d_j and col_j = sum_{i > j} W_ij of W = E S G
// (the diagonal would cancel), and gC', gB' the parts that come from h and gh.
// That sum is closed inside the record, so it does not gather the rounding of
// a long sequence.  Then
//   gd_j = W_jj + col_j + B_j . gB'_j / d_j + A ga_j,   gA = sum d ga,   gdt = gd slope.
//
// A workgroup owns a record of one sequence and a part of one group's heads:
// it goes through the heads (and through P 64 values at a time, which are
// heads of their own as far as the sums are concerned) with the gradients of B
// and C in registers, so that those leave once a part instead of once a head.
// A wave owns 16 tokens: as j for gu and gB, as i for gC; E, S and G are
// formed in the layout of a product's result, twice, once for either side, so
// that each is the next product's operand as it is.
//
// Rounding with bfloat16 streams: S and G are exact products of the streams in
// float32.  What feeds the float32 results (ga, gd and their sums) is float32
// or has h and gh in three bfloat16 parts; what feeds only bfloat16 results
// (E S and E G d in gu, gB, gC; gh in gu) is one.
#include "bssm_select.h"

namespace bssm {
namespace select_scan {

hipError_t launch_adjoints(const SelectArgs& a, hipStream_t stream);  // bssm_select_fwd.hip

namespace {

constexpr int kTileP = 64;
constexpr int kHalf = 32;  // rows of h and gh in LDS at a time

__device__ __forceinline__ bool pieces16(const void* p, int64_t b, int64_t r, int64_t g, int64_t n, int bf16) {
  const int k = bf16 ? 8 : 4;
  return n % k == 0 && b % k == 0 && r % k == 0 && g % k == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// 4 values of a [P, N] record; zeros outside.
__device__ __forceinline__ v4f record_piece(const float* src, int64_t p, int64_t c, int64_t np, int64_t n) {
  v4f o = {0.f, 0.f, 0.f, 0.f};
  if (p >= np || c >= n) return o;
  if (n % 4 == 0) return *reinterpret_cast<const v4f*>(src + p * n + c);
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (c + r < n) o[r] = src[p * n + c + r];
  return o;
}

template <typename T>
struct Sizes {
  static constexpr int kL = sizeof(T) == 2 ? 128 : 64;      // tokens of a record
  static constexpr int kThreads = kL * 4;                   // a wave for 16 tokens
  static constexpr int kPlanes = sizeof(T) == 2 ? 3 : 1;    // parts of h and gh
  static constexpr int kPerLane = kL / kWave;               // tokens a lane of wave 0
};

template <typename T, int NP>
__global__ __launch_bounds__(Sizes<T>::kThreads) void backward_kernel(SelectArgs a, int64_t parts) {
  using Z = Sizes<T>;
  constexpr int L = Z::kL, kThreads = Z::kThreads, kWaves = kThreads / kWave, kPl = pitch<T>(kTileP), nPl = pitch<T>(NP);
  constexpr int kPieces = (kHalf * NP / 4 + kThreads - 1) / kThreads;
  __shared__ __align__(16) T xs[L * kPl], gs[L * kPl], ks[L * nPl], qs[L * nPl], hs[Z::kPlanes][kHalf * nPl], ghs[Z::kPlanes][kHalf * nPl];
  __shared__ __align__(16) float step[L], tok_f[L], tok_b[L], tok_d[L], red[kWaves][2];
  __shared__ Sums<L> sums;
  const int wave = threadIdx.x / kWave, ln = threadIdx.x % kWave, g = ln / 16, own = wave * 16 + ln % 16;
  // Sequences vary fastest, so that a part's neighbours on an XCD share B, C.
  int64_t i = blockIdx.x;
  const int64_t b = i % a.b;
  i /= a.b;
  const int64_t part = i % parts;
  i /= parts;
  const int64_t grp = i % a.g, rec = i / a.g, records = (a.t + L - 1) / L;
  const int64_t per_group = a.h / a.g, h_first = grp * per_group + part * per_group / parts,
                h_last = grp * per_group + (part + 1) * per_group / parts;
  const int64_t t0 = rec * L, live = row_length(a, b) - t0, pn = a.p * a.n;
  {
    const bool vb = pieces16(a.bk, a.bk_batch, a.bk_row, a.bk_group, a.n, a.bf16),
               vc = pieces16(a.cq, a.cq_batch, a.cq_row, a.cq_group, a.n, a.bf16);
    stage<L, NP, kThreads>(ks, static_cast<const T*>(a.bk) + b * a.bk_batch + grp * a.bk_group + t0 * a.bk_row,
                           a.bk_row, live, 0, a.n, vb);
    stage<L, NP, kThreads>(qs, static_cast<const T*>(a.cq) + b * a.cq_batch + grp * a.cq_group + t0 * a.cq_row,
                           a.cq_row, live, 0, a.n, vc);
  }
  const bool vx = pieces16(a.x, a.x_batch, a.x_row, a.x_head, a.p, a.bf16), vg = pieces16(a.gy, a.p, a.p, a.p, a.p, a.bf16);
  v4f gk[NP / 16], gq[NP / 16];  // gradients of B and C, transposed: rows n, column own
#pragma unroll
  for (int n = 0; n < NP / 16; ++n) gk[n] = gq[n] = v4f{0.f, 0.f, 0.f, 0.f};

  for (int64_t h = h_first; h < h_last; ++h) {
    const float rate = a.rate[h], rate2 = rate * lane::kLog2e, skip = a.skip == nullptr ? 0.f : a.skip[h];
    float row = 0.f, col = 0.f, diagonal = 0.f, from_h = 0.f, from_gh = 0.f, dot_h = 0.f, dot_x = 0.f;
    float d_lane[Z::kPerLane], slope[Z::kPerLane];  // wave 0
    for (int64_t p0 = 0; p0 < a.p; p0 += kTileP) {
      __syncthreads();
      stage<L, kTileP, kThreads>(xs, static_cast<const T*>(a.x) + b * a.x_batch + t0 * a.x_row + h * a.x_head, a.x_row,
                                 live, p0, a.p, vx);
      stage<L, kTileP, kThreads>(gs, static_cast<const T*>(a.gy) + ((b * a.t + t0) * a.h + h) * a.p, a.h * a.p, live,
                                 p0, a.p, vg);
      const float* h_rec = a.states + ((b * a.h + h) * records + rec) * pn;
      const float* gh_rec = a.adjoints + ((b * a.h + h) * records + rec) * pn;
      auto stage_half = [&](int64_t from) {
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int at = (k * kThreads + threadIdx.x) * 4, p = at / NP, c = at % NP;
          if (p >= kHalf) break;
          v4f hv = record_piece(h_rec, from + p, c, a.p, a.n), gv = record_piece(gh_rec, from + p, c, a.p, a.n);
#pragma unroll
          for (int r = 0; r < 4; ++r) dot_h = fmaf(hv[r], gv[r], dot_h);
#pragma unroll
          for (int s = 0; s < Z::kPlanes; ++s) {
            Pack<T, 4> o, go;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              o.v[r] = lane::narrow<T>(hv[r]);
              go.v[r] = lane::narrow<T>(gv[r]);
              hv[r] -= lane::widen(o.v[r]);
              gv[r] -= lane::widen(go.v[r]);
            }
            lane::store_pack<T, 4>(hs[s] + p * nPl + c, o);
            lane::store_pack<T, 4>(ghs[s] + p * nPl + c, go);
          }
        }
      };
      stage_half(p0);
      if (wave == 0 && p0 == 0) {
        float log2_fade[Z::kPerLane];
#pragma unroll
        for (int e = 0; e < Z::kPerLane; ++e) {  // lane: tokens kPerLane * ln + e
          const int64_t t = Z::kPerLane * ln + e;
          d_lane[e] = slope[e] = 0.f;
          if (t < live) d_lane[e] = time_step(a, b, t0 + t, h, slope[e]);
          step[t] = d_lane[e];
          log2_fade[e] = d_lane[e] * rate2;
        }
        sums.template fill<Z::kPerLane>(log2_fade);
      }
      __syncthreads();
      const float s_own = sums.near[own], d_own = step[own];
      Operand<T> x_own[2], g_own[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        x_own[k] = along(xs + own * kPl + 32 * k, g);
        g_own[k] = along(gs + own * kPl + 32 * k, g);
      }
      v4f gu[kTileP / 16];  // rows p, column own
#pragma unroll
      for (int k = 0; k < kTileP / 16; ++k) gu[k] = v4f{0.f, 0.f, 0.f, 0.f};
      {  // own = j: rows i
        Operand<T> k_own[NP / 32];
#pragma unroll
        for (int k = 0; k < NP / 32; ++k) k_own[k] = along(ks + own * nPl + 32 * k, g);
        for (int kk = wave / 2; kk < L / 32; ++kk) {
          Computed<T, 1> es, eg;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int i0 = kk * 32 + half * 16;
            v4f s = {0.f, 0.f, 0.f, 0.f}, gx = {0.f, 0.f, 0.f, 0.f};
            if (i0 >= wave * 16) {
#pragma unroll
              for (int k = 0; k < NP / 32; ++k) mma(s, along(qs + (i0 + ln % 16) * nPl + 32 * k, g), k_own[k]);
#pragma unroll
              for (int k = 0; k < 2; ++k) mma(gx, along(gs + (i0 + ln % 16) * kPl + 32 * k, g), x_own[k]);
            }
            const float to = sums.between(i0 / 16, wave) - s_own;
            const v4f si = *reinterpret_cast<const v4f*>(sums.near + i0 + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = i0 + 4 * g + r;
              const float e = at >= own ? lane::exp2_(si[r] + to) : 0.f;
              const float esr = e * s[r];
              es.set(half * 4 + r, esr);
              eg.set(half * 4 + r, e * gx[r] * d_own);
              if (at == own) {
                diagonal = fmaf(esr, gx[r], diagonal);
                dot_x += gx[r];
              } else {
                col = fmaf(esr, gx[r], col);
              }
            }
          }
#pragma unroll
          for (int k = 0; k < kTileP / 16; ++k) mma(gu[k], across<true>(gs + kk * 32 * kPl + 16 * k, kPl, ln), es);
#pragma unroll
          for (int n = 0; n < NP / 16; ++n) mma(gk[n], across<true>(qs + kk * 32 * nPl + 16 * n, nPl, ln), eg);
        }
      }
      {  // own = i: rows j
        Operand<T> q_own[NP / 32];
#pragma unroll
        for (int k = 0; k < NP / 32; ++k) q_own[k] = along(qs + own * nPl + 32 * k, g);
        for (int kk = 0; kk <= wave / 2; ++kk) {
          Computed<T, 1> eg;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int j0 = kk * 32 + half * 16;
            v4f s = {0.f, 0.f, 0.f, 0.f}, gx = {0.f, 0.f, 0.f, 0.f};
            if (j0 <= wave * 16) {
#pragma unroll
              for (int k = 0; k < NP / 32; ++k) mma(s, along(ks + (j0 + ln % 16) * nPl + 32 * k, g), q_own[k]);
#pragma unroll
              for (int k = 0; k < 2; ++k) mma(gx, along(xs + (j0 + ln % 16) * kPl + 32 * k, g), g_own[k]);
            }
            const float from = s_own + sums.between(wave, j0 / 16);
            const v4f sj = *reinterpret_cast<const v4f*>(sums.near + j0 + 4 * g), dj = *reinterpret_cast<const v4f*>(step + j0 + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = j0 + 4 * g + r;
              const float e = at <= own ? lane::exp2_(from - sj[r]) * dj[r] * gx[r] : 0.f;
              eg.set(half * 4 + r, e);
              if (at != own) row = fmaf(e, s[r], row);
            }
          }
#pragma unroll
          for (int n = 0; n < NP / 16; ++n) mma(gq[n], across<true>(ks + kk * 32 * nPl + 16 * n, nPl, ln), eg);
        }
      }
      // From the state before the record, gC: exp(s_i) h^T gy_i; from the adjoint behind it, gu and gB.
      const float before = lane::exp2_(static_cast<float>(sums.at(own))),
                  behind = lane::exp2_(static_cast<float>(sums.at(L - 1) - sums.at(own)));
#pragma unroll
      for (int half = 0; half < kTileP / kHalf; ++half) {
        if (half > 0) {
          if (p0 + half * kHalf >= a.p) break;  // uniform
          __syncthreads();
          stage_half(p0 + half * kHalf);
          __syncthreads();
        }
#pragma unroll
        for (int m = 0; m < kHalf / 16; ++m) {
          v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < NP / 32; ++k)
            mma(o, along(ghs[0] + (16 * m + ln % 16) * nPl + 32 * k, g), along(ks + own * nPl + 32 * k, g));
          gu[half * (kHalf / 16) + m] += o * behind;
        }
#pragma unroll
        for (int n = 0; n < NP / 16; ++n) {
          v4f o = {0.f, 0.f, 0.f, 0.f}, go = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < Z::kPlanes; ++s) {
            mma(o, across<false>(hs[s] + 16 * n, nPl, ln), g_own[half]);
            mma(go, across<false>(ghs[s] + 16 * n, nPl, ln), x_own[half]);
          }
          const Pack<T, 4> q = lane::load_pack<T, 4>(qs + own * nPl + 16 * n + 4 * g),
                           kb = lane::load_pack<T, 4>(ks + own * nPl + 16 * n + 4 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            o[r] *= before;
            go[r] *= behind;
            from_h = fmaf(o[r], lane::widen(q.v[r]), from_h);
            from_gh = fmaf(go[r], lane::widen(kb.v[r]), from_gh);
          }
          gq[n] += o;
          gk[n] += go * d_own;
        }
      }
      if (t0 + own < a.t) {
        T* out = static_cast<T*>(a.gx) + ((b * a.t + t0 + own) * a.h + h) * a.p + p0;
#pragma unroll
        for (int k = 0; k < kTileP / 16; ++k) {
          const int c0 = 16 * k + 4 * g;
          const Pack<T, 4> gi = lane::load_pack<T, 4>(gs + own * kPl + c0);
          Pack<T, 4> o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o.v[r] = lane::narrow<T>(fmaf(d_own, gu[k][r], skip * lane::widen(gi.v[r])));
          if (p0 + c0 + 4 <= a.p && a.p % 4 == 0) {
            lane::store_pack<T, 4>(out + c0, o);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (p0 + c0 + r < a.p) out[c0 + r] = o.v[r];
          }
        }
      }
    }
    // The head's token sums: lanes g = 0..3 of a column hold parts of them.
    auto over_groups = [](float v) {
      v += __shfl_xor(v, 16, kWave);
      return v + __shfl_xor(v, 32, kWave);
    };
    row = over_groups(row);
    col = over_groups(col);
    diagonal = over_groups(diagonal);
    from_h = over_groups(from_h);
    from_gh = over_groups(from_gh);
    const float d_own = step[own];
    if (g == 0) {
      tok_f[own] = row - d_own * col + from_h;
      tok_b[own] = d_own * from_gh;
      tok_d[own] = diagonal + col + from_gh;
    }
    dot_h = lane::lanes_sum(dot_h);
    dot_x = lane::lanes_sum(dot_x);
    if (ln == 0) {
      red[wave][0] = dot_h;
      red[wave][1] = dot_x;
    }
    __syncthreads();
    if (wave == 0) {
      float whole = 0.f, skip_sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        whole += red[w][0];
        skip_sum += red[w][1];
      }
      whole *= lane::exp2_(static_cast<float>(sums.at(L - 1)));
      float f = 0.f, bsum = 0.f;
#pragma unroll
      for (int e = 0; e < Z::kPerLane; ++e) {
        f += tok_f[Z::kPerLane * ln + e];
        bsum += tok_b[Z::kPerLane * ln + e];
      }
      // f of this lane's tokens and later, b of earlier ones
      const float f_up = lanes_prefix(f);
      float later = __shfl(f_up, kWave - 1, kWave) - f_up + f, earlier = lanes_prefix(bsum) - bsum;
      float g_rate = 0.f, g_bias = 0.f;
#pragma unroll
      for (int e = 0; e < Z::kPerLane; ++e) {
        const int t = Z::kPerLane * ln + e;
        const float ga = later + earlier + whole;
        later -= tok_f[t];
        earlier += tok_b[t];
        const float gd = fmaf(rate, ga, tok_d[t]) * slope[e];
        g_rate = fmaf(d_lane[e], ga, g_rate);
        g_bias += gd;
        if (t0 + t < a.t) lane::put_param(a.gdt, (b * a.t + t0 + t) * a.h + h, t < live ? gd : 0.f, a.dt_bf16);
      }
      g_rate = lane::lanes_sum(g_rate);
      g_bias = lane::lanes_sum(g_bias);
      if (ln == 0) {
        float* out = a.rows + (rec * a.b + b) * 3 * a.h + h;
        out[0] = g_rate;
        out[a.h] = skip_sum;
        out[2 * a.h] = g_bias;
      }
    }
  }
  if (t0 + own >= a.t) return;
  const int64_t at = ((b * a.t + t0 + own) * a.g + grp) * a.n, all = a.b * a.t * a.g * a.n;
#pragma unroll
  for (int n = 0; n < NP / 16; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t c = 16 * n + 4 * g + r;
      if (c >= a.n) continue;
      if (parts == 1) {
        static_cast<T*>(a.gbk)[at + c] = lane::narrow<T>(gk[n][r]);
        static_cast<T*>(a.gcq)[at + c] = lane::narrow<T>(gq[n][r]);
      } else {
        a.gparts[(2 * part) * all + at + c] = gk[n][r];
        a.gparts[(2 * part + 1) * all + at + c] = gq[n][r];
      }
    }
}

// Gradients of B and C: their sums over the parts of a group's heads.
template <typename T>
__global__ __launch_bounds__(256) void parts_kernel(SelectArgs a, int64_t parts) {
  const int64_t all = a.b * a.t * a.g * a.n, i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= 2 * all) return;
  float s = 0.f;
  for (int64_t k = 0; k < parts; ++k) s += a.gparts[2 * k * all + i];
  T* out = static_cast<T*>(i < all ? a.gbk : a.gcq);
  out[i < all ? i : i - all] = lane::narrow<T>(s);
}

__global__ __launch_bounds__(256) void heads_kernel(SelectArgs a, int64_t rows) {
  lane::fold_columns(a.rows, rows, 3 * a.h, blockIdx.x, [&](int64_t c, float s) {
    float* out = c < a.h ? a.grate : c < 2 * a.h ? a.gskip : a.gdt_bias;
    if (out != nullptr) out[c % a.h] = s;
  });
}

template <typename T>
hipError_t sizes(const SelectArgs& a, hipStream_t stream) {
  constexpr int L = Sizes<T>::kL;
  const int64_t records = (a.t + L - 1) / L, parts = select_parts(a);
  const dim3 grid(static_cast<unsigned>(a.b * a.g * records * parts)), block(Sizes<T>::kThreads);
  if (records > 0 && a.b > 0) {
    if (hipError_t e = launch_adjoints(a, stream); e != hipSuccess) return e;
    if (a.n <= 32) hipLaunchKernelGGL((backward_kernel<T, 32>), grid, block, 0, stream, a, parts);
    else if (a.n <= 64) hipLaunchKernelGGL((backward_kernel<T, 64>), grid, block, 0, stream, a, parts);
    else hipLaunchKernelGGL((backward_kernel<T, 128>), grid, block, 0, stream, a, parts);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (parts > 1) {
      const int64_t all = 2 * a.b * a.t * a.g * a.n;
      hipLaunchKernelGGL(parts_kernel<T>, dim3(static_cast<unsigned>((all + 255) / 256)), dim3(256), 0, stream, a, parts);
    }
  }
  hipLaunchKernelGGL(heads_kernel, dim3(static_cast<unsigned>((3 * a.h + lane::kFoldColumns - 1) / lane::kFoldColumns)),
                     dim3(256), 0, stream, a, a.b * records);
  return hipGetLastError();
}

}  // namespace
}  // namespace select_scan

// Two workgroups a compute unit where a group has the heads for it.
int64_t select_parts(const SelectArgs& a) {
  const int64_t record = select_record(a.bf16), have = a.b * a.g * ((a.t + record - 1) / record);
  if (have == 0) return 1;
  const int64_t want = (512 + have - 1) / have, most = a.h / a.g;
  return want < most ? want : most;
}

hipError_t launch_select_backward(const SelectArgs& a, hipStream_t stream) {
  if (a.h == 0) return hipSuccess;
  return a.bf16 ? select_scan::sizes<__bf16>(a, stream) : select_scan::sizes<float>(a, stream);
}

}  // namespace bssm
