// Selective state space scan, the passes that carry a state along the time
// axis, gfx950.  Per sequence b, head h (P values, N states, group of B and C
// rows h / (H / G)) and token t, with d = softplus(dt + dt_bias):
//   h[t] = exp(d A) h[t-1] + d x[t] B[t]^T,   y[t] = h[t] C[t] + D x[t].
//
// Chunk form.  With s = running sum of d A inside a chunk of 64 tokens and h0
// the state before it, both rewritten as products of tiles,
//   y_i = exp(s_i) h0 C_i + sum_{j <= i} exp(s_i - s_j) (C_i . B_j) d_j x_j + D x_i
//   h0' = exp(s_64) h0 + sum_j exp(s_64 - s_j) d_j x_j B_j^T
// so a token costs about 4 N P + 64 (N + P) multiply-adds on the matrix units
// where the recurrence costs 5 N P vector operations.  Exponents are
// differences inside a chunk, never products of exponentials that leave the
// range.
//
// A workgroup (4 waves) owns one (sequence, head, 64 values of P) and walks
// its chunks with the state in registers: x, B, C are read once and y is
// written once.  Where there are too few of those for the chip the time axis
// is split into segments: a pass without outputs gives each segment's state
// from zero, and the full pass of a segment starts from the earlier ones'.
// A wave's part: 16 tokens of the outputs, 16 values of P of the state.
//
// Rounding with bfloat16 streams: the chunk's weights exp(s_i - s_j) (C.B) d
// and h0 enter y's products as bfloat16 (y is rounded to it anyway, and their
// errors are of that size); the state, which is a float32 result, takes its
// weighted values in three bfloat16 parts, which is all of their bits (two left
// errors of 2e-6 in the state).  Sums are float32.
#include "bssm_select.h"

namespace bssm {
namespace select_scan {
namespace {

constexpr int kChunk = kSelectChunk;
constexpr int kThreads = 256;
constexpr int kTileP = 64;
constexpr int kRecordsB16 = 128, kRecordsF32 = 64;  // tokens between two kept states

__device__ __forceinline__ bool pieces16(const SelectArgs& a) {
  const int n = a.bf16 ? 8 : 4;
  return a.p % n == 0 && a.x_batch % n == 0 && a.x_row % n == 0 && a.x_head % n == 0 &&
         (reinterpret_cast<uintptr_t>(a.x) & 15u) == 0;
}
__device__ __forceinline__ bool pieces16(const void* p, int64_t b, int64_t r, int64_t g, int64_t n, int bf16) {
  const int k = bf16 ? 8 : 4;
  return n % k == 0 && b % k == 0 && r % k == 0 && g % k == 0 && (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// A wave's 16 values of P of a state, transposed: tile i holds n = 16 i + 4 g + r, p = first + l % 16.
template <int NP>
struct State {
  v4f v[NP / 16];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NP / 16; ++i) v[i] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // fn(element of the tile, pointer to 4 of memory, how many of the 4 exist)
  template <typename Fn>
  __device__ __forceinline__ void each(int64_t p, int64_t np, int64_t n, int g, Fn fn) {
    if (p >= np) return;
#pragma unroll
    for (int i = 0; i < NP / 16; ++i) {
      const int64_t c = 16 * i + 4 * g;
      if (c < n) fn(v[i], p * n + c, n - c < 4 ? static_cast<int>(n - c) : 4);
    }
  }
  __device__ __forceinline__ void add(const float* src, float scale, int64_t p, int64_t np, int64_t n, int g) {
#pragma unroll
    for (int i = 0; i < NP / 16; ++i) v[i] *= scale;
    if (src == nullptr) return;
    each(p, np, n, g, [&](v4f& t, int64_t at, int k) {
      if (k == 4 && n % 4 == 0) {
        t += *reinterpret_cast<const v4f*>(src + at);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < k) t[r] += src[at + r];
      }
    });
  }
  __device__ __forceinline__ void store(float* dst, int64_t p, int64_t np, int64_t n, int g) {
    each(p, np, n, g, [&](v4f& t, int64_t at, int k) {
      if (k == 4 && n % 4 == 0) {
        *reinterpret_cast<v4f*>(dst + at) = t;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < k) dst[at + r] = t[r];
      }
    });
  }
};

// Wave 0: step d and running sums of d A (base 2) of a chunk's tokens, and the weight that a token has in the state
// that the chunk leaves (BACK: in the adjoint before it).  Tokens from `live` on have d = 0.
template <bool BACK>
__device__ __forceinline__ void chunk_steps(const SelectArgs& a, int64_t b, int64_t t0, int64_t h, int64_t live,
                                            float rate2, float* step, Sums<kChunk>& sums, float* weight, float* fade) {
  const int ln = threadIdx.x;
  float slope, d = 0.f;
  if (ln < live) d = time_step(a, b, t0 + ln, h, slope);
  const float log2_fade[1] = {d * rate2};
  sums.fill<1>(log2_fade);
  if (step != nullptr) step[ln] = d;
  const double own = sums.at(ln), all = __shfl(own, kChunk - 1, kWave);
  weight[ln] = BACK ? lane::exp2_(static_cast<float>(own)) : d * lane::exp2_(static_cast<float>(all - own));
  if (ln == 0) *fade = static_cast<float>(all);
}

// state = fade * state + sum_j k_j (w_j u_j)^T over the chunk's tokens j.
template <typename T, int NP>
__device__ __forceinline__ void advance(State<NP>& st, const T* us, const T* ks, const float* weight, float fade,
                                        int p_first, int ln) {
  const int g = ln / 16;
#pragma unroll
  for (int i = 0; i < NP / 16; ++i) st.v[i] *= fade;
#pragma unroll
  for (int kk = 0; kk < kChunk / 32; ++kk) {
    const Operand<T> u = across<true>(us + kk * 32 * pitch<T>(kTileP) + p_first, pitch<T>(kTileP), ln);
    Computed<T, 3> wu;
#pragma unroll
    for (int e = 0; e < 8; ++e) wu.set(e, u.get(e) * weight[kk * 32 + (e < 4 ? 4 * g + e : 12 + 4 * g + e)]);
#pragma unroll
    for (int i = 0; i < NP / 16; ++i)
      mma(st.v[i], across<true>(ks + kk * 32 * pitch<T>(NP) + 16 * i, pitch<T>(NP), ln), wu);
  }
}

struct Block {
  int64_t b, h, p0, seg, first, last;  // chunks [first, last)
  __device__ __forceinline__ Block(const SelectArgs& a, int64_t segs) {
    // Sequences vary fastest, then segments: workgroups of one B and C meet on one XCD's L2.
    int64_t i = blockIdx.x;
    b = i % a.b;
    i /= a.b;
    seg = i % segs;
    i /= segs;
    h = i % a.h;
    p0 = i / a.h * kTileP;
    const int64_t chunks = (a.t + kChunk - 1) / kChunk;
    // Whole records a segment.
    const int64_t per = ((chunks + segs - 1) / segs + 1) / 2 * 2;
    first = seg * per < chunks ? seg * per : chunks;
    last = first + per < chunks ? first + per : chunks;
  }
};

// The workspace of the segments: [segs, B, H, P, N] states, then [segs, B, H] decays.
__device__ __forceinline__ float* segment_state(const SelectArgs& a, int64_t seg, int64_t b, int64_t h) {
  return a.segments + ((seg * a.b + b) * a.h + h) * a.p * a.n;
}
__device__ __forceinline__ float* segment_fade(const SelectArgs& a, int64_t segs, int64_t seg, int64_t b, int64_t h) {
  return a.segments + segs * a.b * a.h * a.p * a.n + (seg * a.b + b) * a.h + h;
}

template <typename T, int NP>
__global__ __launch_bounds__(kThreads) void forward_kernel(SelectArgs a, int64_t segs) {
  __shared__ __align__(16) T xs[kChunk * pitch<T>(kTileP)], ks[kChunk * pitch<T>(NP)], qs[kChunk * pitch<T>(NP)],
      hs[kTileP * pitch<T>(NP)];
  __shared__ __align__(16) float step[kChunk], left[kChunk];
  __shared__ Sums<kChunk> sums;
  __shared__ float log2_fade;
  const Block at(a, segs);
  const int wave = threadIdx.x / kWave, ln = threadIdx.x % kWave, g = ln / 16, own = wave * 16 + ln % 16;
  const int64_t grp = at.h / (a.h / a.g), n_live = row_length(a, at.b), bh = at.b * a.h + at.h;
  const T* x = static_cast<const T*>(a.x) + at.b * a.x_batch + at.h * a.x_head;
  const T* bk = static_cast<const T*>(a.bk) + at.b * a.bk_batch + grp * a.bk_group;
  const T* cq = static_cast<const T*>(a.cq) + at.b * a.cq_batch + grp * a.cq_group;
  const bool vx = pieces16(a), vb = pieces16(a.bk, a.bk_batch, a.bk_row, a.bk_group, a.n, a.bf16),
             vc = pieces16(a.cq, a.cq_batch, a.cq_row, a.cq_group, a.n, a.bf16);
  const float rate2 = a.rate[at.h] * lane::kLog2e, skip = a.skip == nullptr ? 0.f : a.skip[at.h];
  const int64_t p = at.p0 + own, pn = a.p * a.n;
  const int64_t record = sizeof(T) == 2 ? kRecordsB16 : kRecordsF32, ratio = record / kChunk,
                records = (a.t + record - 1) / record;
  State<NP> st;
  st.clear();
  st.add(a.state0 == nullptr ? nullptr : a.state0 + bh * pn, 1.f, p, a.p, a.n, g);
  for (int64_t s = 0; s < at.seg; ++s)
    st.add(segment_state(a, s, at.b, at.h), *segment_fade(a, segs, s, at.b, at.h), p, a.p, a.n, g);
  for (int64_t c = at.first; c < at.last; ++c) {
    const int64_t t0 = c * kChunk, live = n_live - t0;
    if (a.states != nullptr && c % ratio == 0)
      st.store(a.states + (bh * records + c / ratio) * pn, p, a.p, a.n, g);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP / 16; ++i) {
      Pack<T, 4> o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o.v[r] = lane::narrow<T>(st.v[i][r]);
      lane::store_pack<T, 4>(hs + own * pitch<T>(NP) + 16 * i + 4 * g, o);
    }
    stage<kChunk, kTileP, kThreads>(xs, x + t0 * a.x_row, a.x_row, live, at.p0, a.p, vx);
    stage<kChunk, NP, kThreads>(ks, bk + t0 * a.bk_row, a.bk_row, live, 0, a.n, vb);
    stage<kChunk, NP, kThreads>(qs, cq + t0 * a.cq_row, a.cq_row, live, 0, a.n, vc);
    if (wave == 0) chunk_steps<false>(a, at.b, t0, at.h, live, rate2, step, sums, left, &log2_fade);
    __syncthreads();
    // Outputs of the wave's 16 tokens, transposed: rows p, column own.
    Operand<T> q[NP / 32];
#pragma unroll
    for (int k = 0; k < NP / 32; ++k) q[k] = along(qs + own * pitch<T>(NP) + 32 * k, g);
    const float s_own = sums.near[own], since = lane::exp2_(static_cast<float>(sums.at(own)));
    v4f y[kTileP / 16];
#pragma unroll
    for (int i = 0; i < kTileP / 16; ++i) {
      y[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NP / 32; ++k) mma(y[i], along(hs + (16 * i + ln % 16) * pitch<T>(NP) + 32 * k, g), q[k]);
      y[i] *= since;
    }
    for (int kk = 0; kk <= wave / 2; ++kk) {
      Computed<T, 1> m;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int j0 = kk * 32 + half * 16;
        v4f dot = {0.f, 0.f, 0.f, 0.f};
        if (j0 <= wave * 16)
#pragma unroll
          for (int k = 0; k < NP / 32; ++k) mma(dot, along(ks + (j0 + ln % 16) * pitch<T>(NP) + 32 * k, g), q[k]);
        const float from = s_own + sums.between(wave, j0 / 16);
        const v4f sj = *reinterpret_cast<const v4f*>(sums.near + j0 + 4 * g), dj = *reinterpret_cast<const v4f*>(step + j0 + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          m.set(half * 4 + r, j0 + 4 * g + r <= own ? dot[r] * lane::exp2_(from - sj[r]) * dj[r] : 0.f);
      }
#pragma unroll
      for (int i = 0; i < kTileP / 16; ++i)
        mma(y[i], across<true>(xs + kk * 32 * pitch<T>(kTileP) + 16 * i, pitch<T>(kTileP), ln), m);
    }
    const int64_t t = t0 + own;
    if (t < a.t) {
      T* out = static_cast<T*>(a.y) + ((at.b * a.t + t) * a.h + at.h) * a.p + at.p0;
#pragma unroll
      for (int i = 0; i < kTileP / 16; ++i) {
        const int c0 = 16 * i + 4 * g;
        const Pack<T, 4> xi = lane::load_pack<T, 4>(xs + own * pitch<T>(kTileP) + c0);
        Pack<T, 4> o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o.v[r] = lane::narrow<T>(own < live ? fmaf(skip, lane::widen(xi.v[r]), y[i][r]) : 0.f);
        if (at.p0 + c0 + 4 <= a.p && a.p % 4 == 0) {
          lane::store_pack<T, 4>(out + c0, o);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (at.p0 + c0 + r < a.p) out[c0 + r] = o.v[r];
        }
      }
    }
    advance<T, NP>(st, xs, ks, left, lane::exp2_(log2_fade), wave * 16, ln);
  }
  if (at.seg == segs - 1 && a.state_out != nullptr) st.store(a.state_out + bh * pn, p, a.p, a.n, g);
}

// The state alone, along a segment.  Forward (BACK false): from zero, into the
// workspace.  BACK: the adjoint of the state, chunks in reverse,
//   gh0 = exp(s_64) gh0' + sum_i exp(s_i) C_i gy_i^T;
// LOCAL: from zero, into the workspace; else from the later segments', keeping
// the adjoint behind every record's last token and the one before the first.
template <typename T, int NP, bool BACK, bool LOCAL>
__global__ __launch_bounds__(kThreads) void carry_kernel(SelectArgs a, int64_t segs) {
  __shared__ __align__(16) T us[kChunk * pitch<T>(kTileP)], ks[kChunk * pitch<T>(NP)];
  __shared__ __align__(16) float weight[kChunk];
  __shared__ Sums<kChunk> sums;
  __shared__ float log2_fade;
  const Block at(a, segs);
  const int wave = threadIdx.x / kWave, ln = threadIdx.x % kWave, g = ln / 16, own = wave * 16 + ln % 16;
  const int64_t grp = at.h / (a.h / a.g), n_live = row_length(a, at.b), bh = at.b * a.h + at.h;
  const T* u = BACK ? static_cast<const T*>(a.gy) + (at.b * a.t * a.h + at.h) * a.p
                    : static_cast<const T*>(a.x) + at.b * a.x_batch + at.h * a.x_head;
  const int64_t u_row = BACK ? a.h * a.p : a.x_row;
  const T* k = BACK ? static_cast<const T*>(a.cq) + at.b * a.cq_batch + grp * a.cq_group
                    : static_cast<const T*>(a.bk) + at.b * a.bk_batch + grp * a.bk_group;
  const int64_t k_row = BACK ? a.cq_row : a.bk_row;
  const bool vu = BACK ? pieces16(a.gy, a.p, a.p, a.p, a.p, a.bf16) : pieces16(a);
  const bool vk = BACK ? pieces16(a.cq, a.cq_batch, a.cq_row, a.cq_group, a.n, a.bf16)
                       : pieces16(a.bk, a.bk_batch, a.bk_row, a.bk_group, a.n, a.bf16);
  const float rate2 = a.rate[at.h] * lane::kLog2e;
  const int64_t p = at.p0 + own, pn = a.p * a.n;
  const int64_t record = sizeof(T) == 2 ? kRecordsB16 : kRecordsF32, ratio = record / kChunk,
                records = (a.t + record - 1) / record, chunks = (a.t + kChunk - 1) / kChunk;
  State<NP> st;
  st.clear();
  float total = 0.f;
  if constexpr (!LOCAL) {
    st.add(a.gstate_out == nullptr ? nullptr : a.gstate_out + bh * pn, 1.f, p, a.p, a.n, g);
    for (int64_t s = segs - 1; s > at.seg; --s)
      st.add(segment_state(a, s, at.b, at.h), *segment_fade(a, segs, s, at.b, at.h), p, a.p, a.n, g);
  }
  for (int64_t i = 0; i < at.last - at.first; ++i) {
    const int64_t c = BACK ? at.last - 1 - i : at.first + i, t0 = c * kChunk, live = n_live - t0;
    if (!LOCAL && (c % ratio == ratio - 1 || c == chunks - 1))
      st.store(a.adjoints + (bh * records + c / ratio) * pn, p, a.p, a.n, g);
    if (live <= 0) continue;  // uniform: the workgroup has one sequence
    __syncthreads();
    stage<kChunk, kTileP, kThreads>(us, u + t0 * u_row, u_row, live, at.p0, a.p, vu);
    stage<kChunk, NP, kThreads>(ks, k + t0 * k_row, k_row, live, 0, a.n, vk);
    if (wave == 0) chunk_steps<BACK>(a, at.b, t0, at.h, live, rate2, nullptr, sums, weight, &log2_fade);
    __syncthreads();
    total += log2_fade;
    advance<T, NP>(st, us, ks, weight, lane::exp2_(log2_fade), wave * 16, ln);
  }
  if constexpr (LOCAL) {
    st.store(segment_state(a, at.seg, at.b, at.h), p, a.p, a.n, g);
    if (threadIdx.x == 0 && at.p0 == 0) *segment_fade(a, segs, at.seg, at.b, at.h) = lane::exp2_(total);
  } else if (at.seg == 0 && a.gstate0 != nullptr) {
    st.store(a.gstate0 + bh * pn, p, a.p, a.n, g);
  }
}

unsigned blocks(const SelectArgs& a, int64_t segs) {
  return static_cast<unsigned>(a.b * a.h * ((a.p + kTileP - 1) / kTileP) * segs);
}

template <typename T, int NP>
hipError_t forward(const SelectArgs& a, hipStream_t stream) {
  const int64_t segs = select_segments(a);
  if (segs > 1) hipLaunchKernelGGL((carry_kernel<T, NP, false, true>), dim3(blocks(a, segs)), dim3(kThreads), 0, stream, a, segs);
  hipLaunchKernelGGL((forward_kernel<T, NP>), dim3(blocks(a, segs)), dim3(kThreads), 0, stream, a, segs);
  return hipGetLastError();
}
template <typename T, int NP>
hipError_t reverse(const SelectArgs& a, hipStream_t stream) {
  const int64_t segs = select_segments(a);
  if (segs > 1) hipLaunchKernelGGL((carry_kernel<T, NP, true, true>), dim3(blocks(a, segs)), dim3(kThreads), 0, stream, a, segs);
  hipLaunchKernelGGL((carry_kernel<T, NP, true, false>), dim3(blocks(a, segs)), dim3(kThreads), 0, stream, a, segs);
  return hipGetLastError();
}

template <typename T>
hipError_t sizes(const SelectArgs& a, bool back, hipStream_t stream) {
  if (a.n <= 32) return back ? reverse<T, 32>(a, stream) : forward<T, 32>(a, stream);
  if (a.n <= 64) return back ? reverse<T, 64>(a, stream) : forward<T, 64>(a, stream);
  return back ? reverse<T, 128>(a, stream) : forward<T, 128>(a, stream);
}

}  // namespace

// The reverse pass of the state (called by the backward, bssm_select_bwd.hip).
hipError_t launch_adjoints(const SelectArgs& a, hipStream_t stream) {
  return a.bf16 ? sizes<__bf16>(a, true, stream) : sizes<float>(a, true, stream);
}

}  // namespace select_scan

int64_t select_record(int bf16) { return bf16 ? select_scan::kRecordsB16 : select_scan::kRecordsF32; }

// One segment where the sequences, heads and P tiles alone give every compute
// unit a workgroup; else two a unit, each of 8 chunks or more: a segment costs
// the pass that gives its state from zero.
int64_t select_segments(const SelectArgs& a) {
  const int64_t have = a.b * a.h * ((a.p + select_scan::kTileP - 1) / select_scan::kTileP);
  if (have >= 256 || have == 0) return 1;
  const int64_t chunks = (a.t + kSelectChunk - 1) / kSelectChunk, want = (512 + have - 1) / have, most = chunks / 8;
  return want < most ? want : most > 1 ? most : 1;
}
int64_t select_segment_floats(const SelectArgs& a) {
  const int64_t segs = select_segments(a);
  return segs == 1 ? 0 : segs * a.b * a.h * (a.p * a.n + 1);
}

hipError_t launch_select_forward(const SelectArgs& a, hipStream_t stream) {
  if (a.b * a.h * a.p == 0) return hipSuccess;
  return a.bf16 ? select_scan::sizes<__bf16>(a, false, stream) : select_scan::sizes<float>(a, false, stream);
}

}  // namespace bssm
