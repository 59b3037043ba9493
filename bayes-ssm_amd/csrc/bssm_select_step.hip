// One token of a selective state space block from its carried states, gfx950:
// the short filter over the token's channels (values of every head, then B and
// C of every group), its activation, and the recurrence
//   h' = exp(d A) h + d x B^T,   y = h' C + D x,   d = softplus(dt + dt_bias).
//
// Bound by memory: the states, read and written once (float32, 8 N bytes for
// each of the B H P rows), and by latency for a few requests; one launch does
// both operators, so that the filter's output never leaves the chip (and is
// not rounded).  A workgroup owns a strip of a head's P rows: its threads ask
// for the strip's states first, filter the strip's values and the group's B and
// C while those arrive (every strip again: 2 N channels of W taps from the
// caches), and meet in LDS.  LPR lanes share a row of the state.
// Measured with 32 heads of 64 x 128, bfloat16: a batch of 256 123 us (4.4 TB/s
// of the states' 0.54 GB), one request 7 us.
// Every element of the float32 state is read and written by one thread, so
// state_out may be the input; the filter's carried rows are read by many
// workgroups, so theirs may not.
#include "bssm_lane.h"
#include "bssm_sequence.h"

namespace bssm {
namespace select_step {
namespace {

using lane::Pack;
constexpr int kThreads = 256;

// The filter's output for channel c of sequence b; the carried rows move up where `keep`.
template <typename T>
__device__ __forceinline__ float filtered(const SelectStepArgs& a, int64_t b, int64_t c, bool keep) {
  const int64_t channels = a.h * a.p + 2 * a.g * a.n, rows = b * (a.w - 1) * channels + c;
  const T x = static_cast<const T*>(a.row)[b * a.row_batch + c];
  float p = a.conv_bias == nullptr ? 0.f : lane::param(a.conv_bias, c, a.param_bf16);
  for (int j = 0; j < a.w - 1; ++j) {
    const T old = static_cast<const T*>(a.conv_state)[rows + j * channels];
    p = fmaf(lane::param(a.weight, c * a.w + j, a.param_bf16), lane::widen(old), p);
    if (keep && j > 0) static_cast<T*>(a.conv_state_out)[rows + (j - 1) * channels] = old;
  }
  p = fmaf(lane::param(a.weight, c * a.w + a.w - 1, a.param_bf16), lane::widen(x), p);
  if (keep) static_cast<T*>(a.conv_state_out)[rows + (a.w - 2) * channels] = x;
  return a.silu ? p * lane::sigmoid_(p) : p;
}

// V values a lane, LPR lanes a row, K pieces a lane along N, ITER rows a thread.
template <typename T, int V, int LPR, int K, int ITER>
__global__ __launch_bounds__(kThreads) void step_kernel(SelectStepArgs a) {
  constexpr int kRowsAtOnce = kThreads / LPR, kStrip = kRowsAtOnce * ITER;
  __shared__ float xs[kStrip], ks[kSelectMaxState], qs[kSelectMaxState];
  const int64_t strips = (a.p + kStrip - 1) / kStrip;
  int64_t i = blockIdx.x;
  const int64_t p0 = i % strips * kStrip;
  i /= strips;
  const int64_t h = i % a.h, b = i / a.h, grp = h / (a.h / a.g), bh = b * a.h + h;
  const int row = threadIdx.x / LPR, ln = threadIdx.x % LPR;
  Pack<float, V> st[ITER][K];
#pragma unroll
  for (int it = 0; it < ITER; ++it)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t p = p0 + it * kRowsAtOnce + row, n = (k * LPR + ln) * V;
      if (p < a.p && n < a.n) st[it][k] = lane::load_pack<float, V>(a.state + (bh * a.p + p) * a.n + n);
    }
  float v = lane::param(a.dt, b * a.dt_batch + h, a.dt_bf16);
  if (a.dt_bias != nullptr) v += a.dt_bias[h];
  const float d = a.softplus ? lane::softplus_(v) : v, fade = lane::exp_(d * a.rate[h]);
  const float skip = a.skip == nullptr ? 0.f : a.skip[h];
  // The group's B and C are kept by its first head's first strip.
  const bool keep = p0 == 0 && h == grp * (a.h / a.g);
  const int64_t mine = a.p - p0 < kStrip ? a.p - p0 : kStrip;
  for (int64_t c = threadIdx.x; c < mine + 2 * a.n; c += kThreads) {
    if (c < mine) xs[c] = filtered<T>(a, b, h * a.p + p0 + c, true);
    else if (c < mine + a.n) ks[c - mine] = filtered<T>(a, b, a.h * a.p + grp * a.n + c - mine, keep);
    else qs[c - mine - a.n] = filtered<T>(a, b, a.h * a.p + (a.g + grp) * a.n + c - mine - a.n, keep);
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < ITER; ++it) {
    const int local = it * kRowsAtOnce + row;
    const int64_t p = p0 + local;
    const float x = p < a.p ? xs[local] : 0.f, dx = d * x;
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int n = (k * LPR + ln) * V;
      if (p < a.p && n < a.n) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          st[it][k].v[e] = fmaf(fade, st[it][k].v[e], dx * ks[n + e]);
          y = fmaf(st[it][k].v[e], qs[n + e], y);
        }
        lane::store_pack<float, V>(a.state_out + (bh * a.p + p) * a.n + n, st[it][k]);
      }
    }
    y = lane::lanes_sum<LPR>(y);
    if (ln == 0 && p < a.p) static_cast<T*>(a.y)[bh * a.p + p] = lane::narrow<T>(fmaf(skip, x, y));
  }
}

template <typename T, int V, int LPR, int K>
hipError_t launch(const SelectStepArgs& a, hipStream_t stream) {
  // 8 rows a thread keep more loads in flight; with few workgroups, or short
  // heads, 2 rows spread the work over more of the chip.
  constexpr int kLong = kThreads / LPR * 8, kShort = kThreads / LPR * 2;
  const int64_t bh = a.b * a.h, longs = bh * ((a.p + kLong - 1) / kLong), shorts = bh * ((a.p + kShort - 1) / kShort);
  if (a.p >= kLong && longs >= 1024)
    hipLaunchKernelGGL((step_kernel<T, V, LPR, K, 8>), dim3(static_cast<unsigned>(longs)), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((step_kernel<T, V, LPR, K, 2>), dim3(static_cast<unsigned>(shorts)), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}
template <typename T>
hipError_t sizes(const SelectStepArgs& a, hipStream_t stream) {
  const bool vec = a.n % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.state_out)) & 15u) == 0;
  if (!vec) return launch<T, 1, 64, 2>(a, stream);
  if (a.n <= 32) return launch<T, 4, 8, 1>(a, stream);
  if (a.n <= 64) return launch<T, 4, 16, 1>(a, stream);
  return launch<T, 4, 32, 1>(a, stream);
}

}  // namespace
}  // namespace select_step

hipError_t launch_select_step(const SelectStepArgs& a, hipStream_t stream) {
  if (a.b * a.h * a.p == 0) return hipSuccess;
  return a.bf16 ? select_step::sizes<__bf16>(a, stream) : select_step::sizes<float>(a, stream);
}

}  // namespace bssm
