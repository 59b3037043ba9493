// Distillation loss from a teacher's top logits, forward and backward, gfx950.
//
// A row has V student logits x and K listed teacher entries (index i_k, logit
// l_k).  An entry counts if its index lies in [0, V) and its logit is above
// -infinity.  With p = softmax(l / tau) over the entries that count and
// q = softmax(x / tau) over the vocabulary,
//   loss = tau^2 sum_k p_k (log p_k - log q[i_k]),   grad_v = tau (q_v - sum over k with i_k = v of p_k) upstream;
// a row without entries has loss 0 and gradient 0, whatever its logits hold.
// Exponents are taken of (x - max) / tau: a row of the type's lowest value
// stays finite for tau < 1, and a vocabulary entry at -infinity has q = 0.
//
// Bound by memory: the forward reads the logits once (a running maximum and a
// sum that is rescaled when the maximum moves), the backward reads them again
// and writes the gradient.
#include "bssm_lane.h"
#include "bssm_sequence.h"

namespace bssm {
namespace distill {
namespace {

using lane::Pack;
using lane::kWave;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / kWave;

__device__ __forceinline__ float block_sum(float x, float* red) {
  x = lane::lanes_sum(x);
  __syncthreads();
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
  __syncthreads();
  x = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) x += red[w];
  return x;
}
__device__ __forceinline__ float block_max(float x, float* red) {
  x = lane::lanes_max(x);
  __syncthreads();
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
  __syncthreads();
  x = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) x = fmaxf(x, red[w]);
  return x;
}

struct Teacher {
  int64_t at[kDistillMaxTeacher];  // vocabulary index, -1: does not count
  float p[kDistillMaxTeacher];
};

// The row's teacher distribution into LDS; log p_k = (l_k - max) / tau - log sum.
__device__ __forceinline__ bool teacher_row(const DistillArgs& a, int64_t r, Teacher& t, float* red, float& top,
                                            float& sum) {
  const float c = lane::kLog2e / a.tau;
  float m = -INFINITY;
  bool any = false;
  for (int64_t k = threadIdx.x; k < a.k; k += kThreads) {
    const float l = lane::param(a.teacher, r * a.k + k, a.teacher_bf16);
    const int64_t i = a.index[r * a.k + k];
    const bool there = i >= 0 && i < a.v && !(l == -INFINITY);
    t.at[k] = there ? i : -1;
    t.p[k] = l;
    if (there) m = fmaxf(m, l);
    any |= there;
  }
  top = block_max(m, red);
  any = block_max(any ? 1.f : 0.f, red) > 0.f;
  if (top == -INFINITY) top = 0.f;  // every entry that counts is NaN
  float s = 0.f;
  for (int64_t k = threadIdx.x; k < a.k; k += kThreads) {
    const float e = t.at[k] >= 0 ? lane::exp2_((t.p[k] - top) * c) : 0.f;
    t.p[k] = e;
    s += e;
  }
  sum = block_sum(s, red);
  return any;
}

template <typename T>
__device__ __forceinline__ float logit(const DistillArgs& a, int64_t r, int64_t v) {
  return lane::widen(static_cast<const T*>(a.logits)[r * a.logits_row + v]);
}

// lse[r] = (maximum, sum of exponentials, 1 if the row has a teacher).
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void forward_kernel(DistillArgs a) {
  __shared__ Teacher t;
  __shared__ float red[kWaves];
  const int64_t r = blockIdx.x;
  const float c = lane::kLog2e / a.tau;
  const T* x = static_cast<const T*>(a.logits) + r * a.logits_row;
  float m = -INFINITY, s = 0.f;
  for (int64_t v = threadIdx.x * N; v < a.v; v += kThreads * N) {
    const Pack<T, N> p = lane::load_pack<T, N>(x + v);
    float best = m;
#pragma unroll
    for (int i = 0; i < N; ++i) best = fmaxf(best, lane::widen(p.v[i]));
    if (best > m) {
      s = m == -INFINITY ? s : s * lane::exp2_((m - best) * c);
      m = best;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) s += lane::exp2_((lane::widen(p.v[i]) - base) * c);
  }
  float top = block_max(m, red);
  if (top == -INFINITY) top = 0.f;
  const float total = block_sum(m == -INFINITY ? s : s * lane::exp2_((m - top) * c), red);
  float t_top, t_sum;
  const bool any = teacher_row(a, r, t, red, t_top, t_sum);
  float loss = 0.f;
  const float log_t = logf(t_sum), log_s = logf(total), inv_tau = 1.f / a.tau, inv_t = 1.f / t_sum;
  for (int64_t k = threadIdx.x; k < a.k; k += kThreads) {
    if (t.at[k] < 0) continue;
    const float p = t.p[k] * inv_t;
    if (p == 0.f) continue;
    const float l = lane::param(a.teacher, r * a.k + k, a.teacher_bf16);
    const float log_p = (l - t_top) * inv_tau - log_t;
    const float log_q = (logit<T>(a, r, t.at[k]) - top) * inv_tau - log_s;
    loss = fmaf(p, log_p - log_q, loss);
  }
  loss = block_sum(loss, red);
  if (threadIdx.x == 0) {
    a.loss[r] = any ? a.tau * a.tau * loss : 0.f;
    a.lse[3 * r] = top;
    a.lse[3 * r + 1] = total;
    a.lse[3 * r + 2] = any ? 1.f : 0.f;
  }
}

// mean[] = (sum / rows with a teacher, 1 / rows, sum), in a fixed order.
__global__ __launch_bounds__(kThreads) void mean_kernel(DistillArgs a) {
  __shared__ float red[kWaves];
  float s = 0.f, n = 0.f;
  for (int64_t r = threadIdx.x; r < a.r; r += kThreads) {
    s += a.loss[r];
    n += a.lse[3 * r + 2];
  }
  s = block_sum(s, red);
  n = fmaxf(block_sum(n, red), 1.f);
  if (threadIdx.x == 0) {
    a.mean[0] = s / n;
    a.mean[1] = 1.f / n;
    a.mean[2] = s;
  }
}

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void backward_kernel(DistillArgs a) {
  __shared__ Teacher t;
  __shared__ float red[kWaves];
  const int64_t r = blockIdx.x;
  const float c = lane::kLog2e / a.tau;
  const T* x = static_cast<const T*>(a.logits) + r * a.logits_row;
  T* g = static_cast<T*>(a.grad) + r * a.v;
  const float top = a.lse[3 * r], inv_s = 1.f / a.lse[3 * r + 1];
  const bool any = a.lse[3 * r + 2] > 0.f;
  const float u = a.tau * a.upstream[a.upstream_scalar ? 0 : r] * (a.mean == nullptr ? 1.f : a.mean[1]);
  float t_top, t_sum;
  teacher_row(a, r, t, red, t_top, t_sum);
  for (int64_t v = threadIdx.x * N; v < a.v; v += kThreads * N) {
    Pack<T, N> p;
    if (any) {
      p = lane::load_pack<T, N>(x + v);
#pragma unroll
      for (int i = 0; i < N; ++i)
        p.v[i] = lane::narrow<T>(u * (lane::exp2_((lane::widen(p.v[i]) - top) * c) * inv_s));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p.v[i] = lane::narrow<T>(0.f);
    }
    lane::store_pack<T, N>(g + v, p);
  }
  if (!any) return;
  // The listed entries once more, from float32: an index that is listed twice
  // is written by its first place, with the sum of its p.
  __syncthreads();
  const float inv_t = 1.f / t_sum;
  for (int64_t k = threadIdx.x; k < a.k; k += kThreads) {
    const int64_t at = t.at[k];
    if (at < 0) continue;
    float p = 0.f;
    bool first = true;
    for (int64_t j = 0; j < a.k; ++j) {
      if (t.at[j] != at) continue;
      if (j < k) first = false;
      p += t.p[j];
    }
    if (first) g[at] = lane::narrow<T>(u * (lane::exp2_((logit<T>(a, r, at) - top) * c) * inv_s - p * inv_t));
  }
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool vectors(const DistillArgs& a) {
  const int n = a.bf16 ? 8 : 4;
  return a.v % n == 0 && a.logits_row % n == 0 && aligned(a.logits) && aligned(a.grad);
}

template <typename T, int N>
hipError_t launch(const DistillArgs& a, bool back, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.r)), block(kThreads);
  if (back) hipLaunchKernelGGL((backward_kernel<T, N>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((forward_kernel<T, N>), grid, block, 0, stream, a);
  return hipGetLastError();
}
hipError_t types(const DistillArgs& a, bool back, hipStream_t stream) {
  if (a.r == 0) return hipSuccess;
  if (vectors(a)) return a.bf16 ? launch<__bf16, 8>(a, back, stream) : launch<float, 4>(a, back, stream);
  return a.bf16 ? launch<__bf16, 1>(a, back, stream) : launch<float, 1>(a, back, stream);
}

}  // namespace
}  // namespace distill

hipError_t launch_distill_forward(const DistillArgs& a, hipStream_t stream) {
  if (hipError_t e = distill::types(a, false, stream); e != hipSuccess) return e;
  if (a.mean == nullptr) return hipSuccess;
  hipLaunchKernelGGL(distill::mean_kernel, dim3(1), dim3(distill::kThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_distill_backward(const DistillArgs& a, hipStream_t stream) {
  return distill::types(a, true, stream);
}

}  // namespace bssm
