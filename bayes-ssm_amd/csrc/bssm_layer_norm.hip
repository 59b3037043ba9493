// Layer norm over rows of D values, forward and backward, gfx950.
//
//   xh = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = xh w + b
//   gu = gy w,  gx = rstd (gu - mean(gu) - xh mean(gu xh)),  gw = sum gy xh,  gb = sum gy
//
// Bound by memory: the forward reads and writes a stream once, the backward
// reads two and writes one.  A row belongs to one wave, to 4 or to 16 waves
// (the fewest that hold it in kVectors vectors a lane), stays in registers
// between the mean, the centred sum of squares and the output, and is read
// once.  Longer rows (see `fits`) are read again from the caches for each of the three.
// The backward's blocks walk rows a grid apart and keep the column sums of
// their rows in registers: the weight's and the bias's gradient leave a block
// as one row of partials and are folded in a fixed order.
#include "bssm_lane.h"
#include "bssm_sequence.h"

namespace bssm {
namespace layer_norm {
namespace {

using lane::Pack;
using lane::kWave;

constexpr int kVectors = 4;       // vectors of a row that a lane holds
constexpr int kMaxBlocks = 1024;  // blocks of the backward: 4 a compute unit

// Sum over the WAVES waves of a row (all of the block when WAVES > 1).
template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float* red) {
  x = lane::lanes_sum(x);
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == 0) red[wave] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) x += red[w];
  }
  return x;
}
template <int WAVES>
__device__ __forceinline__ void row_sums(float& x, float& z, float* red) {
  x = lane::lanes_sum(x);
  z = lane::lanes_sum(z);
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
      red[wave] = x;
      red[WAVES + wave] = z;
    }
    __syncthreads();
    x = z = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      x += red[w];
      z += red[WAVES + w];
    }
  }
}

// Where the rows of a block lie: rows a block, this thread's row and lane.
template <int WAVES>
struct Place {
  static constexpr int kRows = WAVES == 1 ? 4 : 1;  // 4 waves a block at least
  static constexpr int kLanes = WAVES * kWave;
  int row, ln;
  __device__ __forceinline__ Place() {
    row = WAVES == 1 ? threadIdx.x / kWave : 0;
    ln = WAVES == 1 ? threadIdx.x % kWave : threadIdx.x;
  }
};

template <typename T, int N, int WAVES, bool HELD>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void forward_kernel(LayerNormArgs a) {
  __shared__ float red[2 * WAVES];
  const Place<WAVES> at;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * Place<WAVES>::kRows + at.row;
  if (r >= a.r) return;  // whole waves, and whole blocks where a row is a block's
  const T* x = static_cast<const T*>(a.x) + r * a.x_row;
  T* y = static_cast<T*>(a.y) + r * a.d;
  const int64_t step = Place<WAVES>::kLanes * N, c_first = at.ln * N;
  const float inv_d = 1.f / static_cast<float>(a.d);
  Pack<T, N> held[kVectors];
  float sum = 0.f, sq = 0.f;
  if constexpr (HELD) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d) held[v] = lane::load_pack<T, N>(x + c_first + v * step);
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d)
#pragma unroll
        for (int i = 0; i < N; ++i) sum += lane::widen(held[v].v[i]);
  } else {
    for (int64_t c = c_first; c < a.d; c += step) {
      const Pack<T, N> p = lane::load_pack<T, N>(x + c);
#pragma unroll
      for (int i = 0; i < N; ++i) sum += lane::widen(p.v[i]);
    }
  }
  const float mean = row_sum<WAVES>(sum, red) * inv_d;
  auto centred = [&](const Pack<T, N>& p) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float o = lane::widen(p.v[i]) - mean;
      sq = fmaf(o, o, sq);
    }
  };
  if constexpr (HELD) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d) centred(held[v]);
  } else {
    for (int64_t c = c_first; c < a.d; c += step) centred(lane::load_pack<T, N>(x + c));
  }
  const float rstd = rsqrtf(fmaf(row_sum<WAVES>(sq, red), inv_d, a.eps));
  auto write = [&](const Pack<T, N>& p, int64_t c) {
    Pack<T, N> out;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float o = (lane::widen(p.v[i]) - mean) * rstd;
      if (a.weight != nullptr) o *= lane::param(a.weight, c + i, a.param_bf16);
      if (a.bias != nullptr) o += lane::param(a.bias, c + i, a.param_bf16);
      out.v[i] = lane::narrow<T>(o);
    }
    lane::store_pack<T, N>(y + c, out);
  };
  if constexpr (HELD) {
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d) write(held[v], c_first + v * step);
  } else {
    for (int64_t c = c_first; c < a.d; c += step) write(lane::load_pack<T, N>(x + c), c);
  }
  if (at.ln == 0 && a.mean != nullptr) {
    a.mean[r] = mean;
    a.rstd[r] = rstd;
  }
}

// Gradient of the input and, where a.partials is given, the column sums.
template <typename T, int N, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void backward_kernel(LayerNormArgs a) {
  constexpr int kRows = Place<WAVES>::kRows;
  __shared__ float red[2 * WAVES];
  __shared__ float cols[WAVES == 1 ? kRows - 1 : 1][WAVES == 1 ? kWave * N : 1];
  const Place<WAVES> at;
  const int64_t step = Place<WAVES>::kLanes * N, c_first = at.ln * N;
  const float inv_d = 1.f / static_cast<float>(a.d);
  float gw[kVectors][N], gb[kVectors][N];
#pragma unroll
  for (int v = 0; v < kVectors; ++v)
#pragma unroll
    for (int i = 0; i < N; ++i) gw[v][i] = gb[v][i] = 0.f;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + at.row; r < a.r;
       r += static_cast<int64_t>(gridDim.x) * kRows) {
    const T* x = static_cast<const T*>(a.x) + r * a.x_row;
    const T* gy = static_cast<const T*>(a.gy) + r * a.d;
    const float mean = a.mean[r], rstd = a.rstd[r];
    Pack<T, N> px[kVectors], pg[kVectors];
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d) {
        px[v] = lane::load_pack<T, N>(x + c_first + v * step);
        pg[v] = lane::load_pack<T, N>(gy + c_first + v * step);
      }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float xh = (lane::widen(px[v].v[i]) - mean) * rstd, g = lane::widen(pg[v].v[i]);
          const float w = a.weight == nullptr ? 1.f : lane::param(a.weight, c_first + v * step + i, a.param_bf16);
          gw[v][i] = fmaf(g, xh, gw[v][i]);
          gb[v][i] += g;
          s1 = fmaf(g, w, s1);
          s2 = fmaf(g * w, xh, s2);
        }
    if (a.gx == nullptr) continue;
    row_sums<WAVES>(s1, s2, red);
    s1 *= inv_d;
    s2 *= inv_d;
    T* gx = static_cast<T*>(a.gx) + r * a.d;
#pragma unroll
    for (int v = 0; v < kVectors; ++v)
      if (c_first + v * step < a.d) {
        Pack<T, N> out;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float xh = (lane::widen(px[v].v[i]) - mean) * rstd, g = lane::widen(pg[v].v[i]);
          const float w = a.weight == nullptr ? 1.f : lane::param(a.weight, c_first + v * step + i, a.param_bf16);
          out.v[i] = lane::narrow<T>(rstd * (fmaf(g, w, -s1) - xh * s2));
        }
        lane::store_pack<T, N>(gx + c_first + v * step, out);
      }
  }
  if (a.partials == nullptr) return;
  float* part = a.partials + static_cast<int64_t>(blockIdx.x) * 2 * a.d;
#pragma unroll
  for (int v = 0; v < kVectors; ++v)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float s[N];
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = k == 0 ? gw[v][i] : gb[v][i];
      if constexpr (WAVES == 1) {  // the block's 4 rows at a time meet here
        __syncthreads();
        if (at.row > 0)
#pragma unroll
          for (int i = 0; i < N; ++i) cols[at.row - 1][i * kWave + at.ln] = s[i];
        __syncthreads();
        if (at.row == 0)
#pragma unroll
          for (int w = 0; w < kRows - 1; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] += cols[w][i * kWave + at.ln];
      }
      if (at.row == 0 && c_first + v * step < a.d)
#pragma unroll
        for (int i = 0; i < N; ++i) part[k * a.d + c_first + v * step + i] = s[i];
    }
}

// Rows too long to be held: three passes over a row, and the column sums by
// blocks of their own (256 columns x a share of the rows).
template <typename T>
__global__ __launch_bounds__(1024) void backward_long_kernel(LayerNormArgs a) {
  constexpr int WAVES = 16;
  __shared__ float red[2 * WAVES];
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + r * a.x_row;
  const T* gy = static_cast<const T*>(a.gy) + r * a.d;
  T* gx = static_cast<T*>(a.gx) + r * a.d;
  const float mean = a.mean[r], rstd = a.rstd[r], inv_d = 1.f / static_cast<float>(a.d);
  float s1 = 0.f, s2 = 0.f;
  for (int64_t c = threadIdx.x; c < a.d; c += 1024) {
    const float g = lane::widen(gy[c]) * (a.weight == nullptr ? 1.f : lane::param(a.weight, c, a.param_bf16));
    s1 += g;
    s2 = fmaf(g, (lane::widen(x[c]) - mean) * rstd, s2);
  }
  row_sums<WAVES>(s1, s2, red);
  for (int64_t c = threadIdx.x; c < a.d; c += 1024) {
    const float g = lane::widen(gy[c]) * (a.weight == nullptr ? 1.f : lane::param(a.weight, c, a.param_bf16));
    gx[c] = lane::narrow<T>(rstd * (g - s1 * inv_d - (lane::widen(x[c]) - mean) * rstd * (s2 * inv_d)));
  }
}
template <typename T>
__global__ __launch_bounds__(256) void columns_kernel(LayerNormArgs a, int64_t rows) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= a.d) return;
  float gw = 0.f, gb = 0.f;
  const int64_t first = blockIdx.y * rows, last = first + rows < a.r ? first + rows : a.r;
  for (int64_t r = first; r < last; ++r) {
    const float g = lane::widen(static_cast<const T*>(a.gy)[r * a.d + c]);
    gw = fmaf(g, (lane::widen(static_cast<const T*>(a.x)[r * a.x_row + c]) - a.mean[r]) * a.rstd[r], gw);
    gb += g;
  }
  a.partials[(blockIdx.y * 2) * a.d + c] = gw;
  a.partials[(blockIdx.y * 2 + 1) * a.d + c] = gb;
}

__global__ __launch_bounds__(256) void fold_kernel(LayerNormArgs a, int64_t rows) {
  lane::fold_columns(a.partials, rows, 2 * a.d, blockIdx.x, [&](int64_t c, float sum) {
    if (c < a.d) {
      if (a.gweight != nullptr) lane::put_param(a.gweight, c, sum, a.param_bf16);
    } else if (a.gbias != nullptr) {
      lane::put_param(a.gbias, c - a.d, sum, a.param_bf16);
    }
  });
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool vectors(const LayerNormArgs& a) {
  const int n = a.bf16 ? 8 : 4;
  return a.d % n == 0 && a.x_row % n == 0 && aligned(a.x) && aligned(a.y) && aligned(a.gy) && aligned(a.gx);
}
// Waves of a row with N values a vector: 1, 4 or 16; 0 where 16 do not hold it.
int row_waves(int64_t d, int n) {
  const int64_t one = (int64_t)kVectors * kWave * n;
  return d <= one ? 1 : d <= 4 * one ? 4 : d <= 16 * one ? 16 : 0;
}
// Blocks of the backward, from the sizes alone: each adds a row of partials.
int64_t backward_blocks(int64_t r, int64_t d, int bf16) {
  const int waves = row_waves(d, bf16 ? 8 : 4), rows = waves == 1 ? 4 : 1;
  const int64_t most = waves == 16 ? kMaxBlocks / 4 : waves == 0 ? 64 : kMaxBlocks, want = (r + rows - 1) / rows;
  return want < most ? want : most;
}

hipError_t fold(const LayerNormArgs& a, int64_t rows, hipStream_t s) {
  if (a.gweight == nullptr && a.gbias == nullptr) return hipSuccess;
  const int64_t cols = 2 * a.d;
  hipLaunchKernelGGL(fold_kernel, dim3(static_cast<unsigned>((cols + lane::kFoldColumns - 1) / lane::kFoldColumns)),
                     dim3(256), 0, s, a, rows);
  return hipGetLastError();
}

template <typename T, int N>
hipError_t forward(const LayerNormArgs& a, hipStream_t s) {
  const auto grid = [&](int rows) { return dim3(static_cast<unsigned>((a.r + rows - 1) / rows)); };
  switch (row_waves(a.d, N)) {
    case 1: hipLaunchKernelGGL((forward_kernel<T, N, 1, true>), grid(4), dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL((forward_kernel<T, N, 4, true>), grid(1), dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((forward_kernel<T, N, 16, true>), grid(1), dim3(1024), 0, s, a); break;
    default: hipLaunchKernelGGL((forward_kernel<T, N, 16, false>), grid(1), dim3(1024), 0, s, a); break;
  }
  return hipGetLastError();
}
template <typename T, int N>
hipError_t backward(const LayerNormArgs& a, hipStream_t s) {
  int64_t blocks = backward_blocks(a.r, a.d, a.bf16);
  const dim3 grid(static_cast<unsigned>(blocks));
  switch (row_waves(a.d, N)) {
    case 1: hipLaunchKernelGGL((backward_kernel<T, N, 1>), grid, dim3(256), 0, s, a); break;
    case 4: hipLaunchKernelGGL((backward_kernel<T, N, 4>), grid, dim3(256), 0, s, a); break;
    case 16: hipLaunchKernelGGL((backward_kernel<T, N, 16>), grid, dim3(1024), 0, s, a); break;
    default: {
      if (a.gx != nullptr)
        hipLaunchKernelGGL(backward_long_kernel<T>, dim3(static_cast<unsigned>(a.r)), dim3(1024), 0, s, a);
      if (a.partials != nullptr) {
        const int64_t rows = (a.r + blocks - 1) / blocks;
        hipLaunchKernelGGL(columns_kernel<T>, dim3(static_cast<unsigned>((a.d + 255) / 256), grid.x), dim3(256), 0, s,
                           a, rows);
      }
    }
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  return fold(a, blocks, s);
}

}  // namespace
}  // namespace layer_norm

int64_t layer_norm_partial_rows(int64_t r, int64_t d, int bf16) { return layer_norm::backward_blocks(r, d, bf16); }

hipError_t launch_layer_norm_forward(const LayerNormArgs& a, hipStream_t stream) {
  if (a.r == 0) return hipSuccess;
  if (layer_norm::vectors(a))
    return a.bf16 ? layer_norm::forward<__bf16, 8>(a, stream) : layer_norm::forward<float, 4>(a, stream);
  return a.bf16 ? layer_norm::forward<__bf16, 1>(a, stream) : layer_norm::forward<float, 1>(a, stream);
}

hipError_t launch_layer_norm_backward(const LayerNormArgs& a, hipStream_t stream) {
  if (a.r == 0) return layer_norm::fold(a, 0, stream);  // no rows: zero sums
  if (layer_norm::vectors(a))
    return a.bf16 ? layer_norm::backward<__bf16, 8>(a, stream) : layer_norm::backward<float, 4>(a, stream);
  return a.bf16 ? layer_norm::backward<__bf16, 1>(a, stream) : layer_norm::backward<float, 1>(a, stream);
}

}  // namespace bssm
