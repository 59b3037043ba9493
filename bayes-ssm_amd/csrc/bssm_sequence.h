// Arguments and launchers of the operators around a selective state space
// block: the short causal filter, the scan, its single-token step, layer norm
// and the distillation loss.  Host code only; sizes are checked by the C
// entry points (bssm_capi.hip).
#ifndef BSSM_SEQUENCE_H_
#define BSSM_SEQUENCE_H_

#include <hip/hip_runtime.h>

#include <cstdint>

namespace bssm {

// ---- short causal filter (bssm_short_conv.hip)
struct ShortConvArgs {
  const void* x;
  int64_t x_batch, x_row;        // strides in elements
  const void *weight, *bias;     // [C, W], [C] or null
  const void* state;             // [B, W - 1, C] or null (zeros)
  const int64_t* lengths;        // [B] or null
  void *y, *final_state;         // [B, T, C], [B, W - 1, C]
  const void *gy, *gfinal;       // upstream gradients, either may be null
  void *gx, *gstate;             // gstate may be null
  float* partials;               // [short_conv_partial_rows, W + 1, C]
  void *gweight, *gbias;         // sums of the partials; may be null
  int64_t b, t, c;
  int w, bf16, param_bf16, silu;
};
int64_t short_conv_partial_rows(int64_t b, int64_t t, int64_t c);
hipError_t launch_short_conv_forward(const ShortConvArgs& a, hipStream_t stream);
hipError_t launch_short_conv_backward(const ShortConvArgs& a, hipStream_t stream);

// ---- layer norm (bssm_layer_norm.hip)
struct LayerNormArgs {
  const void* x;
  int64_t x_row;                 // row stride in elements
  const void *weight, *bias;     // [D] or null
  void* y;                       // [R, D]
  float *mean, *rstd;            // [R]; null in a forward that keeps nothing
  const void* gy;                // [R, D]
  void* gx;                      // [R, D] or null
  float* partials;               // [layer_norm_partial_rows, 2, D]
  void *gweight, *gbias;         // may be null
  int64_t r, d;
  float eps;
  int bf16, param_bf16;
};
int64_t layer_norm_partial_rows(int64_t r, int64_t d, int bf16);
hipError_t launch_layer_norm_forward(const LayerNormArgs& a, hipStream_t stream);
hipError_t launch_layer_norm_backward(const LayerNormArgs& a, hipStream_t stream);

// ---- distillation loss (bssm_distill.hip)
constexpr int kDistillMaxTeacher = 1024;
struct DistillArgs {
  const void* logits;
  int64_t logits_row;            // row stride in elements
  const void* teacher;           // [R, K]
  const int64_t* index;          // [R, K]
  float *loss, *stats;           // [R], [R, 3]: maximum, sum of exponentials, 1 if the row has a teacher
  float* counts;                 // workspace of distill_count_floats, where the forward divides its gradient by the rows
  float* mean;                   // [3] or null: mean, 1 / rows with a teacher, sum
  const float* upstream;         // [R] or (upstream_scalar) [1]
  void* grad;                    // [R, V]; null in a forward without gradient
  int64_t r, v, k;
  float tau;
  int bf16, teacher_bf16, upstream_scalar, mean_of_rows, ready;
};
int64_t distill_count_floats();
hipError_t launch_distill_forward(const DistillArgs& a, hipStream_t stream);
hipError_t launch_distill_backward(const DistillArgs& a, hipStream_t stream);

// ---- selective scan (bssm_select_fwd.hip, bssm_select_bwd.hip) and its
// single-token step (bssm_select_step.hip)
constexpr int kSelectMaxState = 128;   // N
constexpr int kSelectChunk = 64;       // tokens of a chunk of the forward
struct SelectArgs {
  // Strides in elements; the innermost axis of each stream is contiguous.
  const void* x;                       // [B, T, H, P]
  int64_t x_batch, x_row, x_head;
  const void* dt;                      // [B, T, H]
  int64_t dt_batch, dt_row;
  const void *bk, *cq;                 // B and C, [B, T, G, N]
  int64_t bk_batch, bk_row, bk_group, cq_batch, cq_row, cq_group;
  const float *rate, *skip, *dt_bias;  // A, D, dt_bias [H]; D and dt_bias may be null
  const float* state0;                 // [B, H, P, N] or null
  const int64_t* lengths;              // [B] or null
  void* y;                             // [B, T, H, P]
  float* state_out;                    // [B, H, P, N] or null
  float* states;                       // [B, H, records, P, N]: state before every record'th token, or null
  float* segments;                     // workspace, see select_segments
  float* steps;                        // the tokens' steps and their sums: written by the forward, read by the backward
  int64_t b, t, h, p, n, g;
  int bf16, dt_bf16, softplus;
  // Backward.
  const void* gy;                      // [B, T, H, P] contiguous
  const float* gstate_out;             // [B, H, P, N] or null
  float* adjoints;                     // [B, H, records, P, N]: adjoint of the state behind a record's tokens
  float* gstate0;                      // [B, H, P, N] or null
  void *gx, *gdt;                      // contiguous
  void *gbk, *gcq;                     // [B, T, G, N] contiguous
  float* gparts;                       // [parts, 2, B, T, G, N]: gradients of B and C by parts of a group's heads
  float* token_sums;                   // workspace of select_token_floats
  float* rows;                         // [B * records, 3, H]: gradients of A, D, dt_bias by records
  float *grate, *gskip, *gdt_bias;     // [H]
};
// Tokens between two kept states; parts that a group's heads are split into by
// the backward; segments that the time axis is split into by the passes that
// carry a state (1: no workspace), and the workspace's floats.
bool select_fast(const SelectArgs& a);
int64_t select_record(int bf16);
int64_t select_parts(const SelectArgs& a);
int64_t select_segments(const SelectArgs& a);
int64_t select_segment_floats(const SelectArgs& a);
int64_t select_step_floats(const SelectArgs& a);
int64_t select_token_floats(const SelectArgs& a);
hipError_t launch_select_forward(const SelectArgs& a, hipStream_t stream);
hipError_t launch_select_backward(const SelectArgs& a, hipStream_t stream);

struct SelectStepArgs {
  const void* row;                     // [B, H * P + 2 G N], the filter's new inputs
  int64_t row_batch;
  const void* dt;                      // [B, H]
  int64_t dt_batch;
  const void* conv_state;              // [B, W - 1, C]
  const float* state;                  // [B, H, P, N]
  const void *weight, *conv_bias;      // [C, W], [C] or null
  const float *rate, *skip, *dt_bias;
  void* y;                             // [B, H, P]
  void* conv_state_out;                // not the input's memory
  float* state_out;                    // may be the input's memory
  int64_t b, h, p, n, g;
  int w, bf16, dt_bf16, param_bf16, silu, softplus;
};
hipError_t launch_select_step(const SelectStepArgs& a, hipStream_t stream);

}  // namespace bssm

#endif  // BSSM_SEQUENCE_H_
