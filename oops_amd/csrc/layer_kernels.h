// Layer operators: launchers behind the oops_rms_norm_*, oops_quantize_int8,
// oops_int8_linear and oops_linear_attn_* C entry points.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/oops_amd.h"

namespace oops {

// ---- error reporting of the C entry points (capi.cpp): the code is returned, the text kept for oops_last_error
int report(int code, const char* fmt, long long a = 0, long long b = 0);
void clear_report();
int report_launch(hipError_t err, const char* what);
int report_workspace(const void* workspace, size_t given, size_t need);

// ---- rms_norm.hip
hipError_t launch_rms_norm_forward(const oops_rms_norm_geometry& g, const void* x, const void* residual,
                                   const void* weight, void* y, void* sum, float* rstd, hipStream_t stream);
hipError_t launch_rms_norm_int8(const oops_rms_norm_geometry& g, const void* x, const void* residual,
                                const void* weight, void* values, float* scales, void* sum, hipStream_t stream);
hipError_t launch_quantize_int8(const oops_rms_norm_geometry& g, const void* x, void* values, float* scales,
                                hipStream_t stream);
int64_t rms_norm_parts(const oops_rms_norm_geometry& g);  // rows of weight-gradient partials
hipError_t launch_rms_norm_backward(const oops_rms_norm_geometry& g, const void* h, const float* rstd,
                                    const void* weight, const void* grad_y, const void* grad_sum, void* grad_x,
                                    float* weight_parts, hipStream_t stream);
// the partials' sum, of the weight's type
hipError_t launch_rms_weight_sum(const oops_rms_norm_geometry& g, const float* parts, void* out, hipStream_t stream);

// ---- int8_linear.hip
size_t int8_linear_workspace_bytes(const oops_int8_geometry& g);
hipError_t launch_int8_linear(const oops_int8_geometry& g, const void* x, const float* x_scale, const void* w,
                              const float* w_scale, const void* bias, void* out, void* workspace, hipStream_t stream);

// ---- linear_attn.hip: one decayed causal walk over tokens, from which the output and every gradient are made.
// For positions p = 0 .. n-1 of a (batch, head) (token p, or n - 1 - p from the end):
//   S_p = l S_(p-1) + b_p^T c_p,   out_p = scale a_p S_p
// with S_(-1) = initial; from the end S_0 = initial + ..., and the last state decays once more.
struct LinearWalk {
  const void *a, *b, *c;  // a, b: `rows` wide, c and out: `cols` wide
  void* out;
  int64_t a_stride[3], b_stride[3], c_stride[3], out_stride[3];  // batch, head, token
  const float* log_decay;
  const void* lengths;
  const float* initial;  // state before the walk, or NULL
  float* final_state;    // state behind the walk, or NULL
  int64_t batch, length;
  int32_t heads, rows, cols, lengths_i64;
  int32_t from_end;       // walk from the last token to the first
  int32_t state_by_cols;  // initial and final_state are [cols][rows]
  float scale;            // of out; of the update in walks from the end (their initial state is not scaled)
};
// A long walk of few heads runs in segments: launch_linear_walk_starts writes the states they start from to the
// workspace (0 bytes: one segment), where launch_linear_walk reads them.  They depend on b, c and the decays alone
// and are laid out like `initial`, so walks over the same state from the same end share them.
size_t linear_walk_workspace_bytes(int dtype, const LinearWalk& w);
hipError_t launch_linear_walk_starts(int dtype, const LinearWalk& w, void* workspace, hipStream_t stream);
hipError_t launch_linear_walk(int dtype, const LinearWalk& w, const void* workspace, hipStream_t stream);
hipError_t launch_linear_attn_step(const oops_linear_attn_geometry& g, const void* q, const void* k, const void* v,
                                   const float* log_decay, float* state, void* out, hipStream_t stream);

}  // namespace oops
