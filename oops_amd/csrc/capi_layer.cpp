// C entry points of the layer operators (root-mean-square norm, 8-bit linear
// layers, linear attention): host checks, then the launchers.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "layer_kernels.h"

namespace {

using oops::report;
using oops::report_launch;

bool known_dtype(int dtype) { return dtype == OOPS_F32 || dtype == OOPS_BF16 || dtype == OOPS_F16; }
size_t align256(size_t b) { return (b + 255) / 256 * 256; }
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1;

// ---- rms_norm
int check_rms(const oops_rms_norm_geometry* g, bool residual) {
  if (!g) return report(OOPS_EINVAL, "rms_norm geometry is NULL");
  if (!known_dtype(g->dtype)) return report(OOPS_EINVAL, "unknown dtype %lld", g->dtype);
  if (g->width <= 0 || g->width > 16384) return report(OOPS_EINVAL, "width must be in 1..16384, got %lld", g->width);
  if (g->rows < 0 || g->rows > kMaxRows) return report(OOPS_EINVAL, "rows must be in 0..2^31-1, got %lld", g->rows);
  if (g->rows > 1 && (g->x_row < g->width || (residual && g->r_row < g->width)))
    return report(OOPS_EINVAL, "row strides (%lld, %lld) must cover the width", g->x_row, g->r_row);
  return OOPS_OK;
}
size_t rms_parts_bytes(const oops_rms_norm_geometry& g) {
  return align256((size_t)oops::rms_norm_parts(g) * (size_t)g.width * sizeof(float));
}


// ---- int8_linear
int check_int8(const oops_int8_geometry* g) {
  if (!g) return report(OOPS_EINVAL, "int8_linear geometry is NULL");
  if (!known_dtype(g->out_dtype) || !known_dtype(g->bias_dtype))
    return report(OOPS_EINVAL, "unknown out_dtype %lld or bias_dtype %lld", g->out_dtype, g->bias_dtype);
  if (g->bias_dtype != OOPS_F32 && g->bias_dtype != g->out_dtype)
    return report(OOPS_EINVAL, "the bias must be float32 or of the output's type");
  if (g->rows < 0 || g->rows > kMaxRows || g->n < 0 || g->n > kMaxRows)
    return report(OOPS_EINVAL, "rows (%lld) and n (%lld) must be in 0..2^31-1", g->rows, g->n);
  // (131072 products of -128 by -128 would pass the 32-bit sums)
  if (g->k < 0 || g->k > 131071) return report(OOPS_EINVAL, "k must be in 0..131071, got %lld", g->k);
  if ((g->rows > 1 && g->x_row < g->k) || (g->n > 1 && g->w_row < g->k))
    return report(OOPS_EINVAL, "row strides (%lld, %lld) must cover k", g->x_row, g->w_row);
  return OOPS_OK;
}

// ---- linear attention
int check_linear(const oops_linear_attn_geometry* g) {
  if (!g) return report(OOPS_EINVAL, "linear attention geometry is NULL");
  if (!known_dtype(g->dtype)) return report(OOPS_EINVAL, "unknown dtype %lld", g->dtype);
  if (g->heads <= 0) return report(OOPS_EINVAL, "heads must be positive, got %lld", g->heads);
  if (g->key_size <= 0 || g->key_size > 128 || g->value_size <= 0 || g->value_size > 128)
    return report(OOPS_EINVAL, "key_size and value_size must be in 1..128, got %lld and %lld", g->key_size,
                  g->value_size);
  if (g->batch < 0 || g->length < 0 || g->length > kMaxRows)
    return report(OOPS_EINVAL, "batch must be >= 0 and length in 0..2^31-1 (%lld, %lld)", g->batch, g->length);
  if (g->batch > 0 && g->heads > kMaxRows / 128 / g->batch)
    return report(OOPS_EINVAL, "too many heads (%lld x %lld)", g->batch, g->heads);
  for (int i = 0; i < OOPS_LA_OPERANDS; ++i)
    for (int d = 0; d < 3; ++d)
      if (g->stride[i][d] < 0) return report(OOPS_EINVAL, "operand %lld has a negative stride", i);
  return OOPS_OK;
}

void set3(int64_t (&to)[3], const int64_t (&from)[3]) { std::copy(from, from + 3, to); }

// operand `id` of the geometry at `p`, as the walk's a, b, c or out
struct Operand {
  const void* p;
  int id;
};
oops::LinearWalk walk(const oops_linear_attn_geometry& g, Operand a, Operand b, Operand c, void* out, int out_id,
                      const float* log_decay, const void* lengths) {
  oops::LinearWalk w{};
  w.a = a.p;
  w.b = b.p;
  w.c = c.p;
  w.out = out;
  set3(w.a_stride, g.stride[a.id]);
  set3(w.b_stride, g.stride[b.id]);
  set3(w.c_stride, g.stride[c.id]);
  set3(w.out_stride, g.stride[out_id]);
  w.log_decay = log_decay;
  w.lengths = lengths;
  w.batch = g.batch;
  w.length = g.length;
  w.heads = g.heads;
  w.lengths_i64 = g.lengths_i64;
  w.scale = g.scale;
  const bool keys = a.id == OOPS_LA_Q || a.id == OOPS_LA_K;  // a and b are key_size wide, c and out value_size
  w.rows = keys ? g.key_size : g.value_size;
  w.cols = keys ? g.value_size : g.key_size;
  w.state_by_cols = !keys;
  return w;
}
// o = walk(q, k, v); dq = walk(do, v, k) on the transposed state; from the end dk = walk(v, do, q) and
// dv = walk(k, q, do), whose state behind the first token is the initial state's gradient
oops::LinearWalk walk_out(const oops_linear_attn_geometry& g, const void* q, const void* k, const void* v, void* out,
                          const float* log_decay, const void* lengths, const float* initial, float* final_state) {
  oops::LinearWalk w = walk(g, {q, OOPS_LA_Q}, {k, OOPS_LA_K}, {v, OOPS_LA_V}, out, OOPS_LA_O, log_decay, lengths);
  w.initial = initial;
  w.final_state = final_state;
  return w;
}
struct GradWalks {
  oops::LinearWalk dq, dk, dv;
};
GradWalks grad_walks(const oops_linear_attn_geometry& g, const void* q, const void* k, const void* v,
                     const float* log_decay, const void* lengths, const float* initial, const void* grad_out,
                     const float* grad_final, void* grad_q, void* grad_k, void* grad_v, float* grad_initial) {
  const Operand Q{q, OOPS_LA_Q}, K{k, OOPS_LA_K}, V{v, OOPS_LA_V}, DO{grad_out, OOPS_LA_DO};
  GradWalks w{walk(g, DO, V, K, grad_q, OOPS_LA_DQ, log_decay, lengths),
              walk(g, V, DO, Q, grad_k, OOPS_LA_DK, log_decay, lengths),
              walk(g, K, Q, DO, grad_v, OOPS_LA_DV, log_decay, lengths)};
  w.dq.initial = initial;
  w.dk.initial = w.dv.initial = grad_final;
  w.dk.from_end = w.dv.from_end = 1;
  w.dv.final_state = grad_initial;
  return w;
}

}  // namespace

extern "C" {

int oops_rms_norm_forward(const oops_rms_norm_geometry* geo, const void* x, const void* residual, const void* weight,
                          void* y, void* sum, float* rstd, void* stream) {
  oops::clear_report();
  if (int rc = check_rms(geo, residual != nullptr)) return rc;
  if (geo->rows == 0) return OOPS_OK;
  if (!x || !y || (residual && !sum)) return report(OOPS_EINVAL, "x, y and, with a residual, sum must be non-NULL");
  return report_launch(oops::launch_rms_norm_forward(*geo, x, residual, weight, y, sum, rstd,
                                                     static_cast<hipStream_t>(stream)),
                       "rms_norm forward");
}

int oops_rms_norm_int8(const oops_rms_norm_geometry* geo, const void* x, const void* residual, const void* weight,
                       void* values, float* scales, void* sum, void* stream) {
  oops::clear_report();
  if (int rc = check_rms(geo, residual != nullptr)) return rc;
  if (geo->rows == 0) return OOPS_OK;
  if (!x || !values || !scales || (residual && !sum))
    return report(OOPS_EINVAL, "x, values, scales and, with a residual, sum must be non-NULL");
  return report_launch(oops::launch_rms_norm_int8(*geo, x, residual, weight, values, scales, sum,
                                                  static_cast<hipStream_t>(stream)),
                       "rms_norm int8");
}

int oops_quantize_int8(const oops_rms_norm_geometry* geo, const void* x, void* values, float* scales, void* stream) {
  oops::clear_report();
  if (int rc = check_rms(geo, false)) return rc;
  if (geo->rows == 0) return OOPS_OK;
  if (!x || !values || !scales) return report(OOPS_EINVAL, "x, values and scales must be non-NULL");
  oops_rms_norm_geometry g = *geo;
  g.r_row = g.width;
  return report_launch(oops::launch_quantize_int8(g, x, values, scales, static_cast<hipStream_t>(stream)),
                       "quantize_int8");
}

size_t oops_rms_norm_backward_workspace_bytes(const oops_rms_norm_geometry* geo) {
  oops::clear_report();
  if (check_rms(geo, false)) return 0;
  return rms_parts_bytes(*geo);
}

int oops_rms_norm_backward(const oops_rms_norm_geometry* geo, const void* h, const float* rstd, const void* weight,
                           const void* grad_y, const void* grad_sum, void* grad_x, void* grad_weight, void* workspace,
                           size_t ws_bytes, void* stream) {
  oops::clear_report();
  if (int rc = check_rms(geo, false)) return rc;
  if (geo->rows == 0) return report(OOPS_EINVAL, "the backward needs rows");
  if (!h || !rstd || !grad_y || !grad_x) return report(OOPS_EINVAL, "h, rstd, grad_y and grad_x must be non-NULL");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (grad_weight)
    if (int rc = oops::report_workspace(workspace, ws_bytes, oops_rms_norm_backward_workspace_bytes(geo))) return rc;
  float* parts = grad_weight ? static_cast<float*>(workspace) : nullptr;
  oops_rms_norm_geometry g = *geo;
  g.r_row = g.width;
  hipError_t e = oops::launch_rms_norm_backward(g, h, rstd, weight, grad_y, grad_sum, grad_x, parts, st);
  if (e == hipSuccess && grad_weight) e = oops::launch_rms_weight_sum(g, parts, grad_weight, st);
  return report_launch(e, "rms_norm backward");
}

size_t oops_int8_linear_workspace_bytes(const oops_int8_geometry* geo) {
  oops::clear_report();
  if (check_int8(geo)) return 0;
  return oops::int8_linear_workspace_bytes(*geo);
}

int oops_int8_linear(const oops_int8_geometry* geo, const void* x, const float* x_scale, const void* w,
                     const float* w_scale, const void* bias, void* out, void* workspace, size_t ws_bytes,
                     void* stream) {
  oops::clear_report();
  if (int rc = check_int8(geo)) return rc;
  if (geo->rows == 0 || geo->n == 0) return OOPS_OK;
  if ((geo->k > 0 && (!x || !w)) || !x_scale || !w_scale || !out)
    return report(OOPS_EINVAL, "x, w, their scales and out must be non-NULL");
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops::int8_linear_workspace_bytes(*geo))) return rc;
  return report_launch(oops::launch_int8_linear(*geo, x, x_scale, w, w_scale, bias, out, workspace,
                                                static_cast<hipStream_t>(stream)),
                       "int8_linear");
}

size_t oops_linear_attn_forward_workspace_bytes(const oops_linear_attn_geometry* geo) {
  oops::clear_report();
  if (check_linear(geo)) return 0;
  float state;
  return oops::linear_walk_workspace_bytes(
      geo->dtype, walk_out(*geo, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, &state));
}

int oops_linear_attn_forward(const oops_linear_attn_geometry* geo, const void* q, const void* k, const void* v,
                             const float* log_decay, const void* lengths, const float* initial, void* out,
                             float* final_state, void* workspace, size_t ws_bytes, void* stream) {
  oops::clear_report();
  if (int rc = check_linear(geo)) return rc;
  if (geo->batch == 0) return OOPS_OK;
  if (!log_decay || (geo->length > 0 && (!q || !k || !v || !out)))
    return report(OOPS_EINVAL, "q, k, v, log_decay and out must be non-NULL");
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops_linear_attn_forward_workspace_bytes(geo))) return rc;
  const oops::LinearWalk w = walk_out(*geo, q, k, v, out, log_decay, lengths, initial, final_state);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = oops::launch_linear_walk_starts(geo->dtype, w, workspace, st);
  if (e == hipSuccess) e = oops::launch_linear_walk(geo->dtype, w, workspace, st);
  return report_launch(e, "linear attention forward");
}

size_t oops_linear_attn_backward_workspace_bytes(const oops_linear_attn_geometry* geo) {
  // (the walks from the start, then those from the end, keep their segments' states there)
  return oops_linear_attn_forward_workspace_bytes(geo);
}

int oops_linear_attn_backward(const oops_linear_attn_geometry* geo, const void* q, const void* k, const void* v,
                              const float* log_decay, const void* lengths, const float* initial,
                              const void* forward_workspace, const void* grad_out, const float* grad_final,
                              void* grad_q, void* grad_k, void* grad_v, float* grad_initial, void* workspace,
                              size_t ws_bytes, void* stream) {
  oops::clear_report();
  if (int rc = check_linear(geo)) return rc;
  if (geo->batch == 0) return OOPS_OK;
  if (!log_decay || (geo->length > 0 && (!q || !k || !v || !grad_out)))
    return report(OOPS_EINVAL, "q, k, v, log_decay and grad_out must be non-NULL");
  if (int rc = oops::report_workspace(workspace, ws_bytes, oops_linear_attn_backward_workspace_bytes(geo))) return rc;
  const GradWalks w = grad_walks(*geo, q, k, v, log_decay, lengths, initial, grad_out, grad_final, grad_q, grad_k,
                                 grad_v, grad_initial);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e = hipSuccess;
  if (grad_q) {
    if (!forward_workspace)
      e = oops::launch_linear_walk_starts(
          geo->dtype, walk_out(*geo, q, k, v, nullptr, log_decay, lengths, initial, nullptr), workspace, st);
    if (e == hipSuccess)
      e = oops::launch_linear_walk(geo->dtype, w.dq, forward_workspace ? forward_workspace : workspace, st);
  }
  const bool dv = grad_v || grad_initial;
  if (e == hipSuccess && (grad_k || dv)) e = oops::launch_linear_walk_starts(geo->dtype, w.dv, workspace, st);
  if (e == hipSuccess && grad_k) e = oops::launch_linear_walk(geo->dtype, w.dk, workspace, st);
  if (e == hipSuccess && dv) e = oops::launch_linear_walk(geo->dtype, w.dv, workspace, st);
  return report_launch(e, "linear attention backward");
}

int oops_linear_attn_step(const oops_linear_attn_geometry* geo, const void* q, const void* k, const void* v,
                          const float* log_decay, float* state, void* out, void* stream) {
  oops::clear_report();
  if (int rc = check_linear(geo)) return rc;
  if (geo->batch == 0) return OOPS_OK;
  if (!q || !k || !v || !log_decay || !state || !out)
    return report(OOPS_EINVAL, "q, k, v, log_decay, state and out must be non-NULL");
  return report_launch(oops::launch_linear_attn_step(*geo, q, k, v, log_decay, state, out,
                                                     static_cast<hipStream_t>(stream)),
                       "linear attention step");
}

}  // extern "C"
