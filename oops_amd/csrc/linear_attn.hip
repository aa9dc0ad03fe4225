// Linear attention with a decay for each head:
//
//   S_t = l S_(t-1) + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log_decay)
//
// and its gradients, all of them one walk (LinearWalk, layer_kernels.h) over
// other operands:
//   o  = walk(q, k, v)       dq = walk(do, v, k) on the transposed state
//   dk = walk(v, do, q) and dv = walk(k, q, do) from the end, where the state
//   R_t = l R_(t+1) + scale q_t^T do_t is the gradient of S_t.
//
// walk_kernel is the recurrence itself: a workgroup holds a (batch, head)'s
// state for 64 columns in registers, a quarter of the rows each wave, and goes
// token by token through chunks staged in LDS.
#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "layer_kernels.h"

namespace oops {
namespace {

constexpr int kThreads = 256;

// exp(log_decay n) for n >= 0: n = 0 gives 1 for every decay, -inf included
__device__ __forceinline__ float log2_decay(float log_decay) { return fmaxf(log_decay * kLog2e, -1e30f); }
__device__ __forceinline__ float decay_power(float l2, float n) { return exp2f(l2 * n); }

__device__ __forceinline__ int64_t walk_length(const LinearWalk& w, int64_t b) {
  if (!w.lengths) return w.length;
  const int64_t n = w.lengths_i64 ? static_cast<const int64_t*>(w.lengths)[b]
                                  : (int64_t) static_cast<const int32_t*>(w.lengths)[b];
  return n < 0 ? 0 : n > w.length ? w.length : n;
}

constexpr int kTok = 16;  // tokens of a chunk

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void walk_kernel(LinearWalk w) {
  constexpr int DG = DP / 4;  // state rows of a wave
  __shared__ float sa[kTok][DP], sb[kTok][DP], sc[kTok][64], red[4][kTok][64];
  const int64_t bh = blockIdx.x;
  const int64_t b = bh / w.heads;
  const int h = (int)(bh % w.heads);
  const int col = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int e = blockIdx.y * 64 + col;
  const int64_t n = walk_length(w, b);
  const float decay = decay_power(log2_decay(w.log_decay[h]), 1.f);
  const T* a = static_cast<const T*>(w.a) + b * w.a_stride[0] + h * w.a_stride[1];
  const T* bb = static_cast<const T*>(w.b) + b * w.b_stride[0] + h * w.b_stride[1];
  const T* c = static_cast<const T*>(w.c) + b * w.c_stride[0] + h * w.c_stride[1];
  T* out = static_cast<T*>(w.out);
  if (out) out += b * w.out_stride[0] + h * w.out_stride[1];
  const int64_t state0 = bh * w.rows * w.cols;
  float s[DG];
#pragma unroll
  for (int i = 0; i < DG; ++i) {
    const int d = g * DG + i;
    const int64_t at = state0 + (w.state_by_cols ? (int64_t)e * w.rows + d : (int64_t)d * w.cols + e);
    s[i] = w.initial && d < w.rows && e < w.cols ? w.initial[at] : 0.f;
  }
  const float up = w.from_end ? w.scale : 1.f, os = w.from_end ? 1.f : w.scale;
  for (int64_t p0 = 0; p0 < n; p0 += kTok) {
    const int m = (int)(n - p0 < kTok ? n - p0 : kTok);
    __syncthreads();
    for (int i = threadIdx.x; i < kTok * DP; i += kThreads) {
      const int t = i / DP, d = i % DP;
      const int64_t tok = w.from_end ? n - 1 - p0 - t : p0 + t;
      const bool in = t < m && d < w.rows;
      sa[t][d] = in ? (float)a[tok * w.a_stride[2] + d] : 0.f;
      sb[t][d] = in ? (float)bb[tok * w.b_stride[2] + d] : 0.f;
    }
    for (int i = threadIdx.x; i < kTok * 64; i += kThreads) {
      const int t = i / 64, d = blockIdx.y * 64 + i % 64;
      const int64_t tok = w.from_end ? n - 1 - p0 - t : p0 + t;
      sc[t][i % 64] = t < m && d < w.cols ? (float)c[tok * w.c_stride[2] + d] * up : 0.f;
    }
    __syncthreads();
    for (int t = 0; t < m; ++t) {
      const float l = w.from_end && p0 + t == 0 ? 1.f : decay;
      const float cv = sc[t][col];
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < DG; ++i) {
        s[i] = __builtin_fmaf(sb[t][g * DG + i], cv, s[i] * l);
        o = __builtin_fmaf(sa[t][g * DG + i], s[i], o);
      }
      red[g][t][col] = o;
    }
    __syncthreads();
    if (out)
      for (int t = g; t < m; t += 4) {
        const int64_t tok = w.from_end ? n - 1 - p0 - t : p0 + t;
        const float o = (red[0][t][col] + red[1][t][col]) + (red[2][t][col] + red[3][t][col]);
        if (e < w.cols) out[tok * w.out_stride[2] + e] = (T)(o * os);
      }
  }
  if (out && e < w.cols)
    for (int64_t t = n + g; t < w.length; t += 4) out[t * w.out_stride[2] + e] = (T)0.f;
  if (w.final_state) {
    const float l = w.from_end && n > 0 ? decay : 1.f;
#pragma unroll
    for (int i = 0; i < DG; ++i) {
      const int d = g * DG + i;
      const int64_t at = state0 + (w.state_by_cols ? (int64_t)e * w.rows + d : (int64_t)d * w.cols + e);
      if (d < w.rows && e < w.cols) w.final_state[at] = s[i] * l;
    }
  }
}

// ---------------------------------------------------------------- one token
//
// The state crosses HBM once each way (8 bytes an element against 6
// operations): a workgroup streams the rows of a (batch, head)'s columns, VW
// columns and up to kStepRows rows in flight a lane.  Few heads are split over
// workgroups by columns, 32 each.
struct StepArgs {
  const void *q, *k, *v;
  void* out;
  const float* log_decay;
  float* state;
  int64_t q_s[2], k_s[2], v_s[2], o_s[2];
  int32_t heads, rows, cols, block_cols;
  float scale;
};
constexpr int kStepRows = 8;

template <typename T, int VW>
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs a) {
  typedef float FV __attribute__((ext_vector_type(VW)));
  __shared__ float sq[128], sk[128];
  __shared__ FV red[kThreads];
  const int64_t bh = blockIdx.x;
  const int64_t b = bh / a.heads;
  const int h = (int)(bh % a.heads), tid = threadIdx.x;
  const int c0 = blockIdx.y * a.block_cols;
  const int cols = a.cols - c0 < a.block_cols ? a.cols - c0 : a.block_cols;
  const int tr = cols / VW, rpp = kThreads / tr;  // lanes of a row, rows of a pass
  const int r0 = tid / tr, col = c0 + tid % tr * VW;
  const bool on = r0 < rpp;
  float* s = a.state + (bh * a.rows) * a.cols + col;
  const T* q = static_cast<const T*>(a.q) + b * a.q_s[0] + h * a.q_s[1];
  const T* k = static_cast<const T*>(a.k) + b * a.k_s[0] + h * a.k_s[1];
  const T* v = static_cast<const T*>(a.v) + b * a.v_s[0] + h * a.v_s[1];
  FV x[kStepRows];
#pragma unroll
  for (int i = 0; i < kStepRows; ++i) {
    const int d = r0 + i * rpp;
    if (on && d < a.rows) x[i] = *reinterpret_cast<const FV*>(s + (int64_t)d * a.cols);
  }
  if (tid < a.rows) {
    sq[tid] = (float)q[tid];
    sk[tid] = (float)k[tid];
  }
  const float decay = decay_power(log2_decay(a.log_decay[h]), 1.f);
  FV vv, o;
#pragma unroll
  for (int j = 0; j < VW; ++j) {
    vv[j] = on ? (float)v[col + j] : 0.f;
    o[j] = 0.f;
  }
  __syncthreads();
  for (int d0 = r0; on && d0 < a.rows; d0 += kStepRows * rpp) {
#pragma unroll
    for (int i = 0; i < kStepRows; ++i) {
      const int d = d0 + i * rpp;
      if (d < a.rows) {
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          x[i][j] = __builtin_fmaf(sk[d], vv[j], x[i][j] * decay);
          o[j] = __builtin_fmaf(sq[d], x[i][j], o[j]);
        }
        *reinterpret_cast<FV*>(s + (int64_t)d * a.cols) = x[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kStepRows; ++i) {
      const int d = d0 + (kStepRows + i) * rpp;
      if (d < a.rows) x[i] = *reinterpret_cast<const FV*>(s + (int64_t)d * a.cols);
    }
  }
  red[tid] = o;
  __syncthreads();
  if (tid < cols) {
    float sum = 0.f;
    for (int r = 0; r < rpp; ++r) sum += red[r * tr + tid / VW][tid % VW];
    T* out = static_cast<T*>(a.out) + b * a.o_s[0] + h * a.o_s[1];
    out[c0 + tid] = (T)(sum * a.scale);
  }
}

template <typename F>
hipError_t by_type(int dtype, F&& f) {
  if (dtype == OOPS_F32) return f(float{});
  if (dtype == OOPS_BF16) return f((__bf16)0.f);
  return f((_Float16)0.f);
}

}  // namespace

size_t linear_walk_workspace_bytes(int, const LinearWalk&) { return 0; }

hipError_t launch_linear_walk(int dtype, const LinearWalk& w, void*, hipStream_t stream) {
  const dim3 grid((unsigned)(w.batch * w.heads), (unsigned)((w.cols + 63) / 64));
  return by_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (w.rows <= 32)
      hipLaunchKernelGGL((walk_kernel<T, 32>), grid, dim3(kThreads), 0, stream, w);
    else if (w.rows <= 64)
      hipLaunchKernelGGL((walk_kernel<T, 64>), grid, dim3(kThreads), 0, stream, w);
    else
      hipLaunchKernelGGL((walk_kernel<T, 128>), grid, dim3(kThreads), 0, stream, w);
    return hipGetLastError();
  });
}

hipError_t launch_linear_attn_step(const oops_linear_attn_geometry& g, const void* q, const void* k, const void* v,
                                   const float* log_decay, float* state, void* out, hipStream_t stream) {
  StepArgs a{q, k, v, out, log_decay, state, {}, {}, {}, {}, g.heads, g.key_size, g.value_size, g.value_size, g.scale};
  for (int i = 0; i < 2; ++i) {
    a.q_s[i] = g.stride[OOPS_LA_Q][i];
    a.k_s[i] = g.stride[OOPS_LA_K][i];
    a.v_s[i] = g.stride[OOPS_LA_V][i];
    a.o_s[i] = g.stride[OOPS_LA_O][i];
  }
  const bool vec = g.value_size % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0;
  if (g.batch * g.heads < 512 && g.value_size > 32) a.block_cols = 32;
  const dim3 grid((unsigned)(g.batch * g.heads), (unsigned)((g.value_size + a.block_cols - 1) / a.block_cols));
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (vec)
      hipLaunchKernelGGL((step_kernel<T, 4>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((step_kernel<T, 1>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace oops
