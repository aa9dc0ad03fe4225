// Root-mean-square norm of rows, with the residual's addition and an 8-bit output.
//
//   h = x + r (rounded to the element type, written back as the new residual stream)
//   y = h rstd w,   rstd = (mean(h^2) + eps)^-1/2
//   8-bit output: q = rint(y 127 / max|y|), scale = max|y| / 127 of the row
// backward, with g = dy w and n = h rstd:
//   dh = dsum + rstd (g - n mean(g n));   dw = sum over rows of dy n
//
// About ten operations an element against 4 to 10 bytes: bound by HBM.  A row
// is held in the registers of TPR lanes (16 bytes a lane and load, CH loads a
// lane), so every tensor is read and written once; statistics, products and
// the maximum are float32.  Rows of up to 256 pieces of 16 bytes (4 KB) stay
// in one wave, of up to 16 pieces in 16 lanes of it (no barrier); longer ones
// take the four waves of a workgroup.  The backward walks its rows with a
// bounded grid, dw in registers, one partial row a workgroup, summed afterwards
// in a fixed order.
//
// Measured (a copy reaches 4.9 TB/s): 8192 x 4096 bfloat16 with the residual's
// addition 50 us forward (5.3 TB/s), 57 backward (4.7), 6.7 the weight's sum;
// 8-bit output of 8192 x 8192 102 (4.6); 65536 x 128 8.3, 10.0 and 3.9; 8-bit
// rows of 8192 x 4096 21 (4.7), 30 where the launch before has left 268 MB of
// output to be written back.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_common.h"
#include "layer_kernels.h"

namespace oops {
namespace {

constexpr int kThreads = 256;

struct RmsArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* y;      // element type, or int8 values
  void* sum;
  float* rstd;  // also the 8-bit scales
  int64_t rows, x_row, r_row;
  int32_t width, weight_f32;
  float eps;
};
struct RmsGradArgs {
  const void* h;
  const float* rstd;
  const void* weight;
  const void* dy;
  const void* dsum;
  void* dx;
  float* parts;
  int64_t rows, h_row;
  int32_t width, weight_f32;
};

// The columns of chunk c of a lane: VE consecutive ones in the vector layout
// (16-byte rows), else VE columns TPR apart, so that a wave's loads are
// consecutive elements at any width and alignment.
template <typename T, int TPR, bool VEC>
struct Cols {
  static constexpr int VE = 16 / sizeof(T);
  static __device__ __forceinline__ int at(int lane, int c, int j) {
    return VEC ? (c * TPR + lane) * VE + j : (c * VE + j) * TPR + lane;
  }
};

template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void load_chunk(const T* row, int width, int lane, int c, float (&v)[16 / sizeof(T)]) {
  constexpr int VE = 16 / sizeof(T);
  using C = Cols<T, TPR, VEC>;
  if constexpr (VEC) {
    const int col = C::at(lane, c, 0);
    uint4 u = make_uint4(0, 0, 0, 0);
    if (col < width) u = *reinterpret_cast<const uint4*>(row + col);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int j = 0; j < VE; ++j) v[j] = (float)e[j];
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const int col = C::at(lane, c, j);
      v[j] = col < width ? (float)row[col] : 0.f;
    }
  }
}

// weight columns (float32 or the element type); none: ones
template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void load_weight(const void* w, int f32, int width, int lane, int c,
                                            float (&v)[16 / sizeof(T)]) {
  constexpr int VE = 16 / sizeof(T);
  using C = Cols<T, TPR, VEC>;
  if (w == nullptr) {
#pragma unroll
    for (int j = 0; j < VE; ++j) v[j] = 1.f;
  } else if (f32) {
    const float* wf = static_cast<const float*>(w);
    if constexpr (VEC) {
      const int col = C::at(lane, c, 0);
#pragma unroll
      for (int j = 0; j < VE; j += 4) {
        f32x4 u = {0.f, 0.f, 0.f, 0.f};
        if (col < width) u = *reinterpret_cast<const f32x4*>(wf + col + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[j + k] = u[k];
      }
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const int col = C::at(lane, c, j);
        v[j] = col < width ? wf[col] : 0.f;
      }
    }
  } else {
    load_chunk<T, TPR, VEC>(static_cast<const T*>(w), width, lane, c, v);
  }
}

template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void store_chunk(T* row, int width, int lane, int c, const float (&v)[16 / sizeof(T)]) {
  constexpr int VE = 16 / sizeof(T);
  using C = Cols<T, TPR, VEC>;
  if constexpr (VEC) {
    const int col = C::at(lane, c, 0);
    typedef T TV __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef float FV __attribute__((ext_vector_type(16 / sizeof(T))));
    FV f;
#pragma unroll
    for (int j = 0; j < VE; ++j) f[j] = v[j];
    if (col < width) *reinterpret_cast<TV*>(row + col) = __builtin_convertvector(f, TV);
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const int col = C::at(lane, c, j);
      if (col < width) row[col] = (T)v[j];
    }
  }
}

template <typename T, int TPR, bool VEC>
__device__ __forceinline__ void store_int8(int8_t* row, int width, int lane, int c, const int (&q)[16 / sizeof(T)]) {
  constexpr int VE = 16 / sizeof(T);
  using C = Cols<T, TPR, VEC>;
  if constexpr (VEC) {
    const int col = C::at(lane, c, 0);
    uint32_t u[VE / 4];
#pragma unroll
    for (int j = 0; j < VE; j += 4)
      u[j / 4] = (q[j] & 255) | (q[j + 1] & 255) << 8 | (q[j + 2] & 255) << 16 | (uint32_t)(q[j + 3] & 255) << 24;
    if (col < width) {
      if constexpr (VE == 8)
        *reinterpret_cast<uint2*>(row + col) = make_uint2(u[0], u[1]);
      else
        *reinterpret_cast<uint32_t*>(row + col) = u[0];
    }
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const int col = C::at(lane, c, j);
      if (col < width) row[col] = (int8_t)q[j];
    }
  }
}

// sum of x / largest of u over a row's TPR lanes, in every one of them.  TPR
// 256: `red` holds the waves' values; the caller passes another array for
// each call between two barriers.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
#pragma unroll
  for (int d = 1; d < (TPR < 64 ? TPR : 64); d *= 2) x += __shfl_xor(x, d, 64);
  if constexpr (TPR == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return x;
}
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x, uint32_t* red) {
#pragma unroll
  for (int d = 1; d < (TPR < 64 ? TPR : 64); d *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)x, d, 64);
    x = o > x ? o : x;
  }
  if constexpr (TPR == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    const uint32_t a = red[0] > red[1] ? red[0] : red[1], b = red[2] > red[3] ? red[2] : red[3];
    x = a > b ? a : b;
  }
  return x;
}

enum { kNorm = 0, kNormInt8 = 1, kInt8 = 2 };

template <typename T, int TPR, int CH, bool VEC, int MODE>
__global__ __launch_bounds__(kThreads) void rms_forward_kernel(RmsArgs a) {
  constexpr int VE = 16 / sizeof(T), RPB = kThreads / TPR;
  __shared__ float red_sum[2][4];
  __shared__ uint32_t red_max[2][4];
  const int lane = threadIdx.x % TPR;
  int turn = 0;
  // (a group of lanes past the rows leaves; TPR 256: the whole workgroup)
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows;
       row += (int64_t)gridDim.x * RPB, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_row;
    float h[CH][VE], ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) load_chunk<T, TPR, VEC>(x, a.width, lane, c, h[c]);
    if (MODE != kInt8 && a.residual) {
      const T* r = static_cast<const T*>(a.residual) + row * a.r_row;
      T* sum = static_cast<T*>(a.sum) + row * a.width;
      float rv[CH][VE];
#pragma unroll
      for (int c = 0; c < CH; ++c) load_chunk<T, TPR, VEC>(r, a.width, lane, c, rv[c]);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int j = 0; j < VE; ++j) h[c][j] = (float)(T)(h[c][j] + rv[c][j]);
        store_chunk<T, TPR, VEC>(sum, a.width, lane, c, h[c]);
      }
    }
    if constexpr (MODE != kInt8) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < VE; ++j) ss = __builtin_fmaf(h[c][j], h[c][j], ss);
      ss = row_sum<TPR>(ss, red_sum[turn]);
      const float rstd = 1.0f / sqrtf(ss / (float)a.width + a.eps);
      if (MODE == kNorm && a.rstd && lane == 0) a.rstd[row] = rstd;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float w[VE];
        load_weight<T, TPR, VEC>(a.weight, a.weight_f32, a.width, lane, c, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) h[c][j] = h[c][j] * rstd * w[j];
      }
    }
    if constexpr (MODE == kNorm) {
      T* y = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
      for (int c = 0; c < CH; ++c) store_chunk<T, TPR, VEC>(y, a.width, lane, c, h[c]);
    } else {
      // The largest magnitude as an integer: the bits of non-negative floats
      // order like their values, an infinity above every number and NaN above
      // that.  A row that holds either gets the scale NaN and zero values.
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const uint32_t b = __builtin_bit_cast(uint32_t, h[c][j]) & 0x7FFFFFFFu;
          top = b > top ? b : top;
        }
      top = row_max<TPR>(top, red_max[turn]);
      const bool fine = top < 0x7F800000u;
      const float amax = __builtin_bit_cast(float, top);
      // (rows of magnitudes far from 1 are scaled first: 1 / amax, or 127 amax, would be infinite)
      const float up = amax < 0x1p-100f ? 0x1p64f : amax > 0x1p100f ? 0x1p-64f : 1.0f;
      const float most = amax * up, inv = fine && top ? 1.0f / most : 0.f;
      if (lane == 0) a.rstd[row] = fine ? amax / 127.0f : __builtin_nanf("");
      int8_t* q = static_cast<int8_t*>(a.y) + row * a.width;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        int qi[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          // The quotient corrected by its residual: 127 x / amax to float32, so that what lies exactly between two
          // steps (half the largest: 63.5) goes to the even one.  (127 x is exact for 16-bit rows.)
          const float x = h[c][j] * up, x127 = x * 127.f, near = x127 * inv;
          float rest = __builtin_fmaf(-near, most, x127);
          if constexpr (MODE != kInt8 || sizeof(T) == 4) rest += __builtin_fmaf(x, 127.f, -x127);
          qi[j] = fine ? (int)__builtin_rintf(__builtin_fmaf(rest, inv, near)) : 0;
        }
        store_int8<T, TPR, VEC>(q, a.width, lane, c, qi);
      }
    }
  }
}

template <typename T, int TPR, int CH, bool VEC>
__global__ __launch_bounds__(kThreads) void rms_backward_kernel(RmsGradArgs a) {
  constexpr int VE = 16 / sizeof(T), RPB = kThreads / TPR;
  __shared__ float red[2][4];
  __shared__ float acc[RPB > 1 ? kThreads * CH * VE : 1];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  float w[CH][VE], dw[CH][VE] = {};
#pragma unroll
  for (int c = 0; c < CH; ++c) load_weight<T, TPR, VEC>(a.weight, a.weight_f32, a.width, lane, c, w[c]);
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows; row0 += (int64_t)gridDim.x * RPB, turn ^= 1) {
    const int64_t row = row0 + group;
    const bool live = row < a.rows;  // (a group of lanes beyond the rows reads and writes nothing)
    const int width = live ? a.width : 0;
    const int64_t r = live ? row : 0;
    const T* hp = static_cast<const T*>(a.h) + r * a.h_row;
    const T* gp = static_cast<const T*>(a.dy) + r * a.width;
    const float rstd = a.rstd[r];
    float n[CH][VE], g[CH][VE], ds[CH][VE], dot = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) load_chunk<T, TPR, VEC>(hp, width, lane, c, n[c]);
#pragma unroll
    for (int c = 0; c < CH; ++c) load_chunk<T, TPR, VEC>(gp, width, lane, c, g[c]);
    if (a.dsum) {
      const T* sp = static_cast<const T*>(a.dsum) + r * a.width;
#pragma unroll
      for (int c = 0; c < CH; ++c) load_chunk<T, TPR, VEC>(sp, width, lane, c, ds[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        n[c][j] *= rstd;
        dw[c][j] = __builtin_fmaf(g[c][j], n[c][j], dw[c][j]);
        g[c][j] *= w[c][j];
        dot = __builtin_fmaf(g[c][j], n[c][j], dot);
      }
    dot = row_sum<TPR>(dot, red[turn]) / (float)a.width;
    T* dx = static_cast<T*>(a.dx) + r * a.width;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float d = rstd * __builtin_fmaf(-dot, n[c][j], g[c][j]);
        g[c][j] = a.dsum ? d + ds[c][j] : d;
      }
      store_chunk<T, TPR, VEC>(dx, width, lane, c, g[c]);
    }
  }
  if (!a.parts) return;
  float* out = a.parts + (int64_t)blockIdx.x * a.width;
  if constexpr (RPB > 1) {
    // the groups' sums of one column, in order
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < VE; ++j) acc[group * (TPR * CH * VE) + Cols<T, TPR, VEC>::at(lane, c, j)] = dw[c][j];
    __syncthreads();
    for (int col = threadIdx.x; col < a.width; col += kThreads) {
      float s = acc[col];
#pragma unroll
      for (int k = 1; k < RPB; ++k) s += acc[k * (TPR * CH * VE) + col];
      out[col] = s;
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const int col = Cols<T, TPR, VEC>::at(lane, c, j);
        if (col < a.width) out[col] = dw[c][j];
      }
  }
}

// The partial rows' sum, in a fixed order and one launch: a workgroup takes 16
// columns, its 64 slices every 64th row each, then the slices in a tree.
template <typename W>
__global__ __launch_bounds__(1024) void rms_weight_sum_kernel(const float* parts, W* out, int rows, int width) {
  __shared__ float sum[64][17];
  const int c = threadIdx.x & 15, slice = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < width) {
#pragma unroll 4
    for (int r = slice; r < rows; r += 64) s += parts[(int64_t)r * width + col];
  }
  sum[slice][c] = s;
  for (int d = 32; d > 0; d /= 2) {
    __syncthreads();
    if (slice < d) sum[slice][c] += sum[slice + d][c];
  }
  if (slice == 0 && col < width) out[col] = (W)sum[0][c];
}

// ------------------------------------------------------------------ launchers

// Lanes and 16-byte chunks a lane of a row: as many lanes as chunks up to a
// wave, then up to four chunks a lane, then the whole workgroup.
struct RmsPlan {
  int tpr, ch;
  bool vec;
};
RmsPlan rms_plan(const oops_rms_norm_geometry& g, std::initializer_list<const void*> ptrs, bool strided = true) {
  const int ve = g.dtype == OOPS_F32 ? 4 : 8;
  const int chunks = (g.width + ve - 1) / ve;
  RmsPlan p{16, 1, g.width % ve == 0};
  if (strided && g.rows > 1 && (g.x_row % ve || g.r_row % ve)) p.vec = false;
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % 16) p.vec = false;
  if (chunks > 16) p.tpr = 64;
  if (chunks > 256) p.tpr = 256;
  while (p.tpr * p.ch < chunks) p.ch *= 2;
  return p;
}

template <typename F>
hipError_t by_type(int dtype, F&& f) {
  if (dtype == OOPS_F32) return f(float{});
  if (dtype == OOPS_BF16) return f((__bf16)0.f);
  return f((_Float16)0.f);
}
template <int TPR_, int CH_>
struct Shape {
  static constexpr int TPR = TPR_, CH = CH_;
};
// the (lanes, chunks) pairs rms_plan makes: 16 x 1, 64 x 1..4, 256 x 2..16 (float32 rows of 16384)
template <typename F>
hipError_t by_shape(const RmsPlan& p, F&& f) {
  if (p.tpr == 16) return f(Shape<16, 1>{});
  if (p.tpr == 64) {
    if (p.ch == 1) return f(Shape<64, 1>{});
    if (p.ch == 2) return f(Shape<64, 2>{});
    return f(Shape<64, 4>{});
  }
  if (p.ch == 2) return f(Shape<256, 2>{});
  if (p.ch == 4) return f(Shape<256, 4>{});
  if (p.ch == 8) return f(Shape<256, 8>{});
  return f(Shape<256, 16>{});
}

template <int MODE>
hipError_t run_forward(const oops_rms_norm_geometry& g, const RmsArgs& a, const RmsPlan& p, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  const int rpb = kThreads / p.tpr;
  // (a launch of more than 2^32 lanes is refused by the runtime: longer inputs are walked)
  const dim3 grid((unsigned)std::min<int64_t>((g.rows + rpb - 1) / rpb, 1 << 22));
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_shape(p, [&](auto s) {
      using S = decltype(s);
      if (p.vec)
        hipLaunchKernelGGL((rms_forward_kernel<T, S::TPR, S::CH, true, MODE>), grid, dim3(kThreads), 0, stream, a);
      else
        hipLaunchKernelGGL((rms_forward_kernel<T, S::TPR, S::CH, false, MODE>), grid, dim3(kThreads), 0, stream, a);
      return hipGetLastError();
    });
  });
}

RmsArgs forward_args(const oops_rms_norm_geometry& g, const void* x, const void* residual, const void* weight,
                     void* y, void* sum, float* rstd) {
  return RmsArgs{x, residual, weight, y, sum, rstd, g.rows, g.x_row, g.r_row, g.width, g.weight_f32, g.eps};
}
}  // namespace

hipError_t launch_rms_norm_forward(const oops_rms_norm_geometry& g, const void* x, const void* residual,
                                   const void* weight, void* y, void* sum, float* rstd, hipStream_t stream) {
  return run_forward<kNorm>(g, forward_args(g, x, residual, weight, y, sum, rstd),
                            rms_plan(g, {x, residual, weight, y, sum}), stream);
}

hipError_t launch_rms_norm_int8(const oops_rms_norm_geometry& g, const void* x, const void* residual,
                                const void* weight, void* values, float* scales, void* sum, hipStream_t stream) {
  return run_forward<kNormInt8>(g, forward_args(g, x, residual, weight, values, sum, scales),
                                rms_plan(g, {x, residual, weight, values, sum}), stream);
}

hipError_t launch_quantize_int8(const oops_rms_norm_geometry& g, const void* x, void* values, float* scales,
                                hipStream_t stream) {
  return run_forward<kInt8>(g, forward_args(g, x, nullptr, nullptr, values, nullptr, scales),
                            rms_plan(g, {x, values}), stream);
}

int64_t rms_norm_parts(const oops_rms_norm_geometry& g) {
  const int rpb = kThreads / rms_plan(g, {}, false).tpr;
  return std::min<int64_t>((g.rows + rpb - 1) / rpb, 1024);
}

hipError_t launch_rms_norm_backward(const oops_rms_norm_geometry& g, const void* h, const float* rstd,
                                    const void* weight, const void* grad_y, const void* grad_sum, void* grad_x,
                                    float* weight_parts, hipStream_t stream) {
  if (g.rows == 0) return hipSuccess;
  const RmsPlan p = rms_plan(g, {h, weight, grad_y, grad_sum, grad_x});
  const RmsGradArgs a{h, rstd, weight, grad_y, grad_sum, grad_x, weight_parts, g.rows, g.x_row, g.width, g.weight_f32};
  const dim3 grid((unsigned)rms_norm_parts(g));
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    return by_shape(p, [&](auto s) {
      using S = decltype(s);
      if (p.vec)
        hipLaunchKernelGGL((rms_backward_kernel<T, S::TPR, S::CH, true>), grid, dim3(kThreads), 0, stream, a);
      else
        hipLaunchKernelGGL((rms_backward_kernel<T, S::TPR, S::CH, false>), grid, dim3(kThreads), 0, stream, a);
      return hipGetLastError();
    });
  });
}

hipError_t launch_rms_weight_sum(const oops_rms_norm_geometry& g, const float* parts, void* out, hipStream_t stream) {
  const int rows = (int)rms_norm_parts(g);
  const dim3 grid((unsigned)(g.width + 15) / 16);
  return by_type(g.weight_f32 ? OOPS_F32 : g.dtype, [&](auto tag) {
    using W = decltype(tag);
    hipLaunchKernelGGL((rms_weight_sum_kernel<W>), grid, dim3(1024), 0, stream, parts, static_cast<W*>(out), rows, g.width);
    return hipGetLastError();
  });
}

}  // namespace oops
