// Linear layer on 8-bit integers:
//
//   out[r][j] = x_scale[r] w_scale[j] sum_k x[r][k] w[j][k] + bias[j]
//
// sums exact in 32-bit integers on the int8 matrix units (32x32x32 MFMA, twice
// the bf16 rate), one rounding at the end.
//
// int8_any_kernel serves every size and alignment: 64 x 64 outputs a
// workgroup, 128 bytes of k a step through LDS, the next step's bytes loaded
// to registers meanwhile.  The weight is MFMA's row operand: a lane then holds
// one output row and four consecutive columns at a time.
#include <hip/hip_runtime.h>

#include "attn_common.h"
#include "layer_kernels.h"

namespace oops {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
constexpr int kStep = 128;  // bytes of k of a step
constexpr int64_t kMaxTiles = (int64_t(1) << 32) / kThreads - 1;  // a launch has less than 2^32 lanes

struct Int8Args {
  const int8_t *x, *w;
  const float *x_scale, *w_scale;
  const void* bias;
  void* out;
  int64_t rows, n, x_row, w_row;
  int32_t k, bias_f32;
};

// bytes col .. col+15 of a row of k bytes, zeros behind it, at any alignment
__device__ __forceinline__ i32x4 load_bytes(const int8_t* row, int col, int k, bool live) {
  i32x4 u = {0, 0, 0, 0};
  if (!live || col >= k) return u;
  if (col + 16 <= k) {
    __builtin_memcpy(&u, row + col, 16);
    return u;
  }
  uint32_t t[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; ++i)
    if (col + i < k) t[i / 4] |= (uint32_t)(uint8_t)row[col + i] << (8 * (i % 4));
  u = i32x4{(int)t[0], (int)t[1], (int)t[2], (int)t[3]};
  return u;
}

// 16-byte slot of chunk c of an LDS row of 8 chunks: the 8 rows of one read phase use all 8 slots
__device__ __forceinline__ int slot(int row, int c) { return row * 8 + (c ^ (row & 7)); }

template <typename T>
__device__ __forceinline__ float bias_at(const Int8Args& a, int64_t j) {
  if (!a.bias) return 0.f;
  return a.bias_f32 ? static_cast<const float*>(a.bias)[j] : (float)static_cast<const T*>(a.bias)[j];
}

template <typename T>
__global__ __launch_bounds__(kThreads) void int8_any_kernel(Int8Args a) {
  __shared__ i32x4 tw[64 * 8], tx[64 * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t tiles = (a.n + 63) / 64;
  const int64_t j0 = (int64_t)blockIdx.x % tiles * 64, r0 = (int64_t)blockIdx.x / tiles * 64;
  const int wj = (wave & 1) * 32, wr = (wave >> 1) * 32, l = lane & 31, half = lane >> 5;
  i32x4 pw[2], px[2];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (tid + i * kThreads) >> 3, col = k0 + (tid & 7) * 16;
      const int64_t j = j0 + row, r = r0 + row;
      pw[i] = load_bytes(a.w + (j < a.n ? j : 0) * a.w_row, col, a.k, j < a.n);
      px[i] = load_bytes(a.x + (r < a.rows ? r : 0) * a.x_row, col, a.k, r < a.rows);
    }
  };
  i32x16 acc = {};
  fetch(0);
  for (int k0 = 0; k0 < a.k; k0 += kStep) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = (tid + i * kThreads) >> 3;
      tw[slot(row, tid & 7)] = pw[i];
      tx[slot(row, tid & 7)] = px[i];
    }
    __syncthreads();
    if (k0 + kStep < a.k) fetch(k0 + kStep);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(tw[slot(wj + l, 2 * c + half)], tx[slot(wr + l, 2 * c + half)], acc,
                                                  0, 0, 0);
  }
  const int64_t r = r0 + wr + l;
  if (r >= a.rows) return;
  const float sx = a.x_scale[r];
  T* out = static_cast<T*>(a.out) + r * a.n;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t j = j0 + wj + kappa(half, i);
    if (j < a.n) out[j] = (T)__builtin_fmaf((float)acc[i] * sx, a.w_scale[j], bias_at<T>(a, j));
  }
}

template <typename F>
hipError_t by_type(int dtype, F&& f) {
  if (dtype == OOPS_F32) return f(float{});
  if (dtype == OOPS_BF16) return f((__bf16)0.f);
  return f((_Float16)0.f);
}

}  // namespace

size_t int8_linear_workspace_bytes(const oops_int8_geometry&) { return 0; }

hipError_t launch_int8_linear(const oops_int8_geometry& g, const void* x, const float* x_scale, const void* w,
                              const float* w_scale, const void* bias, void* out, void*, hipStream_t stream) {
  const Int8Args a{static_cast<const int8_t*>(x), static_cast<const int8_t*>(w), x_scale, w_scale, bias, out, g.rows,
                   g.n, g.x_row, g.w_row, (int32_t)g.k, g.bias_dtype == OOPS_F32};
  const int64_t tiles = ((g.n + 63) / 64) * ((g.rows + 63) / 64);
  if (tiles > kMaxTiles) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)tiles);
  return by_type(g.out_dtype, [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((int8_any_kernel<T>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace oops
