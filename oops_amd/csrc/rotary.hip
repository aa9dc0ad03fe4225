// Root-mean-square norm of queries and keys for each head, with the rotation by their position in the same pass.
//
//   n = x rstd,  rstd = (mean(x^2) + eps)^-1/2,  z = n w
//   y_i = z_i c - z_(i+R/2) s,  y_(i+R/2) = z_(i+R/2) c + z_i s  (i < R/2),  y_i = z_i (i >= R)
// backward, with g the rotation's transpose of dy (the same with -s):
//   dx = rstd (g w - n mean(g w n)),  dw = sum over rows of g n
//
// Bound by HBM: x is read and y written once (the backward reads x and dy and
// writes dx; rstd is made again from x, which costs no byte).  A row of a head
// lies in the registers of 8, 16 or 32 lanes, eight elements each; the other half
// of a pair is another lane's (R/2 a multiple of eight), or, for other sizes,
// strides and alignments, one wave takes a row and reads the other half again.
// Rows are ordered by token, then head, so that a token's cosines and sines are
// read from memory once.  dw stays in registers over a workgroup's rows; the
// workgroups' partial rows are added in a fixed order by a second launch.
#include <algorithm>

#include "attn_common.h"
#include "decoder_kernels.h"

namespace oops {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxParts = 1024;

struct Side {  // the queries or the keys
  const void *x, *weight, *dy;
  void *y, *dx;
  float* parts;
  void* dweight;
  int64_t sx[3], sy[3], sdy[3], sdx[3];
  int64_t rows;
  int32_t heads, weight_f32, parts_count;
};
struct RotaryArgs {
  Side side[2];
  const float* table;
  const void* positions;
  int64_t length, table_rows;
  int32_t size, half, positions_i64;
  float eps;
};

struct RowAt {
  int64_t b, t;
  int h;
};
__device__ __forceinline__ RowAt row_at(uint32_t r, uint32_t heads, uint32_t length) {
  const uint32_t token = r / heads;
  return RowAt{token / length, token % length, (int)(r % heads)};
}
__device__ __forceinline__ int64_t offset(const int64_t (&s)[3], const RowAt& a) { return a.b * s[0] + a.h * s[1] + a.t * s[2]; }
__device__ __forceinline__ const float* angles(const RotaryArgs& a, const RowAt& at) {
  int64_t p = at.t;
  if (a.positions) {
    const int64_t i = at.b * a.length + at.t;
    p = a.positions_i64 ? static_cast<const int64_t*>(a.positions)[i] : static_cast<const int32_t*>(a.positions)[i];
  }
  p = p < 0 ? 0 : p >= a.table_rows ? a.table_rows - 1 : p;
  return a.table + p * 2 * a.half;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)e[i];
  } else {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    union {
      uint4 u;
      T e[8];
    } r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = (T)v[i];
    *reinterpret_cast<uint4*>(p) = r.u;
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int d = LANES / 2; d > 0; d /= 2) x += __shfl_xor(x, d);
  return x;
}
template <typename T>
__device__ __forceinline__ float weight_at(const Side& s, int i) {
  if (!s.weight) return 1.f;
  return s.weight_f32 ? static_cast<const float*>(s.weight)[i] : (float)static_cast<const T*>(s.weight)[i];
}

// ---- eight elements a lane: LANES lanes a row (size <= 8 LANES, a multiple of 8; half too)
template <typename T, int LANES>
struct Piece {
  int lane, first, partner;  // first: of its elements; partner: the lane with the other halves of its pairs
  bool live, turned, upper;
  __device__ __forceinline__ Piece(const RotaryArgs& a) {
    lane = threadIdx.x % LANES;
    first = lane * 8;
    live = first < a.size;
    turned = first < 2 * a.half;
    upper = turned && first >= a.half;
    partner = (int)(threadIdx.x % 64) + (turned ? (upper ? -a.half / 8 : a.half / 8) : 0);
  }
  // v turned by the angle, or back
  template <bool BACK>
  __device__ __forceinline__ void turn(const RotaryArgs& a, const float* row, float (&v)[8]) const {
    float o[8], c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl(v[i], partner);
    if (!turned) return;
    const float* at = row + first - (upper ? a.half : 0);
    load8<float>(at, c);
    load8<float>(at + a.half, s);
    const bool plus = upper != BACK;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(plus ? o[i] : -o[i], s[i], v[i] * c[i]);
  }
};

template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void rotary_forward_kernel(RotaryArgs a) {
  const Side& s = a.side[blockIdx.y];
  const Piece<T, LANES> p(a);
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = p.live ? weight_at<T>(s, p.first + i) : 0.f;
  const uint32_t per = kThreads / LANES;
  // (a row's lanes stay together: what they exchange is theirs)
  for (int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / LANES; r < s.rows; r += (int64_t)gridDim.x * per) {
    const RowAt at = row_at((uint32_t)r, s.heads, (uint32_t)a.length);
    float v[8] = {}, sq = 0.f;
    if (p.live) load8<T>(static_cast<const T*>(s.x) + offset(s.sx, at) + p.first, v);
    const float* row = angles(a, at);
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = __builtin_fmaf(v[i], v[i], sq);
    const float rstd = 1.0f / __builtin_sqrtf(lanes_sum<LANES>(sq) / (float)a.size + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * rstd * w[i];
    p.template turn<false>(a, row, v);
    if (p.live) store8<T>(static_cast<T*>(s.y) + offset(s.sy, at) + p.first, v);
  }
}

template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void rotary_backward_kernel(RotaryArgs a) {
  const Side& s = a.side[blockIdx.y];
  if (!s.dy || blockIdx.x >= s.parts_count) return;
  const Piece<T, LANES> p(a);
  constexpr int per = kThreads / LANES;
  __shared__ float sum[per][LANES * 8];
  float w[8], dw[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = p.live ? weight_at<T>(s, p.first + i) : 0.f;
  for (int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / LANES; r < s.rows; r += (int64_t)s.parts_count * per) {
    const RowAt at = row_at((uint32_t)r, s.heads, (uint32_t)a.length);
    float n[8] = {}, d[8] = {}, sq = 0.f, dot = 0.f;
    if (p.live) {
      load8<T>(static_cast<const T*>(s.x) + offset(s.sx, at) + p.first, n);
      load8<T>(static_cast<const T*>(s.dy) + offset(s.sdy, at) + p.first, d);
    }
    const float* row = angles(a, at);
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = __builtin_fmaf(n[i], n[i], sq);
    const float rstd = 1.0f / __builtin_sqrtf(lanes_sum<LANES>(sq) / (float)a.size + a.eps);
    p.template turn<true>(a, row, d);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      n[i] *= rstd;
      dw[i] = __builtin_fmaf(d[i], n[i], dw[i]);
      d[i] *= w[i];
      dot = __builtin_fmaf(d[i], n[i], dot);
    }
    dot = lanes_sum<LANES>(dot) / (float)a.size;
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = rstd * __builtin_fmaf(-dot, n[i], d[i]);
    if (p.live && s.dx) store8<T>(static_cast<T*>(s.dx) + offset(s.sdx, at) + p.first, d);
  }
  if (!s.parts) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[threadIdx.x / LANES][p.first + i] = dw[i];
  __syncthreads();
  for (int c = threadIdx.x; c < a.size; c += kThreads) {
    float t = sum[0][c];
    for (int k = 1; k < per; ++k) t += sum[k][c];
    s.parts[(int64_t)blockIdx.x * a.size + c] = t;
  }
}

// ---- any size, stride and alignment: a wave a row, four elements a lane, 64 apart
constexpr int kCols = 4;
template <typename T, bool BACK>
__global__ __launch_bounds__(kThreads) void rotary_any_kernel(RotaryArgs a) {
  const Side& s = a.side[blockIdx.y];
  if (BACK && (!s.dy || blockIdx.x >= s.parts_count)) return;
  const int lane = threadIdx.x & 63;
  constexpr int per = kThreads / 64;
  __shared__ float sum[per][64 * kCols];
  float dw[kCols] = {};
  const int64_t step = (BACK ? (int64_t)s.parts_count : (int64_t)gridDim.x) * per;
  for (int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / 64; r < s.rows; r += step) {
    const RowAt at = row_at((uint32_t)r, s.heads, (uint32_t)a.length);
    const T* x = static_cast<const T*>(s.x) + offset(s.sx, at);
    const float* row = angles(a, at);
    float v[kCols] = {}, sq = 0.f;
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
      const int i = lane + 64 * k;
      if (i < a.size) v[k] = (float)x[i];
      sq = __builtin_fmaf(v[k], v[k], sq);
    }
    const float rstd = 1.0f / __builtin_sqrtf(lanes_sum<64>(sq) / (float)a.size + a.eps);
    // element i of a row turned by the angle or back, from the elements e(i)
    auto turned = [&](auto e, int i) {
      const float own = e(i);
      if (i >= 2 * a.half) return own;
      const bool upper = i >= a.half;
      const int j = upper ? i - a.half : i;
      const float other = e(upper ? j : i + a.half);
      return __builtin_fmaf(upper != BACK ? other : -other, row[a.half + j], own * row[j]);
    };
    if constexpr (!BACK) {
      T* y = static_cast<T*>(s.y) + offset(s.sy, at);
      auto z = [&](int i) { return (float)x[i] * rstd * weight_at<T>(s, i); };
#pragma unroll
      for (int k = 0; k < kCols; ++k)
        if (lane + 64 * k < a.size) y[lane + 64 * k] = (T)turned(z, lane + 64 * k);
    } else {
      const T* dy = static_cast<const T*>(s.dy) + offset(s.sdy, at);
      auto e = [&](int i) { return (float)dy[i]; };
      float d[kCols] = {}, dot = 0.f;
#pragma unroll
      for (int k = 0; k < kCols; ++k) {
        const int i = lane + 64 * k;
        v[k] *= rstd;
        if (i < a.size) {
          d[k] = turned(e, i);
          dw[k] = __builtin_fmaf(d[k], v[k], dw[k]);
          d[k] *= weight_at<T>(s, i);
        }
        dot = __builtin_fmaf(d[k], v[k], dot);
      }
      dot = lanes_sum<64>(dot) / (float)a.size;
      if (s.dx) {
        T* dx = static_cast<T*>(s.dx) + offset(s.sdx, at);
#pragma unroll
        for (int k = 0; k < kCols; ++k)
          if (lane + 64 * k < a.size) dx[lane + 64 * k] = (T)(rstd * __builtin_fmaf(-dot, v[k], d[k]));
      }
    }
  }
  if (!BACK || !s.parts) return;
#pragma unroll
  for (int k = 0; k < kCols; ++k) sum[threadIdx.x / 64][lane + 64 * k] = dw[k];
  __syncthreads();
  for (int c = threadIdx.x; c < a.size; c += kThreads) {
    float t = sum[0][c];
    for (int k = 1; k < per; ++k) t += sum[k][c];
    s.parts[(int64_t)blockIdx.x * a.size + c] = t;
  }
}

// The partial rows' sum in a fixed order: 16 columns a workgroup, its 64 slices every 64th row each, then a tree.
template <typename T>
__global__ __launch_bounds__(1024) void rotary_weight_kernel(RotaryArgs a) {
  const Side& s = a.side[blockIdx.y];
  if (!s.parts) return;
  __shared__ float sum[64][17];
  const int c = threadIdx.x & 15, slice = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float t = 0.f;
  if (col < a.size)
    for (int r = slice; r < s.parts_count; r += 64) t += s.parts[(int64_t)r * a.size + col];
  sum[slice][c] = t;
  for (int d = 32; d > 0; d /= 2) {
    __syncthreads();
    if (slice < d) sum[slice][c] += sum[slice + d][c];
  }
  if (slice == 0 && col < a.size) {
    if (s.weight_f32) static_cast<float*>(s.dweight)[col] = sum[0][c];
    else static_cast<T*>(s.dweight)[col] = (T)sum[0][c];
  }
}

RotaryArgs rotary_args(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                       const float* table, const void* positions) {
  RotaryArgs a{};
  for (int i = 0; i < 2; ++i) {
    Side& s = a.side[i];
    s.x = x[i];
    s.weight = weight[i];
    s.heads = g.heads[i];
    s.weight_f32 = g.weight_f32[i];
    s.rows = g.batch * g.length * g.heads[i];
    std::copy(g.stride[OOPS_RO_X][i], g.stride[OOPS_RO_X][i] + 3, s.sx);
    std::copy(g.stride[OOPS_RO_Y][i], g.stride[OOPS_RO_Y][i] + 3, s.sy);
    std::copy(g.stride[OOPS_RO_DY][i], g.stride[OOPS_RO_DY][i] + 3, s.sdy);
    std::copy(g.stride[OOPS_RO_DX][i], g.stride[OOPS_RO_DX][i] + 3, s.sdx);
  }
  a.table = table;
  a.positions = positions;
  a.length = g.length;
  a.table_rows = g.table_rows;
  a.size = g.size;
  a.half = g.rotary / 2;
  a.positions_i64 = g.positions_i64;
  a.eps = g.eps;
  return a;
}

// Whole pieces of eight elements at 16-byte addresses everywhere, the pairs' halves in different pieces
bool pieces(const oops_rotary_geometry& g, const RotaryArgs& a, bool back) {
  const int n = g.dtype == OOPS_F32 ? 4 : 8;
  if (g.size % 8 || (g.rotary / 2) % 8 || reinterpret_cast<uintptr_t>(a.table) % 16) return false;
  auto whole = [&](const void* p, const int64_t(&s)[3]) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % n == 0 && s[1] % n == 0 && s[2] % n == 0;
  };
  for (const Side& s : a.side) {
    if (s.rows == 0) continue;
    if (!whole(s.x, s.sx)) return false;
    if (!back && !whole(s.y, s.sy)) return false;
    if (back && s.dy && !whole(s.dy, s.sdy)) return false;
    if (back && s.dx && !whole(s.dx, s.sdx)) return false;
  }
  return true;
}
template <typename F>
hipError_t by_type(int dtype, F&& f) {
  if (dtype == OOPS_F32) return f(float{});
  if (dtype == OOPS_BF16) return f((__bf16)0.f);
  return f((_Float16)0.f);
}
int lanes_of(int size) { return size <= 64 ? 8 : size <= 128 ? 16 : 32; }

}  // namespace

int rotary_parts(const oops_rotary_geometry& g, int which) {
  const int64_t rows = g.batch * g.length * g.heads[which];
  // (the same for both layouts: with a wave a row the workgroups walk further)
  const int per = kThreads / lanes_of(g.size);
  return (int)std::min<int64_t>((rows + per - 1) / per, kMaxParts);
}

hipError_t launch_rotary_forward(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                                 const float* table, const void* positions, void* const (&y)[2], hipStream_t stream) {
  RotaryArgs a = rotary_args(g, x, weight, table, positions);
  for (int i = 0; i < 2; ++i) a.side[i].y = y[i];
  const bool whole = pieces(g, a, false);
  const int per = whole ? kThreads / lanes_of(g.size) : kThreads / 64;
  const int64_t rows = std::max(a.side[0].rows, a.side[1].rows);
  if (rows == 0) return hipSuccess;
  const dim3 grid((unsigned)std::min<int64_t>((rows + per - 1) / per, 1 << 20), 2);
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (!whole) hipLaunchKernelGGL((rotary_any_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
    else if (lanes_of(g.size) == 8) hipLaunchKernelGGL((rotary_forward_kernel<T, 8>), grid, dim3(kThreads), 0, stream, a);
    else if (lanes_of(g.size) == 16) hipLaunchKernelGGL((rotary_forward_kernel<T, 16>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((rotary_forward_kernel<T, 32>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

hipError_t launch_rotary_backward(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                                  const float* table, const void* positions, const void* const (&dy)[2],
                                  void* const (&dx)[2], float* const (&parts)[2], void* const (&dweight)[2],
                                  hipStream_t stream) {
  RotaryArgs a = rotary_args(g, x, weight, table, positions);
  int most = 0;
  for (int i = 0; i < 2; ++i) {
    Side& s = a.side[i];
    s.dy = dy[i];
    s.dx = dx[i];
    s.parts = dy[i] ? parts[i] : nullptr;
    s.dweight = dweight[i];
    s.parts_count = rotary_parts(g, i);
    most = std::max(most, s.parts_count);
  }
  if (most == 0) return hipSuccess;
  const dim3 grid((unsigned)most, 2);
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (!pieces(g, a, true)) hipLaunchKernelGGL((rotary_any_kernel<T, true>), grid, dim3(kThreads), 0, stream, a);
    else if (lanes_of(g.size) == 8) hipLaunchKernelGGL((rotary_backward_kernel<T, 8>), grid, dim3(kThreads), 0, stream, a);
    else if (lanes_of(g.size) == 16) hipLaunchKernelGGL((rotary_backward_kernel<T, 16>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((rotary_backward_kernel<T, 32>), grid, dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (!a.side[0].parts && !a.side[1].parts)) return e;
    hipLaunchKernelGGL((rotary_weight_kernel<T>), dim3((unsigned)(g.size + 15) / 16, 2), dim3(1024), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace oops
