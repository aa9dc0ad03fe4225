// Root-mean-square norm of queries and keys for each head, with the rotation by their position in the same pass.
//
//   n = x rstd,  rstd = (mean(x^2) + eps)^-1/2,  z = n w
//   y_i = z_i c - z_(i+R/2) s,  y_(i+R/2) = z_(i+R/2) c + z_i s  (i < R/2),  y_i = z_i (i >= R)
// backward, with g the rotation's transpose of dy (the same with -s):
//   dx = rstd (g w - n mean(g w n)),  dw = sum over rows of g n
//
// Bound by HBM: x is read and y written once (the backward reads x and dy and
// writes dx; rstd is made again from x, which costs no byte).  A row of a head
// lies in the registers of 8, 16 or 32 lanes, eight elements each, four heads of a
// token at once, whose cosines and sines are read once; the other half of a pair is
// another lane's (R/2 a multiple of eight).  For other sizes, strides and alignments
// one wave takes a row and reads the other half again.  A bounded grid walks over
// tokens and their groups of heads, queries and keys in one launch; dw stays in
// registers meanwhile, and the workgroups' partial rows are added in a fixed order by
// a second launch.
//
// 8192 tokens of 32 + 8 heads of 128, bfloat16: forward 37 us (4.5 TB/s; one head at a
// time 50, two 43), backward 61 (4.1 TB/s, two heads at a time; one 66) and 7 for the sums
// of dw; a large copy reaches 4.9-5.1.  One token of four sequences: 5.4 us, a launch and
// a chain of loads.
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
  int32_t heads, weight_f32;
};
struct RotaryArgs {
  Side side[2];
  const float* table;
  const void* positions;
  int64_t tokens, length, table_rows;
  int32_t size, half, positions_i64, parts_count;
  float eps, inv_size;
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
// x of another lane of the same 16, by a pattern (no trip through LDS)
template <int PATTERN>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), PATTERN, 0xF, 0xF, true));
}
constexpr int kSwapPairs = 0xB1, kSwapHalfQuads = 0x4E, kReverseQuad = 0x1B;  // lanes ^ 1, ^ 2, ^ 3
constexpr int kReverse8 = 0x141, kReverse16 = 0x140, kTurn8 = 0x128;         // lanes ^ 7, ^ 15, (+ 8) % 16
// the sum over LANES neighbours, in each of them
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp<kSwapPairs>(x);
  x += dpp<kSwapHalfQuads>(x);
  x += dpp<kReverse8>(x);  // (the quads are alike by now)
  if constexpr (LANES >= 16) x += dpp<kReverse16>(x);
#pragma unroll
  for (int d = 16; d < LANES; d *= 2) x += __shfl_xor(x, d);
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
  bool live, turned, upper, across;  // across: every lane is turned, with the one LANES / 2 further
  __device__ __forceinline__ Piece(const RotaryArgs& a) {
    lane = threadIdx.x % LANES;
    first = lane * 8;
    live = first < a.size;
    turned = first < 2 * a.half;
    upper = turned && first >= a.half;
    across = a.half == LANES * 4;
    partner = (int)(threadIdx.x % 64) + (turned ? (upper ? -a.half / 8 : a.half / 8) : 0);
  }
  __device__ __forceinline__ void load(const RotaryArgs& a, const float* row, float (&c)[8], float (&s)[8]) const {
    if (!turned) return;
    const float* at = row + first - (upper ? a.half : 0);
    load8<float>(at, c);
    load8<float>(at + a.half, s);
  }
  // v turned by the angle, or back
  template <bool BACK>
  __device__ __forceinline__ void turn(const float (&c)[8], const float (&s)[8], float (&v)[8]) const {
    const float sign = upper != BACK ? 1.f : -1.f;
    if (LANES < 32 && across) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float o = LANES == 16 ? dpp<kTurn8>(v[i]) : dpp<kReverseQuad>(dpp<kReverse8>(v[i]));  // lanes ^ 8, ^ 4
        v[i] = __builtin_fmaf(o, sign * s[i], v[i] * c[i]);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl(v[i], partner);
      v[i] = turned ? __builtin_fmaf(o, sign * s[i], v[i] * c[i]) : v[i];
    }
  }
};

// heads of a token at once
template <bool BACK>
constexpr int kHeads = BACK ? 2 : 4;

template <typename T, int LANES, bool BACK>
__global__ __launch_bounds__(kThreads, 4) void rotary_kernel(RotaryArgs a) {
  const Piece<T, LANES> p(a);
  constexpr uint32_t per = kThreads / LANES;
  constexpr int H = kHeads<BACK>;
  __shared__ float sum[BACK ? per : 1][BACK ? LANES * 8 : 1];
  // (few workgroups: the sides go to different ones)
#pragma unroll 1
  for (int side = blockIdx.y; side < 2; side += gridDim.y) {
    const Side& s = a.side[side];
    if (BACK && !s.dy) continue;
    float w[8], dw[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = p.live ? weight_at<T>(s, p.first + i) : 0.f;
    const uint32_t groups = (uint32_t)(s.heads + H - 1) / H;
    const uint64_t units = (uint64_t)a.tokens * groups;
    // (a row's lanes stay together: what they exchange is theirs)
    for (uint64_t n = blockIdx.x * per + threadIdx.x / LANES; n < units; n += gridDim.x * per) {
      const uint32_t token = (uint32_t)n / groups;
      const RowAt at{token / (uint32_t)a.length, token % (uint32_t)a.length, (int)((uint32_t)n - token * groups) * H};
      const int count = s.heads - at.h < H ? s.heads - at.h : H;
      const float* row = angles(a, at);
      float x[H][8], d[H][8], c[8], sn[8];
      const T* xp = static_cast<const T*>(s.x) + offset(s.sx, at) + p.first;
      const T* dp = BACK ? static_cast<const T*>(s.dy) + offset(s.sdy, at) + p.first : nullptr;
#pragma unroll
      for (int k = 0; k < H; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = d[k][i] = 0.f;
        if (p.live && k < count) {
          load8<T>(xp + k * s.sx[1], x[k]);
          if constexpr (BACK) load8<T>(dp + k * s.sdy[1], d[k]);
        }
      }
      p.load(a, row, c, sn);
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq = __builtin_fmaf(x[k][i], x[k][i], sq);
        const float rstd = 1.0f / __builtin_sqrtf(lanes_sum<LANES>(sq) * a.inv_size + a.eps);
        if constexpr (!BACK) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[k][i] = x[k][i] * rstd * w[i];
          p.template turn<false>(c, sn, x[k]);
          if (p.live && k < count) store8<T>(static_cast<T*>(s.y) + offset(s.sy, at) + k * s.sy[1] + p.first, x[k]);
        } else {
          p.template turn<true>(c, sn, d[k]);
          float dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[k][i] *= rstd;
            // (a head that is not there has zeros, which eps = 0 makes NaN)
            if (k == 0 || k < count) dw[i] = __builtin_fmaf(d[k][i], x[k][i], dw[i]);
            d[k][i] *= w[i];
            dot = __builtin_fmaf(d[k][i], x[k][i], dot);
          }
          dot = lanes_sum<LANES>(dot) * a.inv_size;
#pragma unroll
          for (int i = 0; i < 8; ++i) d[k][i] = rstd * __builtin_fmaf(-dot, x[k][i], d[k][i]);
          if (p.live && k < count && s.dx) store8<T>(static_cast<T*>(s.dx) + offset(s.sdx, at) + k * s.sdx[1] + p.first, d[k]);
        }
      }
    }
    if constexpr (BACK) {
      if (!s.parts) continue;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[threadIdx.x / LANES][p.first + i] = dw[i];
      __syncthreads();
      for (int c = threadIdx.x; c < a.size; c += kThreads) {
        float t = sum[0][c];
        for (uint32_t k = 1; k < per; ++k) t += sum[k][c];
        s.parts[(int64_t)blockIdx.x * a.size + c] = t;
      }
    }
  }
}

// ---- any size, stride and alignment: a wave a row, four elements a lane, 64 apart
constexpr int kCols = 4;
template <typename T, bool BACK>
__global__ __launch_bounds__(kThreads) void rotary_any_kernel(RotaryArgs a) {
  const Side& s = a.side[blockIdx.y];
  if (BACK && !s.dy) return;
  const int lane = threadIdx.x & 63;
  constexpr int per = kThreads / 64;
  __shared__ float sum[per][64 * kCols];
  float dw[kCols] = {};
  const int64_t step = (int64_t)gridDim.x * per;
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
    for (int r = slice; r < a.parts_count; r += 64) t += s.parts[(int64_t)r * a.size + col];
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
  a.tokens = g.batch * g.length;
  a.length = g.length;
  a.table_rows = g.table_rows;
  a.size = g.size;
  a.half = g.rotary / 2;
  a.positions_i64 = g.positions_i64;
  a.eps = g.eps;
  a.inv_size = 1.0f / (float)g.size;
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
// workgroups for the longer side's groups of heads, four on every CU at most (they stay resident, so that all end together)
template <bool BACK>
int grid_of(const oops_rotary_geometry& g) {
  constexpr int H = kHeads<BACK>;
  const int per = kThreads / lanes_of(g.size);
  const int64_t units = g.batch * g.length * ((std::max(g.heads[0], g.heads[1]) + H - 1) / H);
  return (int)std::min<int64_t>((units + per - 1) / per, kMaxParts);
}
template <typename T, bool BACK>
void launch_pieces(const oops_rotary_geometry& g, const RotaryArgs& a, hipStream_t stream) {
  const int n = grid_of<BACK>(g);
  const dim3 grid((unsigned)n, n < kMaxParts / 2 ? 2 : 1);
  const int lanes = lanes_of(g.size);
  if (lanes == 8) hipLaunchKernelGGL((rotary_kernel<T, 8, BACK>), grid, dim3(kThreads), 0, stream, a);
  else if (lanes == 16) hipLaunchKernelGGL((rotary_kernel<T, 16, BACK>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<T, 32, BACK>), grid, dim3(kThreads), 0, stream, a);
}

}  // namespace

int rotary_parts(const oops_rotary_geometry& g) { return grid_of<true>(g); }

hipError_t launch_rotary_forward(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                                 const float* table, const void* positions, void* const (&y)[2], hipStream_t stream) {
  RotaryArgs a = rotary_args(g, x, weight, table, positions);
  for (int i = 0; i < 2; ++i) a.side[i].y = y[i];
  if (g.batch * g.length == 0) return hipSuccess;
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (pieces(g, a, false)) {
      launch_pieces<T, false>(g, a, stream);
    } else {
      const int64_t rows = std::max(a.side[0].rows, a.side[1].rows);
      const dim3 grid((unsigned)std::min<int64_t>((rows + kThreads / 64 - 1) / (kThreads / 64), 1 << 20), 2);
      hipLaunchKernelGGL((rotary_any_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
    }
    return hipGetLastError();
  });
}

hipError_t launch_rotary_backward(const oops_rotary_geometry& g, const void* const (&x)[2], const void* const (&weight)[2],
                                  const float* table, const void* positions, const void* const (&dy)[2],
                                  void* const (&dx)[2], float* const (&parts)[2], void* const (&dweight)[2],
                                  hipStream_t stream) {
  RotaryArgs a = rotary_args(g, x, weight, table, positions);
  for (int i = 0; i < 2; ++i) {
    Side& s = a.side[i];
    s.dy = dy[i];
    s.dx = dx[i];
    s.parts = dy[i] ? parts[i] : nullptr;
    s.dweight = dweight[i];
  }
  a.parts_count = rotary_parts(g);
  if (g.batch * g.length == 0) return hipSuccess;
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (pieces(g, a, true)) launch_pieces<T, true>(g, a, stream);
    else hipLaunchKernelGGL((rotary_any_kernel<T, true>), dim3((unsigned)a.parts_count, 2), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (!a.side[0].parts && !a.side[1].parts)) return e;
    hipLaunchKernelGGL((rotary_weight_kernel<T>), dim3((unsigned)(g.size + 15) / 16, 2), dim3(1024), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace oops
