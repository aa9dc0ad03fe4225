// Linear layer on 8-bit integers:
//
//   out[r][j] = x_scale[r] w_scale[j] sum_k x[r][k] w[j][k] + bias[j]
//
// sums exact in 32-bit integers on the int8 matrix units (32x32x32 MFMA, twice
// the bf16 rate); scales and bias in float32 (three roundings: the conversion
// of sums above 2^24, the product with x_scale, one fused product and
// addition), then the result's type.
//
// The weight is MFMA's row operand: a lane then holds one output row and four
// consecutive columns at a time.  By size and alignment:
//   up to 16 rows                   int8_few_kernel     the weight read once
//   whole 16-byte pieces a row      int8_tile_kernel    LDS tiles, 64^2 to 256^2
//   else, 10^9 products and more    int8_pad_kernel     copies, then tiles
//   else                            int8_any_kernel, or int8_small_kernel for few
//
// Measured: 8192 x 8192 x 8192 2.25 PFLOP/s (a library's product 2.12),
// rows x n x k of 8192 x 16384 x 4096 1.95; 4 x 16384 x 4096 4.4 TB/s of weight.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_common.h"
#include "attn_fast_common.h"
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
  int32_t* sums;  // parts > 1: [parts][rows][n] sums over part_k bytes of k each
  int32_t parts, part_k;
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

// Every size and alignment: 64 x 64 outputs a workgroup, 128 bytes of k a step
// through LDS, the next step's bytes loaded to registers meanwhile.  Bound by
// the waits of its steps (1001 bytes of k: 15 us up to one tile a CU).
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

// ---------------------------------------------------------------- whole tiles
//
// BM x BN outputs a workgroup of four waves (2 x 2, each BM/2 x BN/2 in 32 x
// 32 accumulator tiles), operands whose rows are whole 16-byte pieces at
// aligned places.  Steps of 128 bytes of k, whole cache lines: NB LDS buffers
// filled by direct global-to-LDS loads NB - 1 steps ahead.  One barrier a step,
// where all of a step's fragments are in registers and the next step's bytes
// have landed: the last slice's MFMAs run behind it while the next step's
// first fragments are read.
constexpr int kTileStep = 128;

// fast::dma16_asm with the LDS address as a number (the conversion of a pointer checks it for NULL in five scalar
// instructions, too many to hide behind an MFMA)
__device__ __forceinline__ void load_lds(const fast::u32x4& r, uint32_t to, uint32_t voff, uint32_t soff) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to),
      "v"(voff), "s"(r), "s"(soff)
      : "memory", "m0");
}

template <typename T, int BM, int BN, int NB>
__global__ __launch_bounds__(kThreads, 1) void int8_tile_kernel(Int8Args a, int tiles_r, int tiles_j,
                                                                               int grid_pad) {
  constexpr int TR = BM / 64, TJ = BN / 64;                  // accumulator tiles of a wave
  constexpr int kRowBytes = kTileStep, kStage = (BM + BN) * kRowBytes;
  constexpr int LR = BM / 32, LJ = BN / 32;                  // loads a wave and step: 8 rows each
  __shared__ __align__(16) char lds[NB * kStage];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Workgroups of one XCD take a contiguous run of tiles, eight rows of tiles
  // deep: the 32 that run at once read 8 + 4 tiles' bytes through its L2.
  const int t_all = (int)xcd_tile(blockIdx.x, grid_pad, 0);
  if (t_all >= tiles_r * tiles_j * a.parts) return;
  const int part = __builtin_amdgcn_readfirstlane(t_all / (tiles_r * tiles_j)), t = t_all - part * tiles_r * tiles_j;
  const int k_begin = part * a.part_k, k_end = a.k - k_begin < a.part_k ? a.k : k_begin + a.part_k;
  const int group = t / (8 * tiles_j), deep = tiles_r - group * 8 < 8 ? tiles_r - group * 8 : 8;
  const int in = t - group * 8 * tiles_j;
  const int64_t r0 = (int64_t)(group * 8 + in % deep) * BM, j0 = (int64_t)(in / deep) * BN;

  const int64_t left_r = a.rows - r0 < BM ? a.rows - r0 : BM, left_j = a.n - j0 < BN ? a.n - j0 : BN;
  // (rows behind the last one lie outside the resource: zeros)
  const fast::u32x4 rx = fast::rsrc_words(a.x + r0 * a.x_row, (uint32_t)((left_r - 1) * a.x_row + a.k));
  const fast::u32x4 rw = fast::rsrc_words(a.w + j0 * a.w_row, (uint32_t)((left_j - 1) * a.w_row + a.k));
  // a load fills 8 rows of eight 16-byte slots; slot c of row r holds bytes 16 (c ^ (r / 2 % 8)) of the step, so that
  // the 16 rows of a read phase use distinct banks (rows r and r + 8 hold it alike: loads i and i + 1 differ by 32 rows)
  uint32_t vx[LR], vw[LJ];
  const int lrow = wave * 8 + (lane >> 3), lc = (lane & 7) ^ ((lrow >> 1) & 7);
#pragma unroll
  for (int i = 0; i < LR; ++i) vx[i] = (uint32_t)((i * 32 + lrow) * (int)a.x_row + lc * 16);
#pragma unroll
  for (int i = 0; i < LJ; ++i) vw[i] = (uint32_t)((i * 32 + lrow) * (int)a.w_row + lc * 16);
  // load i of a step (x's rows, then w's); a scalar offset is never past the resource
  const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)lds + wave * 1024;
  auto load = [&](int step, int i) {
    const int k0 = k_begin + step * kTileStep;
    const uint32_t to = lds0 + (step % NB) * kStage + (i < LR ? i * 4096 : BM * kRowBytes + (i - LR) * 4096);
    const uint32_t at = k0 < k_end ? k0 : 0, v = i < LR ? vx[i < LR ? i : 0] : vw[i < LR ? 0 : i - LR];
    load_lds(i < LR ? rx : rw, __builtin_amdgcn_readfirstlane(to), k0 + lc * 16 < k_end ? v : fast::kOut, at);
  };
  const int steps = (k_end - k_begin + kTileStep - 1) / kTileStep;
#pragma unroll
  for (int s = 0; s < NB - 1; ++s)  // (steps behind k load zeros)
#pragma unroll
    for (int i = 0; i < LR + LJ; ++i) load(s, i);

  const int wr = (wave >> 1) * (BM / 2), wj = (wave & 1) * (BN / 2);
  const int lx = (wr + l) * kRowBytes + ((half ^ ((l >> 1) & 7)) << 4);
  const int lw = BM * kRowBytes + (wj + l) * kRowBytes + ((half ^ ((l >> 1) & 7)) << 4);
  i32x16 acc[TJ][TR];
#pragma unroll
  for (int q = 0; q < TJ; ++q)
#pragma unroll
    for (int p = 0; p < TR; ++p) acc[q][p] = i32x16{};
  i32x4 fx[2][TR], fw[2][TJ];
  auto read = [&](int step, int slice, i32x4(&x)[TR], i32x4(&w)[TJ]) {
    const char* from = lds + (step % NB) * kStage;
#pragma unroll
    for (int q = 0; q < TJ; ++q) w[q] = *reinterpret_cast<const i32x4*>(from + (lw ^ (slice << 5)) + q * 32 * kRowBytes);
#pragma unroll
    for (int p = 0; p < TR; ++p) x[p] = *reinterpret_cast<const i32x4*>(from + (lx ^ (slice << 5)) + p * 32 * kRowBytes);
  };
  // the products of a slice; between them, the loads of a later step
  auto multiply = [&](const i32x4(&x)[TR], const i32x4(&w)[TJ], int step) {
#pragma unroll
    for (int i = 0; i < TJ * TR; ++i) {
      acc[i / TR][i % TR] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[i / TR], x[i % TR], acc[i / TR][i % TR], 0, 0, 0);
      constexpr int kPer = (LR + LJ + TJ * TR - 1) / (TJ * TR);
      if (step >= 0) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = i * kPer; q < (i + 1) * kPer && q < LR + LJ; ++q) load(step, q);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  constexpr int kLater = (NB - 2) * (LR + LJ);  // loads behind the next step's
  fast::vmem_wait<kLater>();
  lds_barrier();
  read(0, 0, fx[0], fw[0]);
  for (int s = 0; s < steps; ++s) {
    read(s, 1, fx[1], fw[1]);
    __builtin_amdgcn_sched_barrier(0);
    multiply(fx[0], fw[0], s + NB - 1);
    read(s, 2, fx[0], fw[0]);
    __builtin_amdgcn_sched_barrier(0);
    multiply(fx[1], fw[1], -1);
    __builtin_amdgcn_sched_barrier(0);
    read(s, 3, fx[1], fw[1]);
    __builtin_amdgcn_sched_barrier(0);
    multiply(fx[0], fw[0], -1);
    __builtin_amdgcn_sched_barrier(0);
    fast::vmem_wait<kLater>();     // step s + 1 has landed (this wave's part)
    lds_barrier();                 // everywhere, and step s is in registers everywhere
    read(s + 1, 0, fx[0], fw[0]);  // (behind the last step: not used)
    __builtin_amdgcn_sched_barrier(0);
    multiply(fx[1], fw[1], -1);
    __builtin_amdgcn_sched_barrier(0);
  }
  fast::vmem_wait<0>();  // (no load may land in LDS that is used otherwise by then, or another workgroup's)
  lds_barrier();

  // out[r0 + wr + 32 p + l][j0 + wj + 32 q + kappa(half, i)]
  if (BM * BN == 64 * 64 && a.parts > 1) {
    int32_t* sums = a.sums + (int64_t)part * a.rows * a.n;
#pragma unroll
    for (int q = 0; q < TJ; ++q)
#pragma unroll
      for (int p = 0; p < TR; ++p) {
        const int64_t r = r0 + wr + 32 * p + l, jq = j0 + wj + 32 * q;
        if (r < a.rows)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (jq + kappa(half, i) < a.n) sums[r * a.n + jq + kappa(half, i)] = acc[q][p][i];
      }
    return;
  }
  // scales and biases without branches: zeros behind the last row and column
  const auto rs_x = make_rsrc(a.x_scale + r0, (uint32_t)left_r * 4), rs_w = make_rsrc(a.w_scale + j0, (uint32_t)left_j * 4);
  const int bias_bytes = a.bias == nullptr ? 0 : a.bias_f32 ? 4 : (int)sizeof(T);
  const auto rs_b = make_rsrc(static_cast<const char*>(a.bias) + j0 * bias_bytes, (uint32_t)(left_j * bias_bytes));
  float scale_x[TR];
#pragma unroll
  for (int p = 0; p < TR; ++p)
    scale_x[p] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs_x, (wr + 32 * p + l) * 4, 0, 0));
  // Whole lines to memory: a wave's rows of 128 bytes (64 outputs of 16 bits, 32 of float32) pass through 16 KB of LDS
  // of its own, from lanes that hold a row each to eight lanes a row; slots are XORed with the row.
  constexpr int V = 16 / sizeof(T), kTilesLine = sizeof(T) == 4 || TJ == 1 ? 1 : 2;  // column tiles of a line
  constexpr int kLanes = kTilesLine * 32 / V;                                        // lanes of a line (64 bytes: TJ 1)
  const bool vec = a.n % V == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  char* line = lds + wave * (BM / 2 * 128);
#pragma unroll
  for (int q = 0; q < TJ; ++q) {
    float scale_w[16], add[16] = {};
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint32_t j = wj + 32 * q + kappa(half, i);
      const f32x4 u = __builtin_bit_cast(f32x4, buffer_load16(rs_w, j * 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) scale_w[i + e] = u[e];
    }
    if (bias_bytes == 4) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 u = __builtin_bit_cast(f32x4, buffer_load16(rs_b, (wj + 32 * q + kappa(half, i)) * 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) add[i + e] = u[e];
      }
    } else if (bias_bytes == 2) {
      if constexpr (sizeof(T) == 2) {
        // (one by one: a pair that straddles the last column would be outside as a whole)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          add[i] = (float)__builtin_bit_cast(
              T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs_b, (wj + 32 * q + kappa(half, i)) * 2, 0, 0));
      }
    }
#pragma unroll
    for (int p = 0; p < TR; ++p) {
      const int64_t r = r0 + wr + 32 * p + l, jq = j0 + wj + 32 * q;
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = __builtin_fmaf((float)acc[q][p][i] * scale_x[p], scale_w[i], add[i]);
      if (!vec) {
        T* row = static_cast<T*>(a.out) + (r < a.rows ? r : 0) * a.n;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (r < a.rows && jq + kappa(half, i) < a.n) row[jq + kappa(half, i)] = (T)y[i];
      } else {
        char* to = line + (32 * p + l) * 128;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<f32x4*>(to + (((i / 2 + half) ^ (l & 7)) << 4)) = f32x4{y[i], y[i + 1], y[i + 2], y[i + 3]};
        } else {
          uint32_t pk[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) pk[i] = fast::pack2<T>(y[2 * i], y[2 * i + 1]);
          uint4 lo, hi;
          fast::trade16(pk, lo, hi);  // this lane: columns 16 half .. and 16 half + 8 .. of its row
          const int c = q % kTilesLine * 4 + 2 * half;
          *reinterpret_cast<uint4*>(to + ((c ^ (l & 7)) << 4)) = lo;
          *reinterpret_cast<uint4*>(to + (((c + 1) ^ (l & 7)) << 4)) = hi;
        }
      }
    }
    if (vec && q % kTilesLine == kTilesLine - 1) {
      const int64_t j = j0 + wj + 32 * (q - kTilesLine + 1) + lane % kLanes * V;
#pragma unroll
      for (int i = 0; i < BM / 2 * kLanes / 64; ++i) {
        const int row = (i * 64 + lane) / kLanes;
        const uint4 u = *reinterpret_cast<const uint4*>(line + row * 128 + ((lane % kLanes ^ (row & 7)) << 4));
        const int64_t r = r0 + wr + row;
        if (r < a.rows && j < a.n) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + r * a.n + j) = u;
      }
    }
  }
}

// ---------------------------------------------------------------- few rows
//
// Up to 16 rows of x: bound by the weight's bytes, each read once.  A
// workgroup takes 16 weight rows; its W waves take whole lines of k in turn, U
// lines in flight each, the operands loaded straight into the 16x16x64 MFMA's
// layout (a quarter wave reads 64 bytes of a row), and join their sums in LDS.
// W U lines are k where it can be had: all loads of a wave then fly at once
// (4 x 4096 x 16384: W, U = 8, 4 16.0 us or 4.2 TB/s; 4, 8 18.4; 16, 4 20.2;
// 8 x 1024 x 50000: 8, 2 15.7; 8, 4 22.6;  4 x 16384 x 4096: 16, 4 16.1; 8, 4 22.3).
// WHOLE: rows of whole 16-byte pieces at aligned places; else any.
template <typename T, int W, int U, bool WHOLE>
__global__ __launch_bounds__(64 * W) void int8_few_kernel(Int8Args a) {
  __shared__ i32x4 red[W][64];
  const int tid = threadIdx.x, lane = tid & 63, row = lane & 15, part = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t j0 = (int64_t)blockIdx.x * 16;
  const int64_t left = a.n - j0 < 16 ? a.n - j0 : 16;
  // (weight rows behind the last one lie outside the resource: zeros)
  const auto rw = make_rsrc(a.w + j0 * a.w_row, (uint32_t)((left - 1) * a.w_row + a.k));
  const auto rx = make_rsrc(a.x, (uint32_t)((a.rows - 1) * a.x_row + a.k));
  const uint32_t vw = row * (uint32_t)a.w_row + part * 16, vx = row * (uint32_t)a.x_row + part * 16;
  const int64_t j = j0 + 4 * part;
  i32x4 acc = {};
  for (int k0 = wave * 128; k0 < a.k; k0 += W * U * 128) {
    i32x4 fw[2 * U], fx[2 * U];
#pragma unroll
    for (int u = 0; u < 2 * U; ++u) {
      const int k = k0 + (u / 2) * W * 128 + (u % 2) * 64;
      if constexpr (WHOLE) {
        const bool in = k + part * 16 < a.k;
        fw[u] = __builtin_bit_cast(i32x4, buffer_load16(rw, in ? vw + k : fast::kOut));
        fx[u] = __builtin_bit_cast(i32x4, buffer_load16(rx, in && row < a.rows ? vx + k : fast::kOut));
      } else {
        fw[u] = load_bytes(a.w + (j0 + (row < left ? row : 0)) * a.w_row, k + part * 16, a.k, row < left);
        fx[u] = load_bytes(a.x + (row < a.rows ? row : 0) * a.x_row, k + part * 16, a.k, row < a.rows);
      }
    }
#pragma unroll
    for (int u = 0; u < 2 * U; ++u) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], fx[u], acc, 0, 0, 0);
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave > 0 || row >= a.rows) return;
  i32x4 sum = red[0][lane];
#pragma unroll
  for (int q = 1; q < W; ++q) sum += red[q][lane];
  // out[row][j0 + 4 part + i]
  const float sx = a.x_scale[row];
  T* out = static_cast<T*>(a.out) + row * a.n + j;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (j + i < a.n) out[i] = (T)__builtin_fmaf((float)sum[i] * sx, a.w_scale[j + i], bias_at<T>(a, j + i));
}

// ---------------------------------------------------------------- few products of odd rows
//
// 32 x 32 outputs a workgroup, whose W waves take lines of k in turn with the
// operands loaded straight into the 32x32x32 MFMA's layout, at any alignment,
// and join their sums in LDS: 64 x 64 tiles would leave most CUs idle and go
// through k one wait after the other.
template <typename T, int W>
__global__ __launch_bounds__(64 * W) void int8_small_kernel(Int8Args a) {
  __shared__ i32x4 red[W][4][64];
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t tiles = (a.n + 31) / 32;
  const int64_t j0 = (int64_t)blockIdx.x % tiles * 32, r0 = (int64_t)blockIdx.x / tiles * 32;
  const bool in_w = j0 + l < a.n, in_x = r0 + l < a.rows;
  const int8_t* w = a.w + (in_w ? j0 + l : 0) * a.w_row;
  const int8_t* x = a.x + (in_x ? r0 + l : 0) * a.x_row;
  i32x16 acc = {};
  for (int k0 = wave * 128; k0 < a.k; k0 += W * 128) {
    i32x4 fw[4], fx[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      fw[c] = load_bytes(w, k0 + 32 * c + 16 * half, a.k, in_w);
      fx[c] = load_bytes(x, k0 + 32 * c + 16 * half, a.k, in_x);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[c], fx[c], acc, 0, 0, 0);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) red[wave][q][lane] = i32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  if (wave >= 4 || !in_x) return;
  i32x4 sum = red[0][wave][lane];
#pragma unroll
  for (int q = 1; q < W; ++q) sum += red[q][wave][lane];
  // out[r0 + l][j0 + 8 wave + 4 half + i]
  const int64_t r = r0 + l, j = j0 + 8 * wave + 4 * half;
  const float sx = a.x_scale[r];
  T* out = static_cast<T*>(a.out) + r * a.n + j;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (j + i < a.n) out[i] = (T)__builtin_fmaf((float)sum[i] * sx, a.w_scale[j + i], bias_at<T>(a, j + i));
}

// ---------------------------------------------------------------- padded operands
//
// Rows that are no whole pieces at aligned places, copied to ones that are
// (zeros behind k): two passes over the bytes, where the products are many
// enough that whole tiles earn them back.
struct PadArgs {
  const int8_t* from[2];
  int8_t* to[2];
  int64_t rows[2], stride[2];
  int32_t k, pieces;  // 16-byte pieces of a padded row
};
__global__ __launch_bounds__(kThreads) void int8_pad_kernel(PadArgs a) {
  const int64_t first = a.rows[0] * a.pieces, all = first + a.rows[1] * a.pieces;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < all; i += (int64_t)gridDim.x * kThreads) {
    const int op = i >= first;
    const int64_t at = op ? i - first : i, row = at / a.pieces;
    const int piece = (int)(at - row * a.pieces);
    reinterpret_cast<i32x4*>(a.to[op])[at] = load_bytes(a.from[op] + row * a.stride[op], piece * 16, a.k, true);
  }
}

// ---------------------------------------------------------------- joined parts
//
// Few tiles and a long k: the tiles' parts of k write their sums, and this
// kernel adds them (whole numbers: in any order) and scales the result.
template <typename T>
__global__ __launch_bounds__(kThreads) void int8_join_kernel(Int8Args a) {
  const int64_t size = a.rows * a.n;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < size; i += (int64_t)gridDim.x * kThreads) {
    int sum = 0;
    for (int p = 0; p < a.parts; ++p) sum += a.sums[p * size + i];
    const int64_t r = i / a.n, j = i - r * a.n;
    static_cast<T*>(a.out)[i] = (T)__builtin_fmaf((float)sum * a.x_scale[r], a.w_scale[j], bias_at<T>(a, j));
  }
}

template <typename F>
hipError_t by_type(int dtype, F&& f) {
  if (dtype == OOPS_F32) return f(float{});
  if (dtype == OOPS_BF16) return f((__bf16)0.f);
  return f((_Float16)0.f);
}

// rows at multiples of 16 bytes, a tile of which spans less than 2 GiB
bool aligned_rows(const void* p, int64_t rows, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || (stride % 16 == 0 && stride < (int64_t(1) << 22)));
}

template <bool WHOLE>
hipError_t run_few(const oops_int8_geometry& g, Int8Args a, hipStream_t stream) {
  if (g.rows == 1) a.x_row = g.k;
  if (g.n == 1) a.w_row = g.k;
  const dim3 grid((unsigned)((g.n + 15) / 16));
  return by_type(g.out_dtype, [&](auto tag) {
    using T = decltype(tag);
    if (g.k <= 2048)
      hipLaunchKernelGGL((int8_few_kernel<T, 8, 2, WHOLE>), grid, dim3(512), 0, stream, a);
    else if (g.k <= 4096)
      hipLaunchKernelGGL((int8_few_kernel<T, 8, 4, WHOLE>), grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((int8_few_kernel<T, 16, 4, WHOLE>), grid, dim3(1024), 0, stream, a);
    return hipGetLastError();
  });
}

// Rows that go to int8_few_kernel: up to 8, or 16 where the weight has few rows (16 x 4096 x 4096: 7.5 us, tiles 10.2;
// 16 x 4096 x 16384: 20.8, tiles 17.6).
bool few_rows(const oops_int8_geometry& g) {
  return g.rows <= (g.n <= 8192 ? 16 : 8) && g.n < kMaxTiles * 8;
}

int64_t tiles_of(const oops_int8_geometry& g, int64_t m, int64_t n) {
  return ((g.n + n - 1) / n) * ((g.rows + m - 1) / m);
}

// Parts of k: where the smallest tiles are too few for the CUs, as many as fill them with at least kMinPart bytes each;
// fewer than four do not pay for the join (48 x 16384 x 4096: 36 us, eight parts 18 + 5; 32 x 4096 x 4096: 10.1, four
// parts 7.2 + 3.4).
constexpr int64_t kMinPart = 2048;
struct KParts {
  int parts, part_k;
};
KParts k_parts(const oops_int8_geometry& g) {
  const int64_t tiles = tiles_of(g, 64, 64);
  int64_t parts = 1;
  if (g.k % 16 == 0 && !few_rows(g) && tiles > 0 && tiles <= 128) parts = std::min(256 / tiles, g.k / kMinPart);
  if (parts < 4) return {1, (int)g.k};
  const int64_t per = ((g.k + parts - 1) / parts + kTileStep - 1) / kTileStep * kTileStep;
  return {(int)((g.k + per - 1) / per), (int)per};
}

// Operands to be copied to padded rows (a size's own: pointers off 16 bytes go to int8_any_kernel).
struct Pads {
  bool x, w;
  int64_t row, x_bytes, w_bytes;
};
Pads pads(const oops_int8_geometry& g) {
  Pads p{g.k % 16 != 0 || (g.rows > 1 && g.x_row % 16 != 0), g.k % 16 != 0 || (g.n > 1 && g.w_row % 16 != 0),
         (g.k + 15) / 16 * 16, 0, 0};
  // (1024 x 4097 x 4096: 40 us, int8_any_kernel 73; 512 x 2001 x 4096: 22.5, 24; 256 x 1001 x 1024: no gain)
  if (few_rows(g) || (double)g.rows * (double)g.n * (double)g.k < 1e9) p.x = p.w = false;
  if (p.x) p.x_bytes = (g.rows * p.row + 255) / 256 * 256;
  if (p.w) p.w_bytes = (g.n * p.row + 255) / 256 * 256;
  return p;
}

template <int BM, int BN, int NB>
hipError_t run_tiles(const oops_int8_geometry& g, Int8Args a, hipStream_t stream) {
  if (g.rows == 1) a.x_row = g.k;
  if (g.n == 1) a.w_row = g.k;
  const int tr = (int)((g.rows + BM - 1) / BM), tj = (int)((g.n + BN - 1) / BN);
  const int grid = (int)xcd_grid((int64_t)tr * tj * a.parts, 0);
  return by_type(g.out_dtype, [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((int8_tile_kernel<T, BM, BN, NB>), dim3((unsigned)grid), dim3(kThreads), 0, stream, a, tr, tj, grid);
    return hipGetLastError();
  });
}

}  // namespace

namespace {

// whole rows: the kernels by size, `sums` for the parts of k
hipError_t run_whole(const oops_int8_geometry& g, Int8Args a, void* sums, hipStream_t stream) {
  if (few_rows(g)) return run_few<true>(g, a, stream);
  // the largest tile that gives (nearly) every CU one, measured in us at rows x n x k:
  //   4096 x 4096 x 4096: 256^2 69, 128^2 83 (two a CU);   2048 x 4096 x 4096: 256^2 56, 128^2 40
  //   1024 x 4096 x 4096: 128^2 24 (four buffers; two: 31), 64 x 128 29;   512 x 4096 x 4096: 128^2 21, 64 x 128 17
  const int64_t t128 = tiles_of(g, 128, 128);
  if (tiles_of(g, 256, 256) >= 192) return run_tiles<256, 256, 2>(g, a, stream);
  if (t128 > 256) return run_tiles<128, 128, 2>(g, a, stream);
  if (t128 >= 192) return run_tiles<128, 128, 4>(g, a, stream);
  if (tiles_of(g, 64, 128) >= 192) return run_tiles<64, 128, 4>(g, a, stream);
  const KParts kp = k_parts(g);
  a.sums = static_cast<int32_t*>(sums);
  a.parts = kp.parts;
  a.part_k = kp.part_k;
  const hipError_t e = run_tiles<64, 64, 4>(g, a, stream);
  if (e != hipSuccess || a.parts == 1) return e;
  return by_type(g.out_dtype, [&](auto tag) {
    using T = decltype(tag);
    const int64_t blocks = std::min<int64_t>((g.rows * g.n + kThreads - 1) / kThreads, 2048);
    hipLaunchKernelGGL((int8_join_kernel<T>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

// The geometry of the padded operands (of the given ones where nothing is padded).
oops_int8_geometry padded(const oops_int8_geometry& g, const Pads& p) {
  oops_int8_geometry t = g;
  if (p.x || p.w) t.k = p.row;  // (a padded row's zeros meet zeros, or bytes of the other operand that is whole)
  if (p.x) t.x_row = p.row;
  if (p.w) t.w_row = p.row;
  return t;
}

}  // namespace

size_t int8_linear_workspace_bytes(const oops_int8_geometry& g) {
  const Pads p = pads(g);
  const int parts = k_parts(padded(g, p)).parts;
  return (size_t)(p.x_bytes + p.w_bytes) + (parts > 1 ? (size_t)parts * (size_t)g.rows * (size_t)g.n * sizeof(int32_t) : 0);
}

hipError_t launch_int8_linear(const oops_int8_geometry& g, const void* x, const float* x_scale, const void* w,
                              const float* w_scale, const void* bias, void* out, void* workspace, hipStream_t stream) {
  Int8Args a{static_cast<const int8_t*>(x), static_cast<const int8_t*>(w), x_scale, w_scale, bias, out, g.rows, g.n,
             g.x_row, g.w_row, (int32_t)g.k, g.bias_dtype == OOPS_F32, nullptr, 1, (int32_t)g.k};
  const int64_t tiles = tiles_of(g, 64, 64);
  const Pads p = pads(g);
  const oops_int8_geometry t = padded(g, p);
  const bool whole = g.k > 0 && t.k % 16 == 0 && (p.x || aligned_rows(x, g.rows, g.x_row)) &&
                     (p.w || aligned_rows(w, g.n, g.w_row)) && tiles < kMaxTiles;
  if (whole) {
    char* ws = static_cast<char*>(workspace);
    if (p.x || p.w) {
      PadArgs pa{{a.x, a.w}, {reinterpret_cast<int8_t*>(ws), reinterpret_cast<int8_t*>(ws + p.x_bytes)},
                 {p.x ? g.rows : 0, p.w ? g.n : 0}, {g.x_row, g.w_row}, (int32_t)g.k, (int32_t)(p.row / 16)};
      const int64_t pieces = (pa.rows[0] + pa.rows[1]) * pa.pieces;
      const dim3 grid((unsigned)std::min<int64_t>((pieces + kThreads - 1) / kThreads, 8192));
      hipLaunchKernelGGL(int8_pad_kernel, grid, dim3(kThreads), 0, stream, pa);
      if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
      if (p.x) a.x = pa.to[0];
      if (p.w) a.w = pa.to[1];
      a.k = a.part_k = (int32_t)t.k;
      a.x_row = t.x_row;
      a.w_row = t.w_row;
    }
    return run_whole(t, a, ws + p.x_bytes + p.w_bytes, stream);
  }
  if (few_rows(g)) return run_few<false>(g, a, stream);
  if (tiles >= kMaxTiles) return hipErrorInvalidConfiguration;
  return by_type(g.out_dtype, [&](auto tag) {
    using T = decltype(tag);
    // up to two 32 x 32 tiles a CU, or 64 x 64 ones (333 x 777 x 1001: 11 us, 15.4;
    // 500 x 1000 x 1001: 12.8, 14.8; 576 x 1000 x 1001: 17.2, 14.8)
    if (tiles <= 128) {
      const dim3 grid((unsigned)tiles_of(g, 32, 32));
      hipLaunchKernelGGL((int8_small_kernel<T, 8>), grid, dim3(512), 0, stream, a);
      return hipGetLastError();
    }
    hipLaunchKernelGGL((int8_any_kernel<T>), dim3((unsigned)tiles), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

}  // namespace oops
