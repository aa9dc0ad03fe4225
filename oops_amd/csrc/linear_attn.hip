// Linear attention with a decay for each head:
//
//   S_t = l S_(t-1) + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log_decay)
//
// and its gradients, all of them one walk (LinearWalk, layer_kernels.h) over
// other operands:
//   o  = walk(q, k, v)       dq = walk(do, v, k) on the transposed state
//   dk = walk(v, do, q) and dv = walk(k, q, do) from the end, where the state
//   R_t = l R_(t+1) + scale q_t^T do_t is the gradient of S_t.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attn_common.h"
#include "attn_fast_common.h"
#include "layer_kernels.h"

namespace oops {
namespace {

constexpr int kThreads = 256;

// exp(log_decay n) for n >= 0: n = 0 gives 1 for every decay, -inf included (a NaN stays one)
__device__ __forceinline__ float log2_decay(float log_decay) {
  const float l2 = log_decay * kLog2e;
  return l2 < -1e30f ? -1e30f : l2;
}
__device__ __forceinline__ float decay_power(float l2, float n) { return exp2f(l2 * n); }

__device__ __forceinline__ int64_t walk_length(const LinearWalk& w, int64_t b) {
  if (!w.lengths) return w.length;
  const int64_t n = w.lengths_i64 ? static_cast<const int64_t*>(w.lengths)[b]
                                  : (int64_t) static_cast<const int32_t*>(w.lengths)[b];
  return n < 0 ? 0 : n > w.length ? w.length : n;
}

// x, of which the compiler no longer knows where it comes from: what is computed from it is computed here, and not
// kept in registers over a loop because an expression before or in the loop looks the same
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// ---------------------------------------------------------------- bfloat16, in chunks
//
// With the state kept one decay ahead in walks from the end (first = 1, else
// 0), a chunk of m <= 64 tokens that starts from state S is
//   out_i = scale sum_(j <= i) l^(i-j) (a_i . b_j) c_j + so l^(i+1-first) a_i S
//   S    := l^m S + sum_j u l^(m-1-j+first) b_j^T c_j
// (so, u) = (scale, 1), or (1, scale) from the end: four products on the
// matrix units for 2 C D + 4 D^2 operations a token instead of the
// recurrence's vector work.  A workgroup walks a segment of a (batch, head)
// with the state in float32 accumulators, 32 columns a wave; the next chunk's
// rows are loaded to registers meanwhile.  Few heads are split into segments:
// walk_chunks_kernel<.., false> makes each segment's state from zero,
// walk_scan_kernel joins them, then every segment starts from its own state.
//
// Measured, 4 x 16 heads x 4096 x 128: 47 us the segments' states, 15 the scan,
// 71 to 85 the outputs and each gradient (the matrix units busy 20% and 17% of
// it): bound by the loads' latency and the LDS exchanges between a chunk's four
// products.  Three workgroups a CU on single direct-to-LDS buffers took 95,
// outputs written in whole rows through LDS 87.
//
// Operand layouts: accumulators hold [row of the state or value][lane], lane =
// value column (state) or token (weights, outputs), so weights and state are
// turned into the next product's operand in registers; the state's rows are
// taken in the order that makes that operand's k run 8 half + 0..7, as a
// 16-byte read of a row gives it (bits 2 and 3 of the row index swapped).
//
// Roundings to bfloat16: the weights scale l^(i-j) (a_i . b_j) and the state
// where they are read by the second products, once each (different terms of
// the output, 2^-8 of each at most, as in softmax attention).  The update's
// operand u l^n c is split into three bfloat16 terms, which hold its float32
// value, where the state is kept (the last state is a float32 result), and into
// two (2^-16) where it only goes into the segment's own outputs: walks in
// several segments have their last state from walk_scan_kernel.
constexpr int kChunk = 64;

struct ChunkArgs {
  LinearWalk w;
  float* starts;       // [batch * heads][segs][state]: segments' own states, then the states they start from
  int64_t seg_tokens;  // whole chunks
  int32_t segs;
};

// byte of a state's element, or an offset past every resource (reads as 0, is not written)
__device__ __forceinline__ uint32_t state_byte(const LinearWalk& w, int row, int col) {
  const int rs = w.state_by_cols ? 1 : w.cols, cs = w.state_by_cols ? w.rows : 1;
  return ((row < w.rows) & (col < w.cols)) ? (uint32_t)(row * rs + col * cs) * 4 : fast::kOut;
}
__device__ __forceinline__ int64_t token_of(const LinearWalk& w, int64_t p, int64_t n) {
  return w.from_end && p < n ? n - 1 - p : p;
}

// 16-byte slot of a tile row, XORed into the chunk index: rows of 256, 128 or
// 64 bytes put the 16 rows of a read phase into distinct slots
template <int D>
__device__ __forceinline__ int row_swizzle(int row) {
  return D == 128 ? row & 15 : D == 64 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// Bits 15 and 31 of the result are set where a 16-bit half of u has its exponent all ones (an infinity or NaN): the
// exponent's bits alone, plus its lowest one, carry out of it.
__device__ __forceinline__ uint32_t non_finite(uint4 u) {
  constexpr uint32_t kExp = 0x7F807F80u, kOne = 0x00800080u;
  return ((u.x & kExp) + kOne) | ((u.y & kExp) + kOne) | ((u.z & kExp) + kOne) | ((u.w & kExp) + kOne);
}

// eight floats in pairs (one conversion instruction each)
__device__ __forceinline__ bf16x8 to_bf16x8(const float (&x)[8]) {
  return __builtin_bit_cast(bf16x8, make_uint4(fast::pack2<__bf16>(x[0], x[1]), fast::pack2<__bf16>(x[2], x[3]),
                                               fast::pack2<__bf16>(x[4], x[5]), fast::pack2<__bf16>(x[6], x[7])));
}

template <int D, bool VEC, bool MAIN, int kTerms>
__global__ __launch_bounds__(2 * D, MAIN || D == 128 ? 2 : 4) void walk_chunks_kernel(ChunkArgs ca) {
  using T = __bf16;
  using Frag = bf16x8;
  constexpr int NT = 2 * D, NW = D / 32;      // threads, waves: 32 columns each
  constexpr int RB = 2 * D, CPR = D / 8;      // bytes and 16-byte chunks of a tile row
  constexpr int NL = kChunk * CPR / NT;       // 16-byte loads a thread and tile
  __shared__ __align__(16) char tb[kChunk * RB], tc[kChunk * RB], ta[MAIN ? kChunk * RB : 16];
  __shared__ __align__(16) char tp[MAIN ? kChunk * kChunk * 2 : 16];  // weights [token i][token j]
  __shared__ __align__(16) float tw[kChunk];                          // decays of the update
  __shared__ float td[MAIN ? 2 * kChunk : 1];                         // scale l^(n - 64), 0 before 64
  __shared__ int bad[2];                                              // c holds an infinity or NaN
  const LinearWalk& w = ca.w;
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t bh = (int64_t)blockIdx.x / ca.segs;
  const int seg = (int)((int64_t)blockIdx.x % ca.segs);
  if (!MAIN && seg == ca.segs - 1 && !w.final_state) return;  // (no segment starts from its state)
  const int64_t b = bh / w.heads;
  const int h = (int)(bh % w.heads);
  const int64_t n = walk_length(w, b);
  const int64_t s0 = seg * ca.seg_tokens;
  const int64_t s1 = s0 + ca.seg_tokens < n ? s0 + ca.seg_tokens : n;  // (s1 <= s0: nothing to walk)
  const int first = w.from_end ? 1 : 0;
  const float l2 = log2_decay(w.log_decay[h]);
  const float up = first ? w.scale : 1.f, so = first ? 1.f : w.scale;
  const T* a = static_cast<const T*>(w.a) + b * w.a_stride[0] + h * w.a_stride[1];
  const T* bp = static_cast<const T*>(w.b) + b * w.b_stride[0] + h * w.b_stride[1];
  const T* c = static_cast<const T*>(w.c) + b * w.c_stride[0] + h * w.c_stride[1];

  // the state: tile rt, register r is row 32 rt + 16 (r / 8) + 8 g + r % 8, column 32 wave + l
  f32x16 S[NW];
  const int col = 32 * wave + l;
  const int64_t state_size = (int64_t)w.rows * w.cols;
  {
    const float* from = nullptr;
    if (MAIN) from = ca.segs > 1 ? ca.starts + (bh * ca.segs + seg) * state_size
                                 : w.initial ? w.initial + bh * state_size : nullptr;
    const auto rsrc = make_rsrc(from, from ? (uint32_t)state_size * 4 : 0u);
#pragma unroll
    for (int rt = 0; rt < NW; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        S[rt][r] = __builtin_bit_cast(
            float, __builtin_amdgcn_raw_buffer_load_b32(
                       rsrc, state_byte(w, 32 * rt + 16 * (r >> 3) + 8 * g + (r & 7), col), 0, 0));
  }

  // lane addresses: rows as they are (16 bytes of row l), and transposed (4 x 4 blocks, see lds_read_tr4)
  const int nat = l * RB + ((g ^ row_swizzle<D>(l)) << 4);
  int tr_c, tr_b;
  {
    const int j = lane & 15, grp = lane >> 4;
    const int row = ((grp >> 1) << 2) + (j >> 2);
    auto at = [&](int cc) { return row * RB + (((cc >> 3) ^ row_swizzle<D>(row)) << 4) + (cc & 7) * 2; };
    tr_c = at(((grp & 1) << 4) + ((j & 3) << 2));
    tr_b = at(((grp & 1) << 4) + ((j & 1) << 3) + ((j & 2) << 1));
  }
  auto rows_frag = [&](const char* t, int tile, int kb) {
    return __builtin_bit_cast(Frag, *reinterpret_cast<const uint4*>(t + tile * 32 * RB + (nat ^ (kb << 5))));
  };
  auto tr_frag = [&](const char* t, int lane_at, int kb, int ct) {
    const int lo = (lane_at ^ (ct << 6)) + kb * 16 * RB, hi = (lane_at ^ (ct << 6) ^ (RB / 2)) + (kb * 16 + 8) * RB;
    const s16x4 x = lds_read_tr4(t + lo), y = lds_read_tr4(t + hi);
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    return __builtin_bit_cast(Frag, v);
  };
  const int pl = l * 128 + ((g ^ ((l >> 1) & 7)) << 4);

  float fo[2];
  if (MAIN) {
    for (int i = tid; i < 2 * kChunk; i += NT) td[i] = i < kChunk ? 0.f : w.scale * decay_power(l2, (float)(i - kChunk));
#pragma unroll
    for (int it = 0; it < 2; ++it) fo[it] = so * decay_power(l2, (float)(32 * it + l + 1 - first));
  }

  // rows row0, row0 + kRows, ..: 16 bytes a lane, zeros behind the segment.  A chunk's resource starts at its lowest
  // row, whichever way the walk goes.
  constexpr int kRows = NT / CPR;
  const int row0 = tid / CPR, cc0 = tid % CPR * 8;
  uint4 ra[NL], rb[NL], rc[NL];
  auto fetch = [&](uint4(&reg)[NL], const T* base, int64_t stride, int width, int64_t p0, int left) {
    if constexpr (VEC) {
      const T* lowest = base + (first ? n - kChunk - p0 : p0) * stride;
      const auto rsrc = make_rsrc(lowest, 0x7FFFFFFFu);
      const int bytes = (int)stride * 2;
      // (row r of a walk from the end is kChunk - 1 - r rows up: kRows - 1 - row0, and whole steps of kRows)
      const uint32_t off = cc0 < width ? (uint32_t)((first ? kRows - 1 - row0 : row0) * bytes + cc0 * 2) : fast::kOut;
#pragma unroll
      for (int i = 0; i < NL; ++i)
        reg[i] = fast::buffer_load16_s(rsrc, row0 + i * kRows < left ? off : fast::kOut,
                                       (uint32_t)((first ? NL - 1 - i : i) * kRows * bytes));
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int row = row0 + i * kRows;
        reg[i] = row < left ? load16(base + token_of(w, p0 + row, n) * stride, cc0, width, false) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto fetch_all = [&](int64_t p0) {
    const int left = s1 - p0 < kChunk ? (int)(s1 - p0) : kChunk;
    if (MAIN) fetch(ra, a, w.a_stride[2], w.rows, p0, left);
    fetch(rb, bp, w.b_stride[2], w.rows, p0, left);
    fetch(rc, c, w.c_stride[2], w.cols, p0, left);
  };
  if (s0 < s1) fetch_all(s0);
  if (tid < 2) bad[tid] = 0;

  int turn = 0;
  for (int64_t p0 = s0; p0 < s1; p0 += kChunk, turn ^= 1) {
    const int m = (int)(s1 - p0 < kChunk ? s1 - p0 : kChunk);
    lds_barrier();  // the tiles have been read
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int idx = tid + i * NT, row = idx / CPR;
      const int at = row * RB + ((idx % CPR ^ row_swizzle<D>(row)) << 4);
      if (MAIN) *reinterpret_cast<uint4*>(ta + at) = ra[i];
      *reinterpret_cast<uint4*>(tb + at) = rb[i];
      *reinterpret_cast<uint4*>(tc + at) = rc[i];
      if (MAIN) odd |= non_finite(rc[i]);
    }
    if (MAIN && (odd & 0x80008000u)) bad[turn] = 1;
    if (MAIN && tid == 0) bad[turn ^ 1] = 0;
    if (tid < kChunk) tw[tid] = tid < m ? up * decay_power(l2, (float)(m - 1 - tid + first)) : 0.f;
    lds_barrier();
    if (p0 + kChunk < s1) fetch_all(p0 + kChunk);

    Frag cf[4];
    if constexpr (MAIN) {
      // weights: [j][i] accumulators, lane i; waves take the tiles (0,0), (1,0), (1,1) in turn
      constexpr int kTiles = (3 + NW - 1) / NW;
#pragma unroll
      for (int q = 0; q < kTiles; ++q) {
        const int tile = wave + q * NW;
        if (tile < 3) {
          const int it = tile > 0, jt = tile > 1;
          f32x16 acc = {};
#pragma unroll
          for (int kb = 0; kb < D / 16; ++kb)
            acc = Elem<T>::mma(rows_frag(tb, jt, kb), rows_frag(ta, it, kb), acc);
          // (a later token's product may be infinite: masked by its bits)
          const int last = opaque(32 * (it - jt) + l);
          const float* f = td + (kChunk + last) - 4 * g;
          float x[2][8];
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int later = (last - 4 * g - kappa(0, r)) >> 31;  // all ones where j > i
            x[r / 8][r % 8] = __builtin_bit_cast(float, __builtin_bit_cast(int, acc[r] * f[-kappa(0, r)]) & ~later);
          }
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
            *reinterpret_cast<Frag*>(tp + it * 32 * 128 + (pl ^ ((jt * 4 + kb * 2) << 4))) = to_bf16x8(x[kb]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (the products' operands are not all held at once)
      // from the state: [value][token] accumulators, lane = token
      f32x16 o[2] = {};
#pragma unroll
      for (int rt = 0; rt < NW; ++rt)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = S[rt][8 * kb + j];
          const Frag sf = to_bf16x8(x);
#pragma unroll
          for (int it = 0; it < 2; ++it) o[it] = Elem<T>::mma(sf, rows_frag(ta, it, 2 * rt + kb), o[it]);
        }
#pragma unroll
      for (int it = 0; it < 2; ++it)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[it][r] *= fo[it];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) cf[kb] = tr_frag(tc, tr_c, kb, wave);
      lds_barrier();
      if (!bad[turn]) {
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int kb = 0; kb < 2 + 2 * it; ++kb) {
            const Frag pfr = __builtin_bit_cast(
                Frag, *reinterpret_cast<const uint4*>(tp + it * 32 * 128 + (pl ^ ((kb * 2) << 4))));
            o[it] = Elem<T>::mma(cf[kb], pfr, o[it]);
          }
      } else {
        // an infinity or NaN among the values: the products that the mask leaves out (0 times it is NaN) must not
        // be made, so that no token sees a later one's
        const int l_ = opaque(l), g_ = opaque(g);
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll 1
          for (int j = 0; j <= 32 * it + l_; ++j) {
            const int jj = j & 31, r = ((jj >> 3) << 2) | (jj & 3);
            const int chunk = (j >> 5) * 4 + (r >> 3) * 2 + ((jj >> 2) & 1);
            const int row = 32 * it + l_;
            const float p = (float)*reinterpret_cast<const T*>(tp + row * 128 + ((chunk ^ ((l_ >> 1) & 7)) << 4) + (r & 7) * 2);
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              const int cc = 32 * wave + kappa(g_, q);
              const float v = (float)*reinterpret_cast<const T*>(tc + j * RB + (((cc >> 3) ^ row_swizzle<D>(j)) << 4) + (cc & 7) * 2);
              o[it][q] = __builtin_fmaf(p, v, o[it][q]);
            }
          }
      }
      if (w.out) {
        T* base = static_cast<T*>(w.out) + b * w.out_stride[0] + h * w.out_stride[1];
        if constexpr (VEC) {
          const auto rsrc = make_rsrc(base + (first ? n - kChunk - p0 : p0) * w.out_stride[2], 0x7FFFFFFFu);
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            uint32_t pk[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) pk[q] = fast::pack2<T>(o[it][2 * q], o[it][2 * q + 1]);
            uint4 lo, hi;
            fast::trade16(pk, lo, hi);  // this lane: its token's columns cc .. cc+7 and cc+8 .. cc+15
            const int i = 32 * it + l, cc = 32 * wave + 16 * g;
            const uint32_t at = (uint32_t)((first ? kChunk - 1 - i : i) * (int)w.out_stride[2] + cc) * 2;
            buffer_store16(rsrc, i < m && cc < w.cols ? at : fast::kOut, lo);
            buffer_store16(rsrc, i < m && cc + 8 < w.cols ? at + 16 : fast::kOut, hi);
          }
        } else {
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            const int i = 32 * it + l;
            T* row = base + token_of(w, i < m ? p0 + i : p0, n) * w.out_stride[2];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int cc = 32 * wave + kappa(g, r);
              if (i < m && cc < w.cols) row[cc] = (T)o[it][r];
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) cf[kb] = tr_frag(tc, tr_c, kb, wave);
    }
    __builtin_amdgcn_sched_barrier(0);
    // the state's update
    const float lm = decay_power(l2, (float)m);
    // An infinity is its own first term: its difference with that is NaN, so a lane that holds one (or a NaN) among
    // its column's tokens has no further terms (4 x 16 heads x 4096 x 128 in training: 373 us, without this 368).
    uint32_t keep = ~0u;
    if (!MAIN || bad[turn]) {
      uint32_t odd = 0;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) odd |= non_finite(__builtin_bit_cast(uint4, cf[kb]));
      keep = odd & 0x80008000u ? 0u : ~0u;
    }
#pragma unroll
    for (int rt = 0; rt < NW; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[rt][r] *= lm;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      // tokens 16 kb + kappa(g, 0..7) of this lane's column, decayed, in kTerms terms
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(tw + 16 * kb + 4 * g);
      const f32x4 w1 = *reinterpret_cast<const f32x4*>(tw + 16 * kb + 8 + 4 * g);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (float)cf[kb][j] * (j < 4 ? w0[j & 3] : w1[j & 3]);
      Frag part[kTerms];
#pragma unroll
      for (int q = 0; q < kTerms; ++q) {
        part[q] = to_bf16x8(x);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] -= (float)part[q][j];
        if (q > 0) {
          uint4 u = __builtin_bit_cast(uint4, part[q]);
          u.x &= keep, u.y &= keep, u.z &= keep, u.w &= keep;
          part[q] = __builtin_bit_cast(Frag, u);
        }
      }
#pragma unroll
      for (int rt = 0; rt < NW; ++rt) {
        const Frag bf = tr_frag(tb, tr_b, kb, rt);
#pragma unroll
        for (int q = 0; q < kTerms; ++q) S[rt] = Elem<T>::mma(bf, part[q], S[rt]);
      }
    }
  }

  // rows behind the sequence are zero
  if (MAIN && w.out) {
    int64_t e1 = s0 + ca.seg_tokens;
    if (e1 > w.length || seg == ca.segs - 1) e1 = w.length;
    T* out = static_cast<T*>(w.out) + b * w.out_stride[0] + h * w.out_stride[1];
    const int64_t z0 = s0 > n ? s0 : n;
    for (int64_t i = tid; i < (e1 - z0) * w.cols; i += NT) out[(z0 + i / w.cols) * w.out_stride[2] + i % w.cols] = (T)0.f;
  }
  // the state behind the segment, or behind the sequence
  float* to = nullptr;
  if (!MAIN) to = ca.starts + (bh * ca.segs + seg) * state_size;
  else if (kTerms == 3 && w.final_state) to = w.final_state + bh * state_size;
  if (to) {
    const int g_ = opaque(g), col_ = opaque(col);
    const auto rsrc = make_rsrc(to, (uint32_t)state_size * 4);
#pragma unroll
    for (int rt = 0; rt < NW; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        buffer_store4(rsrc, state_byte(w, 32 * rt + 16 * (r >> 3) + 8 * g_ + (r & 7), col_), S[rt][r]);
  }
}

// ---------------------------------------------------------------- float32 and float16, in chunks
//
// The same chunks on the float32 matrix units (32x32x2 MFMA, products and
// sums in float32), float16 operands widened on their way into LDS: the
// unnormalised weights and states of linear attention pass float16's range
// where its outputs do not.  Chunks of 32 tokens: a wave makes the whole
// 32 x 32 weight tile for its 32 columns itself and keeps it in registers (an
// accumulator register is the next MFMA's k-operand as it is), so there is no
// exchange between waves: 13% more products than sharing 64-token tiles, no
// barrier between them.  64 heads x 2048 x 128 float32: 70 us the segments'
// states, 14 the scan, 159 the outputs, the matrix units busy 32% and 60% of it
// (their rate is a sixteenth of bfloat16's; the rest is one wave a SIMD waiting
// for its own chain of products; two workgroups a CU spill: 289 us, not 229).
// Small calls are bound by that latency alone: 48 x 777 x 64 in float16 gives
// 864 waves for 1024 SIMDs, busy 5% and 13%.
constexpr int kExactChunk = 32;

template <typename T, int D, bool VEC, bool MAIN>
__global__ __launch_bounds__(2 * D, D == 32 ? 2 : 1) void walk_exact_kernel(ChunkArgs ca) {
  constexpr int NT = 2 * D, NW = D / 32;
  constexpr int VE = 16 / sizeof(T), CPR = D / VE;           // elements of a load, loads of a row
  constexpr int NL = kExactChunk * CPR / NT, kRows = NT / CPR;  // loads a thread and tile, rows of one pass
  constexpr int C4 = D / 4;                                  // float4 slots of a tile row
  __shared__ f32x4 tb[kExactChunk * C4], tc[kExactChunk * C4], ta[MAIN ? kExactChunk * C4 : 1];
  __shared__ float tw[kExactChunk], td[MAIN ? 2 * kExactChunk : 1];  // decays of the update; scale l^(n - 32), 0 before 32
  const LinearWalk& w = ca.w;
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t bh = (int64_t)blockIdx.x / ca.segs;
  const int seg = (int)((int64_t)blockIdx.x % ca.segs);
  if (!MAIN && seg == ca.segs - 1) return;  // (no segment starts from its state)
  const int64_t b = bh / w.heads;
  const int h = (int)(bh % w.heads);
  const int64_t n = walk_length(w, b);
  const int64_t s0 = seg * ca.seg_tokens;
  const int64_t s1 = s0 + ca.seg_tokens < n ? s0 + ca.seg_tokens : n;
  const int first = w.from_end ? 1 : 0;
  const float l2 = log2_decay(w.log_decay[h]);
  const float up = first ? w.scale : 1.f, so = first ? 1.f : w.scale;
  const T* a = static_cast<const T*>(w.a) + b * w.a_stride[0] + h * w.a_stride[1];
  const T* bp = static_cast<const T*>(w.b) + b * w.b_stride[0] + h * w.b_stride[1];
  const T* c = static_cast<const T*>(w.c) + b * w.c_stride[0] + h * w.c_stride[1];

  // the state: tile rt, register r is row 32 rt + kappa(g, r), column 32 wave + l
  f32x16 S[NW];
  const int col = 32 * wave + l;
  const int64_t state_size = (int64_t)w.rows * w.cols;
  {
    const float* from = nullptr;
    if (MAIN) from = ca.segs > 1 ? ca.starts + (bh * ca.segs + seg) * state_size
                                 : w.initial ? w.initial + bh * state_size : nullptr;
    const auto rsrc = make_rsrc(from, from ? (uint32_t)state_size * 4 : 0u);
#pragma unroll
    for (int rt = 0; rt < NW; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        S[rt][r] = __builtin_bit_cast(
            float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, state_byte(w, 32 * rt + kappa(g, r), col), 0, 0));
  }

  // float4 slot of a row: slots are XORed with the row, so that a read phase's rows use distinct banks
  auto slot = [](int row, int c4) { return row * C4 + (c4 ^ (row & (C4 < 16 ? C4 - 1 : 15))); };
  auto value = [&](const f32x4* t, int row, int cc) {
    return reinterpret_cast<const float*>(t)[slot(row, cc >> 2) * 4 + (cc & 3)];
  };

  const int row0 = tid / CPR, cc0 = tid % CPR * VE;
  uint4 ra[NL], rb[NL], rc[NL];
  auto fetch = [&](uint4(&reg)[NL], const T* base, int64_t stride, int width, int64_t p0, int left) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = row0 + i * kRows;
      reg[i] = make_uint4(0, 0, 0, 0);
      if (row < left) {
        const T* q = base + token_of(w, p0 + row, n) * stride;
        if constexpr (VEC) {
          if (cc0 < width) reg[i] = *reinterpret_cast<const uint4*>(q + cc0);
        } else {
          reg[i] = load16(q, cc0, width, false);
        }
      }
    }
  };
  auto fetch_all = [&](int64_t p0) {
    const int left = s1 - p0 < kExactChunk ? (int)(s1 - p0) : kExactChunk;
    if (MAIN) fetch(ra, a, w.a_stride[2], w.rows, p0, left);
    fetch(rb, bp, w.b_stride[2], w.rows, p0, left);
    fetch(rc, c, w.c_stride[2], w.cols, p0, left);
  };
  auto put = [&](f32x4* t, const uint4(&reg)[NL]) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const T* e = reinterpret_cast<const T*>(&reg[i]);
#pragma unroll
      for (int q = 0; q < VE / 4; ++q)
        t[slot(row0 + i * kRows, cc0 / 4 + q)] =
            f32x4{(float)e[4 * q], (float)e[4 * q + 1], (float)e[4 * q + 2], (float)e[4 * q + 3]};
    }
  };
  if (s0 < s1) fetch_all(s0);
  if (MAIN && tid < 2 * kExactChunk)
    td[tid] = tid < kExactChunk ? 0.f : w.scale * decay_power(l2, (float)(tid - kExactChunk));
  const float fo = so * decay_power(l2, (float)(l + 1 - first));

  for (int64_t p0 = s0; p0 < s1; p0 += kExactChunk) {
    const int m = (int)(s1 - p0 < kExactChunk ? s1 - p0 : kExactChunk);
    lds_barrier();  // the tiles have been read
    if (MAIN) put(ta, ra);
    put(tb, rb);
    put(tc, rc);
    if (tid < kExactChunk) tw[tid] = tid < m ? up * decay_power(l2, (float)(m - 1 - tid + first)) : 0.f;
    lds_barrier();
    if (p0 + kExactChunk < s1) fetch_all(p0 + kExactChunk);

    float cv[16];  // this lane's column of tokens kappa(g, r)
#pragma unroll
    for (int r = 0; r < 16; ++r) cv[r] = value(tc, kappa(g, r), col);
    if constexpr (MAIN) {
      // weights [j][i] and outputs from the state [value][i], lane i = l; k-slot g of MFMA (q, t) is column 8 q + 4 g + t
      f32x16 p = {}, o = {};
#pragma unroll
      for (int q = 0; q < D / 8; ++q) {
        const f32x4 av = ta[slot(l, 2 * q + g)], bv = tb[slot(l, 2 * q + g)];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          p = Elem<float>::mma(bv[t], av[t], p);
          o = Elem<float>::mma(S[q / 4][4 * (q % 4) + t], av[t], o);
        }
      }
      const float* f = td + (kExactChunk + l) - 4 * g;
      bool odd = false;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        // (a later token's product may be infinite: masked by its bits)
        const int later = (l - 4 * g - kappa(0, r)) >> 31;
        p[r] = __builtin_bit_cast(float, __builtin_bit_cast(int, p[r] * f[-kappa(0, r)]) & ~later);
        o[r] *= fo;
        odd |= (__builtin_bit_cast(uint32_t, cv[r]) & 0x7F800000u) == 0x7F800000u;
      }
      if (!__any(odd)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) o = Elem<float>::mma(cv[r], p[r], o);
      } else {
        // an infinity or NaN among the values: the products that the mask leaves out (0 times it is NaN) must not be
        // made, so that no token sees a later one's
        const int l_ = opaque(l), g_ = opaque(g);
#pragma unroll 1
        for (int j = 0; j <= l_; ++j) {
          float x = 0.f;
#pragma unroll 1
          for (int d = 0; d < w.rows; ++d) x = __builtin_fmaf(value(ta, l_, d), value(tb, j, d), x);
          x *= td[kExactChunk + l_ - j];
#pragma unroll
          for (int r = 0; r < 16; ++r) o[r] = __builtin_fmaf(x, value(tc, j, 32 * wave + kappa(g_, r)), o[r]);
        }
      }
      if (w.out && l < m) {
        T* row = static_cast<T*>(w.out) + b * w.out_stride[0] + h * w.out_stride[1] +
                 token_of(w, p0 + l, n) * w.out_stride[2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int cc = 32 * wave + 8 * q + 4 * g;
          if constexpr (VEC) {
            if (cc < w.cols) fast::store4(row, cc, o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
          } else {
#pragma unroll
            for (int t = 0; t < 4; ++t)
              if (cc + t < w.cols) row[cc + t] = (T)o[4 * q + t];
          }
        }
      }
    }
    // the state's update: k-slot g of MFMA r is token kappa(g, r)
    const float lm = decay_power(l2, (float)m);
#pragma unroll
    for (int r = 0; r < 16; ++r) cv[r] *= tw[kappa(g, r)];
#pragma unroll
    for (int rt = 0; rt < NW; ++rt) {
#pragma unroll
      for (int r = 0; r < 16; ++r) S[rt][r] *= lm;
#pragma unroll
      for (int r = 0; r < 16; ++r) S[rt] = Elem<float>::mma(value(tb, kappa(g, r), 32 * rt + l), cv[r], S[rt]);
    }
  }

  // rows behind the sequence are zero
  if (MAIN && w.out) {
    int64_t e1 = s0 + ca.seg_tokens;
    if (e1 > w.length || seg == ca.segs - 1) e1 = w.length;
    T* out = static_cast<T*>(w.out) + b * w.out_stride[0] + h * w.out_stride[1];
    const int64_t z0 = s0 > n ? s0 : n;
    for (int64_t i = tid; i < (e1 - z0) * w.cols; i += NT) out[(z0 + i / w.cols) * w.out_stride[2] + i % w.cols] = (T)0.f;
  }
  float* to = nullptr;
  if (!MAIN) to = ca.starts + (bh * ca.segs + seg) * state_size;
  else if (w.final_state && (n > 0 ? s0 < n && n <= s0 + ca.seg_tokens : seg == 0)) to = w.final_state + bh * state_size;
  if (to) {
    const int g_ = opaque(g), col_ = opaque(col);
    const auto rsrc = make_rsrc(to, (uint32_t)state_size * 4);
#pragma unroll
    for (int rt = 0; rt < NW; ++rt)
#pragma unroll
      for (int r = 0; r < 16; ++r) buffer_store4(rsrc, state_byte(w, 32 * rt + kappa(g_, r), col_), S[rt][r]);
  }
}

// Segments' own states to the states they start from, in place and in order:
// start_0 = initial, start_(s+1) = l^(tokens of s) start_s + own_s; the last
// state, where it is wanted here.  Bound by the states' bytes, read and written
// once (64 heads x 8 segments x 128 x 128: 15 us, 4.5 TB/s).
__global__ __launch_bounds__(kThreads) void walk_scan_kernel(ChunkArgs ca, float* last) {
  const LinearWalk& w = ca.w;
  const int64_t size = (int64_t)w.rows * w.cols;
  const int64_t bh = blockIdx.y, at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= size) return;
  const int64_t n = walk_length(w, bh / w.heads);
  const float l2 = log2_decay(w.log_decay[bh % w.heads]);
  float* own = ca.starts + bh * ca.segs * size + at;
  float cur = w.initial ? w.initial[bh * size + at] : 0.f;
  const float whole = decay_power(l2, (float)ca.seg_tokens);
  constexpr int U = 8;
  for (int s0 = 0; s0 < ca.segs; s0 += U) {
    float x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = s0 + i < ca.segs - (last ? 0 : 1) ? own[(s0 + i) * size] : 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (s0 + i >= ca.segs) break;
      own[(s0 + i) * size] = cur;
      const int64_t left = n - (s0 + i) * ca.seg_tokens;
      const float lm = left >= ca.seg_tokens ? whole : left > 0 ? decay_power(l2, (float)left) : 1.f;
      cur = __builtin_fmaf(cur, lm, x[i]);
    }
  }
  if (last) last[bh * size + at] = cur;
}

// ---------------------------------------------------------------- one token
//
// The state crosses HBM once each way (8 bytes an element against 6
// operations): a workgroup streams the rows of a (batch, head)'s columns, VW
// columns and up to kStepRows rows in flight a lane.  Few heads are split over
// workgroups by columns, 32 each.  256 x 32 heads x 128 x 128: 211 us, 5.1 TB/s;
// 16 heads: 4.5 us, a launch's own time.
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

namespace {

// Segments of a walk.  They cost its state's traffic and half its products once
// more, so walks that give most CUs a workgroup go in one (256 heads x 512
// tokens x 128: 42 us, in two segments 91).  Others get segments of at least
// four chunks until there are eight waves a CU, or of two while there are not
// four (16 x 1024 x 128: 34 us, with four chunks 42; 8 x 8192 x 128: 57, 51).
// Below that, single chunks: of 32 tokens in the float32 products, whose time is
// the larger part (training 2 x 300 x 64 in float16 87 us, 192 with segments of
// two 64-token chunks; 48 x 777 x 64 123, 147), of 64 in bfloat16 while there are
// not two waves a CU (2 x 300 x 64 63, 80; 64 x 512 x 64 70, without them 66).
// (At most 256 segments a head are made so: more single chunks are not worth
// their scan, 32768 x 64: 154, 107.  Segments of several chunks have no limit.)
void plan_segments(int dtype, const LinearWalk& w, ChunkArgs& ca) {
  const bool exact = dtype != OOPS_BF16;
  const int64_t tokens = exact ? kExactChunk : kChunk, unit = kChunk / tokens;
  const int64_t chunks = std::max<int64_t>(1, (w.length + tokens - 1) / tokens), bh = w.batch * w.heads;
  const int widest = std::max(w.rows, w.cols);
  const int64_t wide = widest <= 32 ? 4 : widest <= 64 ? 2 : 1;  // workgroups of four waves' worth
  int64_t segs = 1;
  if (bh < 192 * wide) {
    auto split = [&](int64_t target, int64_t least) {
      segs = std::max(segs, std::min((target * wide + bh - 1) / bh, (chunks + least - 1) / least));
    };
    split(512, 4 * unit);
    split(256, 2 * unit);
    if (segs < 256 && (exact || chunks >= 4))
      split(std::min<int64_t>(exact ? 256 : 128, 256 * bh / wide), 1);
  }
  const int64_t per = (chunks + segs - 1) / segs;
  ca.segs = (int32_t)((chunks + per - 1) / per);
  ca.seg_tokens = per * tokens;
}

// rows read and written 16 bytes at a time, whose chunks span less than 2 GiB
bool rows16(const void* p, const int64_t (&stride)[3], int width, int element) {
  const int v = 16 / element;
  return width % v == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride[0] % v == 0 && stride[1] % v == 0 &&
         stride[2] % v == 0 && stride[2] < (int64_t(1) << 31) / (4 * kChunk) - 128;
}

template <typename T, int D, bool VEC, bool MAIN>
void launch_chunks(const ChunkArgs& ca, dim3 grid, hipStream_t stream) {
  if constexpr (!std::is_same_v<T, __bf16>)
    hipLaunchKernelGGL((walk_exact_kernel<T, D, VEC, MAIN>), grid, dim3(2 * D), 0, stream, ca);
  else if (MAIN && ca.segs > 1)
    hipLaunchKernelGGL((walk_chunks_kernel<D, VEC, MAIN, MAIN ? 2 : 3>), grid, dim3(2 * D), 0, stream, ca);
  else
    hipLaunchKernelGGL((walk_chunks_kernel<D, VEC, MAIN, 3>), grid, dim3(2 * D), 0, stream, ca);
}

template <typename T, int D, bool VEC>
hipError_t run_chunks(const ChunkArgs& ca, bool starts, hipStream_t stream) {
  const LinearWalk& w = ca.w;
  const unsigned bh = (unsigned)(w.batch * w.heads);
  const dim3 grid(bh * (unsigned)ca.segs);
  if (starts) {
    launch_chunks<T, D, VEC, false>(ca, grid, stream);
    hipLaunchKernelGGL(walk_scan_kernel, dim3((unsigned)((w.rows * w.cols + kThreads - 1) / kThreads), bh),
                       dim3(kThreads), 0, stream, ca, std::is_same_v<T, __bf16> ? w.final_state : nullptr);
  } else if (w.out || ca.segs == 1 || !std::is_same_v<T, __bf16>) {
    launch_chunks<T, D, VEC, true>(ca, grid, stream);
  }
  return hipGetLastError();
}

// The walk itself (with the states its segments start from in the workspace), or those states.
hipError_t run_walk(int dtype, const LinearWalk& w, void* workspace, bool starts, hipStream_t stream) {
  ChunkArgs ca{};
  ca.w = w;
  plan_segments(dtype, w, ca);
  ca.starts = static_cast<float*>(workspace);
  if (starts && ca.segs == 1) return hipSuccess;
  const int el = dtype == OOPS_F32 ? 4 : 2;
  const bool vec = (starts || (rows16(w.a, w.a_stride, w.rows, el) && rows16(w.out, w.out_stride, w.cols, el))) &&
                   rows16(w.b, w.b_stride, w.rows, el) && rows16(w.c, w.c_stride, w.cols, el);
  const int d = std::max(w.rows, w.cols);
  return by_type(dtype, [&](auto tag) {
    using T = decltype(tag);
    auto run = [&](auto size) {
      constexpr int D = decltype(size)::value;
      return vec ? run_chunks<T, D, true>(ca, starts, stream) : run_chunks<T, D, false>(ca, starts, stream);
    };
    if (d <= 32) return run(std::integral_constant<int, 32>{});
    if (d <= 64) return run(std::integral_constant<int, 64>{});
    return run(std::integral_constant<int, 128>{});
  });
}

}  // namespace

size_t linear_walk_workspace_bytes(int dtype, const LinearWalk& w) {
  if (w.batch == 0) return 0;
  ChunkArgs ca{};
  plan_segments(dtype, w, ca);
  if (ca.segs == 1) return 0;
  return (size_t)(w.batch * w.heads * ca.segs) * (size_t)w.rows * (size_t)w.cols * sizeof(float);
}
hipError_t launch_linear_walk_starts(int dtype, const LinearWalk& w, void* workspace, hipStream_t stream) {
  return run_walk(dtype, w, workspace, true, stream);
}
hipError_t launch_linear_walk(int dtype, const LinearWalk& w, const void* workspace, hipStream_t stream) {
  return run_walk(dtype, w, const_cast<void*>(workspace), false, stream);
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
