// Causal attention over whole prompts, backward.
//
// With P_ij = exp(scale q_i.k_j - LSE_i) and delta_i = sum_d O_id dO_id:
//   dS_ij = P_ij (dO_i.v_j - delta_i)
//   dQ_i = scale sum_j dS_ij k_j,  dK_j = scale sum_i dS_ij q_i,  dV_j = sum_i P_ij dO_i
// the sums of dK and dV also over the query heads that share key head j.
//
// Two kernels, both without atomics, so results do not depend on the order of
// workgroups.  The first is laid out like the forward (128 queries a workgroup,
// dQ^T in registers, K and V in LDS) and writes delta; the second holds 128 keys,
// 32 a wave, with dK^T and dV^T in registers, while queries and dO pass through
// LDS, over the query heads of its group in turn.  P and dS are made twice: seven
// products where five are needed, against partial gradients in memory or atomics.
// Where key blocks and heads are too few to fill the chip, the query heads of a
// group and then the walks are split, and the parts' float32 gradients added in
// order by a third kernel.
//
// Bound by the matrix units, like the forward.  bfloat16, 32 heads on 8 of 8192
// tokens in five packed sequences, 128 channels: dQ 326 us (830 TFLOP/s of the pairs
// that count), dK and dV 414-430 (four products, 860) and 48 for their parts' sums, the
// order of blocks 5.  A group's heads in one part: 1090 (one workgroup walks for 58% of
// the time); in two: 603.  V of the block in LDS and not in registers: 480 spilled before.
#include <algorithm>

#include "causal_common.h"

namespace oops {
namespace causal {
namespace {

template <typename T, int DP>
constexpr int kOcc = sizeof(T) == 4 && DP == 128 ? 1 : 2;

template <typename T, int DP>
__global__ __launch_bounds__(256, (kOcc<T, DP>)) void causal_grad_query_kernel(CausalArgs a) {
  using TL = Tile<T, DP>;
  using A = Att<T>;
  constexpr int KT = TL::kRows, NS = DP / 16, NDT = DP / 32, SUB = KT / 32;
  using Plane = typename TL::Plane;
  using PlaneType = typename TL::PlaneType;
  __shared__ __attribute__((aligned(1024))) char k_lds[A::kBuffers][TL::kBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds[A::kBuffers][TL::kBytes];
  __shared__ uint32_t lost_lds[2];

  const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const Work w = work_of(blockIdx.x, (uint32_t)(a.batch * a.heads * a.key_splits));
  const int split = w.head % a.key_splits, b = w.head / a.key_splits / a.heads, h = w.head / a.key_splits % a.heads;
  const int block = a.order ? a.order[w.rank] : a.blocks - 1 - w.rank;
  const int length = (int)a.length;

  const int block0 = block * kBlock, block1 = std::min(block0 + kBlock, length) - 1;
  const int q0 = block0 + wave * 32, row = q0 + lq;
  const bool idle = q0 >= length;
  const int last = std::min(q0 + 31, length - 1);
  const bool valid = row < length;

  const Rows dor = rows_of<T>(a.dout, a.do_stride, b, h, a.value_size, length);
  float delta = row_dot<T, DP>(rows_of<T>(a.out, a.o_stride, b, h, a.value_size, length), dor, row, valid, g, 0.f);
  if (a.low) delta = row_dot<T, DP>(rows_of<T>(a.low, a.o_stride, b, h, a.value_size, length), dor, row, valid, g, delta);
  delta = fast::sum_halves(delta);
  const float c1 = score_factor(a);
  const int64_t stat = ((int64_t)b * a.heads + h) * length + row;
  const float lse = valid ? a.lse[stat] : 0.f;
  if (valid && g == 0 && split == 0) {
    // (as the second kernel's accumulators start)
    a.neg_delta[stat] = -delta;
    a.neg_lse[stat] = -lse / c1;
  }
  if (!a.dq) return;

  const Spans spans = spans_of(a, block0, block1, std::min(q0, last), last, std::min(row, last));
  const int start = spans.own.start;
  const bool empty = !valid || start > row;
  const uint32_t reach = empty ? 0u : (uint32_t)(row - start);
  const int first_start = __builtin_amdgcn_readlane(start, 0), last_start = __builtin_amdgcn_readlane(start, idle ? 0 : last - q0);
  Frag<T> qf[NS], dof[NS];
  load_row<T, DP>(dof, dor, row, valid, g);
  load_row<T, DP>(qf, rows_of<T>(a.q, a.q_stride, b, h, a.key_size, length), row, valid, g, a.flip);

  const Rows kr = rows_of<T>(a.k, a.k_stride, b, h / a.group, a.key_size, length);
  const Rows vr = rows_of<T>(a.v, a.v_stride, b, h / a.group, a.value_size, length);
  const int tile0 = std::min(spans.first.start, block0) / KT, tiles = block1 / KT + 1 - tile0;
  const int t0 = tile0 + tiles * split / a.key_splits, t1 = tile0 + tiles * (split + 1) / a.key_splits - 1;
  Loader<T, DP> kl, vl;
  kl.init(kr, wave, lane);
  vl.init(vr, wave, lane);
  kl.seek(kr, t0 * KT);
  vl.seek(vr, t0 * KT);
  Reads<T, DP> rd;
  rd.init(lane);

  f32x16 dq[NDT];
#pragma unroll
  for (int t = 0; t < NDT; ++t) dq[t] = f32x16{};

  fast::vmem_wait<0>();  // (the rows, before loads that the compiler does not count)
  if (t0 <= t1) {
    kl.next(k_lds[0]);
    vl.next(v_lds[0]);
  }
  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int buf = decltype(buffer)::value % A::kBuffers, other = (buf + 1) % A::kBuffers;
    const int k0 = t * KT;
    arrived<T>(kl, k_lds[buf], vl, v_lds[buf]);
    if (t < t1) {
      kl.next(k_lds[other]);
      vl.next(v_lds[other]);
    }
    auto keep = [&](int r) { return !empty && (uint32_t)(k0 + r - start) <= reach; };
    uint64_t lost = 0;
    if (k0 < spans.last.start || k0 + KT - 1 > block0) {
      // (masked pairs for some wave)
      if (__syncthreads_or(tile_non_finite<Plane, PlaneType>(k_lds[buf]))) {
        lost = rows_non_finite<Plane, PlaneType>(k_lds[buf], lost_lds);
        add_non_finite<TL, false>(dq, k_lds[buf], g, keep);
        __syncthreads();
        clean_tile<Plane, PlaneType>(k_lds[buf]);
        __syncthreads();
      }
    }
    if (idle || k0 > last || k0 + KT <= first_start) return;
    const bool whole = k0 >= last_start && k0 + KT - 1 <= q0;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      f32x16 s{}, dp{};
#pragma unroll
      for (int i = 0; i < NS; ++i) s = A::mma(rd.row(k_lds[buf], u, i), qf[i], s);
#pragma unroll
      for (int i = 0; i < NS; ++i) dp = A::mma(rd.row(v_lds[buf], u, i), dof[i], dp);
      if constexpr (TL::k16) {
        interleave<6, 2 * NS, 1>();
      } else {
        mend_scores(s, [&] {
          f32x16 f{};
#pragma unroll
          for (int i = 0; i < NS; ++i) f = Elem<__bf16>::mma(rd.row(k_lds[buf], u, i).t[0], qf[i].t[0], f);
          return f;
        });
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], c1, -lse)) * (dp[j] - delta);
      if (lost) {
        // (a pair with a lost key: its weight was 0, or made the row's sum NaN)
        const uint32_t rows = (uint32_t)(lost >> (32 * u)) >> (4 * g);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = rows & (1u << kappa(0, j)) ? 0.f * lse : s[j];
      }
      if (!whole) {
        const uint32_t from = here(k0 + 4 * g - start), far = empty ? 0u : reach + 1;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = from + 32 * u + kappa(0, j) < far ? s[j] : 0.f;
      }
      const Frag<T> ds[2] = {pack<T>(s, 0), pack<T>(s, 1)};
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < NDT; ++d) dq[d] = A::mma(rd.col(k_lds[buf], 2 * u + m, d), ds[m], dq[d]);
      if constexpr (TL::k16) interleave<8, 2 * NDT, 2>();
    }
  };
  for (int t = t0; t <= t1;) {
    step(t, std::integral_constant<int, 0>{});
    if (++t > t1) break;
    step(t, std::integral_constant<int, 1>{});
    if (++t > t1) break;
  }
  if (!valid) return;
  // (a row of one key: its weight is 1 whatever the score, and what dS has is the roundings of two sums)
  const float scale = reach == 0 ? 0.f : a.flip ? -a.scale : a.scale;
  if (a.key_splits > 1) {
    const int64_t at = (((int64_t)split * a.batch + b) * a.heads + h) * length + row;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
      store_columns<float>(reinterpret_cast<char*>(a.dq_parts + at * a.key_size), 32 * d, a.key_size, g, dq[d], scale);
    return;
  }
  char* to = static_cast<char*>(a.dq) + (b * a.dq_stride[0] + h * a.dq_stride[1] + row * a.dq_stride[2]) * (int64_t)sizeof(T);
#pragma unroll
  for (int d = 0; d < NDT; ++d) store_columns<T>(to, 32 * d, a.key_size, g, dq[d], scale);
}

// 4 bytes a lane from a buffer to 64 consecutive words at lds; an offset out of range writes zeros
__device__ __forceinline__ void dma4_asm(const fast::u32x4& r, const void* lds, uint32_t voff) {
  const uint32_t m0 =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)(lds));
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds" ::"s"(m0),
      "v"(voff), "s"(r)
      : "memory", "m0");
}

// (float32: one workgroup a CU, whose waves have 512 registers: 33 us for 2 x 6 heads of 777 tokens and 40 channels before the
// look at dV's sums, 36 with it; with two workgroups 42 of 256 registers spilled and it took 33-34)
template <typename T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) == 4 ? 1 : 2)) void causal_grad_key_value_kernel(CausalArgs a) {
  using TL = Tile<T, DP, 32>;
  using A = Att<T>;
  constexpr int QT = 32, NS = DP / 16, NDT = DP / 32;
  // (registers: with 128 channels dK, dV and K fill them; V is read again from LDS at each step)
  constexpr bool kValuesInLds = DP == 128;
  constexpr bool kAgain = !__is_same(T, __bf16);
  using Plane = typename TL::Plane;
  using PlaneType = typename TL::PlaneType;
  __shared__ __attribute__((aligned(1024))) char q_lds[A::kBuffers][TL::kBytes];
  __shared__ __attribute__((aligned(1024))) char do_lds[A::kBuffers][TL::kBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds[kValuesInLds ? 4 : 1][kValuesInLds ? TL::kBytes : 16];
  __shared__ __attribute__((aligned(1024))) float lse_lds[2][64], delta_lds[2][64];

  const int tid = threadIdx.x, lane = tid & 63, lk = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const int parts = a.parts * a.query_splits;
  const Work w = work_of(blockIdx.x, (uint32_t)(a.batch * a.kv_heads * parts));
  const int part = w.head % parts, hk = w.head / parts % a.kv_heads, b = w.head / parts / a.kv_heads;
  const int heads_part = part / a.query_splits, split = part % a.query_splits;
  const int block = a.order ? a.order[a.blocks + w.rank] : w.rank;
  const int length = (int)a.length;

  const int block0 = block * kBlock, block1 = std::min(block0 + kBlock, length) - 1;
  const int k0 = block0 + wave * 32, key = k0 + lk;
  const bool idle = k0 >= length;
  const int last = std::min(k0 + 31, length - 1);
  const bool valid = key < length;
  const Spans spans = spans_of(a, block0, block1, std::min(k0, last), last, std::min(key, last));
  // queries this lane's key is paired with: [key, key + width)
  const int end = spans.own.end;
  const uint32_t width = valid && end > key ? (uint32_t)(end - key) : 0u;
  const bool alone = valid && spans.own.start == key;  // (the only key of the first row)
  const int first_end = __builtin_amdgcn_readlane(end, 0), last_end = __builtin_amdgcn_readlane(end, idle ? 0 : last - k0);

  Frag<T> kf[NS], vf[kValuesInLds ? 1 : NS];
  load_row<T, DP>(kf, rows_of<T>(a.k, a.k_stride, b, hk, a.key_size, length), key, valid, g, a.flip);
  const Rows vr = rows_of<T>(a.v, a.v_stride, b, hk, a.value_size, length);
  if constexpr (!kValuesInLds) load_row<T, DP>(vf, vr, key, valid, g);

  const int block_end = std::max(spans.last.end, block1 + 1);
  const int tile0 = block0 / QT, tiles = (block_end - 1) / QT + 1 - tile0;
  const int t0 = tile0 + tiles * split / a.query_splits, t1 = tile0 + tiles * (split + 1) / a.query_splits - 1;
  const int h0 = hk * a.group + heads_part * a.group / a.parts, h1 = hk * a.group + (heads_part + 1) * a.group / a.parts;

  f32x16 dk[NDT], dv[NDT];
#pragma unroll
  for (int t = 0; t < NDT; ++t) dk[t] = f32x16{}, dv[t] = f32x16{};
  const float c1 = score_factor(a);
  Reads<T, DP> rd, rv;
  rd.init(lane);
  rv = rd;
  rv.shift_rows(wave * TL::kBytes);

  // the tiles' order: the group's heads, each from the block's first query to the last that is paired with its keys
  Loader<T, DP, 32> ql, dl;
  ql.init(rows_of<T>(a.q, a.q_stride, b, h0, a.key_size, length), wave, lane);
  dl.init(rows_of<T>(a.dout, a.do_stride, b, h0, a.value_size, length), wave, lane);
  int load_h = h0, load_t = t0;
  const float* stats = nullptr;  // of the next tile, for waves 0 and 1
  auto seek = [&] {
    ql.seek(rows_of<T>(a.q, a.q_stride, b, load_h, a.key_size, length), load_t * QT);
    dl.seek(rows_of<T>(a.dout, a.do_stride, b, load_h, a.value_size, length), load_t * QT);
    stats = (wave == 0 ? a.neg_lse : a.neg_delta) + ((int64_t)b * a.heads + load_h) * length + load_t * QT;
  };
  auto load = [&](auto buffer) {
    constexpr int to = decltype(buffer)::value, buf = to % A::kBuffers;
    const int n = std::min(ql.left, QT);
    ql.next(q_lds[buf]);
    dl.next(do_lds[buf]);
    if (wave < 2)
      dma4_asm(fast::rsrc_words(stats, (uint32_t)n * 4), wave == 0 ? lse_lds[to] : delta_lds[to], (uint32_t)lane * 4);
    stats += QT;
    if (++load_t > t1) {
      load_t = t0;
      ++load_h;
      if (load_h < h1) seek();
    }
  };

  fast::vmem_wait<0>();  // (the rows, before loads that the compiler does not count)
  if constexpr (kValuesInLds) {
    Loader<T, DP, 32> vl;
    vl.init(vr, wave, lane);
    vl.seek(vr, block0);
    for (int i = 0; i < 4; ++i) {
      vl.next(v_lds[i]);
      if constexpr (!TL::k16) vl.land(v_lds[i]);
    }
  }
  bool careful = false;  // every tile of queries is looked through
  auto step = [&](int t, auto buffer) __attribute__((always_inline)) {
    constexpr int now = decltype(buffer)::value, buf = now % A::kBuffers;
    const int q0 = t * QT;
    arrived<T>(ql, q_lds[buf], dl, do_lds[buf]);
    if (load_h < h1) load(std::integral_constant<int, now ^ 1>{});
    auto keep = [&](int r) { return (uint32_t)(q0 + r - key) < width; };
    if (careful || q0 < block0 + kBlock - 1 || q0 + QT > spans.first.end) {
      // (masked pairs for some wave; a query that is not finite has made its LSE, a dO its delta, NaN or infinite)
      if (__syncthreads_or(tile_non_finite<Plane, PlaneType>(q_lds[buf]) | tile_non_finite<Plane, PlaneType>(do_lds[buf]))) {
        add_non_finite<TL, false>(dk, q_lds[buf], g, keep);
        add_non_finite<TL, true>(dv, do_lds[buf], g, keep);
        __syncthreads();
        clean_tile<Plane, PlaneType>(q_lds[buf]);
        clean_tile<Plane, PlaneType>(do_lds[buf]);
        __syncthreads();
      }
    }
    if (idle || q0 + QT <= k0 || q0 >= last_end) return;
    // scores and dO.v with -LSE / c1 and -delta in the sums; rows kappa(g, 4 q ..) are consecutive
    f32x16 s, dp;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 lse = *reinterpret_cast<const f32x4*>(&lse_lds[now][8 * q + 4 * g]);
      const f32x4 delta = *reinterpret_cast<const f32x4*>(&delta_lds[now][8 * q + 4 * g]);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * q + i] = lse[i], dp[4 * q + i] = delta[i];
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) s = A::mma(rd.row(q_lds[buf], 0, i), kf[i], s);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if constexpr (kValuesInLds) dp = A::mma(rd.row(do_lds[buf], 0, i), rv.row(v_lds[0], 0, i), dp);
      else dp = A::mma(rd.row(do_lds[buf], 0, i), vf[i], dp);
    }
    if constexpr (TL::k16) {
      // (the statistics' eight reads first)
      interleave<12, NS, 1>();
      interleave<kValuesInLds ? 2 : 0, NS, kValuesInLds ? 2 : 1>();
    } else {
      mend_scores(s, [&] {
        f32x16 f;
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = lse_lds[now][kappa(g, j)];
#pragma unroll
        for (int i = 0; i < NS; ++i) f = Elem<__bf16>::mma(rd.row(q_lds[buf], 0, i).t[0], kf[i].t[0], f);
        return f;
      });
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[j] = __builtin_amdgcn_exp2f(s[j] * c1);
      dp[j] *= s[j];
    }
    if (!(q0 >= k0 + 31 && q0 + QT <= first_end)) {
      const uint32_t from = here(q0 + 4 * g - key);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const bool pair = from + kappa(0, j) < width;
        s[j] = pair ? s[j] : 0.f;
        dp[j] = pair ? dp[j] : 0.f;
      }
    }
    if (__any(alone && key >= q0 && key < q0 + QT)) {
      // (a row of one key has no dS: what is left is the roundings of two sums, or NaN)
      const uint32_t from = here(q0 + 4 * g - key);
#pragma unroll
      for (int j = 0; j < 16; ++j) dp[j] = alone && from + kappa(0, j) == 0 ? 0.f * dp[j] : dp[j];
    }
    const Frag<T> p[2] = {pack<T>(s, 0), pack<T>(s, 1)}, ds[2] = {pack<T>(dp, 0), pack<T>(dp, 1)};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        dv[d] = A::mma(rd.col(do_lds[buf], m, d), p[m], dv[d]);
        dk[d] = A::mma(rd.col(q_lds[buf], m, d), ds[m], dk[d]);
      }
    if constexpr (TL::k16) interleave<8, 4 * NDT, 2>();
  };
  if (t0 > t1) fast::vmem_wait<0>();  // (nothing may land in LDS that is another workgroup's by then)
#pragma unroll 1
  while (t0 <= t1) {
    seek();
    load(std::integral_constant<int, 0>{});
    for (int h = h0, t = t0;;) {
      auto next = [&] {
        if (++t > t1) t = t0, ++h;
        return h < h1;
      };
      step(t, std::integral_constant<int, 0>{});
      if (!next()) break;
      step(t, std::integral_constant<int, 1>{});
      if (!next()) break;
    }
    if constexpr (!kAgain) break;
    // (as in the forward: an infinity of dO that nothing masks has met lower terms of a weight, or one that underflowed)
    float any = 0.f;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) any += dv[d][j];
    if (careful || !a.dv || !__syncthreads_or(any != any && width > 0)) break;
    careful = true;
    load_h = h0;
    load_t = t0;
#pragma unroll
    for (int t = 0; t < NDT; ++t) dk[t] = f32x16{}, dv[t] = f32x16{};
  }
  if (!valid) return;
  // (a token of no sequence has zeros, whatever the scale)
  const float scale = width == 0 ? 0.f : a.flip ? -a.scale : a.scale;
  if (parts > 1) {
    const int64_t at = (((int64_t)part * a.batch + b) * a.kv_heads + hk) * length + key;
#pragma unroll
    for (int d = 0; d < NDT; ++d) {
      if (a.dk) store_columns<float>(reinterpret_cast<char*>(a.dk_parts + at * a.key_size), 32 * d, a.key_size, g, dk[d], scale);
      if (a.dv) store_columns<float>(reinterpret_cast<char*>(a.dv_parts + at * a.value_size), 32 * d, a.value_size, g, dv[d], 1.f);
    }
    return;
  }
  char* to_k = static_cast<char*>(a.dk) + (b * a.dk_stride[0] + hk * a.dk_stride[1] + key * a.dk_stride[2]) * (int64_t)sizeof(T);
  char* to_v = static_cast<char*>(a.dv) + (b * a.dv_stride[0] + hk * a.dv_stride[1] + key * a.dv_stride[2]) * (int64_t)sizeof(T);
#pragma unroll
  for (int d = 0; d < NDT; ++d) {
    if (a.dk) store_columns<T>(to_k, 32 * d, a.key_size, g, dk[d], scale);
    if (a.dv) store_columns<T>(to_v, 32 * d, a.value_size, g, dv[d], 1.f);
  }
}

// Blocks of packed sequences by their work, the heaviest first: [blocks] for blocks of queries (tiles of keys up to the
// block's last), then [blocks] for blocks of keys (tiles of queries to the end of the last key's sequence).  A
// counting sort by blocks of 128 tokens; equal ones in any order.
__global__ __launch_bounds__(1024) void causal_order_kernel(CausalArgs a, int32_t* order) {
  __shared__ int start[kMaxOrder + 1];
  for (int side = 0; side < 2; ++side) {
    for (int i = threadIdx.x; i <= a.blocks; i += 1024) start[i] = 0;
    __syncthreads();
    auto weight = [&](int block) {
      const int block0 = block * kBlock, block1 = std::min(block0 + kBlock, (int)a.length) - 1, token = side ? block1 : block0;
      int lo = 0, hi = a.sequences + 1;  // the first bound above the token
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (bound(a, mid, a.length) > token) hi = mid;
        else lo = mid + 1;
      }
      const Span s = span_at(a, token, lo);
      const int tokens = side ? std::max(s.end, block1 + 1) - block0 : block1 + 1 - std::min(s.start, block0);
      return (tokens + kBlock - 1) / kBlock;  // 1 .. blocks
    };
    for (int i = threadIdx.x; i < a.blocks; i += 1024) atomicAdd(&start[a.blocks - weight(i)], 1);
    __syncthreads();
    if (threadIdx.x < 64) {
      // where each weight's blocks begin: a scan, 64 at a time
      int sum = 0;
      for (int i = 0; i < a.blocks; i += 64) {
        const int at = i + (int)threadIdx.x, own = at < a.blocks ? start[at] : 0;
        int x = own;
        for (int d = 1; d < 64; d *= 2) {
          const int y = __shfl_up(x, d);
          if ((int)threadIdx.x >= d) x += y;
        }
        if (at < a.blocks) start[at] = sum + x - own;
        sum += __shfl(x, 63);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.blocks; i += 1024) order[side * a.blocks + atomicAdd(&start[a.blocks - weight(i)], 1)] = i;
    __syncthreads();
  }
}

// The parts' gradients (part, batch, head, token, size), added in order; four elements a thread.
template <typename T>
__global__ __launch_bounds__(256) void causal_parts_kernel(const float* parts, void* out, int64_t s0, int64_t s1, int64_t s2,
                                                           int64_t heads, int64_t length, int size, int count, int64_t cells) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= cells) return;
  f32x4 s = *reinterpret_cast<const f32x4*>(parts + i);
  for (int p = 1; p < count; ++p) s += *reinterpret_cast<const f32x4*>(parts + p * cells + i);
  const int64_t rows = i / size, t = rows % length, h = rows / length % heads, b = rows / length / heads;
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 y;
#pragma unroll
  for (int k = 0; k < 4; ++k) y[k] = (T)s[k];
  *reinterpret_cast<v4*>(static_cast<T*>(out) + b * s0 + h * s1 + t * s2 + i % size) = y;
}

}  // namespace
}  // namespace causal

// Whether blocks of packed sequences are put in order first (a launch of some microseconds): where there are more
// workgroups than places on the chip, so that a heavy block that starts late would be waited for.
bool causal_ordered(const oops_causal_geometry& g) {
  const int64_t blocks = (g.length + causal::kBlock - 1) / causal::kBlock;
  return blocks <= causal::kMaxOrder && blocks * g.batch * g.heads > 512;
}
hipError_t launch_causal_order(const CausalArgs& a, int32_t* order, hipStream_t stream) {
  hipLaunchKernelGGL(causal::causal_order_kernel, dim3(1), dim3(1024), 0, stream, a, order);
  return hipGetLastError();
}

// Parts of a group's query heads: workgroups for every CU's two places four times over, so that the heavy blocks (the first
// keys, paired with every query) find light ones to even them out (32 heads on 8 of 8192 tokens: 1090 us for places once,
// 603 twice, 414-430 and 24 more for the sums four times over).
int causal_grad_parts(const oops_causal_geometry& g) {
  const int64_t blocks = (g.length + causal::kBlock - 1) / causal::kBlock * g.batch * g.kv_heads;
  const int64_t want = blocks > 0 ? (2048 + blocks - 1) / blocks : 1;
  return (int)std::min<int64_t>(want, g.heads / g.kv_heads);
}

hipError_t launch_causal_backward(int dtype, const CausalArgs& a, hipStream_t stream) {
  if (a.length == 0 || a.batch == 0) return hipSuccess;
  const uint32_t blocks = (uint32_t)a.blocks;
  const bool wide = a.key_size > 64 || a.value_size > 64;
  const dim3 grid_q(blocks * (uint32_t)(a.batch * a.heads * a.key_splits));
  const int parts = a.parts * a.query_splits;
  const dim3 grid_kv(blocks * (uint32_t)(a.batch * a.kv_heads * parts));
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (wide) hipLaunchKernelGGL((causal::causal_grad_query_kernel<T, 128>), grid_q, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((causal::causal_grad_query_kernel<T, 64>), grid_q, dim3(256), 0, stream, a);
    hipError_t e = hipGetLastError();
    auto add = [&](const float* from, void* out, const int64_t(&s)[3], int heads, int size, int count) {
      const int64_t cells = a.batch * heads * a.length * size;
      hipLaunchKernelGGL((causal::causal_parts_kernel<T>), dim3((uint32_t)((cells / 4 + 255) / 256)), dim3(256), 0, stream, from,
                         out, s[0], s[1], s[2], (int64_t)heads, a.length, size, count, cells);
      return hipGetLastError();
    };
    if (e == hipSuccess && a.dq && a.key_splits > 1) e = add(a.dq_parts, a.dq, a.dq_stride, a.heads, a.key_size, a.key_splits);
    if (e != hipSuccess || (!a.dk && !a.dv)) return e;
    if (wide) hipLaunchKernelGGL((causal::causal_grad_key_value_kernel<T, 128>), grid_kv, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((causal::causal_grad_key_value_kernel<T, 64>), grid_kv, dim3(256), 0, stream, a);
    e = hipGetLastError();
    if (e == hipSuccess && parts > 1 && a.dk) e = add(a.dk_parts, a.dk, a.dk_stride, a.kv_heads, a.key_size, parts);
    if (e == hipSuccess && parts > 1 && a.dv) e = add(a.dv_parts, a.dv, a.dv_stride, a.kv_heads, a.value_size, parts);
    return e;
  };
  if (dtype == OOPS_F32) return go(float{});
  if (dtype == OOPS_BF16) return go((__bf16)0.f);
  return go((_Float16)0.f);
}

}  // namespace oops
