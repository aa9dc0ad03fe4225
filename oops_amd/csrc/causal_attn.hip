// Causal attention over whole prompts, forward: grouped heads, packed sequences.
//
//   O_i = sum_j P_ij V_j,  P_ij = exp(scale q_i.k_j - LSE_i),  j from the start of i's sequence to i
//
// A workgroup takes 128 queries of a head, 32 a wave, in the registers of its
// lanes (a lane: one query); keys and values pass in tiles of 64 rows through two
// LDS buffers, the next tile's loads in flight behind the products (float32: 32
// rows and one buffer, the next tile in registers until it becomes terms).  S^T = K Q^T leaves each lane the scores of its own query, so the
// running maximum and sum need one exchange between the two halves of a wave,
// and P^T is the second product's operand without leaving its registers:
// O^T += V^T P^T, V^T by transposed LDS reads.  The maximum is raised only where
// it grows by more than 2^8 (sums and O are float32 and the difference is
// exact), so O is rarely rescaled.
//
// Sequences: token i knows its sequence's bounds from `offsets`; blocks of
// queries and tiles of keys lie at multiples of their size in the packed row,
// tiles before a block's first sequence and behind its last query are not read,
// and a tile is masked pair by pair only where a bound or the diagonal crosses
// it for this wave.  Such tiles are looked through for infinities and NaN, which 0
// times them would spread; in float16 and float32 a walk whose sums come out NaN
// is made again with every tile looked through (a microsecond of a small call's
// time for the look at the sums).
//
// Bound by the matrix units and what stands between their two products.  bfloat16,
// 16 heads of 16384 tokens and 128 channels: 1040-1065 us, 1040 TFLOP/s of a
// library's square product's 1380 (matrix units 60% busy, no bank conflicts); five
// packed sequences of 8192 tokens in all, 32 heads: 231-245 us, 770 TFLOP/s of the
// pairs that count (9% of the products lie in masked halves of tiles, the rest
// is four times as many blocks' first tiles and ends).  What it took: the order of
// LDS reads and products given by hand (1303 -> 1130), padded tiles with constant
// addresses (-> 1053), heaviest blocks first.  A loop that makes the next 32 keys'
// scores beside the weights of the last ones: 1070 without spills, 1863 with.
#include <algorithm>

#include "causal_common.h"

namespace oops {
namespace causal {
namespace {

// A row's LSE from its maximum and its sum, and what its O is multiplied with.  Logits that are all -inf have weights 0 / 0, so
// both are NaN: with -inf, a score that the backward makes of cleaned operands would have a weight of infinity, and with
// 1 / 0 an infinite value would stay one.
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? __builtin_nanf("") : m + __builtin_amdgcn_logf(l); }
__device__ __forceinline__ float one_over(float l) { return l == 0.f ? __builtin_nanf("") : 1.0f / l; }

template <typename T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void causal_forward_kernel(CausalArgs a) {
  using TL = Tile<T, DP>;
  using A = Att<T>;
  constexpr int KT = TL::kRows, NS = DP / 16, NDT = DP / 32, SUB = KT / 32;
  // float16's weights as two terms: O, and with it the backward's delta, then has no rounding but its own.  (With one, dQ
  // of short rows is off by as much again as by the roundings of dS and of dQ.)
  constexpr bool TWO = __is_same(T, _Float16);
  constexpr bool kAgain = !__is_same(T, __bf16);  // (one term, with float32's exponents: an infinity times a weight is one)
  using Plane = typename TL::Plane;
  using PlaneType = typename TL::PlaneType;
  __shared__ __attribute__((aligned(1024))) char k_lds[A::kBuffers][TL::kBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds[A::kBuffers][TL::kBytes];

  const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const Work w = work_of(blockIdx.x, (uint32_t)(a.batch * a.heads * a.key_splits));
  const int split = w.head % a.key_splits, b = w.head / a.key_splits / a.heads, h = w.head / a.key_splits % a.heads;
  const int block = a.order ? a.order[w.rank] : a.blocks - 1 - w.rank;
  const int length = (int)a.length;

  const int block0 = block * kBlock, block1 = std::min(block0 + kBlock, length) - 1;
  const int q0 = block0 + wave * 32, row = q0 + lq;
  const bool idle = q0 >= length;  // (a wave behind the last token has no pairs)
  const int last = std::min(q0 + 31, length - 1);
  const bool valid = row < length;
  const Spans spans = spans_of(a, block0, block1, std::min(q0, last), last, std::min(row, last));
  // keys this lane's query is paired with: [start, row]
  const int start = spans.own.start;
  const bool empty = !valid || start > row;
  const uint32_t reach = empty ? 0u : (uint32_t)(row - start);
  const int first_start = __builtin_amdgcn_readlane(start, 0), last_start = __builtin_amdgcn_readlane(start, idle ? 0 : last - q0);

  const Rows kr = rows_of<T>(a.k, a.k_stride, b, h / a.group, a.key_size, length);
  const Rows vr = rows_of<T>(a.v, a.v_stride, b, h / a.group, a.value_size, length);
  Frag<T> qf[NS];
  load_row<T, DP>(qf, rows_of<T>(a.q, a.q_stride, b, h, a.key_size, length), row, valid, g, a.flip);

  const int tile0 = std::min(spans.first.start, block0) / KT, tiles = block1 / KT + 1 - tile0;
  const int t0 = tile0 + tiles * split / a.key_splits, t1 = tile0 + tiles * (split + 1) / a.key_splits - 1;
  Loader<T, DP> kl, vl;
  kl.init(kr, wave, lane);
  vl.init(vr, wave, lane);
  kl.seek(kr, t0 * KT);
  vl.seek(vr, t0 * KT);
  Reads<T, DP> rd;
  rd.init(lane);

  float m_run = kNegInf, neg_m = 0.f, l_run = 0.f;
  f32x16 o[NDT];
#pragma unroll
  for (int t = 0; t < NDT; ++t) o[t] = f32x16{};
  const float c1 = score_factor(a);

  fast::vmem_wait<0>();  // (the queries, before loads that the compiler does not count)
  bool careful = false;  // every tile's values are looked through
  // (the buffer is a constant, so that its address is part of the instructions)
  auto step = [&](int t, auto buffer) {
    constexpr int buf = decltype(buffer)::value % A::kBuffers, other = (buf + 1) % A::kBuffers;
    const int k0 = t * KT;
    arrived<T>(kl, k_lds[buf], vl, v_lds[buf]);
    if (t < t1) {
      kl.next(k_lds[other]);
      vl.next(v_lds[other]);
    }
    auto keep = [&](int r) { return !empty && (uint32_t)(k0 + r - start) <= reach; };
    const bool mine = !(idle || k0 > last || k0 + KT <= first_start);
    f32x16 s[SUB];
    // this tile's scores, and the running maximum with them
    auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        s[u] = f32x16{};
#pragma unroll
        for (int i = 0; i < NS; ++i) s[u] = A::mma(rd.row(k_lds[buf], u, i), qf[i], s[u]);
      }
      if constexpr (TL::k16) {
        interleave<6, SUB * NS, 1>();
      } else {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
          mend_scores(s[u], [&] {
            f32x16 f{};
#pragma unroll
            for (int i = 0; i < NS; ++i) f = Elem<__bf16>::mma(rd.row(k_lds[buf], u, i).t[0], qf[i].t[0], f);
            return f;
          });
      }
      if (k0 < last_start || k0 + KT - 1 > q0) {
        const uint32_t from = here(k0 + 4 * g - start), far = empty ? 0u : reach + 1;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[u][j] = from + 32 * u + kappa(0, j) < far ? s[u][j] : kNegInf;
      }
      float mx = s[0][0];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[u][j]);
      mx = fast::max_halves(mx) * c1;
      const bool grow = mx > m_run + fast::kLazyRescale;
      if (__any(grow)) {
        const float m_new = grow ? mx : m_run;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
        m_run = m_new;
        neg_m = m_run == kNegInf ? 0.f : -m_run;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < NDT; ++d) o[d] *= alpha;
      }
    };
    // What is not finite in a tile with masked pairs (for some wave) is added before its weights are multiplied, but behind
    // the maximum, whose factor for the sums may be 0.  In 16 bits such a tile's scores are made twice; in float32 the look
    // through the tile waits for the scores.  (16 heads of 128, this way and the other: 8192 tokens in float16 451 and 461 us,
    // 4096 in float32 567 and 592.)
    if constexpr (!TL::k16)
      if (mine) scores();
    if (careful || k0 < spans.last.start || k0 + KT - 1 > block0) {
      if (__syncthreads_or(tile_non_finite<Plane, PlaneType>(v_lds[buf]))) {
        if constexpr (TL::k16)
          if (mine) scores();
        add_non_finite<TL, true>(o, v_lds[buf], g, keep);
        __syncthreads();
        clean_tile<Plane, PlaneType>(v_lds[buf]);
        __syncthreads();
      }
    }
    if (!mine) return;
    if constexpr (TL::k16) scores();
    Frag<T> p[KT / 16], rest[TWO ? KT / 16 : 1];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
#pragma unroll
      for (int j = 0; j < 16; ++j) s[u][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], c1, neg_m));
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        p[2 * u + m] = pack<T>(s[u], m);
        if constexpr (TWO) rest[2 * u + m] = pack_rest<T>(s[u], m, p[2 * u + m]);
        // (the sum of what is multiplied: a rounding that all weights share leaves no trace)
        if constexpr (TL::k16 && !TWO) l_run = add_elements<T>(p[2 * u + m], l_run);
      }
      if constexpr (!TL::k16 || TWO) {
#pragma unroll
        for (int j = 0; j < 16; ++j) l_run += s[u][j];
      }
    }
#pragma unroll
    for (int m = 0; m < KT / 16; ++m)
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        const Frag<T> v = rd.col(v_lds[buf], m, d);
        if constexpr (TWO) o[d] = A::mma(v, rest[m], o[d]);
        o[d] = A::mma(v, p[m], o[d]);
      }
    if constexpr (TL::k16 && !TWO) {
      __builtin_amdgcn_sched_group_barrier(0x002, 12, 0);
      interleave<8, NDT * (KT / 16), 2, 5>();
    }
  };
  float l;
#pragma unroll 1
  while (true) {
    if (t0 <= t1) {
      kl.next(k_lds[0]);
      vl.next(v_lds[0]);
    }
    for (int t = t0; t <= t1;) {
      step(t, std::integral_constant<int, 0>{});
      if (++t > t1) break;
      step(t, std::integral_constant<int, 1>{});
      if (++t > t1) break;
    }
    l = fast::sum_halves(l_run);
    if constexpr (!kAgain) break;
    // In a tile that nothing masks an infinite value has met a weight's lower terms, which are zero or of either sign, or a
    // first one that underflowed: NaN.  Then the walk is made again, and such values are added one by one in every tile.
    // (Where the row's weights are NaN, so is the result.)
    float any = 0.f;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) any += o[d][j];
    if (careful || !__syncthreads_or(any != any && l == l && !empty)) break;
    careful = true;
    m_run = kNegInf, neg_m = 0.f, l_run = 0.f;
#pragma unroll
    for (int d = 0; d < NDT; ++d) o[d] = f32x16{};
    kl.seek(kr, t0 * KT);
    vl.seek(vr, t0 * KT);
  }
  // (a row without keys: zeros; one whose logits are all -inf: 0 / 0)
  const float inv = empty ? 0.f : one_over(l);
  if (!valid) return;
  if (a.key_splits > 1) {
    const int64_t at = (((int64_t)split * a.batch + b) * a.heads + h) * length + row;
    if (g == 0) a.stat_parts[2 * at] = m_run, a.stat_parts[2 * at + 1] = empty ? -1.f : l;
#pragma unroll
    for (int d = 0; d < NDT; ++d)
      store_columns<float>(reinterpret_cast<char*>(a.o_parts + at * a.value_size), 32 * d, a.value_size, g, o[d], 1.f);
    return;
  }
  if (a.lse && g == 0) a.lse[((int64_t)b * a.heads + h) * length + row] = empty ? 0.f : log_sum(m_run, l);
  const int64_t at = (b * a.o_stride[0] + h * a.o_stride[1] + row * a.o_stride[2]) * (int64_t)sizeof(T);
#pragma unroll
  for (int d = 0; d < NDT; ++d) {
    if (empty) o[d] = f32x16{};
    store_columns<T>(static_cast<char*>(a.out) + at, 32 * d, a.value_size, g, o[d], inv,
                     a.low ? static_cast<char*>(a.low) + at : nullptr);
  }
}

// Rows whose keys were split: the parts by their maxima and sums, in order; four elements a thread.
template <typename T>
__global__ __launch_bounds__(256) void causal_join_kernel(CausalArgs a, int64_t cells) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= cells) return;
  const int64_t rows = cells / a.value_size, row = i / a.value_size;
  const int d = (int)(i - row * a.value_size);
  float m = kNegInf;
  for (int s = 0; s < a.key_splits; ++s) m = fmaxf(m, a.stat_parts[2 * (s * rows + row)]);
  const bool empty = a.stat_parts[2 * row + 1] == -1.f;
  float l = 0.f;
  f32x4 x{};
  for (int s = 0; s < a.key_splits; ++s) {
    const float part = a.stat_parts[2 * (s * rows + row)], by = part == m ? 1.f : __builtin_amdgcn_exp2f(part - m);
    l = __builtin_fmaf(a.stat_parts[2 * (s * rows + row) + 1], by, l);
    const f32x4 o = *reinterpret_cast<const f32x4*>(a.o_parts + s * cells + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = __builtin_fmaf(o[k], by, x[k]);
  }
  const float inv = empty ? 0.f : one_over(l);
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 y, low;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float v = empty ? 0.f : x[k] * inv;
    y[k] = (T)v;
    const float r = v - (float)y[k];
    low[k] = (T)(__builtin_isfinite(r) ? r : 0.f);
  }
  const int64_t token = row % a.length, h = row / a.length % a.heads, b = row / a.length / a.heads;
  const int64_t at = b * a.o_stride[0] + h * a.o_stride[1] + token * a.o_stride[2] + d;
  *reinterpret_cast<v4*>(static_cast<T*>(a.out) + at) = y;
  if (a.low) *reinterpret_cast<v4*>(static_cast<T*>(a.low) + at) = low;
  if (a.lse && d == 0) a.lse[row] = empty ? 0.f : log_sum(m, l);
}

}  // namespace
}  // namespace causal

// Parts of the axis that a workgroup walks along (keys for queries, queries for keys), so that few workgroups fill the
// chip's 512 places and its longest walk gets shorter; parts of fewer than four tiles cost more in joining than they
// save.  us of kernels, forward / with the backward, in one part and in parts:
//   1 head of 16384 tokens, 128 channels, bf16   315 / 1350   119 / 469   (for 1024 places 105 / 428)
//   2 heads of 4096                               88 /  373    38 / 138   (49 / 185)
//   8 heads of 2048, float32                     253 /  912   100 / 359   (123 / 460)
//   2 x 6 heads of 777, 40 channels, float32      60 /  230    37 / 103
//   the same in bf16: three parts 19 / 61, one 21 / 74, six (of two tiles) 22 / 62
int causal_splits(const oops_causal_geometry& g, int64_t workgroups) {
  const int64_t tokens = g.length / std::max(g.sequences, 1), tile = g.dtype == OOPS_F32 ? 32 : 64;
  return workgroups < 1 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({(511 + workgroups) / workgroups, tokens / (4 * tile), 16}));
}

hipError_t launch_causal_forward(int dtype, const CausalArgs& a, hipStream_t stream) {
  if (a.length == 0 || a.batch == 0) return hipSuccess;
  const dim3 grid((uint32_t)a.blocks * (uint32_t)(a.batch * a.heads * a.key_splits));
  const int64_t cells = a.batch * a.heads * a.length * a.value_size;
  const bool wide = a.key_size > 64 || a.value_size > 64;
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (wide) hipLaunchKernelGGL((causal::causal_forward_kernel<T, 128>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((causal::causal_forward_kernel<T, 64>), grid, dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.key_splits == 1) return e;
    hipLaunchKernelGGL((causal::causal_join_kernel<T>), dim3((uint32_t)((cells / 4 + 255) / 256)), dim3(256), 0, stream, a, cells);
    return hipGetLastError();
  };
  if (dtype == OOPS_F32) return go(float{});
  if (dtype == OOPS_BF16) return go((__bf16)0.f);
  return go((_Float16)0.f);
}

}  // namespace oops
