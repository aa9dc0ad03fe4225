// Causal attention over whole prompts, forward: grouped heads, packed sequences.
//
//   O_i = sum_j P_ij V_j,  P_ij = exp(scale q_i.k_j - LSE_i),  j from the start of i's sequence to i
//
// A workgroup takes 128 queries of a head, 32 a wave, in the registers of its
// lanes (a lane: one query); keys and values pass in tiles of 64 rows (float32:
// 32) through two LDS buffers, the next tile's loads in flight behind the
// products.  S^T = K Q^T leaves each lane the scores of its own query, so the
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
// it for this wave.
#include <algorithm>

#include "causal_common.h"

namespace oops {
namespace causal {
namespace {

template <typename T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) == 4 && DP == 128 ? 1 : 2)) void causal_forward_kernel(CausalArgs a) {
  using TL = Tile<T, DP>;
  using A = Att<T>;
  constexpr int KT = TL::kRows, NS = DP / 16, NDT = DP / 32, SUB = KT / 32;
  // float16's weights as two terms: O, and with it the backward's delta, then has no rounding but its own.  (With one, dQ
  // of short rows is off by as much again as by the roundings of dS and of dQ.)
  constexpr bool TWO = __is_same(T, _Float16);
  using Plane = typename TL::Plane;
  using PlaneType = typename TL::PlaneType;
  __shared__ __attribute__((aligned(1024))) char k_lds[A::kBuffers][TL::kBytes];
  __shared__ __attribute__((aligned(1024))) char v_lds[A::kBuffers][TL::kBytes];

  const int tid = threadIdx.x, lane = tid & 63, lq = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
  const Work w = work_of(blockIdx.x, (uint32_t)(a.batch * a.heads));
  const int b = w.head / a.heads, h = w.head % a.heads;
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

  const int t0 = std::min(spans.first.start, block0) / KT, t1 = block1 / KT;
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
  // (a scale of zero: a product too small to count, that leaves the masked pairs' -inf one)
  const float c1 = fmaxf(a.scale * kLog2e, 0x1p-120f);

  fast::vmem_wait<0>();  // (the queries, before loads that the compiler does not count)
  kl.next(k_lds[0]);
  vl.next(v_lds[0]);
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
    if (k0 < spans.last.start || k0 + KT - 1 > block0) {
      // (masked pairs for some wave)
      if (__syncthreads_or(tile_non_finite<Plane, PlaneType>(v_lds[buf]))) {
        add_non_finite<TL, true>(o, v_lds[buf], g, keep);
        __syncthreads();
        clean_tile<Plane, PlaneType>(v_lds[buf]);
        __syncthreads();
      }
    }
    if (idle || k0 > last || k0 + KT <= first_start) return;

    f32x16 s[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      s[u] = f32x16{};
#pragma unroll
      for (int i = 0; i < NS; ++i) s[u] = A::mma(rd.row(k_lds[buf], u, i), qf[i], s[u]);
    }
    if constexpr (TL::k16) interleave<6, SUB * NS, 1>();
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
  for (int t = t0;;) {
    step(t, std::integral_constant<int, 0>{});
    if (++t > t1) break;
    step(t, std::integral_constant<int, 1>{});
    if (++t > t1) break;
  }

  const float l = fast::sum_halves(l_run);
  // (a row without keys: zeros; one whose logits are all -inf: 0 / 0)
  const float inv = empty ? 0.f : 1.0f / l;
  if (!valid) return;
  if (a.lse && g == 0) a.lse[((int64_t)b * a.heads + h) * length + row] = empty ? 0.f : m_run + __builtin_amdgcn_logf(l);
  const int64_t at = (b * a.o_stride[0] + h * a.o_stride[1] + row * a.o_stride[2]) * (int64_t)sizeof(T);
#pragma unroll
  for (int d = 0; d < NDT; ++d) {
    if (empty) o[d] = f32x16{};
    store_columns<T>(static_cast<char*>(a.out) + at, 32 * d, a.value_size, g, o[d], inv,
                     a.low ? static_cast<char*>(a.low) + at : nullptr);
  }
}

}  // namespace
}  // namespace causal

hipError_t launch_causal_forward(int dtype, const CausalArgs& a, hipStream_t stream) {
  if (a.length == 0 || a.batch == 0) return hipSuccess;
  const dim3 grid((uint32_t)a.blocks * (uint32_t)(a.batch * a.heads));
  const bool wide = a.key_size > 64 || a.value_size > 64;
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if (wide) hipLaunchKernelGGL((causal::causal_forward_kernel<T, 128>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((causal::causal_forward_kernel<T, 64>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
  };
  if (dtype == OOPS_F32) return go(float{});
  if (dtype == OOPS_BF16) return go((__bf16)0.f);
  return go((_Float16)0.f);
}

}  // namespace oops
