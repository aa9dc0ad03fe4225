// The paged key/value cache in 4 bits: written, read back, and attended to by single tokens.
//
// A token of a head is size / 2 bytes of codes and one exponent byte a block of
// 32 channels, for its key and its value: 136 bytes at 128 channels where
// bfloat16 takes 512.
//
// Writing and reading move each byte once (HBM): a lane takes eight channels,
// four lanes a block.  The scaled conversions make two codes an instruction and
// round to nearest even, saturating, so the codes are those of exact arithmetic
// (by comparisons in float32, 12 operations a code, the writing took 63 us for
// 30011 tokens of 8 heads of 128 and was bound by them).
//
// Attention: a workgroup takes one key head, up to 16 query heads that share it,
// and a range of the sequence; each of its waves passes tiles of 32 tokens.  Codes
// become bfloat16 (exact: a code has two significant bits) with the scaled
// conversion, one instruction for two values.  S^T = K Q^T by 16 x 16 x 32 MFMAs:
// a lane loads its token's codes as they lie in memory, and the channels' order is
// the query's fragments'.  S^T leaves the probabilities as the second product's
// operand; V^T comes from LDS by transposed reads (each wave has a region of its
// own, so there is no barrier in the loop).  float16 and float32 queries are split
// into two and three bfloat16 terms, probabilities into two (three for float32),
// whose products are exact and added in float32: a result has its own type's
// precision whatever the cache's.  Few sequences are split over their length; a second launch joins the
// parts by their maxima and sums.
//
// bfloat16, 8 key heads of 128, 32 query heads: writing 30011 tokens 48 us (157 MB at
// 3.3 TB/s) and 4 for the slots' owners, reading them 37 (4.3 TB/s); attention of 64
// sequences of up to 16384 tokens 178 us (4.0 TB/s; 222 and 230 with float16 and
// float32 queries) and 6 for the join, one sequence of 32768 17.6 (2.0 TB/s: 256
// tokens a workgroup, two steps of each wave) and 6.
#include <algorithm>

#include "attn_common.h"
#include "decoder_kernels.h"

namespace oops {
namespace {

constexpr int kThreads = 256;
constexpr int kScanTokens = 1024;  // up to here later tokens of the same slot are looked for by reading the slots

template <typename F>
hipError_t by_type(int dtype, F&& f) {
  if (dtype == OOPS_F32) return f(float{});
  if (dtype == OOPS_BF16) return f((__bf16)0.f);
  return f((_Float16)0.f);
}

struct CacheArgs {
  uint8_t *codes, *scales;
  const void *key, *value;
  void *key_out, *value_out;
  const void* slots;
  const int32_t* owner;
  int64_t stride[2][3];
  int64_t slots_count, tokens, length;
  int32_t heads, size, page, slots_i64, whole;
  int32_t lanes, together;  // lanes of a token, and tokens at once (1: the lanes of one may take several workgroups)
  int64_t run;              // tokens of a workgroup, one after the other: neighbours fill lines of the cache together
};
__device__ __forceinline__ int64_t slot_of(const void* slots, int i64, int64_t t) {
  return i64 ? static_cast<const int64_t*>(slots)[t] : static_cast<const int32_t*>(slots)[t];
}
// One lane's eight channels of keys or values: the same for all tokens that it passes.
struct Lane {
  int which, head, piece, ahead;  // ahead: of the workgroup's first token
  bool live;
};
__device__ __forceinline__ Lane lane_of(const CacheArgs& a) {
  const int i = blockIdx.y * kThreads + threadIdx.x, pieces = a.size / 8;
  const int ahead = a.together > 1 ? i / a.lanes : 0, n = i - ahead * a.lanes;
  return Lane{n / (pieces * a.heads), n / pieces % a.heads, n % pieces, ahead < a.together ? ahead : a.together - 1,
              ahead < a.together && n < a.lanes};
}
__device__ __forceinline__ int64_t valid_slot(const CacheArgs& a, int64_t token) {
  const int64_t s = slot_of(a.slots, a.slots_i64, token);
  return s >= 0 && s < a.slots_count ? s : -1;
}
// row of the codes and scales
__device__ __forceinline__ int64_t cache_row(const CacheArgs& a, const Lane& l, int64_t slot) {
  const uint32_t page = (uint32_t)slot / (uint32_t)a.page;
  return (((int64_t)page * a.heads + l.head) * 2 + l.which) * a.page + ((uint32_t)slot - page * (uint32_t)a.page);
}
__device__ __forceinline__ int64_t operand_at(const CacheArgs& a, const Lane& l, int64_t token) {
  const int64_t* s = a.stride[l.which];
  const uint32_t b = a.tokens > a.length ? (uint32_t)token / (uint32_t)a.length : 0;
  return b * s[0] + l.head * s[1] + (token - b * a.length) * s[2] + l.piece * 8;
}

// ---- of tokens with the same slot the last is kept (long calls: owners are settled first)
__global__ __launch_bounds__(kThreads) void slot_clear_kernel(const void* slots, int i64, int64_t tokens, int64_t count, int32_t* owner) {
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (t >= tokens) return;
  const int64_t s = slot_of(slots, i64, t);
  if (s >= 0 && s < count) owner[s] = -1;
}
__global__ __launch_bounds__(kThreads) void slot_owner_kernel(const void* slots, int i64, int64_t tokens, int64_t count, int32_t* owner) {
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (t >= tokens) return;
  const int64_t s = slot_of(slots, i64, t);
  // (the largest token: any order of the additions gives it)
  if (s >= 0 && s < count) atomicMax(&owner[s], (int32_t)t);
}

// the largest magnitude of eight elements, as a float32's bits
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const uint32_t (&u)[2 * sizeof(T)]) {
  uint32_t top = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = std::max(top, u[i] & 0x7FFFFFFFu);
    return top;
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 t = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, u[i] & 0x7FFF7FFFu));
    const uint16_t m = std::max(t[0], t[1]);
    return __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(T, m));
  }
}
// eight codes: the elements over the scale, to the nearest, ties to even, at most 6
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const uint32_t (&u)[2 * sizeof(T)], float scale) {
  uint32_t w = 0;
  if constexpr (sizeof(T) == 4) {
    auto f = [&](int i) { return __builtin_bit_cast(float, u[i]); };
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(0), f(1), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(2), f(3), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(4), f(5), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f(6), f(7), scale, 3);
  } else if constexpr (__is_same(T, __bf16)) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2, u[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2, u[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2, u[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(v2, u[3]), scale, 3);
  } else {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2, u[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2, u[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2, u[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(v2, u[3]), scale, 3);
  }
  return w;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(CacheArgs a) {
  const Lane l = lane_of(a);
  const int lane = threadIdx.x & 63;
  constexpr int kWords = 2 * (int)sizeof(T);
  const int64_t first_token = (int64_t)blockIdx.x * a.run, end = std::min(first_token + a.run, a.tokens);
  const T* operand = static_cast<const T*>(l.which ? a.value : a.key);
  // (a token's slot, and its elements beside it, a turn before they are used)
  int64_t next_slot;
  uint32_t next[kWords];
  auto fetch = [&](int64_t token) __attribute__((always_inline)) {
    const bool there = l.live && token < end;
    next_slot = there ? valid_slot(a, token) : -1;
#pragma unroll
    for (int i = 0; i < kWords; ++i) next[i] = 0;
    if (!there) return;
    const T* x = operand + operand_at(a, l, token);
    if (a.whole) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(x)[i];
        next[4 * i] = q.x, next[4 * i + 1] = q.y, next[4 * i + 2] = q.z, next[4 * i + 3] = q.w;
      }
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = x[i];
      __builtin_memcpy(next, e, sizeof(next));
    }
  };
  fetch(first_token + l.ahead);
  for (int64_t base = first_token; base < end; base += a.together) {
    const int64_t token = base + l.ahead, slot = next_slot;
    uint32_t u[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) u[i] = next[i];
    fetch(token + a.together);
    bool write = slot >= 0;
    if (a.owner) {
      write = write && a.owner[slot] == (int32_t)token;
    } else {
      // the wave's tokens one after the other, the later slots 64 at a time
      const int first = __builtin_amdgcn_readlane((int)token, 0), last = __builtin_amdgcn_readlane((int)token, 63);
      for (int t = first; t <= last && t < a.tokens; ++t) {
        const int64_t mine = slot_of(a.slots, a.slots_i64, t);
        bool again = false;
        for (int64_t v = t + 1 + lane; v < a.tokens; v += 64) again |= slot_of(a.slots, a.slots_i64, v) == mine;
        if (__any(again) && token == t) write = false;
      }
    }
    // the block's largest magnitude as a bit pattern (a NaN's is above infinity's); its lanes are four neighbours
    uint32_t top = top_bits<T>(u);
    top = std::max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = std::max(top, (uint32_t)__shfl_xor((int)top, 2));
    if (!write) continue;
    // top = 1.f * 2^(exp - 127) <= 6 * 2^e = 1.5 * 2^(e + 2)
    const int exp = (int)(top >> 23);
    const bool lost = exp == 255;
    int e = exp - ((top & 0x7FFFFFu) > 0x400000u ? 1 : 2);
    e = lost ? 255 : e < 1 ? 1 : e > 252 ? 252 : e;
    const uint32_t word = lost ? 0 : codes_of<T>(u, __builtin_bit_cast(float, (uint32_t)e << 23));
    const int64_t row = cache_row(a, l, slot);
    *reinterpret_cast<uint32_t*>(a.codes + row * (a.size / 2) + l.piece * 4) = word;
    if (l.piece % 4 == 0) a.scales[row * (a.size / 32) + l.piece / 4] = (uint8_t)e;
  }
}

__device__ __forceinline__ float scale_value(uint32_t e) {
  return __builtin_bit_cast(float, e == 255 ? 0x7FC00000u : e == 0 ? 0x00400000u : e << 23);
}
__device__ __forceinline__ float code_value(uint32_t c, float scale) {
  const uint32_t m = c & 7;
  const float v = m < 2 ? 0.5f * (float)m : __builtin_bit_cast(float, (((m >> 1) + 126) << 23) | ((m & 1) << 22));
  return (c & 8 ? -v : v) * scale;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(CacheArgs a) {
  const Lane l = lane_of(a);
  if (!l.live) return;
  const int64_t first_token = (int64_t)blockIdx.x * a.run, end = std::min(first_token + a.run, a.tokens);
  for (int64_t token = first_token + l.ahead; token < end; token += a.together) {
    const int64_t slot = valid_slot(a, token);
    uint32_t word = 0, e = 1;
    if (slot >= 0) {
      const int64_t row = cache_row(a, l, slot);
      word = *reinterpret_cast<const uint32_t*>(a.codes + row * (a.size / 2) + l.piece * 4);
      e = a.scales[row * (a.size / 32) + l.piece / 4];
    }
    const float scale = scale_value(e);
    union {
      uint4 u[sizeof(T) / 2];
      T y[8];
    } r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.y[i] = (T)code_value(word >> (4 * i) & 15, scale);
    // (results are allocated in whole pieces)
    uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(l.which ? a.value_out : a.key_out) + operand_at(a, l, token));
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) to[i] = r.u[i];
  }
}

// ------------------------------------------------------------------ attention

constexpr int kTile = 32;      // tokens of a wave's step
constexpr int kHeadTile = 16;  // query heads of a workgroup
constexpr int64_t kMaxSplits = 256;

struct DecodeArgs {
  const void *query, *lengths;
  const uint8_t *codes, *scales;
  const int32_t* table;
  void* out;
  float* parts;  // (batch, heads, splits, size + 2): O, maximum, sum (-1: no token)
  int64_t pages, batch, max_pages, q_batch, q_head;
  int32_t heads, kv_heads, group, tiles, page, lengths_i64, splits;
  uint32_t page16, per16;  // a page in 16 tokens, and 2^32 over that, rounded down
  float scale;
};

// Terms of a query's elements, and of weights: bfloat16's have two like float16's, 16 bits.  (One would round the weights but
// not their sum, and a rounding that many weights share would stay in the result: up to half a step of bfloat16 beside the
// result's own, for 174 us in place of 178 of 64 sequences of up to 16384 tokens, 8 key heads of 128.)
template <typename T> struct Terms { static constexpr int N = 2, kWeight = 2; };
template <> struct Terms<__bf16> { static constexpr int N = 1, kWeight = 2; };
template <> struct Terms<float> { static constexpr int N = 3, kWeight = 3; };

// x as bfloat16 terms, whose sum is x for the types above (an infinity or a NaN is the first term's alone; FINITE: x is no
// infinity, and a NaN may be every term).  A finite number above bfloat16's largest has that for its first term.
template <int N, bool FINITE = false>
__device__ __forceinline__ void split(float x, __bf16 (&t)[N]) {
  constexpr float kTop = 3.3895313892515355e38f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = (__bf16)(N == 3 && !FINITE && i == 0 && __builtin_isfinite(x) ? __builtin_fminf(__builtin_fmaxf(x, -kTop), kTop) : x);
    x -= (float)t[i];
    if (!FINITE && !__builtin_isfinite(x)) x = 0.f;
  }
}

typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
// a wave's tile as loaded: token lane % 16 of each half, 8 NS channels a lane; the halves whose page is there
template <int NS>
struct Raw {
  static constexpr int kScales = NS == 4 ? 1 : NS;
  uint32_t k[2][NS], v[2][NS];
  uint32_t ks[2][kScales], vs[2][kScales];
  bool have[2];
};

// eight codes to bfloat16, times the scale
__device__ __forceinline__ bf16x8 values8(uint32_t word, float scale) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float max_rows(float x) {  // over the four 16-lane rows, in every lane
  const int i = __builtin_bit_cast(int, x);
  const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
  const int y = __builtin_bit_cast(int, fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1])));
  const auto s = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(__builtin_bit_cast(float, (int)s[0]), __builtin_bit_cast(float, (int)s[1]));
}
__device__ __forceinline__ float sum_rows(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <typename T, int NS>
__global__ __launch_bounds__(kThreads, 3) void cache_attn_kernel(DecodeArgs a) {
  constexpr int N = Terms<T>::N, W = Terms<T>::kWeight, D = 32 * NS, ND = D / 16;
  // channels of step s of lane group g: with four steps a lane's sixteen bytes lie together
  auto channel = [](int s, int g) { return NS == 4 ? 32 * g + 8 * s : 32 * s + 8 * g; };
  constexpr int kPitch = 2 * D + 32;  // bytes: 8 rows' pieces of 32 bytes lie in different banks
  constexpr int kRegion = std::max(kTile * kPitch, kHeadTile * (D + 2) * 4);
  __shared__ __attribute__((aligned(16))) char lds[4][kRegion];

  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int split_at = blockIdx.x % a.splits, job = blockIdx.x / a.splits;
  const int tile_at = job % a.tiles, hk = job / a.tiles % a.kv_heads, b = job / a.tiles / a.kv_heads;
  const int h = hk * a.group + tile_at * kHeadTile + c;  // this lane's query head
  const bool head_live = tile_at * kHeadTile + c < a.group;

  const int64_t given = a.lengths_i64 ? static_cast<const int64_t*>(a.lengths)[b] : static_cast<const int32_t*>(a.lengths)[b];
  const int count = (int)std::min<int64_t>(std::max<int64_t>(given, 0), a.max_pages * a.page);
  const int steps = (count + kTile - 1) / kTile, per = (steps + a.splits - 1) / a.splits;
  const int from = split_at * per, to = std::min(steps, from + per);

  bf16x8 q[NS][N];
  {
    const T* x = static_cast<const T*>(a.query) + b * a.q_batch + h * a.q_head;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __bf16 t[N];
        split<N>(head_live ? (float)x[channel(s, g) + i] : 0.f, t);
#pragma unroll
        for (int n = 0; n < N; ++n) q[s][n][i] = t[n];
      }
  }

  // 16 tokens: their page in the sequence and their place there, in units of 16 (the quotient is at most one short)
  auto divided = [&](int t16, uint32_t& place) {
    uint32_t n = __umulhi((uint32_t)t16, a.per16);
    place = (uint32_t)t16 - n * a.page16;
    if (place >= a.page16) ++n, place -= a.page16;
    return n;
  };
  // a tile's pages, or -1; read a step before they are used
  const int32_t* table = a.table + b * a.max_pages;
  auto pages_of = [&](int step, int32_t (&id)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t place;
      const uint32_t n = divided(2 * step + i, place);
      id[i] = step < to && step * kTile + 16 * i < count ? table[n] : -1;
    }
  };
  auto load = [&](int step, const int32_t (&id)[2], Raw<NS>& r) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int s = 0; s < NS; ++s) r.k[i][s] = r.v[i][s] = 0;
#pragma unroll
      for (int s = 0; s < Raw<NS>::kScales; ++s) r.ks[i][s] = r.vs[i][s] = 127;
      r.have[i] = id[i] >= 0 && id[i] < a.pages;
      if (!r.have[i]) continue;
      uint32_t place;
      divided(2 * step + i, place);
      // (places behind the last token lie in the page: what they hold is taken out below)
      const int64_t row = ((int64_t)id[i] * a.kv_heads + hk) * 2 * a.page + place * 16 + c;
      const uint8_t* kc = a.codes + row * (D / 2);
      const uint8_t* vc = kc + (int64_t)a.page * (D / 2);
      const uint8_t* ks = a.scales + row * NS;
      const uint8_t* vs = ks + (int64_t)a.page * NS;
      if constexpr (NS == 4) {
        const u32x4v k = *reinterpret_cast<const u32x4v*>(kc + 16 * g), v = *reinterpret_cast<const u32x4v*>(vc + 16 * g);
#pragma unroll
        for (int s = 0; s < 4; ++s) r.k[i][s] = k[s], r.v[i][s] = v[s];
        r.ks[i][0] = ks[g];
        r.vs[i][0] = vs[g];
      } else {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          r.k[i][s] = *reinterpret_cast<const uint32_t*>(kc + 16 * s + 4 * g);
          r.v[i][s] = *reinterpret_cast<const uint32_t*>(vc + 16 * s + 4 * g);
          r.ks[i][s] = ks[s];
          r.vs[i][s] = vs[s];
        }
      }
    }
  };

  float m_run = kNegInf, neg_m = 0.f, l_run = 0.f;
  bool seen = false;
  f32x4 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4{};
  const float c1 = a.scale * kLog2e;
  char* mine = lds[wave];

  Raw<NS> raw;
  int32_t id[2];
  pages_of(from + wave, id);
  load(from + wave, id, raw);
  pages_of(from + wave + 4, id);
  for (int step = from + wave; step < to; step += 4) {
    Raw<NS> now = raw;
    load(step + 4, id, raw);
    pages_of(step + 8, id);
    if (!now.have[0] && !now.have[1]) continue;
    seen = true;
    const int left = std::min(count - step * kTile, kTile);
    // values behind the last token (absent pages have zeros)
    if (left < kTile)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool live = c + 16 * i < left;
#pragma unroll
      for (int s = 0; s < NS; ++s) now.v[i][s] = live ? now.v[i][s] : 0;
#pragma unroll
      for (int s = 0; s < Raw<NS>::kScales; ++s) now.vs[i][s] = live ? now.vs[i][s] : 127;
    }
    // V to LDS in bfloat16
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s)
        *reinterpret_cast<bf16x8*>(mine + (c + 16 * i) * kPitch + channel(s, g) * 2) =
            values8(now.v[i][s], scale_value(now.vs[i][NS == 4 ? 0 : s]));
    // S^T: rows (registers) tokens 16 i + 4 g + r, columns (lanes) query heads
    f32x4 st[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      st[i] = f32x4{};
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const bf16x8 k = values8(now.k[i][s], scale_value(now.ks[i][NS == 4 ? 0 : s]));
#pragma unroll
        for (int n = 0; n < N; ++n) st[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[s][n], st[i], 0, 0, 0);
      }
    }
    if (left < kTile || !now.have[0] || !now.have[1]) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) st[i][r] = now.have[i] && 16 * i + 4 * g + r < left ? st[i][r] * c1 : kNegInf;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) st[i] *= c1;
    }
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, st[i][r]);
    mx = max_rows(mx);
    const bool grow = mx > m_run + 8.0f;  // (a difference of 2^8 is nothing to float32 sums)
    if (__any(grow)) {
      const float m_new = grow ? mx : m_run;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      m_run = m_new;
      neg_m = m_run == kNegInf ? 0.f : -m_run;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
    }
    bf16x8 p[W];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = __builtin_amdgcn_exp2f(st[i][r] + neg_m);
        l_run += x;
        __bf16 t[W];
        split<W, true>(x, t);
#pragma unroll
        for (int n = 0; n < W; ++n) p[n][4 * i + r] = t[n];
      }
    // O^T += V^T P^T; lane (c, g) gets V[4 g + k][16 d + c] for k = 0..3, then rows + 16
    asm volatile("" ::: "memory");
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const char* at = mine + (4 * g + (c >> 2)) * kPitch + (16 * d + 4 * (c & 3)) * 2;
      const s16x4 lo = lds_read_tr4(at), hi = lds_read_tr4(at + 16 * kPitch);
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const bf16x8 v = __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
#pragma unroll
      for (int n = 0; n < W; ++n) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[n], o[d], 0, 0, 0);
    }
    // (two of V's fragments ahead of the products: left alone, the compiler waits for each, 8 us of such a batch's)
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      __builtin_amdgcn_sched_group_barrier(0x008, W, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    asm volatile("" ::: "memory");
  }

  // the waves' parts: maximum and sum of each query head, then O, joined in order
  l_run = sum_rows(l_run);
  __syncthreads();
  float* part = reinterpret_cast<float*>(mine);
  if (g == 0) part[c] = m_run, part[16 + c] = seen ? l_run : -1.f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[32 + c * D + 16 * d + 4 * g + r] = o[d][r];
  __syncthreads();
  for (int i = threadIdx.x; i < kHeadTile * D; i += kThreads) {
    const int col = i / D, d = i % D;
    if (tile_at * kHeadTile + col >= a.group) continue;
    float m = kNegInf, l = 0.f, x = 0.f;
    bool any = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float* f = reinterpret_cast<const float*>(lds[w]);
      if (f[16 + col] != -1.f) m = fmaxf(m, f[col]), any = true;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float* f = reinterpret_cast<const float*>(lds[w]);
      if (f[16 + col] == -1.f) continue;
      const float by = f[col] == m && m == kNegInf ? 1.f : __builtin_amdgcn_exp2f(f[col] - m);
      l = __builtin_fmaf(f[16 + col], by, l);
      x = __builtin_fmaf(f[32 + col * D + d], by, x);
    }
    const int64_t row = (int64_t)b * a.heads + hk * a.group + tile_at * kHeadTile + col;
    if (a.splits == 1) {
      // (no token: zeros; every logit -inf: 0 / 0)
      static_cast<T*>(a.out)[row * D + d] = (T)(any ? x / l : 0.f);
    } else {
      float* to_part = a.parts + (row * a.splits + split_at) * (D + 2);
      to_part[d] = x;
      if (d == 0) to_part[D] = m, to_part[D + 1] = any ? l : -1.f;
    }
  }
}

// The splits of one row, joined: the parts' factors first (a part a lane), then O, four threads a channel, each every
// fourth part, added in order.
template <typename T>
__global__ __launch_bounds__(512) void cache_join_kernel(const float* parts, void* out, int splits, int size) {
  __shared__ float by[kMaxSplits], sums[4][128], total[2];
  const float* p = parts + (int64_t)blockIdx.x * splits * (size + 2);
  const int tid = threadIdx.x;
  if (tid < 64) {
    float m = kNegInf, l = 0.f;
    bool any = false;
    for (int s = tid; s < splits; s += 64) {
      const float *f = p + s * (size + 2) + size;
      if (f[1] != -1.f) m = fmaxf(m, f[0]), any = true;
    }
    for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
    for (int s = tid; s < splits; s += 64) {
      const float *f = p + s * (size + 2) + size;
      const float w = f[1] == -1.f ? 0.f : m == kNegInf ? 1.f : __builtin_amdgcn_exp2f(f[0] - m);
      by[s] = w;
      if (f[1] != -1.f) l = __builtin_fmaf(f[1], w, l);
    }
    for (int d = 32; d > 0; d /= 2) l += __shfl_xor(l, d);
    if (tid == 0) total[0] = l;
    const bool some = __any(any);
    if (tid == 0) total[1] = some ? 1.f : 0.f;
  }
  __syncthreads();
  const int d = tid & 127, quarter = tid >> 7;
  float x = 0.f;
  if (d < size) {
#pragma unroll 4
    // (a part without tokens has O = 0)
    for (int s = quarter; s < splits; s += 4) x = __builtin_fmaf(p[s * (size + 2) + d], by[s], x);
  }
  sums[quarter][d] = x;
  __syncthreads();
  if (tid >= size) return;
  x = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
  static_cast<T*>(out)[(int64_t)blockIdx.x * size + tid] = (T)(total[1] > 0.f ? x / total[0] : 0.f);
}

// Parts of the length: workgroups for eight on every CU, so that sequences of different lengths even out, but no part
// shorter than two steps of each wave where a sequence fills its page table (8 key heads of 128, one sequence of 32768 or of
// 4096 tokens, us with the join: two steps 28 and 16, one 37 and 15, four 27-30 and 18, eight 30 and 23).  The host knows
// the table's width and not the lengths: few sequences that are short for their table have shorter parts and empty ones.
// us of a call in a graph with a table that the sequence fills, 4 and 32 times as wide: one sequence of 1024 tokens 11, 10
// and 18, of 4096 11, 13 and 28, of 32768 23, 32 and 32, four of 2048 12, 16 and 23, 16 of 4096 30 each.
int decode_splits(const oops_cache_attn_geometry& g) {
  const int64_t group = g.heads / g.kv_heads;
  const int64_t jobs = g.batch * g.kv_heads * ((group + kHeadTile - 1) / kHeadTile);
  if (jobs == 0) return 1;
  const int64_t most = (g.max_pages * g.page + 8 * kTile - 1) / (8 * kTile);
  return (int)std::max<int64_t>(1, std::min<int64_t>({(2048 + jobs - 1) / jobs, most, kMaxSplits}));
}

}  // namespace

size_t cache_write_workspace_bytes(const oops_cache_geometry& g) {
  return g.batch * g.length > kScanTokens ? (size_t)(g.pages * g.page) * sizeof(int32_t) : 0;
}

namespace {
CacheArgs cache_args(const oops_cache_geometry& g, const void* codes, const void* scales, const void* slots) {
  CacheArgs a{};
  a.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  a.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  a.slots = slots;
  for (int i = 0; i < 2; ++i) std::copy(g.stride[i], g.stride[i] + 3, a.stride[i]);
  a.slots_count = g.pages * g.page;
  a.tokens = g.batch * g.length;
  a.length = g.length;
  a.heads = g.heads;
  a.size = g.size;
  a.page = g.page;
  a.slots_i64 = g.slots_i64;
  a.lanes = 2 * g.heads * (g.size / 8);
  a.together = std::max(1, kThreads / a.lanes);
  return a;
}
// lanes of a token along y, tokens along x, sixteen workgroups on every CU at most
dim3 cache_grid(CacheArgs& a) {
  const unsigned y = a.together > 1 ? 1 : (unsigned)((a.lanes + kThreads - 1) / kThreads);
  const int64_t turns = (a.tokens + a.together - 1) / a.together, most = std::max(1u, 4096 / y);
  a.run = (turns + most - 1) / most * a.together;
  return dim3((unsigned)((a.tokens + a.run - 1) / a.run), y);
}
}  // namespace

hipError_t launch_cache_write(const oops_cache_geometry& g, void* codes, void* scales, const void* key, const void* value,
                              const void* slots, void* workspace, hipStream_t stream) {
  CacheArgs a = cache_args(g, codes, scales, slots);
  a.key = key;
  a.value = value;
  const int n = g.dtype == OOPS_F32 ? 4 : 8;
  a.whole = reinterpret_cast<uintptr_t>(key) % 16 == 0 && reinterpret_cast<uintptr_t>(value) % 16 == 0;
  for (int i = 0; i < 2; ++i)
    for (int d = 0; d < 3; ++d) a.whole = a.whole && g.stride[i][d] % n == 0;
  if (a.tokens > kScanTokens) {
    int32_t* owner = static_cast<int32_t*>(workspace);
    const dim3 grid((unsigned)((a.tokens + kThreads - 1) / kThreads));
    hipLaunchKernelGGL(slot_clear_kernel, grid, dim3(kThreads), 0, stream, slots, g.slots_i64, a.tokens, a.slots_count, owner);
    hipLaunchKernelGGL(slot_owner_kernel, grid, dim3(kThreads), 0, stream, slots, g.slots_i64, a.tokens, a.slots_count, owner);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.owner = owner;
  }
  return by_type(g.dtype, [&](auto tag) {
    const dim3 grid = cache_grid(a);
    hipLaunchKernelGGL((cache_write_kernel<decltype(tag)>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

hipError_t launch_cache_read(const oops_cache_geometry& g, const void* codes, const void* scales, const void* slots,
                             void* key, void* value, hipStream_t stream) {
  CacheArgs a = cache_args(g, codes, scales, slots);
  a.key_out = key;
  a.value_out = value;
  return by_type(g.dtype, [&](auto tag) {
    const dim3 grid = cache_grid(a);
    hipLaunchKernelGGL((cache_read_kernel<decltype(tag)>), grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  });
}

size_t cache_attn_workspace_bytes(const oops_cache_attn_geometry& g) {
  const int splits = decode_splits(g);
  return splits > 1 ? (size_t)(g.batch * g.heads) * splits * (g.size + 2) * sizeof(float) : 0;
}

hipError_t launch_cache_attn(const oops_cache_attn_geometry& g, const void* query, const void* codes, const void* scales,
                             const int32_t* pages, const void* lengths, void* out, void* workspace, hipStream_t stream) {
  DecodeArgs a{};
  a.query = query;
  a.lengths = lengths;
  a.codes = static_cast<const uint8_t*>(codes);
  a.scales = static_cast<const uint8_t*>(scales);
  a.table = pages;
  a.out = out;
  a.parts = static_cast<float*>(workspace);
  a.pages = g.pages;
  a.batch = g.batch;
  a.max_pages = g.max_pages;
  a.q_batch = g.stride[0];
  a.q_head = g.stride[1];
  a.heads = g.heads;
  a.kv_heads = g.kv_heads;
  a.group = g.heads / g.kv_heads;
  a.tiles = (a.group + kHeadTile - 1) / kHeadTile;
  a.page = g.page;
  a.lengths_i64 = g.lengths_i64;
  a.splits = decode_splits(g);
  a.page16 = (uint32_t)g.page / 16;
  a.per16 = a.page16 == 1 ? 0xFFFFFFFFu : (uint32_t)((uint64_t(1) << 32) / a.page16);
  a.scale = g.scale;
  const dim3 grid((unsigned)(g.batch * g.kv_heads * a.tiles * a.splits));
  return by_type(g.dtype, [&](auto tag) {
    using T = decltype(tag);
    if (g.size == 32) hipLaunchKernelGGL((cache_attn_kernel<T, 1>), grid, dim3(kThreads), 0, stream, a);
    else if (g.size == 64) hipLaunchKernelGGL((cache_attn_kernel<T, 2>), grid, dim3(kThreads), 0, stream, a);
    else if (g.size == 96) hipLaunchKernelGGL((cache_attn_kernel<T, 3>), grid, dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((cache_attn_kernel<T, 4>), grid, dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    hipLaunchKernelGGL((cache_join_kernel<T>), dim3((unsigned)(g.batch * g.heads)), dim3(512), 0, stream, a.parts, out, a.splits,
                       g.size);
    return hipGetLastError();
  });
}

}  // namespace oops
