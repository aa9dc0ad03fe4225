// Device code shared by the causal attention kernels (forward and backward).
//
// Every product is a 32 x 32 x 16 step on fragments of eight elements a lane: one
// MFMA of a 16-bit type.  float32 operands are three bfloat16 terms, their sum
// exactly (above 2^-110 in magnitude: the terms have float32's exponents, and their
// smallest number is 2^-133), and a step is six MFMAs, the terms' products down to
// 2^-16 of the largest (what is left out is below 2^-23, and 2^-26 on average): 192
// cycles where the float32 matrix unit takes 512.  Lane (c = lane % 32, g = lane / 32)
// holds elements 16 s + 8 g .. + 7 of row c along the contracted axis.  An
// accumulator's rows are kappa(g, j), so eight of its registers are the other
// operand of the next product as they stand, if the tile in LDS is read in the same
// order (Reads::col).
//
// Tiles of 32 or 64 rows go from memory straight to LDS in 16-byte pieces, a
// kilobyte at a time (4 rows of 128 elements of 16 bits, 8 of 64).  Inside it a
// row's 64-byte windows change places by the row's lower bits, and kilobytes lie 16
// or 32 bytes more than their size apart: 16 lanes that read the same piece of 16
// rows meet 16 different groups of four banks, and so do the 4 rows x 64 bytes of a
// transposed read.  A lane's addresses are then two or four registers and constants,
// which the instructions hold themselves.
#pragma once
#include "attn_fast_common.h"
#include "decoder_kernels.h"

namespace oops {
namespace causal {

using fast::kOut;

constexpr int kBlock = 128;      // queries, or keys, of a workgroup
constexpr int kMaxOrder = 8192;  // blocks that are put in order by their work

// float32 in three bfloat16 terms
struct Terms3 {
  bf16x8 t[3];
};
template <typename T> struct Att {
  using Frag = typename Elem<T>::Frag;
  static constexpr int kRows = 64;    // rows of a tile in LDS
  static constexpr int kBuffers = 2;  // tiles filled while others are read
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) { return Elem<T>::mma(a, b, c); }
};
template <> struct Att<float> {
  using Frag = Terms3;
  static constexpr int kRows = 32;
  static constexpr int kBuffers = 1;  // (filled from registers, where the next tile waits)
  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    using E = Elem<__bf16>;
    c = E::mma(a.t[1], b.t[1], c);
    c = E::mma(a.t[0], b.t[2], c);
    c = E::mma(a.t[2], b.t[0], c);
    c = E::mma(a.t[0], b.t[1], c);
    c = E::mma(a.t[1], b.t[0], c);
    return E::mma(a.t[0], b.t[0], c);
  }
};
template <typename T> using Frag = typename Att<T>::Frag;

// eight floats in three terms; an infinity or a NaN is the first term's alone.  CLAMP: finite values above bfloat16's
// largest stay finite.
template <bool CLAMP>
__device__ __forceinline__ Terms3 split3(const float (&x)[8]) {
  constexpr float kTop = 3.3895313892515355e38f;
  Terms3 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = x[i];
    if (CLAMP && fabsf(v) > kTop && fabsf(v) < -kNegInf) v = __builtin_copysignf(kTop, v);
    f.t[0][i] = (__bf16)v;
    float r = x[i] - (float)f.t[0][i];
    r = __builtin_isfinite(r) ? r : 0.f;
    f.t[1][i] = (__bf16)r;
    f.t[2][i] = (__bf16)(r - (float)f.t[1][i]);
  }
  return f;
}

// ---- tiles in LDS: ROWS rows of DP elements
template <typename T, int DP, int ROWS = Att<T>::kRows>
struct Tile {
  using Plane = Tile;  // what holds the elements' largest terms
  using PlaneType = T;
  static constexpr int kRows = ROWS;
  static constexpr bool k16 = true;
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kPieces = kRowBytes / 16;            // of a row
  static constexpr int kChunks = kRows * kRowBytes / 1024;  // kilobytes
  static constexpr int kLoads = kChunks / 4;                // of a wave, four waves a tile
  static constexpr int kPitch = 1024 + (DP == 128 ? 16 : 32);  // between kilobytes
  static constexpr int kBytes = kChunks * kPitch;
  static constexpr int kWindows = DP / 32;

  // piece of row r that lies at place p of the row (its own inverse)
  static __device__ __forceinline__ int placed(int r, int p) {
    if constexpr (DP == 128) return p ^ ((r & 3) << 2);
    else return p ^ (((r >> 1) & 1) << 2) ^ ((r >> 2) & 1);
  }
  static __device__ __forceinline__ int at(int r, int piece) {
    constexpr int n = 1024 / kRowBytes;  // rows of a kilobyte
    return r / n * kPitch + r % n * kRowBytes + (placed(r, piece) << 4);
  }
  // the n-th 16-byte piece in the order of places
  static __device__ __forceinline__ int nth(int n) { return (n >> 6) * kPitch + (n & 63) * 16; }
  static __device__ __forceinline__ float element(const char* tile, int r, int c) {
    return (float)*reinterpret_cast<const T*>(tile + at(r, c >> 3) + (c & 7) * 2);
  }
};
// float32: a tile for each term
template <int DP, int ROWS>
struct Tile<float, DP, ROWS> {
  using Plane = Tile<__bf16, DP, ROWS>;
  using PlaneType = __bf16;
  static constexpr int kRows = ROWS;
  static constexpr bool k16 = false;
  static constexpr int kBytes = 3 * Plane::kBytes;
  static constexpr int kWindows = Plane::kWindows;
  static __device__ __forceinline__ float element(const char* tile, int r, int c) {
    return Plane::element(tile, r, c) + (Plane::element(tile + Plane::kBytes, r, c) + Plane::element(tile + 2 * Plane::kBytes, r, c));
  }
};

// A lane's fragments of tiles
template <typename T, int DP>
struct Reads {
  using TL = Tile<T, DP, 32>;  // (32 rows are a multiple of every pattern)
  static constexpr int kStep16 = 16 / (1024 / TL::kRowBytes) * TL::kPitch;  // bytes of 16 rows
  int row_at[TL::kWindows], col_at[TL::kWindows];
  __device__ __forceinline__ void init(int lane) {
    const int lq = lane & 31, g = lane >> 5, j = lane & 15, half = lane >> 4 & 1, r = 4 * g + (j >> 2);
#pragma unroll
    for (int w = 0; w < TL::kWindows; ++w) {
      row_at[w] = TL::at(lq, 4 * w + g);
      col_at[w] = TL::at(r, 4 * w + 2 * half + ((j & 3) >> 1)) + (j & 1) * 8;
    }
  }
  // the rows of another tile, `bytes` further on
  __device__ __forceinline__ void shift_rows(int bytes) {
#pragma unroll
    for (int w = 0; w < TL::kWindows; ++w) row_at[w] += bytes;
  }
  // elements 16 s + 8 g .. + 7 of row 32 u + lane % 32
  __device__ __forceinline__ Frag<T> row(const char* tile, int u, int s) const {
    return __builtin_bit_cast(Frag<T>, *reinterpret_cast<const uint4*>(tile + row_at[s >> 1] + (s & 1) * 32 + 2 * u * kStep16));
  }
  // column 32 t + lane % 32 of rows 16 m + kappa(g, 0..7)
  __device__ __forceinline__ Frag<T> col(const char* tile, int m, int t) const {
    constexpr int n = 1024 / TL::kRowBytes;
    const char* at = tile + col_at[t] + m * kStep16;
    const s16x4 lo = lds_read_tr4(at), hi = lds_read_tr4(at + 8 / n * TL::kPitch);
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(Frag<T>, v);
  }
};
template <int DP>
struct Reads<float, DP> {
  using Plane = typename Tile<float, DP, 32>::Plane;
  Reads<__bf16, DP> plane;
  __device__ __forceinline__ void init(int lane) { plane.init(lane); }
  __device__ __forceinline__ void shift_rows(int bytes) { plane.shift_rows(bytes); }
  __device__ __forceinline__ Terms3 row(const char* tile, int u, int s) const {
    return Terms3{plane.row(tile, u, s), plane.row(tile + Plane::kBytes, u, s), plane.row(tile + 2 * Plane::kBytes, u, s)};
  }
  __device__ __forceinline__ Terms3 col(const char* tile, int m, int t) const {
    return Terms3{plane.col(tile, m, t), plane.col(tile + Plane::kBytes, m, t), plane.col(tile + 2 * Plane::kBytes, m, t)};
  }
};

// Rows of an operand of one (batch, head): 64-bit base, row pitch in bytes, row length in bytes.
struct Rows {
  const char* base;
  int64_t pitch;
  int32_t bytes;
  int64_t count;
};
template <typename T>
__device__ __forceinline__ Rows rows_of(const void* p, const int64_t (&stride)[3], int64_t b, int64_t h, int size, int64_t count) {
  return Rows{static_cast<const char*>(p) + (b * stride[0] + h * stride[1]) * (int64_t)sizeof(T),
              stride[2] * (int64_t)sizeof(T), size * (int)sizeof(T), count};
}
// Rows of an operand to a tile, tile after tile; rows behind the last and columns behind the size are zeros.  The
// resource starts at the tile's first row, so that offsets stay small however long the operand is (the host refuses row
// pitches of 2^24 bytes and more).
template <typename T, int DP, int ROWS = Att<T>::kRows>
struct Loader {
  using TL = Tile<T, DP, ROWS>;
  uint32_t off[TL::kLoads];
  const char* base;  // of the next tile
  int64_t step;
  int left, bytes, pitch, wave;  // left: rows from there on
  __device__ __forceinline__ void init(const Rows& r, int wave_, int lane) {
    wave = wave_;
    bytes = r.bytes;
    pitch = (int)r.pitch;
    step = r.pitch * ROWS;
#pragma unroll
    for (int i = 0; i < TL::kLoads; ++i) {
      const int n = (wave * TL::kLoads + i) * 64 + lane, row = n / TL::kPieces;
      const int col = TL::placed(row, n % TL::kPieces) * 16;
      off[i] = col < r.bytes ? (uint32_t)(row * pitch + col) : kOut;
    }
  }
  __device__ __forceinline__ void seek(const Rows& r, int row0) {
    base = r.base + row0 * r.pitch;
    left = (int)r.count - row0;
  }
  __device__ __forceinline__ void next(const char* lds) {
    const int n = left < ROWS ? left : ROWS;  // (none or fewer behind the last row: the resource is empty)
    const fast::u32x4 rs = fast::rsrc_words(base, n > 0 ? (uint32_t)((n - 1) * pitch + bytes) : 0u);
#pragma unroll
    for (int i = 0; i < TL::kLoads; ++i) fast::dma16_asm(rs, lds + (wave * TL::kLoads + i) * TL::kPitch, off[i], 0);
    base += step;
    left -= ROWS;
  }
};

// float32: the next tile's elements wait in registers, and become terms when the tile before has been read
template <int DP>
struct Loader<float, DP, 32> {
  using Plane = typename Tile<float, DP, 32>::Plane;
  static constexpr int kN = DP / 64;  // pieces of eight elements a thread
  float v[kN][8];
  const char* base;
  int64_t pitch;
  int left, bytes, row[kN], piece[kN];
  __device__ __forceinline__ void init(const Rows& r, int, int) {
    pitch = r.pitch;
    bytes = r.bytes;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int n = (int)threadIdx.x + 256 * i;
      row[i] = n / (DP / 8);
      piece[i] = n % (DP / 8);
    }
  }
  __device__ __forceinline__ void seek(const Rows& r, int row0) {
    base = r.base + row0 * r.pitch;
    left = (int)r.count - row0;
  }
  __device__ __forceinline__ void next(const char*) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const char* p = base + row[i] * pitch;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = piece[i] * 32 + 16 * h;
        f32x4 x{};
        if (row[i] < left && col < bytes) x = *reinterpret_cast<const f32x4*>(p + col);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i][4 * h + k] = x[k];
      }
    }
    base += pitch * 32;
    left -= 32;
  }
  __device__ __forceinline__ void land(char* tile) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const Terms3 f = split3<true>(v[i]);
#pragma unroll
      for (int t = 0; t < 3; ++t) *reinterpret_cast<bf16x8*>(tile + t * Plane::kBytes + Plane::at(row[i], piece[i])) = f.t[t];
    }
  }
};
// The tile that was asked for last is there, for all waves, in buffer `to` (one tile or two)
template <typename T, typename L>
__device__ __forceinline__ void arrived(const L& first, char* to_first, const L& second, char* to_second) {
  if constexpr (sizeof(T) == 4) {
    lds_barrier();  // (the tiles before have been read)
    first.land(to_first);
    second.land(to_second);
  }
  fast::vmem_wait<0>();
  lds_barrier();
}

// A row's fragments from memory (zeros behind the size and for absent rows); `flip` changes the sign.
template <typename T, int DP>
__device__ __forceinline__ void load_row(Frag<T> (&f)[DP / 16], const Rows& r, int64_t row, bool valid, int g, bool flip = false) {
  const char* p = r.base + row * r.pitch;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    constexpr int n = 8 * (int)sizeof(T) / 16;
    const int col = (16 * s + 8 * g) * (int)sizeof(T);
    uint4 u[n];
#pragma unroll
    for (int i = 0; i < n; ++i) {
      u[i] = make_uint4(0, 0, 0, 0);
      if (valid && col + 16 * i < r.bytes) u[i] = *reinterpret_cast<const uint4*>(p + col + 16 * i);
      if (flip) {
        constexpr uint32_t m = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
        u[i].x ^= m, u[i].y ^= m, u[i].z ^= m, u[i].w ^= m;
      }
    }
    if constexpr (sizeof(T) == 2) {
      __builtin_memcpy(&f[s], u, sizeof(f[s]));
    } else {
      float x[8];
      __builtin_memcpy(x, u, sizeof(x));
      f[s] = split3<true>(x);
    }
  }
}
// sum + the product of two rows (this lane's half of their pieces)
template <typename T, int DP>
__device__ __forceinline__ float row_dot(const Rows& a, const Rows& b, int64_t row, bool valid, int g, float sum) {
  constexpr int n = 16 / (int)sizeof(T);
  const char *p = a.base + row * a.pitch, *q = b.base + row * b.pitch;
#pragma unroll
  for (int s = 0; s < DP / (2 * n); ++s) {
    const int col = (2 * s + g) * 16;
    uint4 u = make_uint4(0, 0, 0, 0), v = u;
    if (valid && col < a.bytes) u = *reinterpret_cast<const uint4*>(p + col), v = *reinterpret_cast<const uint4*>(q + col);
    const T *x = reinterpret_cast<const T*>(&u), *y = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < n; ++i) sum = __builtin_fmaf((float)x[i], (float)y[i], sum);
  }
  return sum;
}

// The order of a block's instructions: AHEAD LDS reads first, then after each of PRODUCTS matrix instructions READS more,
// VECTOR vector ones and EXP exponentials.  (Left alone, the compiler reads two fragments, waits for both and multiplies.)
template <int AHEAD, int PRODUCTS, int READS, int VECTOR = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (AHEAD > 0) __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    if constexpr (VECTOR > 0) __builtin_amdgcn_sched_group_barrier(0x002, VECTOR, 0);
  }
}

// ---- packed sequences: bounds offsets[0 .. n] along the tokens
__device__ __forceinline__ int64_t bound(const CausalArgs& a, int i, int64_t length) {
  const int64_t v = a.offsets_i64 ? static_cast<const int64_t*>(a.offsets)[i] : static_cast<const int32_t*>(a.offsets)[i];
  return v < 0 ? 0 : v > length ? length : v;
}
// Numbers of bounds at or before tokens i[0 .. K-1] (the same for all lanes of the wave): 64 bounds at a time, loads that
// do not wait for each other.
template <int K>
__device__ __forceinline__ void bounds_before(const CausalArgs& a, const int (&i)[K], int (&count)[K]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < K; ++k) count[k] = 0;
  for (int n = 0; n <= a.sequences; n += 64) {
    const bool there = n + lane <= a.sequences;
    const int64_t v = there ? bound(a, n + lane, a.length) : 0;
#pragma unroll
    for (int k = 0; k < K; ++k) count[k] += __builtin_popcountll(__ballot(there && v <= i[k]));
  }
}
// The sequence that holds token i: [start, end); a token of none has start = i + 1 and end = i.
struct Span {
  int start, end;
};
// (bounds that do not increase: what is read stays inside the operands)
__device__ __forceinline__ Span span_at(const CausalArgs& a, int i, int before) {
  if (before == 0 || before > a.sequences) return Span{i + 1, i};
  const int start = (int)bound(a, before - 1, a.length), end = (int)bound(a, before, a.length);
  return Span{start < i ? start : i, end > i ? end : i + 1};
}
// For a workgroup's block of tokens [first, last] and this wave's [w0, w1], of which this lane has `token`
struct Spans {
  Span first, last, own;
};
__device__ __forceinline__ Spans spans_of(const CausalArgs& a, int first, int last, int w0, int w1, int token) {
  const int length = (int)a.length;
  if (!a.offsets) return Spans{{0, length}, {0, length}, {0, length}};
  const int at[3] = {first, last, w0};
  int n[3];
  bounds_before<3>(a, at, n);
  Spans s{span_at(a, first, n[0]), span_at(a, last, n[1]), {token + 1, token}};
  // the wave's tokens: one sequence after the other
  int before = n[2], lo = before ? (int)bound(a, before - 1, length) : 0;
  while (true) {
    const int hi = before <= a.sequences ? (int)bound(a, before, length) : length;
    if (before > 0 && before <= a.sequences && token >= lo && token < hi) s.own = Span{lo, hi};
    if (hi > w1 || before > a.sequences) break;
    lo = hi;
    ++before;
  }
  return s;
}

// eight of the accumulator's registers as the other operand
template <typename T>
__device__ __forceinline__ Frag<T> pack(const f32x16& x, int m) {
  if constexpr (sizeof(T) == 2) {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (T)x[8 * m + i];
    return f;
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[8 * m + i];
    return split3<false>(v);
  }
}
// what the rounding of pack took away (16-bit types)
template <typename T>
__device__ __forceinline__ Frag<T> pack_rest(const f32x16& x, int m, const Frag<T>& f) {
  Frag<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[8 * m + i] - (float)f[i];
    r[i] = (T)(__builtin_isfinite(d) ? d : 0.f);
  }
  return r;
}

// float32: a score that holds an infinity has met the other operand's lower terms, of either sign, and is NaN; such a
// score is taken from the largest terms alone, where it is what the formula has.  first(): those products' sum.
template <typename First>
__device__ __forceinline__ void mend_scores(f32x16& s, First first) {
  float t = s[0];
#pragma unroll
  for (int j = 1; j < 16; ++j) t += s[j];
  if (__any(t != t)) {
    const f32x16 f = first();
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = s[j] != s[j] ? f[j] : s[j];
  }
}

// x, as a value that the compiler does not know more about: what is computed from it stays where it is written (it would
// else keep sixteen sums in registers, or in scratch, for masked tiles to come)
__device__ __forceinline__ uint32_t here(int x) {
  asm volatile("" : "+v"(x));
  return (uint32_t)x;
}
// The scores' factor, in log2 units.  A scale of zero is a product too small to count, that leaves the masked pairs' -inf
// one; one that is NaN stays it.
__device__ __forceinline__ float score_factor(const CausalArgs& a) {
  const float c = a.scale * kLog2e;
  return c < 0x1p-120f ? 0x1p-120f : c;
}
// sum + the elements of f, a fragment of 16 bits (two a step)
template <typename T>
__device__ __forceinline__ float add_elements(const Frag<T>& f, float sum) {
  using P2 = typename fast::Pair<T>::v2;
  P2 x[4], ones;
  __builtin_memcpy(x, &f, sizeof(f));
  ones[0] = ones[1] = (T)1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = fast::Pair<T>::dot(x[i], ones, sum);
  return sum;
}

// ---- tiles where some pairs are masked
//
// A masked pair's weight is 0, but 0 times an infinity or a NaN in the tile
// is NaN.  So a tile that is not whole for every wave of the workgroup is looked
// through first (all threads, once: 1/256 of it each); where it holds such an
// element, what these add to the pairs that are not masked is added to the
// accumulators one by one, and they become zeros in LDS.
template <typename T> struct Bits;
template <> struct Bits<__bf16> { static constexpr uint32_t kExp = 0x7F80u; };
template <> struct Bits<_Float16> { static constexpr uint32_t kExp = 0x7C00u; };
// two elements of 16 bits, zero where they are not finite
template <typename T>
__device__ __forceinline__ uint32_t finite_word(uint32_t u) {
  constexpr uint32_t e = Bits<T>::kExp;
  const uint32_t lo = (u & e) == e ? 0u : u & 0xFFFFu;
  return (u >> 16 & e) == e ? lo : lo | (u & 0xFFFF0000u);
}
template <typename TL, typename T>
__device__ __forceinline__ bool tile_non_finite(const char* tile) {
  bool bad = false;
#pragma unroll 2
  for (int i = 0; i < TL::kChunks / 4; ++i) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile + TL::nth(i * 256 + threadIdx.x));
    bad |= ((u.x ^ finite_word<T>(u.x)) | (u.y ^ finite_word<T>(u.y)) | (u.z ^ finite_word<T>(u.z)) | (u.w ^ finite_word<T>(u.w))) != 0;
  }
  return bad;
}
// the tile's rows with such elements, as bits (two words of LDS, written by all threads)
template <typename TL, typename T>
__device__ __forceinline__ uint64_t rows_non_finite(const char* tile, uint32_t* words) {
  if (threadIdx.x < 2) words[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < TL::kChunks / 4; ++i) {
    const uint4 u = *reinterpret_cast<const uint4*>(tile + TL::nth(i * 256 + threadIdx.x));
    const int row = (i * 256 + (int)threadIdx.x) / TL::kPieces;
    if (((u.x ^ finite_word<T>(u.x)) | (u.y ^ finite_word<T>(u.y)) | (u.z ^ finite_word<T>(u.z)) | (u.w ^ finite_word<T>(u.w))) != 0)
      atomicOr(&words[row >> 5], 1u << (row & 31));
  }
  __syncthreads();
  return fast::uniform64((uint64_t)words[1] << 32 | words[0]);
}
template <typename TL, typename T>
__device__ __forceinline__ void clean_tile(char* tile) {
#pragma unroll 1
  for (int i = 0; i < TL::kChunks / 4; ++i) {
    uint4& u = *reinterpret_cast<uint4*>(tile + TL::nth(i * 256 + threadIdx.x));
    u = make_uint4(finite_word<T>(u.x), finite_word<T>(u.y), finite_word<T>(u.z), finite_word<T>(u.w));
  }
}
// SIGNED: the weights are positive, an infinity stays one (acc must not be rescaled for this tile any more); else what is not
// finite makes NaN.  keep(row): whether the
// tile's row is paired with this lane's column.
template <typename TL, bool SIGNED, int NDT, typename Keep>
__device__ __forceinline__ void add_non_finite(f32x16 (&acc)[NDT], const char* tile, int g, Keep keep) {
#pragma unroll 1
  for (int r = 0; r < TL::kRows; ++r) {
    const bool pair = keep(r);
#pragma unroll
    for (int t = 0; t < NDT; ++t) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float x = TL::element(tile, r, 32 * t + kappa(g, j));
        if (pair && !__builtin_isfinite(x)) acc[t][j] += SIGNED ? x : __builtin_nanf("");
      }
      asm volatile("" ::: "memory");  // (few of these rare reads in flight: they would take registers from the loop)
    }
  }
}

// A 32 x 32 accumulator tile (rows: elements d0 ..+31, this lane's column: one row of the result) to row[d0 ..], times
// s, where below `size`; `low` (16-bit types, optional) takes what the rounding left.
template <typename T>
__device__ __forceinline__ void store_columns(char* row, int d0, int size, int g, const f32x16& acc, float s, char* low = nullptr) {
  if constexpr (sizeof(T) == 2) {
    f32x16 y;
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = acc[j] * s;
    fast::store_tile<T>(reinterpret_cast<T*>(row), d0, size, g, y, 1.0f);
    if (low) {
      // (an infinity or a NaN leaves no remainder)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float r = y[j] - (float)(T)y[j];
        y[j] = __builtin_isfinite(r) ? r : 0.f;
      }
      fast::store_tile<T>(reinterpret_cast<T*>(low), d0, size, g, y, 1.0f);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = d0 + 8 * q + 4 * g;
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[4 * q + i] * s;
      if (d < size) *reinterpret_cast<f32x4*>(row + d * 4) = v;
    }
  }
}

// Workgroup `id` of `heads` (batch, head) pairs: the longest blocks first, and, where the heads can be dealt evenly, those
// of one XCD (workgroups id % 8) next to each other, so that heads that share keys meet in one L2.  rank counts the
// blocks from the heaviest.
struct Work {
  int head, rank;
};
__device__ __forceinline__ Work work_of(uint32_t id, uint32_t heads) {
  if (heads % kNumXcds == 0) {
    const uint32_t per = heads / kNumXcds, x = id % kNumXcds, r = id / kNumXcds;
    return Work{(int)(x * per + r % per), (int)(r / per)};
  }
  return Work{(int)(id % heads), (int)(id / heads)};
}

}  // namespace causal
}  // namespace oops
