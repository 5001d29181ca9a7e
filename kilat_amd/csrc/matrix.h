// matrix.h — tiles for the matrix instructions: how the kernels of the gated delta
// rule and of attention lay operands out in registers, and how they carry 32-bit
// values through 16-bit products.
//
// v_mfma_f32_16x16x32_*: D[16x16] += A[16x32] B[32x16].  Lane l holds row l%16 of
// A (column l%16 of B) at eight of the 32 inner indices, and of D column l%16 at rows
// 4(l/16) .. +3.  The order of the inner index is free as long as A and B agree,
// so lane group g = l/16 takes the indices 4g..4g+3 and 16+4g..16+4g+3: then
// two D tiles, one above the other, are a B operand of the next product as they
// stand (or an A operand, transposed), with no exchange between lanes.
#pragma once

#include "kdecay_internal.h"

namespace kd {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// A 32-bit value as a sum of N bfloat16 terms.  Every term but the last keeps
// the upper half of what is left (exact: the difference has no more digits), the
// last one rounds to nearest: 1 term is the rounding to bfloat16 (exact for
// bfloat16 inputs), 2 are exact for float16 inputs and otherwise off by at most
// 2^-17 relative, 3 hold all 24 digits of a float32.
template <int N>
struct Terms {
  bf16x8 t[N];
};

// The upper halves of a and b, a's in the lower half.
__device__ __forceinline__ unsigned upper_halves(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

__device__ __forceinline__ float upper_half(float a) { return __uint_as_float(__float_as_uint(a) & 0xffff0000u); }

template <int N>
__device__ __forceinline__ Terms<N> split(const float (&x)[8]) {
  Terms<N> r;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x[i];
#pragma unroll
  for (int n = 0; n + 1 < N; ++n) {
    unsigned w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = upper_halves(y[2 * i], y[2 * i + 1]);
    r.t[n] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] -= upper_half(y[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) r.t[N - 1][i] = (__bf16)y[i];
  return r;
}

template <int N>
__device__ __forceinline__ Terms<N> split(f32x4 a, f32x4 b) {
  const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return split<N>(x);
}

// acc += A B over the terms of both: the products whose terms' places add up to at
// most ORDER, smallest first.  ORDER 2 leaves out what is below 2^-24 of the
// product, ORDER 1 what is below 2^-16.
template <int ORDER, int NA, int NB>
__device__ __forceinline__ f32x4 product(const Terms<NA>& a, const Terms<NB>& b, f32x4 acc) {
#pragma unroll
  for (int s = ORDER; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) acc = mfma(a.t[i], b.t[s - i < NB ? (s - i >= 0 ? s - i : 0) : 0], acc);
  return acc;
}

// Terms that an input of type T has, exactly.
template <typename T>
inline constexpr int kInputTerms = 3;
template <>
inline constexpr int kInputTerms<__bf16> = 1;
template <>
inline constexpr int kInputTerms<_Float16> = 2;

// p[0..3] as floats, zero from element n on.  vec: p is aligned to four elements.
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int64_t n, bool vec) {
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
  if (vec && n >= 4) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T4 x = *reinterpret_cast<const T4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (float)x[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) r[i] = (float)p[i];
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 x, int64_t n, bool vec) {
  if (vec && n >= 4) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (T)x[i];
    *reinterpret_cast<T4*>(p) = y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = (T)x[i];
  }
}

// One lane's eight values of a row: inner indices k0 + 4g + i and k0 + 16 + 4g + i, zero
// from index `width` on.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int k0, int g, int width, bool vec, float (&x)[8]) {
  const int a = k0 + 4 * g;
  const f32x4 lo = load4(row + a, width - a, vec), hi = load4(row + a + 16, width - a - 16, vec);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = lo[i], x[4 + i] = hi[i];
}

// Sum over the four lane groups (lanes l, l^16, l^32, l^48).
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// The rows of one sequence: cu == null for sequence s of rows 0..N-1 of batch
// entry s, else rows cu[s]..cu[s+1] of batch entry 0, whatever cu holds inside 0..N.
struct Rows {
  int64_t first;
  int64_t n;
  int64_t batch;
};

__device__ __forceinline__ int64_t clamp_row(int64_t x, int64_t N) { return x < 0 ? 0 : x > N ? N : x; }

__device__ __forceinline__ Rows rows_of(const int32_t* cu, int64_t s, int64_t N) {
  if (!cu) return Rows{0, N, s};
  const int64_t a = clamp_row(cu[s], N), b = clamp_row(cu[s + 1], N);
  return Rows{a, b > a ? b - a : 0, 0};
}

// Tiles of C rows are numbered so that a kernel finds its rows without a list of the
// sequences' tiles: sequence s of a packed batch starts at tile first / C + s. That
// leaves room for ceil(n / C) tiles before the next one, and N / C + sequences
// tiles hold all of them.
struct TileOf {
  int64_t seq;
  int64_t index;  // of the sequence's tiles
  Rows rows;
};

template <int C>
__device__ __forceinline__ int64_t first_tile(const int32_t* cu, int64_t s, const Rows& r, int64_t N) {
  return cu ? r.first / C + s : s * ((N + C - 1) / C);
}

// Tile `tile`, by bisection; rows.n <= index * C where it is none.
template <int C>
__device__ __forceinline__ TileOf tile_of(const int32_t* cu, int64_t sequences, int64_t tile, int64_t N) {
  int64_t s;
  if (!cu) {
    s = tile / ((N + C - 1) / C);
  } else {
    int64_t lo = 0, hi = sequences;  // the last s whose first tile is not behind `tile`
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (clamp_row(cu[mid], N) / C + mid <= tile)
        lo = mid;
      else
        hi = mid;
    }
    s = lo;
  }
  const Rows r = rows_of(cu, s, N);
  return TileOf{s, tile - first_tile<C>(cu, s, r, N), r};
}

template <int C>
inline int64_t tile_count(const int32_t* cu, int64_t B, int64_t N, int64_t sequences) {
  return cu ? N / C + sequences : B * ((N + C - 1) / C);
}

// Zeroes columns col .. col + step*... of the rows C*tile.. of batch entry 0 that belong to no
// sequence of a packed batch.  The tiles of a packed batch are at least as many
// as the rows' own, so one call per tile reaches every row.
template <int C, typename T>
__device__ __forceinline__ void zero_outside(const int32_t* cu, int64_t sequences, int64_t tile, int64_t N, T* x,
                                             int64_t row_stride, int width, int thread, int threads) {
  if (!cu || tile * C >= N) return;
  const int64_t lo = clamp_row(cu[0], N), hi = clamp_row(cu[sequences], N);
  const int64_t end = tile * C + C < N ? tile * C + C : N;
  if (tile * C >= lo && end <= hi) return;
  for (int64_t r = tile * C; r < end; ++r)
    if (r < lo || r >= hi)
      for (int d = thread; d < width; d += threads) x[r * row_stride + d] = (T)0.f;
}

}  // namespace kd
