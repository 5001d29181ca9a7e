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

// The same for M accumulators with one B each: neighbouring instructions are independent of each
// other (one that adds to the result of the one before it waits for it).
template <int ORDER, int M, int NA, int NB>
__device__ __forceinline__ void products(const Terms<NA> (&a)[M], const Terms<NB>& b, f32x4* acc) {
#pragma unroll
  for (int s = ORDER; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB)
#pragma unroll
        for (int m = 0; m < M; ++m) acc[m] = mfma(a[m].t[i], b.t[s - i >= 0 && s - i < NB ? s - i : 0], acc[m]);
}

// Terms that an input of type T has, exactly.
template <typename T>
inline constexpr int kInputTerms = 3;
template <>
inline constexpr int kInputTerms<__bf16> = 1;
template <>
inline constexpr int kInputTerms<_Float16> = 2;

// Rows are whole eights of elements, aligned to 16 bytes (the hosts' checks and copies see to it),
// so four or eight elements are all there or none of them is: n, the elements left, is 0 or less,
// or 4 (8) or more.
template <typename T>
using Raw4 = T __attribute__((ext_vector_type(4)));

template <typename T>
using Raw8 = T __attribute__((ext_vector_type(8)));

// Loads that are to stay in flight: no branch that depends on the lane, and no conversion,
// until the values are used.  base itself is read where there is nothing to read.
template <typename T>
__device__ __forceinline__ Raw4<T> fetch4(const T* base, int64_t at, int n) {
  return *reinterpret_cast<const Raw4<T>*>(base + (n > 0 ? at : 0));
}

template <typename T>
__device__ __forceinline__ Raw8<T> fetch8(const T* base, int64_t at, int n) {
  return *reinterpret_cast<const Raw8<T>*>(base + (n > 0 ? at : 0));
}

template <typename T>
__device__ __forceinline__ f32x4 fetched(Raw4<T> x, int n) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = n > 0 ? (float)x[i] : 0.f;
  return r;
}

template <typename T>
__device__ __forceinline__ f32x4 load4(const T* base, int64_t at, int n) {
  return fetched<T>(fetch4(base, at, n), n);
}

template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4 x) {
  Raw4<T> y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (T)x[i];
  *reinterpret_cast<Raw4<T>*>(p) = y;
}

// Results of matrix instructions are written up to 16 passes after they issue, and nothing in
// the hardware holds back an instruction that reads or overwrites them earlier.  The
// compiler keeps the distance inside a basic block only (measured: a loop-carried
// accumulator copied at the head of the next block held its old value), so results
// that are used, or whose registers are reused, behind a branch, barrier or loop end are settled
// first.
__device__ __forceinline__ void settle(f32x4& x) { asm volatile("s_nop 7\n\ts_nop 7" : "+v"(x)); }
__device__ __forceinline__ void settle(f32x16& x) { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" : "+v"(x)); }
template <typename V, int N>
__device__ __forceinline__ void settle(V (&x)[N]) {
#pragma unroll
  for (int i = 1; i < N; ++i) asm volatile("" : "+v"(x[i]));
  settle(x[0]);
}

typedef __attribute__((address_space(3))) void* LdsPtr;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// 16 bytes per lane from global memory to LDS, at `to` + 16 lane.  In assembly, because the compiler
// takes the LDS that its own form of it writes for any LDS that is read later, and
// waits for rows that are still to come before it reads those that are there; who
// calls this waits itself (lds_copies_done, then a barrier).  (M0 has no other use in these kernels.)
__device__ __forceinline__ void copy_to_lds(const void* from, const void* to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(LdsPtr)(void*)to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory");
}
__device__ __forceinline__ void lds_copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Eight bytes per lane, transposed among each 16 lanes: these read four rows of 16 16-bit values (lane j
// the four at row j / 4, columns 4 (j % 4)..), and lane j gets column j's four.
__device__ __forceinline__ u32x2 read_transposed(const void* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(LdsPtr)(void*)p));
}

// The wavefront's number in its workgroup, known to the compiler to be one for all its
// lanes: branches on it are scalar, and barriers behind them are reached by whole wavefronts.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64); }

// 2^x, by the instruction.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

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

// Tile `tile`; rows.n <= index * C where it is none.  A wavefront probes 64 sequences at a time: one round of
// loads for up to 64 of them, two for up to 4096 (bisection takes six and twelve, one behind the
// other, of a microsecond or so each where the offsets are not in the L2).
template <int C>
__device__ __forceinline__ TileOf tile_of(const int32_t* cu, int64_t sequences, int64_t tile, int64_t N) {
  int64_t s;
  if (!cu) {
    s = (unsigned)tile / (unsigned)((N + C - 1) / C);  // (tiles are fewer than 2^31)
  } else {
    int64_t lo = 0, count = sequences;  // the last s whose first tile is not behind `tile` is one of these
    const int lane = threadIdx.x & 63;
    while (count > 1) {
      const int64_t step = (count + 63) / 64, at = lane * step;
      const bool ahead = at < count && clamp_row(cu[lo + (at < count ? at : 0)], N) / C + lo + at <= tile;
      const int last = 63 - __clzll(__ballot(lane == 0 || ahead));
      lo += last * step;
      count = count - last * step < step ? count - last * step : step;
    }
    s = lo;
  }
  const Rows r = rows_of(cu, s, N);
  const int64_t index = tile - first_tile<C>(cu, s, r, N);
  return index < 0 ? TileOf{s, 0, Rows{r.first, 0, r.batch}} : TileOf{s, index, r};  // (before the first sequence)
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

// The hosts' check of one tensor of rows: channels adjacent, every row aligned to 16 bytes.
inline int check_rows(const void* p, const int64_t* strides, int dtype, const char* name) {
  if (strides[3] != 1) return fail(KDECAY_ELAYOUT, "%s: channel (d) stride must be 1", name);
  const int n = dtype == KDECAY_F32 ? 4 : 8;
  if (((uintptr_t)p & 15u) || strides[0] % n || strides[1] % n || strides[2] % n)
    return fail(KDECAY_ELAYOUT, "%s: base and strides must be multiples of 16 bytes", name);
  return 0;
}

}  // namespace kd
