// attention.hip — causal attention over whole prompts (include/kattn.h).
//
//     o_i = sum_{j <= i} exp(x_ij - m_i) v_j / sum_{j <= i} exp(x_ij - m_i),   x_ij = scale q_i.k_j
//
// in one pass over the keys, with the running maximum m_i and sum of every row.  A
// workgroup has 128 rows of one head, 32 per wavefront, and goes through the keys
// 64 at a time, through LDS.  Scores are computed transposed (keys are the rows of
// the matrix instruction's result, queries its columns), so that a lane holds
// scores of one query only: the maximum takes one exchange between two lanes, the
// factor that rescales earlier sums none, and the probabilities are the next
// product's operand as they stand.
#include "matrix.h"

#include "kattn.h"

namespace kd {
namespace attn {

constexpr int BQ = 128;  // rows of a workgroup
constexpr int BK = 64;   // keys of a step
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 512;  // values of one operand tile (64 lanes of 8)

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <typename T>
struct Vec8;
template <>
struct Vec8<__bf16> {
  typedef bf16x8 type;
};
template <>
struct Vec8<_Float16> {
  typedef f16x8 type;
};

// A product of float32 operands as three bfloat16 terms each (matrix.h), kept to 2^-24.
__device__ __forceinline__ f32x16 product32(const Terms<3>& a, const Terms<3>& b, f32x16 acc) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i) acc = mfma32(a.t[i], b.t[s - i], acc);
  return acc;
}

template <int N>
struct Int {
  static constexpr int value = N;
};

struct Args {
  const void *q, *k, *v;
  void* o;
  const int32_t* cu;
  int64_t qb, qh, qn, kb, kh, kn, vb, vh, vn, ob, oh, on;
  int64_t N, sequences, tiles;
  int H, Dk, Dv, group;
  float scale;
};

// Eight elements from base + at, n of them there.
__device__ __forceinline__ void load_row8(const float* base, int64_t at, int n, float (&x)[8]) {
  const f32x4 a = load4(base, at, n), b = load4(base, at + 4, n - 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

template <bool B>
struct Bool {
  static constexpr bool value = B;
};

// float32: rows pass registers, where they are split into terms.  Six matrix instructions for one, and as many
// vector instructions for the splits: 16 heads of 4096 rows, Dk = Dv = 64: 401 us, 86 TFLOP/s of
// float32; 128: 912 us, 75 (a large product of torch's in float32 reaches 154).  Two workgroups per CU
// where registers allow (Dv <= 64): 546 us with one.
// KS: steps of 16 channels of q and k; VT: tiles of 32 channels of v.
template <int KS, int VT>
__global__ __launch_bounds__(kThreads, VT == 2 ? 2 : 1) void forward(Args a) {
  constexpr int N = 3;  // terms
  __shared__ __bf16 ks[N][2 * KS * kTile];  // keys: two tiles of 32 keys, KS steps
  __shared__ __bf16 vs[N][4 * VT * kTile];  // values, transposed: VT tiles of 32 channels, four steps of 16 keys
  __shared__ int odd;                  // a value of a step that masks keys is not finite
  const int64_t tile = a.tiles - 1 - blockIdx.x;  // a sequence's last rows, which have the most keys, first
  const int h = blockIdx.y, hk = h / a.group;
  const int tid = threadIdx.x, w = tid / 64, lane = tid & 63, n32 = lane & 31, half = lane >> 5;
  zero_outside<BQ>(a.cu, a.sequences, tile, a.N, (float*)a.o + h * a.oh, a.on, a.Dv, tid, kThreads);
  const TileOf at = tile_of<BQ>(a.cu, a.sequences, tile, a.N);
  const int64_t q0 = at.index * BQ;
  if (at.rows.n <= q0) return;
  const float* kp = (const float*)a.k + at.rows.batch * a.kb + hk * a.kh + at.rows.first * a.kn;
  const float* vp = (const float*)a.v + at.rows.batch * a.vb + hk * a.vh + at.rows.first * a.vn;
  const int64_t row = q0 + 32 * w + n32;  // of the sequence
  const bool live = row < at.rows.n;
  Terms<3> q[KS];
  {
    const float* p = (const float*)a.q + at.rows.batch * a.qb + h * a.qh + at.rows.first * a.qn;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load_row8(p, row * a.qn + 16 * s + 8 * half, live ? a.Dk - 16 * s - 8 * half : 0, x);
      q[s] = split<3>(x);
    }
  }
  f32x16 O[VT];
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[t][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float to2 = a.scale * 1.44269504088896340736f;  // scores in powers of 2
  const int64_t last = q0 + BQ < at.rows.n ? q0 + BQ : at.rows.n;
  for (int64_t k0 = 0; k0 < last; k0 += BK) {
    const bool masked = k0 + BK > q0;  // keys behind some row, or behind the sequence
    // All of the step's loads first: one wait for memory.
    constexpr int KI = BK * 2 * KS / kThreads, VI = BK / 4 * 8 * VT / kThreads;
    Raw8<float> kr[KI];
    Raw4<float> vr[VI][4];
#pragma unroll
    for (int x = 0; x < KI; ++x) {
      const int i = tid + x * kThreads, key = i / (2 * KS), c = i % (2 * KS);
      kr[x] = fetch8(kp, (k0 + key) * a.kn + 8 * c, k0 + key < at.rows.n ? a.Dk - 8 * c : 0);
    }
#pragma unroll
    for (int x = 0; x < VI; ++x) {
      const int i = tid + x * kThreads, kg = i / (8 * VT), c = (i % (8 * VT)) * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t key = k0 + 4 * kg + j;
        vr[x][j] = fetch4(vp, key * a.vn + c, key < at.rows.n ? a.Dv - c : 0);
      }
    }
    __syncthreads();
    if (tid == 0) odd = 0;
    // keys
#pragma unroll
    for (int z = 0; z < KI; ++z) {
      const int i = tid + z * kThreads, key = i / (2 * KS), c = i % (2 * KS);
      const bool there = k0 + key < at.rows.n && a.Dk > 8 * c;
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = there ? (float)kr[z][j] : 0.f;
      const Terms<3> y = split<3>(x);
      const int slot = ((key & 31) + 32 * (c & 1)) ^ (c & 15);
#pragma unroll
      for (int t = 0; t < N; ++t)
        *reinterpret_cast<bf16x8*>(&ks[t][((key >> 5) * KS + (c >> 1)) * kTile + slot * 8]) = y.t[t];
    }
    __syncthreads();
    // values: four keys of four channels at a time, transposed
#pragma unroll
    for (int z = 0; z < VI; ++z) {
      const int i = tid + z * kThreads, kg = i / (8 * VT), c = (i % (8 * VT)) * 4;
      f32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t key = k0 + 4 * kg + j;
        x[j] = fetched<float>(vr[z][j], key < at.rows.n ? a.Dv - c : 0);
        if (masked) {
#pragma unroll
          for (int d = 0; d < 4; ++d)
            if (!finite(x[j][d])) x[j][d] = 0.f, odd = 1;
        }
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        // channel c + d, keys 4 kg ..: step kg / 4, lane half kg & 1, upper or lower four
        const int slot = ((c + d) & 31) + 32 * (kg & 1);
        const int at8 = (((c + d) >> 5) * 4 + (kg >> 2)) * kTile + slot * 8 + 4 * ((kg >> 1) & 1);
        float y[4] = {x[0][d], x[1][d], x[2][d], x[3][d]};
#pragma unroll
        for (int t = 0; t < N; ++t) {
          bf16x4 e;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (t + 1 < N) {
              const float u = upper_half(y[j]);
              e[j] = (__bf16)u;
              y[j] -= u;
            } else {
              e[j] = (__bf16)y[j];
            }
          }
          *reinterpret_cast<bf16x4*>(&vs[t][at8]) = e;
        }
      }
    }
    __syncthreads();
    if (k0 > q0 + 32 * w + 31) continue;  // every key is behind this wavefront's rows
    f32x16 S[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        Terms<3> x;
#pragma unroll
        for (int y = 0; y < N; ++y)
          x.t[y] = *reinterpret_cast<const bf16x8*>(
              &ks[y][(t * KS + s) * kTile + (lane ^ ((2 * s + half) & 15)) * 8]);
        S[t] = product32(x, q[s], S[t]);
      }
    }
    float top = -INFINITY;
    const int upto = (int)(row - k0) - 4 * half;  // the last key that the row sees
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        S[t][r] *= to2;
        if (masked) S[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) <= upto ? S[t][r] : -INFINITY;
        top = fmaxf(top, S[t][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m1 = fmaxf(m, top), base = m1 == -INFINITY ? 0.f : m1;
    if (__any(m1 > m)) {
      const float f = exp2_fast(m - base);
      l *= f;
#pragma unroll
      for (int t = 0; t < VT; ++t) O[t] *= f;
      m = m1;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = exp2_fast(S[t][r] - base);
        l += p[r];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float x[8] = {p[8 * s], p[8 * s + 1], p[8 * s + 2], p[8 * s + 3], p[8 * s + 4], p[8 * s + 5], p[8 * s + 6], p[8 * s + 7]};
        const Terms<3> pt = split<3>(x);
#pragma unroll
        for (int vt = 0; vt < VT; ++vt) {
          Terms<3> y;
#pragma unroll
          for (int z = 0; z < N; ++z)
            y.t[z] = *reinterpret_cast<const bf16x8*>(&vs[z][(vt * 4 + 2 * t + s) * kTile + lane * 8]);
          O[vt] = product32(y, pt, O[vt]);
        }
      }
    }
    if (masked && odd) {
      // Values that are not finite were taken as 0; they count for the rows from their own on only.
      for (int key = 0; key < BK; ++key)
        if (k0 + key <= row && k0 + key < at.rows.n)
#pragma unroll
          for (int vt = 0; vt < VT; ++vt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int c = 32 * vt + 8 * (r >> 2) + 4 * half + (r & 3);
              const float x = c < a.Dv ? (float)vp[(k0 + key) * a.vn + c] : 0.f;
              if (!finite(x)) O[vt][r] += x;
            }
    }
  }
  l += __shfl_xor(l, 32);
  if (!live) return;
  float* p = (float*)a.o + at.rows.batch * a.ob + h * a.oh + (at.rows.first + row) * a.on;
#pragma unroll
  for (int vt = 0; vt < VT; ++vt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * vt + 2 * r + 4 * half;
      const f32x4 x = {O[vt][r] / l, O[vt][r + 1] / l, O[vt][r + 2] / l, O[vt][r + 3] / l};
      if (c < a.Dv) store4(p + c, x);
    }
}

// --------------------------------------------------------------------------
// 16-bit types
// --------------------------------------------------------------------------
// Keys and values go from global memory to LDS without passing registers, the next 64
// rows while these are computed on (two buffers, one barrier per step), as rows of
// 16-byte chunks; a row's chunks are permuted by an exclusive or with its number, so
// that neither the 32 rows that a key operand reads nor the eight that a value
// operand reads lie in the same banks.  Values are transposed by the LDS read.
//
// Bound by vector issue beside the matrix instructions: per 64 keys and 32 rows a wavefront issues 240 vector
// instructions, 32 of them exponentials at a quarter of the rate, for 16 (Dk = Dv = 64) or 32 (128)
// matrix instructions.  16384 rows, 16 heads (4 key heads), 128, bfloat16: 1342 us, 820 TFLOP/s (a large matrix
// product of torch's reaches 1222); eight sequences of 1024 rows, 6 heads, 64: 23.8 us, of which the
// longest rows' 8 rounds of twice 64 keys take 12 and the launch 6.
template <int CPR, bool VALUES>
__device__ __forceinline__ int swizzle(int row) {
  if (VALUES) return CPR == 16 ? (row & 3) << 2 : (row & 2) << 1;  // four rows by four adjacent chunks
  return CPR == 16 ? row & 15 : (row >> 1) & 7;                    // 16 rows by one chunk
}

// The halves of a word that are infinite or NaN, as masks of 16 bits.
template <typename T>
__device__ __forceinline__ unsigned not_finite(unsigned x) {
  constexpr unsigned top = __is_same(T, __bf16) ? 0x00800080u : 0x04000400u;
  return (((x & 0x7fff7fffu) + top) >> 15 & 0x00010001u) * 0xffffu;
}

// One wavefront's share of a tile of 64 rows of CPR chunks: NL instructions of 64 chunks.
template <typename T, int CPR, bool VALUES>
struct Stage {
  static constexpr int NL = CPR / kWaves;
  const T* p[NL];
  int row[NL];
  bool on[NL];  // the channels are the tensor's, not the tile's padding
  __device__ __forceinline__ void init(const T* base, int64_t stride, int width, int w, int lane) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = (w * NL + i) * 64 + lane, chunk = c % CPR;
      row[i] = c / CPR;
      const int d = (chunk ^ swizzle<CPR, VALUES>(row[i])) * 8;
      on[i] = d < width;
      p[i] = base + row[i] * stride + d;
    }
  }
  // Rows k0.. of n, into `to`; rows behind the last are copies of it.
  // The next call's are G steps on.
  template <int G>
  __device__ __forceinline__ void load(T* to, int64_t k0, int64_t n, int64_t stride, int w) {
    if (k0 + BK <= n) {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (on[i]) copy_to_lds(p[i], to + (w * NL + i) * 512);
    } else {
      const int last = (int)(n - 1 - k0);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int over = row[i] > last ? row[i] - last : 0;
        if (on[i]) copy_to_lds(p[i] - over * stride, to + (w * NL + i) * 512);
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) p[i] += G * BK * stride;
  }
  // Zeroes what is not finite in this wavefront's share; whether there was any.
  __device__ __forceinline__ bool clean(T* at, int w, int lane) {
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      uint4* x = reinterpret_cast<uint4*>(at + (w * NL + i) * 512 + lane * 8);
      const uint4 y = *x;
      const unsigned a = not_finite<T>(y.x), b = not_finite<T>(y.y), c = not_finite<T>(y.z), d = not_finite<T>(y.w);
      if (a | b | c | d) *x = make_uint4(y.x & ~a, y.y & ~b, y.z & ~c, y.w & ~d);
      bad |= a | b | c | d;
    }
    return __any(bad);
  }
};

// The larger of x in this lane and in the one 32 from it.
__device__ __forceinline__ float max_of_halves(float x) {
  const unsigned y = __float_as_uint(x);
  const auto z = __builtin_amdgcn_permlane32_swap(y, y, false, false);
  return fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
}

// What the `order`-th workgroup of a head takes in a packed batch of up to 64 sequences: the longest
// sequence's tiles first, each sequence's last tile first, so that what is left at the end
// is short.  A lane has a sequence.
__device__ __forceinline__ TileOf longest_first(const Args& a, int64_t order, int lane) {
  const Rows rows = lane < a.sequences ? rows_of(a.cu, lane, a.N) : Rows{0, 0, 0};
  const int tiles = (int)((rows.n + BQ - 1) / BQ);  // (fewer than 2^31)
  int before = 0;                                   // tiles of longer sequences
  for (int s = 0; s < (int)a.sequences; ++s) {
    const int other = __builtin_amdgcn_readlane(tiles, s);
    before += other > tiles || (other == tiles && s < lane) ? other : 0;
  }
  const unsigned long long found = __ballot(order >= before && order < before + tiles);
  const int s = found ? __ffsll(found) - 1 : 0;
  const auto of = [&](int64_t x) {
    return (int64_t)(((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), s) << 32) |
                     (unsigned)__builtin_amdgcn_readlane((int)x, s));
  };
  return TileOf{s, found ? of(before + tiles - 1 - order) : 0, Rows{of(rows.first), found ? of(rows.n) : 0, 0}};
}

template <typename T, int KS, int VT, int G>
__global__ __launch_bounds__(kThreads * G, 2) void forward16(Args a) {
  typedef typename Vec8<T>::type V8;
  constexpr int KC = 2 * KS, VC = 4 * VT;  // chunks of a row
  constexpr int kKeys = BK * KC * 8, kValues = BK * VC * 8;
  __shared__ __align__(16) T lds[G * 2 * (kKeys + kValues)];
  __shared__ int odd[G][2];  // the last step with a masked key in the buffer and a value that is not finite
  // Workgroups go to the eight XCDs in turn.  With a multiple of eight heads each XCD has heads of
  // its own, so the keys that its workgroups read at the same time are the same; the tiles
  // with the most keys go first.
  const unsigned id = blockIdx.x, H = a.H, tiles = (unsigned)a.tiles;
  const unsigned per = a.H % 8 ? H : H / 8, lane_of = a.H % 8 ? id : id / 8;
  const unsigned order = lane_of / per;
  const int h = (int)((a.H % 8 ? 0 : id % 8 * per) + lane_of % per);
  int64_t tile = tiles - 1 - order;
  if (!a.cu) {
    const unsigned seqs = (unsigned)a.sequences, each = tiles / seqs;
    tile = order % seqs * (int64_t)each + (each - 1 - order / seqs);
  }
  const int hk = h / a.group;
  const int tid = threadIdx.x, lane = tid & 63, n32 = lane & 31, half = lane >> 5;
  const int part = G == 1 ? 0 : wave_index() / kWaves, w = wave_index() % kWaves;  // steps part, part + G, ...; rows 32w..
  T *kbuf = lds + part * 2 * (kKeys + kValues), *vbuf = kbuf + 2 * kKeys;
  zero_outside<BQ>(a.cu, a.sequences, tile, a.N, (T*)a.o + h * a.oh, a.on, a.Dv, tid, kThreads * G);
  const TileOf at = a.cu && a.sequences <= 64 ? longest_first(a, order, lane) : tile_of<BQ>(a.cu, a.sequences, tile, a.N);
  const int64_t q0 = at.index * BQ, n = at.rows.n;
  if (n <= q0) return;
  const T* kp = (const T*)a.k + at.rows.batch * a.kb + hk * a.kh + at.rows.first * a.kn;
  const T* vp = (const T*)a.v + at.rows.batch * a.vb + hk * a.vh + at.rows.first * a.vn;
  if (a.Dk < KS * 16 || a.Dv < VT * 32) {  // padding chunks are zero throughout
    for (int i = tid; i < G * 2 * BK * (KC + VC); i += kThreads * G) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  Stage<T, KC, false> sk;
  Stage<T, VC, true> sv;
  sk.init(kp + part * BK * a.kn, a.kn, a.Dk, w, lane);
  sv.init(vp + part * BK * a.vn, a.vn, a.Dv, w, lane);
  sk.template load<G>(kbuf, part * BK, n, a.kn, w);
  sv.template load<G>(vbuf, part * BK, n, a.vn, w);
  const int64_t row = q0 + 32 * w + n32;  // of the sequence
  const bool live = row < n;
  const bool flip = a.scale < 0.f;  // scores of -q and the scale's size
  V8 q[KS];
  {
    const T* p = (const T*)a.q + at.rows.batch * a.qb + h * a.qh + at.rows.first * a.qn;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int left = live ? a.Dk - 16 * s - 8 * half : 0;
      const Raw8<T> x = fetch8(p, row * a.qn + 16 * s + 8 * half, left);
      uint4 y = __builtin_bit_cast(uint4, x);
      const unsigned sign = flip ? 0x80008000u : 0u;
      y = left > 0 ? make_uint4(y.x ^ sign, y.y ^ sign, y.z ^ sign, y.w ^ sign) : make_uint4(0, 0, 0, 0);
      q[s] = __builtin_bit_cast(V8, y);
      if (a.scale == 0.f) q[s] *= (T)0.f;  // (scores of 0, or NaN: `to2` is 1 then)
    }
  }
  // Where this lane reads: key operands, row n32 of a tile of 32, chunk 2s + half; value operands, by
  // 16 lanes, four keys (of half's four) of 16 channels.
  const int kat = n32 * KC * 16, kx = half ^ swizzle<KC, false>(n32);
  const int j = lane & 15, vrow = 4 * half + (j >> 2);
  const int vat = vrow * VC * 16 + (j & 1) * 8, vx = (2 * ((lane >> 4) & 1) + ((j >> 1) & 1)) ^ swizzle<VC, true>(vrow);
  f32x16 O[VT];
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) O[t][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (tid < 2 * G) odd[tid / 2][tid % 2] = -1;
  __syncthreads();
  const float to2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.44269504088896340736f;  // scores in powers of 2
  const int64_t last = q0 + BQ < n ? q0 + BQ : n;
  const int steps = (int)((last + BK - 1) / BK), mine = (int)((q0 + 32 * w + 32 + BK - 1) / BK);  // of this wavefront's rows

  const auto step = [&](int i, auto masked_of) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_of)::value;
    const char* kl = reinterpret_cast<const char*>(kbuf + (G == 1 ? i & 1 : i / G & 1) * kKeys);
    const char* vl = reinterpret_cast<const char*>(vbuf + (G == 1 ? i & 1 : i / G & 1) * kValues);
    const int seen = masked ? (int)(row - (int64_t)i * BK) : 0, upto = seen - 4 * half;  // the last key that the row sees
    f32x16 S[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[t][r] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        S[t] = mfma32(*reinterpret_cast<const V8*>(kl + t * 32 * KC * 16 + kat + ((kx ^ (2 * s)) << 4)), q[s], S[t]);
    if (masked) settle(S);
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (masked) S[t][r] = 32 * t + 8 * (r >> 2) + (r & 3) <= upto ? S[t][r] : -INFINITY;
        top = fmaxf(top, S[t][r]);
      }
    top = max_of_halves(top) * to2;
    // The maximum that is subtracted may be up to 8 (in powers of 2) below the true one: sums stay
    // far from 32 bits' end, and the rescaling of earlier sums is rare.
    // (Row by row: what one row's scores are changes no digit of another's result.)
    const bool raise = top > m + 8.f || (m == -INFINITY && top > m);
    if (__any(raise)) {
      const float m1 = raise ? top : m, f = !raise ? 1.f : m == -INFINITY ? 0.f : exp2_fast(m - m1);
      l *= f;
#pragma unroll
      for (int t = 0; t < VT; ++t) O[t] *= f;
      m = m1;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        V8 p;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float x = exp2_fast(fmaf(S[t][8 * s + r], to2, -base));
          l += x;
          p[r] = (T)x;
        }
#pragma unroll
        for (int vt = 0; vt < VT; ++vt) {
          u32x2 y[2];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            y[b] = read_transposed(vl + (32 * t + 16 * s + 8 * b) * VC * 16 + vat + ((vx ^ (4 * vt)) << 4));
          const uint4 z = make_uint4(y[0].x, y[0].y, y[1].x, y[1].y);
          O[vt] = mfma32(__builtin_bit_cast(V8, z), p, O[vt]);
        }
      }
    }
    settle(O);
    if (masked) {
      if (__builtin_amdgcn_readfirstlane(odd[part][i / G & 1]) == i) {
        // Values that are not finite were taken as 0: they count for the rows from their own on only.
        const int64_t k0 = (int64_t)i * BK;
        for (int key = 0; key < BK; ++key)
          if (key <= seen && k0 + key < n)
#pragma unroll
            for (int vt = 0; vt < VT; ++vt)
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                const int c = 32 * vt + 8 * (r >> 2) + 4 * half + (r & 3);
                const float x = c < a.Dv ? (float)vp[(k0 + key) * a.vn + c] : 0.f;
                if (!finite(x)) O[vt][r] += x;
              }
      }
    }
  };
  for (int it = 0; it * G < steps; ++it) {
    const int i = it * G + part;
    lds_copies_done();  // this wavefront's rows of the step are in LDS
    // Where some row does not see some key, values that are not finite become 0 (0 times one is none
    // either); each wavefront looks at the rows that it has copied.
    if ((int64_t)(i + 1) * BK > q0 && sv.clean(vbuf + (G == 1 ? i & 1 : i / G & 1) * kValues, w, lane) && lane == 0)
      odd[part][i / G & 1] = i;
    __syncthreads();
    if (i + G < steps) {
      sk.template load<G>(kbuf + ((it + 1) & 1) * kKeys, (int64_t)(i + G) * BK, n, a.kn, w);
      sv.template load<G>(vbuf + ((it + 1) & 1) * kValues, (int64_t)(i + G) * BK, n, a.vn, w);
    }
    if (i >= mine) continue;  // every key is behind this wavefront's rows
    const int64_t end = (int64_t)(i + 1) * BK;
    if (end <= q0 || (end <= q0 + 32 * w && __builtin_amdgcn_readfirstlane(odd[part][i / G & 1]) != i))
      step(i, Bool<false>());
    else
      step(i, Bool<true>());
  }
  settle(O);
  l += __shfl_xor(l, 32);
  if (G > 1) {
    // The other part's sums, through LDS, to the larger maximum of the two.
    f32x4* sums = reinterpret_cast<f32x4*>(lds) + w * (4 * VT * 64);
    float2* ends = reinterpret_cast<float2*>(reinterpret_cast<f32x4*>(lds) + kWaves * 4 * VT * 64) + w * 64;
    __syncthreads();  // what lds held is read
    if (part == 1) {
#pragma unroll
      for (int vt = 0; vt < VT; ++vt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          sums[(vt * 4 + r) * 64 + lane] = f32x4{O[vt][4 * r], O[vt][4 * r + 1], O[vt][4 * r + 2], O[vt][4 * r + 3]};
      ends[lane] = make_float2(m, l);
    }
    __syncthreads();
    if (part == 1) return;
    const float2 y = ends[lane];
    const float top = fmaxf(m, y.x), base = top == -INFINITY ? 0.f : top;
    const float f0 = exp2_fast(m - base), f1 = exp2_fast(y.x - base);
    l = l * f0 + y.y * f1;
#pragma unroll
    for (int vt = 0; vt < VT; ++vt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const f32x4 x = sums[(vt * 4 + r) * 64 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) O[vt][4 * r + i] = O[vt][4 * r + i] * f0 + x[i] * f1;
      }
  }
  if (!live) return;
  T* p = (T*)a.o + at.rows.batch * a.ob + h * a.oh + (at.rows.first + row) * a.on;
  const float il = 1.f / l;
#pragma unroll
  for (int vt = 0; vt < VT; ++vt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * vt + 2 * r + 4 * half;
      const f32x4 x = {O[vt][r] * il, O[vt][r + 1] * il, O[vt][r + 2] * il, O[vt][r + 3] * il};
      if (c < a.Dv) store4(p + c, x);
    }
}

template <int BLOCK>
int64_t tiles_of(const kattn_problem* p) {
  return p->cu_seqlens ? p->N / BLOCK + p->sequences : p->B * ((p->N + BLOCK - 1) / BLOCK);
}

int check(const kattn_problem* p, const void* o, const int64_t* o_strides) {
  if (!p) return fail(KDECAY_EINVAL, "null problem");
  if (p->B < 0 || p->Hk < 0 || p->H < 0 || p->N < 0 || p->Dk < 0 || p->Dv < 0 || p->sequences < 0)
    return fail(KDECAY_EINVAL, "negative size");
  if (p->dtype != KDECAY_F32 && p->dtype != KDECAY_BF16 && p->dtype != KDECAY_F16)
    return fail(KDECAY_EDTYPE, "q, k and v must be float32, bfloat16 or float16 (code %d)", p->dtype);
  if (p->Dk < 1 || p->Dk > KATTN_MAX_DK || p->Dv < 1 || p->Dv > KATTN_MAX_DV)
    return fail(KDECAY_ESHAPE, "head dims Dk=%lld, Dv=%lld are not 1..%d and 1..%d", (long long)p->Dk,
                (long long)p->Dv, KATTN_MAX_DK, KATTN_MAX_DV);
  if (p->Hk < 1 || p->H < 1 || p->H % p->Hk)
    return fail(KDECAY_ESHAPE, "H=%lld is no multiple of Hk=%lld", (long long)p->H, (long long)p->Hk);
  if (p->H > 65535) return fail(KDECAY_ESHAPE, "more than 65535 heads");
  if (p->cu_seqlens && (p->B != 1 || p->sequences < 1))
    return fail(KDECAY_ESHAPE, "cu_seqlens takes B=1 and at least one sequence");
  if (!p->cu_seqlens && p->sequences != p->B) return fail(KDECAY_EINVAL, "sequences must be B without cu_seqlens");
  if (p->sequences > 0x7fffffff || tiles_of<BQ>(p) * p->H > 0x7fffffff)
    return fail(KDECAY_ESHAPE, "too many sequences or rows");
  if (p->Dk % 8 || p->Dv % 8)
    return fail(KDECAY_ESHAPE, "head dims Dk=%lld, Dv=%lld are not multiples of 8", (long long)p->Dk, (long long)p->Dv);
  if (!p->B || !p->N) return 0;
  if (!p->q || !p->k || !p->v || !o || !o_strides) return fail(KDECAY_EINVAL, "null pointer argument");
  if (const int rc = check_rows(p->q, p->q_strides, p->dtype, "q")) return rc;
  if (const int rc = check_rows(p->k, p->k_strides, p->dtype, "k")) return rc;
  if (const int rc = check_rows(p->v, p->v_strides, p->dtype, "v")) return rc;
  if (const int rc = check_rows(o, o_strides, p->dtype, "o")) return rc;
  return 0;
}

}  // namespace attn
}  // namespace kd

using namespace kd;
using namespace kd::attn;

extern "C" int kattn_fwd(const kattn_problem* p, void* o, const int64_t* o_strides, void* stream) {
  if (const int rc = check(p, o, o_strides)) return rc;
  if (!p->B || !p->N) return 0;
  Args a = {};
  a.q = p->q, a.k = p->k, a.v = p->v, a.o = o, a.cu = p->cu_seqlens;
  a.qb = p->q_strides[0], a.qh = p->q_strides[1], a.qn = p->q_strides[2];
  a.kb = p->k_strides[0], a.kh = p->k_strides[1], a.kn = p->k_strides[2];
  a.vb = p->v_strides[0], a.vh = p->v_strides[1], a.vn = p->v_strides[2];
  a.ob = o_strides[0], a.oh = o_strides[1], a.on = o_strides[2];
  a.N = p->N, a.sequences = p->sequences, a.tiles = tiles_of<BQ>(p);
  a.H = (int)p->H, a.Dk = (int)p->Dk, a.Dv = (int)p->Dv, a.group = (int)(p->H / p->Hk);
  a.scale = p->scale;
  const auto launch = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const hipStream_t s = (hipStream_t)stream;
    const auto with = [&](auto ks, auto vt) {
      constexpr int KS = decltype(ks)::value, VT = decltype(vt)::value;
      if constexpr (sizeof(T) == 2)
        // Keys in two parts where no compute unit has more than two workgroups: 16 heads of 4096 rows (512
        // workgroups), Dk = Dv = 64: 66 us, else 92; 128: 112 and 148.  With more, the units are full, and
        // the joining counts: 12 heads of eight sequences of 1024 rows (768), 64: 40 us, else 32.
        if (a.tiles * a.H <= 512)
          forward16<T, KS, VT, 2><<<dim3((unsigned)(a.tiles * a.H)), kThreads * 2, 0, s>>>(a);
        else
          forward16<T, KS, VT, 1><<<dim3((unsigned)(a.tiles * a.H)), kThreads, 0, s>>>(a);
      else
        forward<KS, VT><<<dim3((unsigned)a.tiles, a.H), kThreads, 0, s>>>(a);
    };
    if (a.Dk <= 64 && a.Dv <= 64)
      with(Int<4>(), Int<2>());
    else if (a.Dk <= 64)
      with(Int<4>(), Int<4>());
    else if (a.Dv <= 64)
      with(Int<8>(), Int<2>());
    else
      with(Int<8>(), Int<4>());
    return hip_check("kattn_fwd launch");
  };
  if (p->dtype == KDECAY_BF16) return launch((__bf16*)nullptr);
  if (p->dtype == KDECAY_F16) return launch((_Float16*)nullptr);
  return launch((float*)nullptr);
}
