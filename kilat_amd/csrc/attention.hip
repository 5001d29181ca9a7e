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

// What the matrix instructions take for inputs of type T: 16-bit types as they are,
// float32 as three bfloat16 terms (matrix.h), products kept to 2^-24.
template <typename T>
struct Op {
  typedef T E;
  static constexpr int N = 1, ORDER = 0;
};
template <>
struct Op<float> {
  typedef __bf16 E;
  static constexpr int N = 3, ORDER = 2;
};

__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <typename E>
struct Vec8;
template <>
struct Vec8<__bf16> {
  typedef bf16x8 type;
  typedef bf16x4 half;
};
template <>
struct Vec8<_Float16> {
  typedef f16x8 type;
  typedef _Float16 half __attribute__((ext_vector_type(4)));
};

// Eight values of an operand, by terms.
template <typename T>
struct Operand {
  typedef typename Vec8<typename Op<T>::E>::type V;
  V t[Op<T>::N];
};

template <typename T>
__device__ __forceinline__ Operand<T> to_operand(const float (&x)[8]) {
  Operand<T> r;
  if constexpr (Op<T>::N == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.t[0][i] = (T)x[i];
  } else {
    const Terms<3> s = split<3>(x);
#pragma unroll
    for (int i = 0; i < 3; ++i) r.t[i] = s.t[i];
  }
  return r;
}

template <typename T>
__device__ __forceinline__ f32x16 product32(const Operand<T>& a, const Operand<T>& b, f32x16 acc) {
  constexpr int N = Op<T>::N;
#pragma unroll
  for (int s = Op<T>::ORDER; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (s - i >= 0 && s - i < N) acc = mfma32(a.t[i], b.t[s - i >= 0 && s - i < N ? s - i : 0], acc);
  return acc;
}

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
template <typename T>
__device__ __forceinline__ void load_row8(const T* base, int64_t at, int n, float (&x)[8]) {
  const f32x4 a = load4(base, at, n), b = load4(base, at + 4, n - 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// KS: steps of 16 channels of q and k; VT: tiles of 32 channels of v.
template <typename T, int KS, int VT>
__global__ __launch_bounds__(kThreads) void forward(Args a) {
  typedef typename Op<T>::E E;
  typedef typename Vec8<E>::half E4;
  constexpr int N = Op<T>::N;
  __shared__ E ks[N][2 * KS * kTile];  // keys: two tiles of 32 keys, KS steps
  __shared__ E vs[N][4 * VT * kTile];  // values, transposed: VT tiles of 32 channels, four steps of 16 keys
  __shared__ int odd;                  // a value of a step that masks keys is not finite
  const int64_t tile = blockIdx.x;
  const int h = blockIdx.y, hk = h / a.group;
  const int tid = threadIdx.x, w = tid / 64, lane = tid & 63, n32 = lane & 31, half = lane >> 5;
  zero_outside<BQ>(a.cu, a.sequences, tile, a.N, (T*)a.o + h * a.oh, a.on, a.Dv, tid, kThreads);
  const TileOf at = tile_of<BQ>(a.cu, a.sequences, tile, a.N);
  const int64_t q0 = at.index * BQ;
  if (at.rows.n <= q0) return;
  const T* kp = (const T*)a.k + at.rows.batch * a.kb + hk * a.kh + at.rows.first * a.kn;
  const T* vp = (const T*)a.v + at.rows.batch * a.vb + hk * a.vh + at.rows.first * a.vn;
  const int64_t row = q0 + 32 * w + n32;  // of the sequence
  const bool live = row < at.rows.n;
  Operand<T> q[KS];
  {
    const T* p = (const T*)a.q + at.rows.batch * a.qb + h * a.qh + at.rows.first * a.qn;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8];
      load_row8(p, row * a.qn + 16 * s + 8 * half, live ? a.Dk - 16 * s - 8 * half : 0, x);
      q[s] = to_operand<T>(x);
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
    __syncthreads();
    if (tid == 0) odd = 0;
    // keys
    for (int i = tid; i < BK * 2 * KS; i += kThreads) {
      const int key = i / (2 * KS), c = i % (2 * KS);
      float x[8];
      load_row8(kp, (k0 + key) * a.kn + 8 * c, k0 + key < at.rows.n ? a.Dk - 8 * c : 0, x);
      const Operand<T> y = to_operand<T>(x);
      const int slot = ((key & 31) + 32 * (c & 1)) ^ (c & 15);
#pragma unroll
      for (int t = 0; t < N; ++t)
        *reinterpret_cast<typename Operand<T>::V*>(&ks[t][((key >> 5) * KS + (c >> 1)) * kTile + slot * 8]) = y.t[t];
    }
    __syncthreads();
    // values: four keys of four channels at a time, transposed
    for (int i = tid; i < (BK / 4) * 8 * VT; i += kThreads) {
      const int kg = i / (8 * VT), c = (i % (8 * VT)) * 4;
      f32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t key = k0 + 4 * kg + j;
        x[j] = load4(vp, key * a.vn + c, key < at.rows.n ? a.Dv - c : 0);
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
          E4 e;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (t + 1 < N) {
              const float u = upper_half(y[j]);
              e[j] = (E)u;
              y[j] -= u;
            } else {
              e[j] = (E)y[j];
            }
          }
          *reinterpret_cast<E4*>(&vs[t][at8]) = e;
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
        Operand<T> x;
#pragma unroll
        for (int y = 0; y < N; ++y)
          x.t[y] = *reinterpret_cast<const typename Operand<T>::V*>(
              &ks[y][(t * KS + s) * kTile + (lane ^ ((2 * s + half) & 15)) * 8]);
        S[t] = product32<T>(x, q[s], S[t]);
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t key = k0 + 32 * t + 8 * (r >> 2) + 4 * half + (r & 3);
        if (masked && key > row) S[t][r] = -INFINITY;
        S[t][r] *= to2;
        top = fmaxf(top, S[t][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 32));
    const float m1 = fmaxf(m, top), base = m1 == -INFINITY ? 0.f : m1;
    if (__any(m1 > m)) {
      const float f = exp2f(m - base);
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
        p[r] = exp2f(S[t][r] - base);
        l += p[r];
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float x[8] = {p[8 * s], p[8 * s + 1], p[8 * s + 2], p[8 * s + 3], p[8 * s + 4], p[8 * s + 5], p[8 * s + 6], p[8 * s + 7]};
        const Operand<T> pt = to_operand<T>(x);
#pragma unroll
        for (int vt = 0; vt < VT; ++vt) {
          Operand<T> y;
#pragma unroll
          for (int z = 0; z < N; ++z)
            y.t[z] = *reinterpret_cast<const typename Operand<T>::V*>(&vs[z][(vt * 4 + 2 * t + s) * kTile + lane * 8]);
          O[vt] = product32<T>(y, pt, O[vt]);
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
  T* p = (T*)a.o + at.rows.batch * a.ob + h * a.oh + (at.rows.first + row) * a.on;
#pragma unroll
  for (int vt = 0; vt < VT; ++vt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * vt + 2 * r + 4 * half;
      const f32x4 x = {O[vt][r] / l, O[vt][r + 1] / l, O[vt][r + 2] / l, O[vt][r + 3] / l};
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
  if (p->sequences > 0x7fffffff || tiles_of<32>(p) > 0x7fffffff)
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
    const dim3 grid((unsigned)a.tiles, a.H);
    const hipStream_t s = (hipStream_t)stream;
    if (a.Dk <= 64 && a.Dv <= 64)
      forward<T, 4, 2><<<grid, kThreads, 0, s>>>(a);
    else if (a.Dk <= 64)
      forward<T, 4, 4><<<grid, kThreads, 0, s>>>(a);
    else if (a.Dv <= 64)
      forward<T, 8, 2><<<grid, kThreads, 0, s>>>(a);
    else
      forward<T, 8, 4><<<grid, kThreads, 0, s>>>(a);
    return hip_check("kattn_fwd launch");
  };
  if (p->dtype == KDECAY_BF16) return launch((__bf16*)nullptr);
  if (p->dtype == KDECAY_F16) return launch((_Float16*)nullptr);
  return launch((float*)nullptr);
}
