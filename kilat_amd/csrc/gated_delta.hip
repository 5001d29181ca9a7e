// gated_delta.hip — the gated delta rule (include/kdelta.h).
//
// Per head, S_t = a_t (S_{t-1} - b_t k_t (k_t' S_{t-1})) + b_t k_t v_t', o_t = scale S_t' q_t.
// What token t writes is k_t u_t' with u_t = b_t (v_t - a_t S_{t-1}' k_t), so over a chunk
// of 64 tokens that starts from S, with G_i = g_1 + .. + g_i inside the chunk,
//
//     (I + A) U = R,   R_i = b_i (v_i - e^{G_i} S' k_i),   A_ij = b_i e^{G_i - G_j} k_i.k_j  (j < i)
//     o_i = scale e^{G_i} S' q_i + sum_{j <= i} P_ij u_j,  P_ij = scale e^{G_i - G_j} q_i.k_j
//     S  <- e^{G_64} S + sum_j e^{G_64 - G_j} k_j u_j'
//
// T = (I + A)^-1 and P do not depend on S: prep() computes them for every chunk
// at once.  chain() then goes through a sequence's chunks; a wavefront keeps
// 16 columns of S in registers and needs no other wavefront: every product
// above leaves those columns where they are.
#include "matrix.h"

#include "kdelta.h"

namespace kd {
namespace delta {

constexpr int C = 64;       // tokens of a chunk
constexpr int NX = 3;       // terms of a 32-bit value that reaches the state or a gradient
constexpr int kFrag = 512;  // bfloat16 values of one operand tile (64 lanes of 8)
// An operand with zeros above its diagonal of 16-row tiles: tiles of rows 0, 1 need
// the first 32 inner indices only (transposed: rows 2, 3 the last 32 only).
constexpr int kTri = 6;
__host__ __device__ constexpr int tri_lower(int mt, int kb) { return mt < 2 ? mt : 2 * (mt - 1) + kb; }
__host__ __device__ constexpr int tri_upper(int mt, int kb) { return mt < 2 ? 2 * mt + kb : mt + 2; }

// Terms of P, and products kept, in what reaches o only.
template <typename T>
constexpr int kOutTerms = sizeof(T) == 4 ? 3 : 2;
template <typename T>
constexpr int kOutOrder = sizeof(T) == 4 ? 2 : 1;

// Per token of a chunk, floats: b e^G, b, e^G, e^(G_64 - G), and G log2(e) as the sum of two.
enum Vec { V_BG, V_BETA, V_SINCE, V_LEFT, V_G, V_GLOW, V_COUNT };
constexpr int V_CHAIN = 4;  // what chain() reads of them

struct Args {
  const void *q, *k, *v;
  const float *g, *beta;
  const int32_t* cu;
  const float* init;
  int64_t qb, qh, qn, kb, kh, kn, vb, vh, vn, gb, gh, gn, bb, bh, bn;
  int64_t N, sequences, tiles;
  int Hk, H, Dk, Dv, group;  // group: value heads of a key head
  int blocks, groups;        // blocks of 32 columns of v, and their groups of 16
  float scale;
  // scratch, by tile and head
  __bf16* tris;     // [tiles][H][kTri * (NX + kOutTerms)][kFrag]: T and P (backward: [kTri * NX], T's transpose)
  float* vecs;      // [tiles][H][V_COUNT][C]
  // Kept for the backward, as planes of terms (see plane_at): S at the chunk's start and u, saved
  __bf16* states;   // [tiles][H][blocks][NX][32][32 KB]
  __bf16* us;       // [tiles][H][blocks][NX][32][C]
  void* o;
  int64_t ob, oh, on;
  float* final;
  // A sequence in `segs` pieces (1: whole): per sequence, head and piece, the state that
  // a piece leaves of zero, how it carries a state over (planes, by its columns), and its first state
  int segs;
  float *seg_n, *seg_s;  // [sequences][H][segs][groups][2 KB][64][4]
  __bf16* seg_m;         // [sequences][H][segs][KB][NX][32][32 KB]
  // backward
  const void* d_o;
  int64_t dob, doh, don;
  const float* d_final;
  float* d_init;
  float* ys;        // [tiles][H][groups][4][64][4]: P' dO, as it lies in registers
  float* zs;        // [tiles][H][groups][2 KB][64][4]: scale Q' (e^G dO)
  __bf16* dstates;  // like states: the gradient of the state at the chunk's end
  __bf16* drs;      // like us: the gradient of R
  void *dq, *dk, *dv;
  int64_t dqb, dqh, dqn, dkb, dkh, dkn, dvb, dvh, dvn;
  float *dg, *dbeta;
};

// The channel of k that row r of the 16-row tile dt of a state (or of K transposed) is. In steps of 32,
// the order in which lane group g's eight inner indices of an operand, tiles 2kb and 2kb+1 of
// a state, are the channels 8g..8g+7: an operand of k's rows is loaded as they lie.
__host__ __device__ constexpr int channel(int dt, int r) { return 32 * (dt >> 1) + 8 * (r >> 2) + 4 * (dt & 1) + (r & 3); }

template <typename T, bool BWD>
constexpr int kTriSize = kTri * (NX + (BWD ? 0 : kOutTerms<T>)) * kFrag;
template <typename T, bool BWD>
__device__ __forceinline__ __bf16* tri_tiles(const Args& a, int64_t tile, int h) {
  return a.tris + (tile * a.H + h) * (int64_t)kTriSize<T, BWD>;
}
__device__ __forceinline__ float* vec_of(const Args& a, int64_t tile, int h) {
  return a.vecs + (tile * a.H + h) * (int64_t)(V_COUNT * C);
}

// States, u and the gradient of R are kept for grads() as 16-bit planes, one per term, of 32
// columns: rows are the columns, and in a row lie the channels (tokens) in order, in
// chunks of eight.  So a wavefront that has 16 columns writes chunks, and the
// transposing LDS read gives operands whose inner index is the column.  A row's
// chunks are permuted by an exclusive or with its number, so that the 16 rows that
// one such read takes lie in different banks.
template <int KB>
__device__ __forceinline__ int plane_swizzle(int row) {
  const int a = (row >> 3) & 1;
  return KB == 2 ? 2 * (((row >> 1) & 1) | a << 1) : KB == 4 ? 2 * ((row & 3) | a << 2) : 2 * a;
}
// Element of row `row`, channel (token) `at`, in a plane of 32 KB of them per row.
template <int KB>
__device__ __forceinline__ int plane_at(int row, int at) {
  return row * 32 * KB + (((at >> 3) ^ plane_swizzle<KB>(row)) << 3) + (at & 7);
}
// Operand with rows 16 rt + lane % 16 of the channels (tokens), inner indices the 32 columns.
template <int KB>
__device__ __forceinline__ Terms<NX> load_plane(const __bf16* planes, int rt, int lane) {
  const int j = lane & 15, row = 8 * (lane >> 4) + (j >> 2);
  Terms<NX> r;
#pragma unroll
  for (int n = 0; n < NX; ++n) {
    const __bf16* p = planes + n * 32 * 32 * KB;
    const u32x2 a = read_transposed(p + plane_at<KB>(row, 16 * rt + 4 * (j & 3)));
    const u32x2 b = read_transposed(p + plane_at<KB>(row + 4, 16 * rt + 4 * (j & 3)));
    r.t[n] = __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
  }
  return r;
}
// A wavefront's 16 columns (group cg) of `x`, rows in the order of registers, as terms to their planes.
template <int KB>  // x: a state's terms
__device__ __forceinline__ void keep_state(__bf16* planes, int cg, int m, int g, const Terms<NX> (&x)[KB]) {
  const int row = 16 * (cg & 1) + m;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int n = 0; n < NX; ++n)
      *reinterpret_cast<bf16x8*>(planes + n * 32 * 32 * KB + plane_at<KB>(row, 32 * kb + 8 * g)) = x[kb].t[n];
}
__device__ __forceinline__ void keep_rows(__bf16* planes, int cg, int m, int g, const Terms<NX> (&x)[2]) {
  const int row = 16 * (cg & 1) + m;
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int n = 0; n < NX; ++n) {
      const uint4 y = __builtin_bit_cast(uint4, x[kb].t[n]);
      __bf16* p = planes + n * 32 * C;
      *reinterpret_cast<u32x2*>(p + plane_at<2>(row, 32 * kb + 4 * g)) = u32x2{y.x, y.y};
      *reinterpret_cast<u32x2*>(p + plane_at<2>(row, 32 * kb + 16 + 4 * g)) = u32x2{y.z, y.w};
    }
}
// The planes of a tile, head and block of 32 columns.
template <int KB>
__device__ __forceinline__ int64_t planes_of(const Args& a, int64_t tile, int h, int block) {
  return ((tile * a.H + h) * a.blocks + block) * (int64_t)(NX * 32 * 32 * KB);
}

template <int N>
__device__ __forceinline__ Terms<N> load_terms(const __bf16* p, int lane) {
  Terms<N> r;
#pragma unroll
  for (int n = 0; n < N; ++n) r.t[n] = *reinterpret_cast<const bf16x8*>(p + n * kFrag + lane * 8);
  return r;
}
template <int N>
__device__ __forceinline__ void store_terms(__bf16* p, int lane, const Terms<N>& x) {
#pragma unroll
  for (int n = 0; n < N; ++n) *reinterpret_cast<bf16x8*>(p + n * kFrag + lane * 8) = x.t[n];
}

// The terms of one lane's fetched eight of a row, of which there are n (0 or less, or 8).
template <typename T>
__device__ __forceinline__ Terms<kInputTerms<T>> terms_of(Raw8<T> x, int n) {
  if constexpr (kInputTerms<T> == 1) {
    const uint4 y = __builtin_bit_cast(uint4, x);
    Terms<1> r;
    r.t[0] = __builtin_bit_cast(bf16x8, make_uint4(n > 0 ? y.x : 0u, n > 0 ? y.y : 0u, n > 0 ? y.z : 0u, n > 0 ? y.w : 0u));
    return r;
  } else {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = n > 0 ? (float)x[i] : 0.f;
    return split<kInputTerms<T>>(y);
  }
}

// A product with one of these picks 16 of an operand's 32 inner indices as they are: rows that lie
// along lanes come out along registers, so it transposes a tile.  This one picks index `inner` in
// the result's column m.
__device__ __forceinline__ bf16x8 selector(int inner, int g) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (__bf16)(8 * g + i == inner ? 1.f : 0.f);
  return r;
}

// A barrier that orders LDS accesses only: loads from global memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// e^x for a difference of sums of log decays (positive for a growing state only).
__device__ __forceinline__ float fade(double x) {
  const float hi = (float)x, e = expf(hi);
  return fmaf(e, (float)(x - (double)hi), e);
}

// --------------------------------------------------------------------------
// prep: T of one chunk and value head (BWD: what the backward's products take)
// --------------------------------------------------------------------------
// Grid (tiles, H), four wavefronts; wavefront w has tokens 16w..16w+15 of the chunk.
// Forward: T and P, as operand tiles of terms.  BWD: T transposed, and what of the gradients does
// not depend on a state: P' dO and scale Q' (e^G dO).
//
// log decays are added up in 64 bits: the sums over a chunk can be far larger than
// the differences that count.  One below -128 is taken as -128: e^-128 is 0 in 32 bits,
// and no difference becomes inf - inf.
//
// Bound by the latency of one workgroup's own steps (loads, K K', the inverse by tiles, stores) and, on
// full grids, by memory: B=8 H=12 N=4096 D=64 bfloat16, 6144 tiles, takes 72 us for 290 MB
// (4.0 TB/s), BWD 140 us for 460 MB (3.3); 768 tiles (one round of workgroups) take 14 us.
template <typename T, int KB, bool BWD>
__global__ __launch_bounds__(256) void prep(Args a) {
  constexpr int NI = kInputTerms<T>;
  constexpr int LD = C + 4;
  constexpr int kKeys = 4 * KB * NI * kFrag, kQt = 4 * KB * NX * kFrag, kDo = 8 * NI * kFrag;
  // K (and Q); BWD: later Q transposed and 64 columns of dO transposed
  __shared__ __align__(16) __bf16 kq[!BWD ? kKeys : 2 * kKeys > kQt + kDo ? 2 * kKeys : kQt + kDo];
  __shared__ __align__(16) float As[C * LD], Ts[C * LD];
  __shared__ __align__(16) float Gh[C], Gl[C], bs[C], es[C];  // G log2(e) as the sum of two, b, e^G
  const int64_t tile = blockIdx.x;
  const int h = blockIdx.y, hk = h / a.group;
  const int w = wave_index(), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  if (!BWD)
    zero_outside<C>(a.cu, a.sequences, tile, a.N, (T*)a.o + h * a.oh, a.on, a.Dv, threadIdx.x, 256);
  else
    zero_outside<C>(a.cu, a.sequences, tile, a.N, (T*)a.dv + h * a.dvh, a.dvn, a.Dv, threadIdx.x, 256);
  const TileOf at = tile_of<C>(a.cu, a.sequences, tile, a.N);
  const int64_t left_rows = at.rows.n - at.index * C;
  if (left_rows <= 0) return;
  const int n = left_rows < C ? (int)left_rows : C;
  const int64_t row0 = at.rows.first + at.index * C;
  // Operand tiles of K (and Q): lane (m, g) has token 16w + m.
  const int t = 16 * w + m;
  const T* kbase = (const T*)a.k + at.rows.batch * a.kb + hk * a.kh + row0 * a.kn;
  const T* qbase = (const T*)a.q + at.rows.batch * a.qb + hk * a.qh + row0 * a.qn;
  Raw8<T> kr[KB], qr[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int d = 32 * kb + 8 * g, left = t < n ? a.Dk - d : 0;
    kr[kb] = fetch8(kbase, t * a.kn + d, left);
    qr[kb] = fetch8(qbase, t * a.qn + d, left);
  }
  if (w == 0) {
    const bool in = lane < n;
    double G = 0.;
    float b = 0.f;
    if (in) {
      const float x = a.g[at.rows.batch * a.gb + h * a.gh + (row0 + lane) * a.gn];
      G = x < -128.f ? -128. : (double)x;
      b = a.beta[at.rows.batch * a.bb + h * a.bh + (row0 + lane) * a.bn];
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const double y = __shfl_up(G, d);
      if (lane >= d) G += y;
    }
    const double all = __shfl(G, 63);
    float* vec = vec_of(a, tile, h);
    const float since = fade(G);
    vec[V_BG * C + lane] = b * since;
    vec[V_BETA * C + lane] = b;
    vec[V_SINCE * C + lane] = since;
    vec[V_LEFT * C + lane] = fade(all - G);
    const double G2 = G * 1.4426950408889634074;
    const float high = (float)G2, low = (float)(G2 - (double)high);
    vec[V_G * C + lane] = high;
    vec[V_GLOW * C + lane] = low;
    Gh[lane] = high, Gl[lane] = low, bs[lane] = b, es[lane] = since;
  }
  Terms<NI> kt[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int left = t < n ? a.Dk - 32 * kb - 8 * g : 0;
    kt[kb] = terms_of<T>(kr[kb], left);
    store_terms<NI>(kq + (w * KB + kb) * NI * kFrag, lane, kt[kb]);
    if constexpr (BWD) store_terms<NI>(kq + kKeys + (w * KB + kb) * NI * kFrag, lane, terms_of<T>(qr[kb], left));
  }
  __syncthreads();
  // A and P, with one e^{G_i - G_j} for both: lane m has this wavefront's token t as i and the rows of the
  // result as j (BWD: t as j, rows as i).  Differences of the high parts are exact where they count, so an
  // exponential is off by its own rounding (1 to 2 units of 2^-24) only.
  Terms<BWD ? NX : 1> pt[2] = {};  // BWD: P transposed
  {
    const float gh = Gh[t], gl = Gl[t], bt = bs[t];
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2) {
      if (BWD ? kb2 < w / 2 : kb2 > w / 2) continue;
      f32x4 p[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, aa[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        Terms<NI> y[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) y[x] = load_terms<NI>(kq + ((2 * kb2 + x) * KB + kb) * NI * kFrag, lane);
        products<2>(y, kt[kb], aa);
        if constexpr (BWD) {
#pragma unroll
          for (int x = 0; x < 2; ++x) y[x] = load_terms<NI>(kq + kKeys + ((2 * kb2 + x) * KB + kb) * NI * kFrag, lane);
          products<2>(y, kt[kb], p);
        } else {
          products<2>(y, terms_of<T>(qr[kb], t < n ? a.Dk - 32 * kb - 8 * g : 0), p);
        }
      }
      settle(p), settle(aa);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int o = 32 * kb2 + 16 * x + 4 * g;
        const f32x4 oh = *reinterpret_cast<const f32x4*>(Gh + o), ol = *reinterpret_cast<const f32x4*>(Gl + o);
        const f32x4 ob = *reinterpret_cast<const f32x4*>(bs + o);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = BWD ? o + r : t, j = BWD ? t : o + r;
          const float d = BWD ? (oh[r] - gh) + (ol[r] - gl) : (gh - oh[r]) + (gl - ol[r]), e = exp2_fast(d);
          p[x][r] = j <= i ? a.scale * e * p[x][r] : 0.f;
          aa[x][r] = j < i ? (BWD ? ob[r] : bt) * e * aa[x][r] : 0.f;
          if (BWD) As[i * LD + j] = aa[x][r];
        }
        if (!BWD) *reinterpret_cast<f32x4*>(As + t * LD + o) = aa[x];
      }
      if constexpr (BWD) {
        pt[kb2] = split<NX>(p[0], p[1]);
      } else {
        constexpr int NO = kOutTerms<T>;
        store_terms<NO>(tri_tiles<T, false>(a, tile, h) + (kTri * NX + tri_lower(w, kb2) * NO) * kFrag, lane, split<NO>(p[0], p[1]));
      }
    }
  }
  __syncthreads();
  // T = (I + A)^-1.  The 16 x 16 diagonal blocks by forward substitution, a column per
  // lane; below them T_ij = -T_ii sum_k A_ik T_kj, in 32-bit products.
  {
    float x[16];
    const float* A = As + (16 * w) * LD + 16 * w;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == m ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-A[i * LD + j], x[j], s);
      x[i] = s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i / 4 == g) Ts[(16 * w + i) * LD + 16 * w + m] = x[i];
    for (int jt = w + 1; jt < 4; ++jt)  // zeros above
#pragma unroll
      for (int i = 0; i < 4; ++i) Ts[(16 * w + 4 * g + i) * LD + 16 * jt + m] = 0.f;
  }
  __syncthreads();
  {
    f32x4 col[4];  // T's tiles of columns 16w.., rows w..3
#pragma unroll
    for (int x = 0; x < 4; ++x) col[0][x] = Ts[(16 * w + 4 * g + x) * LD + 16 * w + m];
#pragma unroll
    for (int d = 1; d < 4; ++d) {
      const int it = w + d;
      if (it < 4) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f}, z = y;
#pragma unroll
        for (int e = 0; e < d; ++e) {
          const float* r = As + (16 * it + m) * LD + 16 * (w + e) + 4 * g;
#pragma unroll
          for (int x = 0; x < 4; ++x) y = __builtin_amdgcn_mfma_f32_16x16x4f32(r[x], col[e][x], y, 0, 0, 0);
        }
        const float* r = Ts + (16 * it + m) * LD + 16 * it + 4 * g;
#pragma unroll
        for (int x = 0; x < 4; ++x) z = __builtin_amdgcn_mfma_f32_16x16x4f32(r[x], -y[x], z, 0, 0, 0);
        settle(z);
        col[d] = z;
#pragma unroll
        for (int x = 0; x < 4; ++x) Ts[(16 * it + 4 * g + x) * LD + 16 * w + m] = z[x];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int kb2 = 0; kb2 < 2; ++kb2) {
    if (BWD ? kb2 < w / 2 : kb2 > w / 2) continue;
    f32x4 x[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int o = 32 * kb2 + 4 * g + (i & 3) + 16 * (i >> 2);
      x[i >> 2][i & 3] = BWD ? Ts[o * LD + t] : Ts[t * LD + o];
    }
    const int f = BWD ? tri_upper(w, kb2) : tri_lower(w, kb2);
    store_terms<NX>(tri_tiles<T, BWD>(a, tile, h) + f * NX * kFrag, lane, split<NX>(x[0], x[1]));
  }
  if constexpr (BWD) {
    __bf16 *Qt = kq, *Do = kq + kQt;
    const f32x4 since = a.scale * *reinterpret_cast<const f32x4*>(es + 16 * w + 4 * g);
    // Q transposed, rows in the order of a state's.
    const bf16x8 ksel[2] = {selector(channel(0, m), g), selector(channel(1, m), g)};
    const bf16x8 vsel[2] = {selector(m, g), selector(16 + m, g)};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Terms<NI> q = terms_of<T>(qr[kb], t < n ? a.Dk - 32 * kb - 8 * g : 0);
      f32x4 y[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        y[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = NI - 1; j >= 0; --j) y[x] = mfma(q.t[j], ksel[x], y[x]);
      }
      settle(y);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const Terms<NX> e = split<NX>(y[x] * since, y[x]);
#pragma unroll
        for (int j = 0; j < NX; ++j) {
          const uint4 z = __builtin_bit_cast(uint4, e.t[j]);
          *reinterpret_cast<u32x2*>(Qt + (((2 * kb + x) * 2 + (w >> 1)) * NX + j) * kFrag + lane * 8 + 4 * (w & 1)) = u32x2{z.x, z.y};
        }
      }
    }
    const T* obase = (const T*)a.d_o + at.rows.batch * a.dob + h * a.doh + row0 * a.don;
    for (int c0 = 0; c0 < 16 * a.groups; c0 += 64) {
      Raw8<T> raw[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) raw[b] = fetch8(obase, t * a.don + c0 + 32 * b + 8 * g, t < n ? a.Dv - c0 - 32 * b - 8 * g : 0);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const Terms<NI> o = terms_of<T>(raw[b], t < n ? a.Dv - c0 - 32 * b - 8 * g : 0);
        f32x4 y[2 * NI];
#pragma unroll
        for (int x = 0; x < 2 * NI; ++x) y[x] = mfma(o.t[x % NI], vsel[x / NI], f32x4{0.f, 0.f, 0.f, 0.f});
        settle(y);
#pragma unroll
        for (int x = 0; x < 2 * NI; ++x) {
          const u32x2 r = {upper_halves(y[x][0], y[x][1]), upper_halves(y[x][2], y[x][3])};
          *reinterpret_cast<u32x2*>(Do + (((2 * b + x / NI) * 2 + (w >> 1)) * NI + x % NI) * kFrag + lane * 8 + 4 * (w & 1)) = r;
        }
      }
      __syncthreads();
      const int64_t cg = (tile * a.H + h) * a.groups + (c0 >> 4);
      const auto times_do = [&](const Terms<NX> (&x)[2], float* to, int64_t step) __attribute__((always_inline)) {
        f32x4 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb2 = 0; kb2 < 2; ++kb2) {
          Terms<NI> o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = load_terms<NI>(Do + (i * 2 + kb2) * NI * kFrag, lane);
#pragma unroll
          for (int ord = 2; ord >= 0; --ord)
#pragma unroll
            for (int j = 0; j < NX; ++j)
              if (ord - j >= 0 && ord - j < NI)
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = mfma(x[kb2].t[j], o[i].t[ord - j >= 0 && ord - j < NI ? ord - j : 0], y[i]);
        }
        settle(y);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((c0 >> 4) + i < a.groups) *reinterpret_cast<f32x4*>(to + i * step) = y[i];
      };
      times_do(pt, a.ys + (cg * 4 + w) * 256 + lane * 4, 4 * 256);
      for (int dt = w; dt < 2 * KB; dt += 4) {
        const Terms<NX> q[2] = {load_terms<NX>(Qt + (dt * 2) * NX * kFrag, lane), load_terms<NX>(Qt + (dt * 2 + 1) * NX * kFrag, lane)};
        times_do(q, a.zs + (cg * 2 * KB + dt) * 256 + lane * 4, 2 * KB * 256);
      }
      __syncthreads();
    }
  }
}

// What a pass of chain() leaves: o (and the last state); what the backward reads as well; or, of a
// piece of a sequence, how it carries states over.
enum Mode { PLAIN, SAVE, TRANS };

// --------------------------------------------------------------------------
// chain: the chunks of one sequence and head, 16 columns of the state per wavefront
// --------------------------------------------------------------------------
// A chunk token by token, for the chunks that hold a value that is not finite: a
// product with the zeros of T and P would carry it to earlier tokens.
template <typename T, int KB, int MODE>
__device__ __forceinline__ void chunk_by_token(const Args& a, const Rows& rows, int64_t row0, int n, int h, int col,
                                            int64_t tile, f32x4 (&S)[2 * KB]) {
  const int hk = h / a.group, lane = threadIdx.x & 63, g = lane >> 4;
  for (int t = 0; t < n; ++t) {
    const T* krow = (const T*)a.k + rows.batch * a.kb + hk * a.kh + (row0 + t) * a.kn;
    const T* qrow = (const T*)a.q + rows.batch * a.qb + hk * a.qh + (row0 + t) * a.qn;
    const float dec = expf(a.g[rows.batch * a.gb + h * a.gh + (row0 + t) * a.gn]);
    const float b = a.beta[rows.batch * a.bb + h * a.bh + (row0 + t) * a.bn];
    float x = 0.f;
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) {
      const f32x4 k = load4(krow, channel(dt, 4 * g), a.Dk - channel(dt, 4 * g));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (channel(dt, 4 * g) < a.Dk) {
          S[dt][i] *= dec;
          x = fmaf(k[i], S[dt][i], x);
        }
      }
    }
    x = group_sum(x);
    const float v = col < a.Dv ? (float)((const T*)a.v)[rows.batch * a.vb + h * a.vh + (row0 + t) * a.vn + col] : 0.f;
    const float u = b * (v - x);
    float o = 0.f;
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) {
      const f32x4 k = load4(krow, channel(dt, 4 * g), a.Dk - channel(dt, 4 * g));
      const f32x4 q = load4(qrow, channel(dt, 4 * g), a.Dk - channel(dt, 4 * g));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (channel(dt, 4 * g) < a.Dk) {
          S[dt][i] = fmaf(k[i], u, S[dt][i]);
          o = fmaf(q[i], S[dt][i], o);
        }
      }
    }
    if (MODE == TRANS) continue;
    o = group_sum(o);
    if (g == 0 && col < a.Dv) {
      ((T*)a.o)[rows.batch * a.ob + h * a.oh + (row0 + t) * a.on + col] = (T)(a.scale * o);
      if (MODE == SAVE) {
        const float y[8] = {u};
        const Terms<NX> e = split<NX>(y);
#pragma unroll
        for (int j = 0; j < NX; ++j) a.us[planes_of<2>(a, tile, h, col >> 5) + j * 32 * C + plane_at<2>(col & 31, t)] = e.t[j][0];
      }
    }
  }
}

// A workgroup has 16 NW columns of one head's state: NW wavefronts that keep 16 each
// (in registers, 32 bits), and four that feed them and write o.  What one chunk
// costs is the chain S -> K S -> R -> U -> S, so everything else is taken off it:
// the feeders fetch the next chunk's rows, lay K and its transpose, T and V out in LDS as
// the chain reads them, and compute o from S and U, which the chain leaves in LDS as terms.
// Two barriers per chunk, so that one buffer each is enough (two of U where LDS has room:
// then the products of P and U are off the first part, the shorter one of the chain's):
//   first part   chain: splits S, K S     feeders: T, V and K' of this chunk to LDS
//   second part  chain: R, U, S           feeders: fetch the next chunk, P U of the one before,
//                                         q S of this one, K of the next to LDS
// Measured: 3.4 us per chunk at D=64 in bfloat16 (41 chunks 140 us), of which the chain's own matrix
// products, splits and LDS reads, one after another, are 2.3; about 55 KB come from memory per
// chunk, and the feeders' fetch is the rest.  B=8 H=12 N=4096 D=64, 2 pieces: 170 us with what
// the backward reads (49 KB per chunk and head, 300 MB), and 72 for what the pieces carry over.
template <typename T, int KB, int NW, int MODE>
__global__ __launch_bounds__(64 * (NW + 4)) void chain(Args a) {
  constexpr int NI = kInputTerms<T>, NO = kOutTerms<T>, ORD = kOutOrder<T>;
  __shared__ __bf16 Kf[4 * KB * NI * kFrag], Kt[4 * KB * NI * kFrag], Tf[kTri * NX * kFrag];
  __shared__ float Vf[NW * 4 * 256];
  constexpr int kLds = (8 * KB * NI + kTri * NX + NW * KB * NO) * 1024 + NW * 4096 + 2 * V_CHAIN * C * 4 + 64;
  constexpr int UB = kLds + 2 * NW * 2 * NO * 1024 <= 160 * 1024 ? 2 : 1;  // buffers of U's terms
  __shared__ __bf16 Sf[MODE == TRANS ? 1 : NW * KB * NO * kFrag], Uf[UB][MODE == TRANS ? 1 : NW * 2 * NO * kFrag];
  __shared__ float vecs[2][V_CHAIN * C];
  __shared__ int by_token[2][NW];
  // (the last piece of a sequence carries nothing over)
  const int pieces = MODE == TRANS ? a.segs - 1 : a.segs;
  const int64_t seq = blockIdx.x / pieces;
  const int seg = blockIdx.x % pieces;
  const int h = blockIdx.y, hk = h / a.group;
  const int wave = wave_index(), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const Rows rows = rows_of(a.cu, seq, a.N);
  const int64_t tile0 = first_tile<C>(a.cu, seq, rows, a.N), all = (rows.n + C - 1) / C;
  const int64_t each = a.segs == 1 ? all : ((unsigned)all + a.segs - 1) / (unsigned)a.segs;  // chunks of a piece
  const int64_t first = seg * each < all ? seg * each : all, nch = first + each < all ? first + each : all;
  // TRANS: workgroups of v's columns, from zero (the first piece: from the state before it), then of the
  // identity's with no v, which the first piece needs none of.
  const int zv = (a.groups + NW - 1) / NW;
  const bool unit = MODE == TRANS && (int)blockIdx.z >= zv;
  if (unit && seg == 0) return;
  const int col0 = ((int)blockIdx.z - (unit ? zv : 0)) * 16 * NW, width = unit ? 0 : a.Dv;  // columns of v there are
  const int64_t piece = (seq * a.H + h) * a.segs + seg;
  if (wave < NW) {
    const int col = col0 + 16 * wave + m;
    const int cg = (col0 >> 4) + wave;
    const bool in = col < width, any = cg < (unit ? 2 * KB : a.groups);
    f32x4 S[2 * KB];
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) {
      if (MODE != TRANS && seg > 0) {
        S[dt] = *reinterpret_cast<const f32x4*>(a.seg_s + ((piece * a.groups + (any ? cg : 0)) * 2 * KB + dt) * 256 + lane * 4);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = channel(dt, 4 * g + i);
          S[dt][i] = unit ? (d == col ? 1.f : 0.f)
                     : a.init && seg == 0 && in && d < a.Dk ? a.init[((seq * a.H + h) * a.Dk + d) * a.Dv + col]
                                                            : 0.f;
        }
      }
    }
    if (first < nch) lds_barrier();
    for (int64_t c = first; c < nch; ++c) {
      const int64_t tile = tile0 + c;
      const float* vec = vecs[c & 1];
      f32x4 X[4];
      if (any) {
        Terms<NX> s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          s[kb] = split<NX>(S[2 * kb], S[2 * kb + 1]);
          if (MODE != TRANS) {
#pragma unroll
            for (int j = 0; j < NO; ++j)
              *reinterpret_cast<bf16x8*>(Sf + ((wave * KB + kb) * NO + j) * kFrag + lane * 8) = s[kb].t[j];
          }
        }
        if (MODE == SAVE) keep_state<KB>(a.states + planes_of<KB>(a, tile, h, cg >> 1), cg, m, g, s);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) X[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          Terms<NI> k[4];
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) k[mt] = load_terms<NI>(Kf + (mt * KB + kb) * NI * kFrag, lane);
          products<2>(k, s[kb], X);
        }
        settle(X);
      }
      lds_barrier();
      if (any) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const f32x4 bg = *reinterpret_cast<const f32x4*>(vec + V_BG * C + 16 * mt + 4 * g);
          const f32x4 b = *reinterpret_cast<const f32x4*>(vec + V_BETA * C + 16 * mt + 4 * g);
          const f32x4 v = *reinterpret_cast<const f32x4*>(Vf + (wave * 4 + mt) * 256 + lane * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) X[mt][i] = fmaf(-bg[i], X[mt][i], b[i] * v[i]);
        }
        const Terms<NX> r[2] = {split<NX>(X[0], X[1]), split<NX>(X[2], X[3])};
        f32x4 U[4];
        float odd = 0.f;
        {
          Terms<NX> x[4], y[2];
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            U[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
            x[mt] = load_terms<NX>(Tf + tri_lower(mt, 0) * NX * kFrag, lane);
          }
          products<2>(x, r[0], U);
#pragma unroll
          for (int mt = 2; mt < 4; ++mt) y[mt - 2] = load_terms<NX>(Tf + tri_lower(mt, 1) * NX * kFrag, lane);
          products<2>(y, r[1], U + 2);
        }
        settle(U);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int i = 0; i < 4; ++i) odd += U[mt][i];
        const bool slow = __any(!(fabsf(odd) <= 3.402823466e38f));  // something is not finite
        if (lane == 0) by_token[c & 1][wave] = slow;
        if (slow) {
          chunk_by_token<T, KB, MODE>(a, rows, rows.first + c * C, rows.n - c * C < C ? (int)(rows.n - c * C) : C, h,
                                      unit ? a.Dv : col, tile, S);  // (column Dv: v is 0)
        } else {
          if (MODE != TRANS) {
            const Terms<MODE == SAVE ? NX : NO> u[2] = {split<MODE == SAVE ? NX : NO>(U[0], U[1]), split<MODE == SAVE ? NX : NO>(U[2], U[3])};
            if constexpr (MODE == SAVE) keep_rows(a.us + planes_of<2>(a, tile, h, cg >> 1), cg, m, g, u);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int j = 0; j < NO; ++j)
                *reinterpret_cast<bf16x8*>(Uf[c & (UB - 1)] + ((wave * 2 + kb) * NO + j) * kFrag + lane * 8) = u[kb].t[j];
          }
          const float whole = vec[V_SINCE * C + C - 1];
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) U[mt] *= *reinterpret_cast<const f32x4*>(vec + V_LEFT * C + 16 * mt + 4 * g);
          const Terms<NX> ul[2] = {split<NX>(U[0], U[1]), split<NX>(U[2], U[3])};
#pragma unroll
          for (int dt = 0; dt < 2 * KB; ++dt) S[dt] *= whole;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) {
            Terms<NI> k[2 * KB];
#pragma unroll
            for (int dt = 0; dt < 2 * KB; ++dt) k[dt] = load_terms<NI>(Kt + (dt * 2 + kb) * NI * kFrag, lane);
            products<2>(k, ul[kb], S);
          }
          settle(S);
        }
      }
      lds_barrier();
    }
    if (MODE == TRANS) {
      if (!any) return;
      if (unit) {
        Terms<NX> s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = split<NX>(S[2 * kb], S[2 * kb + 1]);
        keep_state<KB>(a.seg_m + (piece * KB + (cg >> 1)) * (int64_t)(NX * 32 * 32 * KB), cg, m, g, s);
      } else {
#pragma unroll
        for (int dt = 0; dt < 2 * KB; ++dt)
          *reinterpret_cast<f32x4*>(a.seg_n + ((piece * a.groups + cg) * 2 * KB + dt) * 256 + lane * 4) = S[dt];
      }
    } else if (a.final && seg + 1 == a.segs) {
#pragma unroll
      for (int dt = 0; dt < 2 * KB; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = channel(dt, 4 * g + i);
          if (in && d < a.Dk) a.final[((seq * a.H + h) * a.Dk + d) * a.Dv + col] = S[dt][i];
        }
    }
    return;
  }
  if (first >= nch) return;
  // A feeder: tokens 16w + m of each chunk.
  const int w = wave - NW, t = 16 * w + m, ft = threadIdx.x - 64 * NW;
  const T* kbase = (const T*)a.k + rows.batch * a.kb + hk * a.kh + rows.first * a.kn;
  const T* qbase = (const T*)a.q + rows.batch * a.qb + hk * a.qh + rows.first * a.qn;
  const T* vbase = (const T*)a.v + rows.batch * a.vb + h * a.vh + rows.first * a.vn;
  T* obase = (T*)a.o + rows.batch * a.ob + h * a.oh + rows.first * a.on;
  constexpr int VB = (NW + 1) / 2;             // 32-column blocks of V
  constexpr int TP = (kTri * NX + 3) / 4;      // planes of T per feeder: w, w + 4, ...
  const int64_t t0 = first * C + t;
  const T *kp = kbase + t0 * a.kn + 8 * g, *qp = qbase + t0 * a.qn + 8 * g, *vp = vbase + t0 * a.vn + col0 + 8 * g;
  const __bf16* ip = tri_tiles<T, false>(a, tile0 + first, h) + w * kFrag + lane * 8;
  const __bf16* pp = tri_tiles<T, false>(a, tile0 + first, h) + (kTri * NX + tri_lower(w, 0) * NO) * kFrag + lane * 8;
  const float* ep = vec_of(a, tile0 + first, h) + (ft % (V_CHAIN * C / 4)) * 4;
  Raw8<T> kr[KB], qr[KB], vr[VB];
  bf16x8 tr[TP];
  Terms<NO> pr[2] = {};
  f32x4 er;
  int left = rows.n < t0 ? 0 : rows.n - t0 < 0x7fffffff ? (int)(rows.n - t0) : 0x7fffffff;  // rows from this lane's on
  const auto fetch = [&]() __attribute__((always_inline)) {  // the next chunk's
    const int dk = left > 0 ? a.Dk - 8 * g : 0, dv = left > 0 ? width - col0 - 8 * g : 0;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      kr[kb] = *reinterpret_cast<const Raw8<T>*>(32 * kb < dk ? kp + 32 * kb : kbase);
      if (MODE != TRANS) qr[kb] = *reinterpret_cast<const Raw8<T>*>(32 * kb < dk ? qp + 32 * kb : qbase);
    }
#pragma unroll
    for (int b = 0; b < VB; ++b) vr[b] = *reinterpret_cast<const Raw8<T>*>(32 * b < dv ? vp + 32 * b : vbase);
#pragma unroll
    for (int x = 0; x < TP; ++x)
      if (4 * x + 4 <= kTri * NX || w + 4 * x < kTri * NX) tr[x] = *reinterpret_cast<const bf16x8*>(ip + 4 * x * kFrag);
    if (MODE != TRANS) pr[0] = load_terms<NO>(pp, 0);
    if (MODE != TRANS && w >= 2) pr[1] = load_terms<NO>(pp + NO * kFrag, 0);
    er = *reinterpret_cast<const f32x4*>(ep);
    kp += C * a.kn, qp += C * a.qn, vp += C * a.vn;
    ip += a.H * (int64_t)kTriSize<T, false>, pp += a.H * (int64_t)kTriSize<T, false>, ep += a.H * (int64_t)(V_COUNT * C);
  };
  Terms<NI> kt[KB];
  const auto put_keys = [&](int64_t c) __attribute__((always_inline)) {
    const int dk = left > 0 ? a.Dk - 8 * g : 0;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      kt[kb] = terms_of<T>(kr[kb], dk - 32 * kb);
      store_terms<NI>(Kf + (w * KB + kb) * NI * kFrag, lane, kt[kb]);
    }
    if (ft < V_CHAIN * C / 4) *reinterpret_cast<f32x4*>(vecs[c & 1] + ft * 4) = er;
  };
  // Columns of a 32-channel block of K in the order of a state's rows, and of V in its own.
  const bf16x8 ksel[2] = {selector(channel(0, m), g), selector(channel(1, m), g)};
  const bf16x8 vsel[2] = {selector(m, g), selector(16 + m, g)};
  fetch();
  put_keys(first);
  lds_barrier();
  Terms<NO> p[2];  // P of the last chunk: lane m = token i, inner indices j
  f32x4 O[NW];     // scale e^G S' q of it
  const auto write_out = [&](int64_t c, const Terms<NO> (&p)[2], const f32x4 (&O)[NW]) __attribute__((always_inline)) {
    f32x4 y[NW];
#pragma unroll
    for (int x = 0; x < NW; ++x) y[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      Terms<NO> u[NW];
#pragma unroll
      for (int x = 0; x < NW; ++x) u[x] = load_terms<NO>(Uf[c & (UB - 1)] + (x * 2 + kb) * NO * kFrag, lane);
      products<ORD>(u, p[kb], y);
    }
    settle(y);
    T* row = obase + (c * C + t) * a.on + col0 + 4 * g;
#pragma unroll
    for (int x = 0; x < NW; ++x)
      if (c * C + t < rows.n && col0 + 16 * x + 4 * g < a.Dv && !by_token[c & 1][x]) store4(row + 16 * x, O[x] + y[x]);
  };
  for (int64_t c = first; c < nch; ++c) {
    const float* vec = vecs[c & 1];
#pragma unroll
    for (int x = 0; x < TP; ++x)
      if (4 * x + 4 <= kTri * NX || w + 4 * x < kTri * NX)
        *reinterpret_cast<bf16x8*>(Tf + (w + 4 * x) * kFrag + lane * 8) = tr[x];
    // K and V transposed, q
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x4 y[2 * NI];
#pragma unroll
      for (int x = 0; x < 2 * NI; ++x) y[x] = mfma(kt[kb].t[x % NI], ksel[x / NI], f32x4{0.f, 0.f, 0.f, 0.f});
      settle(y);
#pragma unroll
      for (int x = 0; x < 2 * NI; ++x) {
        const u32x2 r = {upper_halves(y[x][0], y[x][1]), upper_halves(y[x][2], y[x][3])};
        *reinterpret_cast<u32x2*>(Kt + (((2 * kb + x / NI) * 2 + (w >> 1)) * NI + x % NI) * kFrag + lane * 8 + 4 * (w & 1)) = r;
      }
    }
    const int dv = left > 0 ? width - col0 - 8 * g : 0;
#pragma unroll
    for (int b = 0; b < VB; ++b) {
      const Terms<NI> v = terms_of<T>(vr[b], dv - 32 * b);
      f32x4 z[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        z[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = NI - 1; j >= 0; --j) z[x] = mfma(v.t[j], vsel[x], z[x]);
      }
      settle(z);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (2 * b + x < NW) *reinterpret_cast<f32x4*>(Vf + ((2 * b + x) * 4 + w) * 256 + lane * 4) = z[x];
    }
    Terms<NI> q[KB];
    if (MODE != TRANS) {
      const int dk = left > 0 ? a.Dk - 8 * g : 0;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) q[kb] = terms_of<T>(qr[kb], dk - 32 * kb);
    }
    left -= C;
    if (MODE != TRANS && UB == 1 && c > first) write_out(c - 1, p, O);
    // The next chunk is fetched as early as registers allow: with one term per input, before P U, whose P
    // then has to be another than the one that comes.
    constexpr bool early = NI == 1;
    Terms<NO> p1[2];
    if (early) p1[0] = pr[0], p1[1] = pr[1];
    lds_barrier();
    if ((early || MODE == TRANS) && c + 1 < nch) fetch();
    if (MODE != TRANS) {
      if (UB == 2 && c > first) write_out(c - 1, p, O);
      p[0] = early ? p1[0] : pr[0], p[1] = early ? p1[1] : pr[1];
      if (!early && c + 1 < nch) fetch();
      const float since = a.scale * vec[V_SINCE * C + t];
#pragma unroll
      for (int x = 0; x < NW; ++x) O[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        Terms<NO> y[NW];
#pragma unroll
        for (int x = 0; x < NW; ++x) y[x] = load_terms<NO>(Sf + (x * KB + kb) * NO * kFrag, lane);
        products<ORD>(y, q[kb], O);
      }
      settle(O);
#pragma unroll
      for (int x = 0; x < NW; ++x) O[x] *= since;
    }
    if (c + 1 < nch) put_keys(c + 1);
    lds_barrier();
  }
  if (MODE != TRANS) write_out(nch - 1, p, O);
}

// The first state of every piece, one piece after another: S <- M S + N.  A wavefront has 16 columns; M comes
// through LDS, 32 of its columns at a time, the next ones while these are multiplied.
// A chain of segs - 2 products of [Dk, Dk] by [Dk, 16]: 1.2 to 1.8 us each at D=64, 5 us for 4 pieces.
template <int KB>
__global__ __launch_bounds__(256) void join(Args a) {
  constexpr int kBlock = NX * 32 * 32 * KB;
  __shared__ __align__(16) __bf16 Ms[2][kBlock];
  const int64_t seq = blockIdx.x;
  const int h = blockIdx.y;
  const int w = wave_index(), lane = threadIdx.x & 63, j = lane & 15, row = 8 * (lane >> 4) + (j >> 2);
  const int cg = blockIdx.z * 4 + w, cgr = cg < a.groups ? cg : 0;
  const int64_t piece0 = (seq * a.H + h) * a.segs;
  const auto at = [&](int seg) __attribute__((always_inline)) { return (((piece0 + seg) * a.groups + cgr) * 2 * KB) * 256 + lane * 4; };
  const int steps = (a.segs - 2) * KB;  // pieces 1 .. segs - 2
  const auto copy = [&](int i) __attribute__((always_inline)) {
    const __bf16* from = a.seg_m + ((piece0 + 1) * KB + i) * (int64_t)kBlock + lane * 8;
    for (int x = w; x < kBlock / kFrag; x += 4) copy_to_lds(from + x * kFrag, Ms[i & 1] + x * kFrag);
  };
  if (steps) copy(0);
  f32x4 S[2 * KB];
#pragma unroll
  for (int dt = 0; dt < 2 * KB; ++dt) S[dt] = *reinterpret_cast<const f32x4*>(a.seg_n + at(0) + dt * 256);
  for (int seg = 1; seg < a.segs; ++seg) {
    if (cg < a.groups) {
#pragma unroll
      for (int dt = 0; dt < 2 * KB; ++dt) *reinterpret_cast<f32x4*>(a.seg_s + at(seg) + dt * 256) = S[dt];
    }
    if (seg + 1 == a.segs) break;
    Terms<NX> s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = split<NX>(S[2 * kb], S[2 * kb + 1]);
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) S[dt] = *reinterpret_cast<const f32x4*>(a.seg_n + at(seg) + dt * 256);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int i = (seg - 1) * KB + kb;
      lds_copies_done();
      __syncthreads();
      if (i + 1 < steps) copy(i + 1);
#pragma unroll
      for (int dt = 0; dt < 2 * KB; ++dt) {
        // M's rows in the order of a state's: each lane reads the four channels that come next in it
        Terms<NX> x;
#pragma unroll
        for (int n = 0; n < NX; ++n) {
          const __bf16* p = Ms[i & 1] + n * 32 * 32 * KB;
          const u32x2 y = read_transposed(p + plane_at<KB>(row, channel(dt, 4 * (j & 3))));
          const u32x2 z = read_transposed(p + plane_at<KB>(row + 4, channel(dt, 4 * (j & 3))));
          x.t[n] = __builtin_bit_cast(bf16x8, make_uint4(y.x, y.y, z.x, z.y));
        }
        S[dt] = product<2>(x, s[kb], S[dt]);
      }
      settle(S);
    }
  }
}

// --------------------------------------------------------------------------
// Backward.  With dS the gradient of the state at a chunk's end (P with scale):
//     dU = P' dO + e^{G_64 - G} (K dS)          dR = T' dU
//     dS <- e^{G_64} dS + scale Q' (e^G dO) - K' (b e^G dR)
// prep() leaves P' dO and scale Q' (e^G dO) of every chunk; chain_back() goes through the chunks
// from the last to the first as chain() does and leaves dR and each chunk's dS;
// grads() then has everything of its chunk:
//     dq = scale e^G (S dO) + (dP o D) K           dP_ij = dO_i.u_j,  D_ij = scale e^{G_i - G_j}, j <= i
//     dk = b rho + kw                              dA_ij = -dR_i.u_j (over b_i: below)
//     rho_i = -e^{G_i} S dR_i + sum_{j<i} dA_ij e^{G_i-G_j} k_j
//     kw_j  = e^{G_64-G_j} dS u_j + sum_{i>=j} dP_ij D_ij q_i + sum_{i>j} b_i dA_ij e^{G_i-G_j} k_i
//     dv = b dR        db_i = dR_i.v_i + k_i.rho_i
//     dG_i = q_i.dq_i + b_i k_i.rho_i - k_i.kw_i,  and at i = 64 also
//            e^{G_64} <S, dS> + sum_j e^{G_64-G_j} k_j.(dS u_j)
//     dg_i = sum of dG_i.. to the chunk's end
// --------------------------------------------------------------------------
// Few streams are cut into pieces as chain()'s are: numbered from the sequence's end, each first with nothing
// behind it and with the identity's columns (MODE TRANS: N and M of dS <- M dS + N), join()ed.
// Bound as chain() is: B=8 H=12 N=4096 D=64 bfloat16, 2 pieces, 132 us and 82 for the carrying; whole 256.
template <typename T, int KB, int MODE>
__global__ __launch_bounds__(512) void chain_back(Args a) {
  constexpr int NI = kInputTerms<T>, NW = 4;
  __shared__ __bf16 Kf[4 * KB * NI * kFrag], Kt[4 * KB * NI * kFrag], Tf[kTri * NX * kFrag];
  __shared__ float vecs[2][V_CHAIN * C];
  const int pieces = MODE == TRANS ? a.segs - 1 : a.segs;
  const int64_t seq = blockIdx.x / pieces;
  const int seg = blockIdx.x % pieces;
  const int h = blockIdx.y, hk = h / a.group;
  const int wave = wave_index(), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  const Rows rows = rows_of(a.cu, seq, a.N);
  const int64_t tile0 = first_tile<C>(a.cu, seq, rows, a.N), all = (rows.n + C - 1) / C;
  const int64_t each = a.segs == 1 ? all : ((unsigned)all + a.segs - 1) / (unsigned)a.segs;  // chunks of a piece
  const int64_t low = (a.segs - 1 - seg) * each, first = low < all ? low : all, nch = first + each < all ? first + each : all;
  const int zv = (a.groups + NW - 1) / NW;
  const bool unit = MODE == TRANS && (int)blockIdx.z >= zv;
  if (unit && seg == 0) return;
  const int64_t piece = (seq * a.H + h) * a.segs + seg;
  if (wave < NW) {
    const int cg = ((int)blockIdx.z - (unit ? zv : 0)) * NW + wave, col = 16 * cg + m;
    const bool in = !unit && col < a.Dv, any = cg < (unit ? 2 * KB : a.groups);
    f32x4 S[2 * KB], Y[4], Z[2 * KB];
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) {
      Z[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (MODE != TRANS && seg > 0) {
        S[dt] = *reinterpret_cast<const f32x4*>(a.seg_s + ((piece * a.groups + (any ? cg : 0)) * 2 * KB + dt) * 256 + lane * 4);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = channel(dt, 4 * g + i);
          S[dt][i] = unit ? (d == col ? 1.f : 0.f)
                     : a.d_final && seg == 0 && in && d < a.Dk ? a.d_final[((seq * a.H + h) * a.Dk + d) * a.Dv + col]
                                                               : 0.f;
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) Y[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto fetch = [&](int64_t c) __attribute__((always_inline)) {
      if (unit) return;  // (dO is none of M's)
      const int64_t at = ((tile0 + c) * a.H + h) * a.groups + (any ? cg : 0);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) Y[mt] = *reinterpret_cast<const f32x4*>(a.ys + (at * 4 + mt) * 256 + lane * 4);
#pragma unroll
      for (int dt = 0; dt < 2 * KB; ++dt) Z[dt] = *reinterpret_cast<const f32x4*>(a.zs + (at * 2 * KB + dt) * 256 + lane * 4);
    };
    if (first < nch) {
      fetch(nch - 1);
      lds_barrier();
    }
    for (int64_t c = nch - 1; c >= first; --c) {
      const int64_t tile = tile0 + c;
      const float* vec = vecs[c & 1];
      f32x4 X[4];
      if (any) {
        Terms<NX> s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = split<NX>(S[2 * kb], S[2 * kb + 1]);
        if (MODE != TRANS) keep_state<KB>(a.dstates + planes_of<KB>(a, tile, h, cg >> 1), cg, m, g, s);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) X[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          Terms<NI> k[4];
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) k[mt] = load_terms<NI>(Kf + (mt * KB + kb) * NI * kFrag, lane);
          products<2>(k, s[kb], X);
        }
        settle(X);
      }
      lds_barrier();
      if (any) {
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          const f32x4 left = *reinterpret_cast<const f32x4*>(vec + V_LEFT * C + 16 * mt + 4 * g);
#pragma unroll
          for (int i = 0; i < 4; ++i) X[mt][i] = fmaf(left[i], X[mt][i], Y[mt][i]);
        }
        const float whole = vec[V_SINCE * C + C - 1];
#pragma unroll
        for (int dt = 0; dt < 2 * KB; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) S[dt][i] = fmaf(whole, S[dt][i], Z[dt][i]);
        if (c > first) fetch(c - 1);
        const Terms<NX> u[2] = {split<NX>(X[0], X[1]), split<NX>(X[2], X[3])};
        f32x4 R[4];
        {
          Terms<NX> x[4], y[2];
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            R[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
            x[mt] = load_terms<NX>(Tf + tri_upper(mt, 1) * NX * kFrag, lane);
          }
          products<2>(x, u[1], R);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) y[mt] = load_terms<NX>(Tf + tri_upper(mt, 0) * NX * kFrag, lane);
          products<2>(y, u[0], R);
        }
        settle(R);
        if (MODE != TRANS) {
          const Terms<NX> r[2] = {split<NX>(R[0], R[1]), split<NX>(R[2], R[3])};
          keep_rows(a.drs + planes_of<2>(a, tile, h, cg >> 1), cg, m, g, r);
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) R[mt] *= -*reinterpret_cast<const f32x4*>(vec + V_BG * C + 16 * mt + 4 * g);
        const Terms<NX> r[2] = {split<NX>(R[0], R[1]), split<NX>(R[2], R[3])};
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          Terms<NI> k[2 * KB];
#pragma unroll
          for (int dt = 0; dt < 2 * KB; ++dt) k[dt] = load_terms<NI>(Kt + (dt * 2 + kb) * NI * kFrag, lane);
          products<2>(k, r[kb], S);
        }
        settle(S);
      }
      lds_barrier();
    }
    if (MODE == TRANS) {
      if (!any) return;
      if (unit) {
        Terms<NX> s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = split<NX>(S[2 * kb], S[2 * kb + 1]);
        keep_state<KB>(a.seg_m + (piece * KB + (cg >> 1)) * (int64_t)(NX * 32 * 32 * KB), cg, m, g, s);
      } else {
#pragma unroll
        for (int dt = 0; dt < 2 * KB; ++dt)
          *reinterpret_cast<f32x4*>(a.seg_n + ((piece * a.groups + cg) * 2 * KB + dt) * 256 + lane * 4) = S[dt];
      }
    } else if (a.d_init && seg + 1 == a.segs) {
#pragma unroll
      for (int dt = 0; dt < 2 * KB; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = channel(dt, 4 * g + i);
          if (in && d < a.Dk) a.d_init[((seq * a.H + h) * a.Dk + d) * a.Dv + col] = S[dt][i];
        }
    }
    return;
  }
  if (first >= nch) return;
  // A feeder: tokens 16w + m of each chunk, as in chain().
  const int w = wave - NW, t = 16 * w + m, ft = threadIdx.x - 64 * NW;
  constexpr int TP = (kTri * NX + 3) / 4;
  const T* kbase = (const T*)a.k + rows.batch * a.kb + hk * a.kh + rows.first * a.kn;
  Raw8<T> kr[KB];
  bf16x8 tr[TP];
  f32x4 er;
  const auto left_of = [&](int64_t c) __attribute__((always_inline)) { return c * C + t < rows.n ? a.Dk - 8 * g : 0; };
  const auto fetch = [&](int64_t c) __attribute__((always_inline)) {
    const int dk = left_of(c);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) kr[kb] = fetch8(kbase, (c * C + t) * a.kn + 32 * kb + 8 * g, dk - 32 * kb);
    const __bf16* tri = tri_tiles<T, true>(a, tile0 + c, h) + w * kFrag + lane * 8;
#pragma unroll
    for (int x = 0; x < TP; ++x)
      if (4 * x + 4 <= kTri * NX || w + 4 * x < kTri * NX) tr[x] = *reinterpret_cast<const bf16x8*>(tri + 4 * x * kFrag);
    er = *reinterpret_cast<const f32x4*>(vec_of(a, tile0 + c, h) + (ft % (V_CHAIN * C / 4)) * 4);
  };
  Terms<NI> kt[KB];
  const auto put_keys = [&](int64_t c) __attribute__((always_inline)) {
    const int dk = left_of(c);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      kt[kb] = terms_of<T>(kr[kb], dk - 32 * kb);
      store_terms<NI>(Kf + (w * KB + kb) * NI * kFrag, lane, kt[kb]);
    }
    if (ft < V_CHAIN * C / 4) *reinterpret_cast<f32x4*>(vecs[c & 1] + ft * 4) = er;
  };
  const bf16x8 ksel[2] = {selector(channel(0, m), g), selector(channel(1, m), g)};
  fetch(nch - 1);
  put_keys(nch - 1);
  lds_barrier();
  for (int64_t c = nch - 1; c >= first; --c) {
#pragma unroll
    for (int x = 0; x < TP; ++x)
      if (4 * x + 4 <= kTri * NX || w + 4 * x < kTri * NX) *reinterpret_cast<bf16x8*>(Tf + (w + 4 * x) * kFrag + lane * 8) = tr[x];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x4 y[2 * NI];
#pragma unroll
      for (int x = 0; x < 2 * NI; ++x) y[x] = mfma(kt[kb].t[x % NI], ksel[x / NI], f32x4{0.f, 0.f, 0.f, 0.f});
      settle(y);
#pragma unroll
      for (int x = 0; x < 2 * NI; ++x) {
        const u32x2 r = {upper_halves(y[x][0], y[x][1]), upper_halves(y[x][2], y[x][3])};
        *reinterpret_cast<u32x2*>(Kt + (((2 * kb + x / NI) * 2 + (w >> 1)) * NI + x % NI) * kFrag + lane * 8 + 4 * (w & 1)) = r;
      }
    }
    if (c > first) fetch(c - 1);
    lds_barrier();
    if (c > first) put_keys(c - 1);
    lds_barrier();
  }
}

// Grid (tiles, Hk), four wavefronts; wavefront w has tokens 16w..16w+15, lane m the token 16w + m, and
// channels 4g.. of each 16-channel tile: no product's result crosses wavefronts.  First the
// products over v's columns, 32 at a time (their planes go to LDS as they lie), then
// those over the chunk's tokens, whose factors dO_i.u_j and dR_i.u_j are computed
// both ways round, so that either is an operand as it stands.
// Bound by memory and by one workgroup's steps in turn (copies, then products): B=8 H=12 N=4096 D=64
// bfloat16 340 us for 830 MB (2.4 TB/s), 98 KB of each tile's 135 the planes of states, u and their
// gradients.  Two workgroups per CU (KB <= 2; 256 registers, a few spilled) against one: 340 and 475.
template <typename T, int KB, bool GROUPED>
__global__ __launch_bounds__(256, KB <= 2 ? 2 : 1) void grads(Args a) {
  constexpr int NI = kInputTerms<T>;
  constexpr int SP = NX * 32 * 32 * KB, UP = NX * 32 * C, kKt = 4 * KB * NI * kFrag;
  constexpr int kPlanes = 2 * SP + 2 * UP + 4 * NI * kFrag;
  __shared__ __align__(16) __bf16 lds[kPlanes > 2 * kKt ? kPlanes : 2 * kKt];
  __bf16 *Sp = lds, *dSp = lds + SP, *Up = lds + 2 * SP, *Rp = Up + UP, *Of = Rp + UP;  // planes, and rows of dO
  __bf16 *Kt = lds, *Qt = lds + kKt;                                                    // later: K and Q transposed
  __shared__ float dGs[C], ends[4];
  const int64_t tile = blockIdx.x;
  const int hk = blockIdx.y;
  const int w = wave_index(), lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
  zero_outside<C>(a.cu, a.sequences, tile, a.N, (T*)a.dq + hk * a.dqh, a.dqn, a.Dk, threadIdx.x, 256);
  zero_outside<C>(a.cu, a.sequences, tile, a.N, (T*)a.dk + hk * a.dkh, a.dkn, a.Dk, threadIdx.x, 256);
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    zero_outside<C>(a.cu, a.sequences, tile, a.N, a.dg + h * a.N, 1, 1, threadIdx.x, 256);
    zero_outside<C>(a.cu, a.sequences, tile, a.N, a.dbeta + h * a.N, 1, 1, threadIdx.x, 256);
  }
  const TileOf at = tile_of<C>(a.cu, a.sequences, tile, a.N);
  const int64_t left_rows = at.rows.n - at.index * C;
  if (left_rows <= 0) return;
  const int n = left_rows < C ? (int)left_rows : C;
  const int64_t row0 = at.rows.first + at.index * C, bt = at.rows.batch;
  const int t = 16 * w + m;
  const T* kbase = (const T*)a.k + bt * a.kb + hk * a.kh + row0 * a.kn;
  const T* qbase = (const T*)a.q + bt * a.qb + hk * a.qh + row0 * a.qn;
  const bf16x8 sel[2] = {selector(m, g), selector(16 + m, g)};
  f32x4 dq[GROUPED ? 2 * KB : 1], dk[GROUPED ? 2 * KB : 1];
  if (GROUPED) {
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) dq[GROUPED ? dt : 0] = dk[GROUPED ? dt : 0] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    const float* vec = vec_of(a, tile, h);
    const T* obase = (const T*)a.d_o + bt * a.dob + h * a.doh + row0 * a.don;
    const T* vbase = (const T*)a.v + bt * a.vb + h * a.vh + row0 * a.vn;
    const float bt_ = vec[V_BETA * C + t];
    f32x4 hq[2 * KB], rho[2 * KB], kw[2 * KB];
    f32x4 E1[4], E2[4], F1[4], F2[4];  // dO_i.u_j and dR_i.u_j: lane = i, rows j <= i; lane = j, rows i >= j
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) hq[dt] = rho[dt] = kw[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 4; ++x) E1[x] = E2[x] = F1[x] = F2[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    float db = 0.f, ss = 0.f;
    for (int b = 0; b < a.blocks; ++b) {
      const int c0 = 32 * b, dv = t < n ? a.Dv - c0 - 8 * g : 0;
      __syncthreads();  // what lds held is read
      const Raw8<T> oraw = fetch8(obase, t * a.don + c0 + 8 * g, dv), vraw = fetch8(vbase, t * a.vn + c0 + 8 * g, dv);
      const int64_t so = planes_of<KB>(a, tile, h, b), uo = planes_of<2>(a, tile, h, b);
      constexpr int SN = SP / kFrag, UN = UP / kFrag;  // copies of 1 KiB
      for (int i = w; i < SN; i += 4) {
        copy_to_lds(a.states + so + i * kFrag + lane * 8, Sp + i * kFrag);
        copy_to_lds(a.dstates + so + i * kFrag + lane * 8, dSp + i * kFrag);
      }
      for (int i = w; i < UN; i += 4) {
        copy_to_lds(a.us + uo + i * kFrag + lane * 8, Up + i * kFrag);
        copy_to_lds(a.drs + uo + i * kFrag + lane * 8, Rp + i * kFrag);
      }
      const Terms<NI> o = terms_of<T>(oraw, dv);
      store_terms<NI>(Of + w * NI * kFrag, lane, o);
      lds_copies_done();
      __syncthreads();
      const Terms<NX> u = load_plane<2>(Up, w, lane), r = load_plane<2>(Rp, w, lane);
      {
        float x[8];
        Raw8<T> dvs;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = t < n ? ((float)r.t[2][i] + (float)r.t[1][i]) + (float)r.t[0][i] : 0.f;
          db = fmaf(x[i], dv > 0 ? (float)vraw[i] : 0.f, db);
          dvs[i] = (T)(bt_ * x[i]);
        }
        if (dv > 0)
          *reinterpret_cast<Raw8<T>*>((T*)a.dv + bt * a.dvb + h * a.dvh + (row0 + t) * a.dvn + c0 + 8 * g) = dvs;
      }
#pragma unroll
      for (int dt = 0; dt < 2 * KB; ++dt) {
        const Terms<NX> s = load_plane<KB>(Sp, dt, lane), ds = load_plane<KB>(dSp, dt, lane);
        hq[dt] = product<2>(s, o, hq[dt]);
        rho[dt] = product<2>(s, r, rho[dt]);
        kw[dt] = product<2>(ds, u, kw[dt]);
      }
      settle(hq), settle(rho), settle(kw);
      for (int dt = w; dt < 2 * KB; dt += 4) {  // <S, dS>: every fourth tile
        const Terms<NX> s = load_plane<KB>(Sp, dt, lane), ds = load_plane<KB>(dSp, dt, lane);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          ss = fmaf(((float)s.t[2][i] + (float)s.t[1][i]) + (float)s.t[0][i],
                    ((float)ds.t[2][i] + (float)ds.t[1][i]) + (float)ds.t[0][i], ss);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (x <= w) {
          const Terms<NX> uj = load_plane<2>(Up, x, lane);
          E1[x] = product<2>(uj, o, E1[x]);
          E2[x] = product<2>(uj, r, E2[x]);
          asm volatile("" : "+v"(E1[x]));
          settle(E2[x]);
        }
        if (x >= w) {
          F1[x] = product<2>(load_terms<NI>(Of + x * NI * kFrag, lane), u, F1[x]);
          F2[x] = product<2>(load_plane<2>(Rp, x, lane), u, F2[x]);
          asm volatile("" : "+v"(F1[x]));
          settle(F2[x]);
        }
      }
    }
    // K and Q transposed
    __syncthreads();
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int d = 32 * kb + 8 * g, left = t < n ? a.Dk - d : 0;
      const Terms<NI> kt = terms_of<T>(fetch8(kbase, t * a.kn + d, left), left), qt = terms_of<T>(fetch8(qbase, t * a.qn + d, left), left);
      f32x4 y[4 * NI];
#pragma unroll
      for (int x = 0; x < 2 * NI; ++x) {
        y[x] = mfma(kt.t[x % NI], sel[x / NI], f32x4{0.f, 0.f, 0.f, 0.f});
        y[2 * NI + x] = mfma(qt.t[x % NI], sel[x / NI], f32x4{0.f, 0.f, 0.f, 0.f});
      }
      settle(y);
#pragma unroll
      for (int x = 0; x < 4 * NI; ++x) {
        const int z = x % (2 * NI);
        __bf16* to = (x < 2 * NI ? Kt : Qt) + (((2 * kb + z / NI) * 2 + (w >> 1)) * NI + z % NI) * kFrag + lane * 8 + 4 * (w & 1);
        *reinterpret_cast<u32x2*>(to) = u32x2{upper_halves(y[x][0], y[x][1]), upper_halves(y[x][2], y[x][3])};
      }
    }
    const float Gt = vec[V_G * C + t], Gl = vec[V_GLOW * C + t];
    const float since = vec[V_SINCE * C + t], left = vec[V_LEFT * C + t], whole = vec[V_SINCE * C + C - 1];
    // k.(the state's part of kw), q.dq, k.rho, k.kw
    float kend = 0.f, qq = 0.f, kr = 0.f, kk = 0.f;
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) {
      hq[dt] *= a.scale * since;
      rho[dt] *= -since;
      kw[dt] *= left;
      const f32x4 k = load4(kbase, t * a.kn + 16 * dt + 4 * g, t < n ? a.Dk - 16 * dt - 4 * g : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) kend = fmaf(k[i], kw[dt][i], kend);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const f32x4 Gy = *reinterpret_cast<const f32x4*>(vec + V_G * C + 16 * x + 4 * g);
      const f32x4 Ly = *reinterpret_cast<const f32x4*>(vec + V_GLOW * C + 16 * x + 4 * g);
      const f32x4 by = *reinterpret_cast<const f32x4*>(vec + V_BETA * C + 16 * x + 4 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int y = 16 * x + 4 * g + i;
        const float d = (Gt - Gy[i]) + (Gl - Ly[i]);
        const float fi = exp2_fast(d), fj = exp2_fast(-d);
        E1[x][i] = y <= t ? a.scale * fi * E1[x][i] : 0.f;
        E2[x][i] = y < t ? -fi * E2[x][i] : 0.f;
        F1[x][i] = y >= t ? a.scale * fj * F1[x][i] : 0.f;
        F2[x][i] = y > t ? -by[i] * fj * F2[x][i] : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const bool lo = kb <= w / 2, hi = kb >= w / 2;
      const Terms<NX> e1 = split<NX>(E1[2 * kb], E1[2 * kb + 1]), e2 = split<NX>(E2[2 * kb], E2[2 * kb + 1]);
      const Terms<NX> f1 = split<NX>(F1[2 * kb], F1[2 * kb + 1]), f2 = split<NX>(F2[2 * kb], F2[2 * kb + 1]);
      if (lo) {
#pragma unroll
        for (int dt = 0; dt < 2 * KB; ++dt) {
          const Terms<NI> kT = load_terms<NI>(Kt + (dt * 2 + kb) * NI * kFrag, lane);
          hq[dt] = product<2>(kT, e1, hq[dt]);
          rho[dt] = product<2>(kT, e2, rho[dt]);
        }
        settle(hq), settle(rho);
      }
      if (hi) {
#pragma unroll
        for (int dt = 0; dt < 2 * KB; ++dt) {
          kw[dt] = product<2>(load_terms<NI>(Qt + (dt * 2 + kb) * NI * kFrag, lane), f1, kw[dt]);
          kw[dt] = product<2>(load_terms<NI>(Kt + (dt * 2 + kb) * NI * kFrag, lane), f2, kw[dt]);
        }
        settle(kw);
      }
    }
    T* dqrow = (T*)a.dq + bt * a.dqb + hk * a.dqh + (row0 + t) * a.dqn;
    T* dkrow = (T*)a.dk + bt * a.dkb + hk * a.dkh + (row0 + t) * a.dkn;
    const bool done = !GROUPED || h + 1 == (hk + 1) * a.group;
#pragma unroll
    for (int dt = 0; dt < 2 * KB; ++dt) {
      const int d = 16 * dt + 4 * g, ok = t < n ? a.Dk - d : 0;
      const f32x4 k = load4(kbase, t * a.kn + d, ok), q = load4(qbase, t * a.qn + d, ok);
      f32x4 dqs = hq[dt], dks;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qq = fmaf(q[i], hq[dt][i], qq);
        kr = fmaf(k[i], rho[dt][i], kr);
        kk = fmaf(k[i], kw[dt][i], kk);
        dks[i] = fmaf(bt_, rho[dt][i], kw[dt][i]);
      }
      if (GROUPED) {
        dqs = dq[GROUPED ? dt : 0] += dqs;
        dks = dk[GROUPED ? dt : 0] += dks;
      }
      if (done && ok > 0) {
        store4(dqrow + d, dqs);
        store4(dkrow + d, dks);
      }
    }
    kend = group_sum(kend), qq = group_sum(qq), kr = group_sum(kr), kk = group_sum(kk), db = group_sum(db);
    // Over the tokens (kend) and channels (ss) of this wavefront.
#pragma unroll
    for (int x = 1; x < 16; x *= 2) {
      kend += __shfl_xor(kend, x);
      ss += __shfl_xor(ss, x);
    }
    ss = group_sum(ss);
    if (g == 0) {
      dGs[t] = qq + bt_ * kr - kk;
      if (t < n) a.dbeta[(bt * a.H + h) * a.N + row0 + t] = db + kr;
    }
    if (lane == 0) ends[w] = kend + whole * ss;
    __syncthreads();  // (and one before they are written again: the next head's blocks begin with it)
    if (w == 0) {
      float x = dGs[lane];
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const float y = __shfl_down(x, d);
        if (lane + d < 64) x += y;
      }
      if (lane < n) a.dg[(bt * a.H + h) * a.N + row0 + lane] = x + ((ends[0] + ends[1]) + (ends[2] + ends[3]));
    }
  }
}

// --------------------------------------------------------------------------
// One token.  Bound by the state, read and written once: a workgroup has 32
// columns of one head's state, in registers between the two.
//     x = k'S, y = q'S;  u = b (v - a x);  S <- a S + k u';  o = scale (a y + (q.k) u)
// 256 sequences of 12 heads, D=64: 25.7 us a call for 102 MB (4.0 TB/s; a large copy reaches 5.1); one
// sequence of 6 heads 6.3, a launch and two memory round trips.
// --------------------------------------------------------------------------
constexpr int kStepCols = 32;

// Up to four elements, n of them there.  vec: in one access where all are.
template <typename T>
__device__ __forceinline__ f32x4 load_some(const T* p, int n, bool vec) {
  if (vec) return load4(p, 0, n);
  f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) r[i] = (float)p[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, f32x4 x, int n, bool vec) {
  if (vec) {
    if (n > 0) store4(p, x);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = (T)x[i];
}

template <typename T, typename TO>
__global__ __launch_bounds__(256) void step(const T* q, const T* k, const T* v, const float* gs, const float* betas,
                                            const float* in, float* out_state, TO* out, int Hk, int H, int Dk, int Dv,
                                            float scale, bool vec_in, bool vec_out) {
  // Eight lanes of four columns; 32 rows at a time.
  __shared__ float xs[4][kStepCols], ys[4][kStepCols], dots[4];
  const int64_t bh = blockIdx.x;
  const int64_t b = bh / H, h = bh % H;
  const T* kp = k + (b * Hk + h / (H / Hk)) * Dk;
  const T* qp = q + (b * Hk + h / (H / Hk)) * Dk;
  const int c = blockIdx.y * kStepCols + (threadIdx.x & 7) * 4, r0 = threadIdx.x >> 3, w = threadIdx.x >> 6;
  const float dec = expf(gs[bh]), beta = betas[bh];
  constexpr int R = KDELTA_MAX_DK / 32;
  f32x4 S[R];
  float kk[R], qk = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int r = r0 + 32 * j;
    const bool on = r < Dk;
    S[j] = load_some(in + (bh * Dk + (on ? r : 0)) * (int64_t)Dv + c, on ? Dv - c : 0, vec_in);
    kk[j] = on ? (float)kp[r] : 0.f;
    const float qq = on ? (float)qp[r] : 0.f;
    qk = fmaf(kk[j], qq, qk);
    if (on) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        S[j][i] *= dec;
        x[i] = fmaf(kk[j], S[j][i], x[i]);
        y[i] = fmaf(qq, S[j][i], y[i]);
      }
    }
  }
  // over the rows: lanes 8 apart, then the four wavefronts
#pragma unroll
  for (int d = 8; d < 64; d *= 2) {
    qk += __shfl_xor(qk, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] += __shfl_xor(x[i], d);
      y[i] += __shfl_xor(y[i], d);
    }
  }
  if ((threadIdx.x & 63) < 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xs[w][(threadIdx.x & 7) * 4 + i] = x[i];
      ys[w][(threadIdx.x & 7) * 4 + i] = y[i];
    }
    if ((threadIdx.x & 7) == 0) dots[w] = qk;
  }
  __syncthreads();
  qk = (dots[0] + dots[1]) + (dots[2] + dots[3]);
  const f32x4 vv = load_some(v + bh * Dv + c, Dv - c, false);
  f32x4 u, o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int cc = (threadIdx.x & 7) * 4 + i;
    const float xx = (xs[0][cc] + xs[1][cc]) + (xs[2][cc] + xs[3][cc]);
    const float yy = (ys[0][cc] + ys[1][cc]) + (ys[2][cc] + ys[3][cc]);
    u[i] = beta * (vv[i] - xx);
    o[i] = scale * (yy + qk * u[i]);
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int r = r0 + 32 * j;
    if (r >= Dk) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[j][i] = fmaf(kk[j], u[i], S[j][i]);
    store_some(out_state + (bh * Dk + r) * (int64_t)Dv + c, S[j], Dv - c, vec_out);
  }
  asm volatile("" : "+v"(o));  // a multiply that rounds to 16 bits by itself would skip the rounding to 32
  if (threadIdx.x < 8) store_some(out + bh * Dv + c, o, Dv - c, false);
}

// --------------------------------------------------------------------------
// Host
// --------------------------------------------------------------------------
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

int64_t tiles_of(const kdelta_problem* p) {
  return p->cu_seqlens ? p->N / C + p->sequences : p->B * ((p->N + C - 1) / C);
}

int64_t blocks_of(const kdelta_problem* p) { return (p->Dv + 31) / 32; }

// Wavefronts of a workgroup of chain(): four, and fewer where three terms of wide keys leave no room in
// LDS for as many.
constexpr int chain_waves(int element_size, int KB) { return element_size == 2 || KB <= 2 ? 4 : KB == 3 ? 2 : 1; }

// Pieces that a sequence is cut into. A workgroup of chain() takes 3 to 5 us per chunk in 16-bit types (about 9
// in float32) and fills a CU, so few streams leave most of the card idle; pieces cost a
// pass over all of them but the last first (about 0.65 of that per chunk, and as many more
// workgroups as a state has columns of its own), a join of 1 to 3 us per piece and two launches.
// Measured (us, whole / pieces): B=1 H=16 N=65536 D=128 bf16 4212 / 1461 with 8, 1896 with 4, 1653 with 16;
// B=8 H=6 N=1024 D=64 64 / 52 with 4, 69 with 6; B=4 H=16 N=2047 D=80 fp16 202 / 179
// with 2, 221 with 4; B=2 H=6 N=1024 D=64 float32 (with the backward) 266 / 163 with 8.  The backward's chain, the same call:
// 132 then 157; B=8 H=12 N=4096 D=64 bf16, 2 pieces: 1055 and 1084. (A packed batch: by the mean length.)
int pieces_of(const kdelta_problem* p, bool backward) {
  constexpr double kCus = 256, kPass = 0.65, kFixed = 4;
  if (!p->sequences) return 1;
  const int64_t KB = (p->Dk + 31) / 32, NW = backward ? 4 : chain_waves(p->dtype == KDECAY_F32 ? 4 : 2, (int)KB);
  const int64_t zv = (2 * ((p->Dv + 31) / 32) + NW - 1) / NW, zk = (2 * KB + NW - 1) / NW;
  const int64_t chunks = (p->N / (p->cu_seqlens ? p->sequences : 1) + C - 1) / C;
  const double streams = (double)p->sequences * p->H, join = 0.75 * KB;
  const double step = p->dtype == KDECAY_F32 ? 9 : (KB <= 2 ? 3 : 4) + (p->dtype == KDECAY_F16 ? 1 : 0);
  const auto rounds = [](double n) { return ceil(n / kCus); };
  int best = 1;
  double least = 0.9 * rounds(streams * zv) * chunks * step;
  for (int n = 2; n <= 16 && 2 * n <= chunks; ++n) {
    const double each = (double)((chunks + n - 1) / n);
    const double cost = each * step * (rounds(streams * zv * n) + kPass * rounds(streams * (n - 1) * (zv + zk))) + join * n + kFixed;
    if (cost < least) least = cost, best = n;
  }
  return best;
}

struct Sizes {  // bytes
  size_t vecs, tris, back_tris, ys, zs, states, rows, seg_n, seg_m;
};

Sizes sizes_of(const kdelta_problem* p, bool backward) {
  const size_t heads = (size_t)tiles_of(p) * p->H, KB = (p->Dk + 31) / 32, blocks = blocks_of(p);
  Sizes s;
  s.vecs = up256(heads * V_COUNT * C * 4);
  s.tris = up256(heads * kTri * (NX + (p->dtype == KDECAY_F32 ? 3 : 2)) * kFrag * 2);
  s.back_tris = up256(heads * kTri * NX * kFrag * 2);
  s.ys = up256(heads * 2 * blocks * 4 * 256 * 4);
  s.zs = up256(heads * 2 * blocks * 2 * KB * 256 * 4);
  s.states = up256(heads * blocks * NX * 32 * 32 * KB * 2);
  s.rows = up256(heads * blocks * NX * 32 * C * 2);
  const size_t segs = pieces_of(p, backward), pieces = segs > 1 ? (size_t)p->sequences * p->H * segs : 0;
  s.seg_n = up256(pieces * 2 * blocks * 2 * KB * 256 * 4);
  s.seg_m = up256(pieces * KB * NX * 32 * 32 * KB * 2);
  return s;
}

int check(const kdelta_problem* p) {
  if (!p) return fail(KDECAY_EINVAL, "null problem");
  if (p->B < 0 || p->Hk < 0 || p->H < 0 || p->N < 0 || p->Dk < 0 || p->Dv < 0 || p->sequences < 0)
    return fail(KDECAY_EINVAL, "negative size");
  if (p->dtype != KDECAY_F32 && p->dtype != KDECAY_BF16 && p->dtype != KDECAY_F16)
    return fail(KDECAY_EDTYPE, "q, k and v must be float32, bfloat16 or float16 (code %d)", p->dtype);
  if (p->Dk < 1 || p->Dk > KDELTA_MAX_DK || p->Dv < 1 || p->Dv > KDELTA_MAX_DV)
    return fail(KDECAY_ESHAPE, "head dims Dk=%lld, Dv=%lld are not 1..%d and 1..%d", (long long)p->Dk,
                (long long)p->Dv, KDELTA_MAX_DK, KDELTA_MAX_DV);
  if (p->Hk < 1 || p->H < 1 || p->H % p->Hk) return fail(KDECAY_ESHAPE, "H=%lld is no multiple of Hk=%lld", (long long)p->H, (long long)p->Hk);
  if (p->H > 65535) return fail(KDECAY_ESHAPE, "more than 65535 heads");
  if (p->cu_seqlens && (p->B != 1 || p->sequences < 1))
    return fail(KDECAY_ESHAPE, "cu_seqlens takes B=1 and at least one sequence");
  if (!p->cu_seqlens && p->sequences != p->B) return fail(KDECAY_EINVAL, "sequences must be B without cu_seqlens");
  if (p->sequences > 0x7fffffff || tiles_of(p) > 0x7fffffff) return fail(KDECAY_ESHAPE, "too many sequences or rows");
  if (p->B && p->N && (!p->q || !p->k || !p->v || !p->g || !p->beta)) return fail(KDECAY_EINVAL, "null pointer argument");
  if (p->Dk % 8 || p->Dv % 8)
    return fail(KDECAY_ESHAPE, "head dims Dk=%lld, Dv=%lld are not multiples of 8", (long long)p->Dk, (long long)p->Dv);
  if (!p->B || !p->N) return 0;
  if (const int rc = check_rows(p->q, p->q_strides, p->dtype, "q")) return rc;
  if (const int rc = check_rows(p->k, p->k_strides, p->dtype, "k")) return rc;
  return check_rows(p->v, p->v_strides, p->dtype, "v");
}

Args args_of(const kdelta_problem* p, void* workspace, const float* saved, bool backward) {
  Args a = {};
  a.q = p->q, a.k = p->k, a.v = p->v, a.g = p->g, a.beta = p->beta, a.cu = p->cu_seqlens, a.init = p->init;
  a.qb = p->q_strides[0], a.qh = p->q_strides[1], a.qn = p->q_strides[2];
  a.kb = p->k_strides[0], a.kh = p->k_strides[1], a.kn = p->k_strides[2];
  a.vb = p->v_strides[0], a.vh = p->v_strides[1], a.vn = p->v_strides[2];
  a.gb = p->g_strides[0], a.gh = p->g_strides[1], a.gn = p->g_strides[2];
  a.bb = p->beta_strides[0], a.bh = p->beta_strides[1], a.bn = p->beta_strides[2];
  a.N = p->N, a.sequences = p->sequences, a.tiles = tiles_of(p);
  a.Hk = (int)p->Hk, a.H = (int)p->H, a.Dk = (int)p->Dk, a.Dv = (int)p->Dv, a.group = (int)(p->H / p->Hk);
  a.scale = p->scale;
  a.blocks = (int)blocks_of(p);
  a.groups = 2 * a.blocks;
  const Sizes s = sizes_of(p, backward);
  char* w = (char*)workspace;
  a.vecs = (float*)w, w += s.vecs;
  a.tris = (__bf16*)w;
  a.segs = pieces_of(p, backward);
  if (!backward) {
    w += s.tris;
  } else {
    w += s.back_tris;
    a.ys = (float*)w, w += s.ys;
    a.zs = (float*)w, w += s.zs;
    a.dstates = (__bf16*)w, w += s.states;
    a.drs = (__bf16*)w, w += s.rows;
  }
  a.seg_n = (float*)w, w += s.seg_n;
  a.seg_s = (float*)w, w += s.seg_n;
  a.seg_m = (__bf16*)w;
  a.states = (__bf16*)saved;
  a.us = saved ? (__bf16*)((char*)saved + s.states) : nullptr;
  return a;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == KDECAY_BF16) return f((__bf16*)nullptr);
  if (dtype == KDECAY_F16) return f((_Float16*)nullptr);
  return f((float*)nullptr);
}
template <int N>
struct Int {
  static constexpr int value = N;
};
template <typename F>
int by_blocks(int64_t Dk, F f) {
  switch ((Dk + 31) / 32) {
    case 1: return f(Int<1>());
    case 2: return f(Int<2>());
    case 3: return f(Int<3>());
    default: return f(Int<4>());
  }
}

dim3 chain_grid(const Args& a, int waves) {
  return dim3((unsigned)(a.sequences * a.segs), a.H, (a.groups + waves - 1) / waves);
}
}  // namespace delta
}  // namespace kd

using namespace kd;
using namespace kd::delta;

extern "C" size_t kdelta_scan_workspace_bytes(const kdelta_problem* p) {
  if (check(p)) return 0;
  const Sizes s = sizes_of(p, false);
  return s.vecs + s.tris + 2 * s.seg_n + s.seg_m;
}

extern "C" size_t kdelta_scan_bwd_workspace_bytes(const kdelta_problem* p) {
  if (check(p)) return 0;
  const Sizes s = sizes_of(p, true);
  return s.vecs + s.back_tris + s.ys + s.zs + s.states + s.rows + 2 * s.seg_n + s.seg_m;
}

extern "C" size_t kdelta_scan_saved_floats(const kdelta_problem* p) {
  if (check(p)) return 0;
  const Sizes s = sizes_of(p, false);
  return (s.states + s.rows) / 4;
}

extern "C" int kdelta_scan_fwd(const kdelta_problem* p, void* o, const int64_t* o_strides, float* final, float* saved,
                               void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(p)) return rc;
  if (p->sequences == 0) return 0;
  const bool rows = p->B && p->N;
  if (rows && (!o || !o_strides)) return fail(KDECAY_EINVAL, "null pointer argument");
  if (rows)
    if (const int rc = check_rows(o, o_strides, p->dtype, "o")) return rc;
  if (workspace_bytes < kdelta_scan_workspace_bytes(p) || (!workspace && rows) || ((uintptr_t)workspace & 15))
    return fail(KDECAY_EWORKSPACE, "scan workspace of %zu bytes missing, small or not 16-byte aligned",
                kdelta_scan_workspace_bytes(p));
  if ((uintptr_t)saved & 15) return fail(KDECAY_ELAYOUT, "saved is not 16-byte aligned");
  Args a = args_of(p, workspace, saved, false);
  a.o = o, a.final = final;
  if (rows) a.ob = o_strides[0], a.oh = o_strides[1], a.on = o_strides[2];
  const hipStream_t s = (hipStream_t)stream;
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_blocks(p->Dk, [&](auto kb) {
      constexpr int KB = decltype(kb)::value;
      if (rows) {
        prep<T, KB, false><<<dim3((unsigned)a.tiles, a.H), 256, 0, s>>>(a);
        if (const int rc = hip_check("kdelta prep launch")) return rc;
      }
      constexpr int NW = chain_waves(sizeof(T), KB);
      const dim3 grid = chain_grid(a, NW);
      if (a.segs > 1) {
        const dim3 pieces((unsigned)(a.sequences * (a.segs - 1)), a.H, grid.z + (2 * KB + NW - 1) / NW);
        chain<T, KB, NW, TRANS><<<pieces, 64 * (NW + 4), 0, s>>>(a);
        if (const int rc = hip_check("kdelta chain launch")) return rc;
        join<KB><<<dim3((unsigned)a.sequences, a.H, (a.groups + 3) / 4), 256, 0, s>>>(a);
        if (const int rc = hip_check("kdelta join launch")) return rc;
      }
      if (saved)
        chain<T, KB, NW, SAVE><<<grid, 64 * (NW + 4), 0, s>>>(a);
      else
        chain<T, KB, NW, PLAIN><<<grid, 64 * (NW + 4), 0, s>>>(a);
      return hip_check("kdelta chain launch");
    });
  });
}

extern "C" int kdelta_scan_bwd(const kdelta_problem* p, const void* d_o, const int64_t* do_strides,
                               const float* d_final, const float* saved, void* dq, const int64_t* dq_strides, void* dk,
                               const int64_t* dk_strides, void* dv, const int64_t* dv_strides, float* dg, float* dbeta,
                               float* d_init, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(p)) return rc;
  if (p->sequences == 0) return 0;
  const bool rows = p->B && p->N;
  if (rows && (!d_o || !do_strides || !saved || !dq || !dq_strides || !dk || !dk_strides || !dv || !dv_strides || !dg || !dbeta))
    return fail(KDECAY_EINVAL, "null pointer argument");
  if (rows) {
    const struct {
      const void* p;
      const int64_t* strides;
      const char* name;
    } all[] = {{d_o, do_strides, "d_o"}, {dq, dq_strides, "dq"}, {dk, dk_strides, "dk"}, {dv, dv_strides, "dv"}};
    for (const auto& x : all)
      if (const int rc = check_rows(x.p, x.strides, p->dtype, x.name)) return rc;
  }
  if (workspace_bytes < kdelta_scan_bwd_workspace_bytes(p) || (!workspace && rows) || ((uintptr_t)workspace & 15))
    return fail(KDECAY_EWORKSPACE, "backward workspace of %zu bytes missing, small or not 16-byte aligned",
                kdelta_scan_bwd_workspace_bytes(p));
  if ((uintptr_t)saved & 15) return fail(KDECAY_ELAYOUT, "saved is not 16-byte aligned");
  Args a = args_of(p, workspace, saved, true);
  a.d_o = d_o, a.d_final = d_final, a.d_init = d_init, a.dq = dq, a.dk = dk, a.dv = dv, a.dg = dg, a.dbeta = dbeta;
  if (rows) {
    a.dob = do_strides[0], a.doh = do_strides[1], a.don = do_strides[2];
    a.dqb = dq_strides[0], a.dqh = dq_strides[1], a.dqn = dq_strides[2];
    a.dkb = dk_strides[0], a.dkh = dk_strides[1], a.dkn = dk_strides[2];
    a.dvb = dv_strides[0], a.dvh = dv_strides[1], a.dvn = dv_strides[2];
  }
  const hipStream_t s = (hipStream_t)stream;
  return by_type(p->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_blocks(p->Dk, [&](auto kb) {
      constexpr int KB = decltype(kb)::value;
      if (rows) {
        prep<T, KB, true><<<dim3((unsigned)a.tiles, a.H), 256, 0, s>>>(a);
        if (const int rc = hip_check("kdelta prep launch")) return rc;
      }
      const dim3 grid = chain_grid(a, 4);
      if (a.segs > 1) {
        const dim3 pieces((unsigned)(a.sequences * (a.segs - 1)), a.H, grid.z + (2 * KB + 3) / 4);
        chain_back<T, KB, TRANS><<<pieces, 512, 0, s>>>(a);
        if (const int rc = hip_check("kdelta chain_back launch")) return rc;
        join<KB><<<dim3((unsigned)a.sequences, a.H, (a.groups + 3) / 4), 256, 0, s>>>(a);
        if (const int rc = hip_check("kdelta join launch")) return rc;
      }
      chain_back<T, KB, PLAIN><<<grid, 512, 0, s>>>(a);
      if (const int rc = hip_check("kdelta chain_back launch")) return rc;
      if (!rows) return 0;
      if (a.group > 1)
        grads<T, KB, true><<<dim3((unsigned)a.tiles, a.Hk), 256, 0, s>>>(a);
      else
        grads<T, KB, false><<<dim3((unsigned)a.tiles, a.Hk), 256, 0, s>>>(a);
      return hip_check("kdelta grads launch");
    });
  });
}

extern "C" int kdelta_step(const void* q, const void* k, const void* v, int dtype, const float* g, const float* beta,
                           const float* state_in, float* state_out, void* out, int out_dtype, int64_t B, int64_t Hk,
                           int64_t H, int64_t Dk, int64_t Dv, float scale, void* stream) {
  if (B < 0 || Hk < 0 || H < 0 || Dk < 0 || Dv < 0) return fail(KDECAY_EINVAL, "negative size");
  if (dtype != KDECAY_F32 && dtype != KDECAY_BF16 && dtype != KDECAY_F16)
    return fail(KDECAY_EDTYPE, "q, k and v must be float32, bfloat16 or float16 (code %d)", dtype);
  if (out_dtype != dtype && out_dtype != KDECAY_F32) return fail(KDECAY_EDTYPE, "out must have v's type or float32");
  if (Dk < 1 || Dk > KDELTA_MAX_DK || Dv < 1 || Dv > KDELTA_MAX_DV)
    return fail(KDECAY_ESHAPE, "head dims Dk=%lld, Dv=%lld are not 1..%d and 1..%d", (long long)Dk, (long long)Dv,
                KDELTA_MAX_DK, KDELTA_MAX_DV);
  if (Hk < 1 || H < 1 || H % Hk) return fail(KDECAY_ESHAPE, "H=%lld is no multiple of Hk=%lld", (long long)H, (long long)Hk);
  if (B == 0) return 0;
  if (B * H > 0x7fffffff) return fail(KDECAY_ESHAPE, "too many heads");
  if (!q || !k || !v || !g || !beta || !state_in || !state_out || !out) return fail(KDECAY_EINVAL, "null pointer argument");
  const bool vec_in = Dv % 4 == 0 && ((uintptr_t)state_in & 15) == 0, vec_out = Dv % 4 == 0 && ((uintptr_t)state_out & 15) == 0;
  const dim3 grid((unsigned)(B * H), (unsigned)((Dv + kStepCols - 1) / kStepCols));
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (out_dtype == dtype)
      step<T, T><<<grid, 256, 0, (hipStream_t)stream>>>((const T*)q, (const T*)k, (const T*)v, g, beta, state_in,
                                                        state_out, (T*)out, (int)Hk, (int)H, (int)Dk, (int)Dv, scale, vec_in, vec_out);
    else
      step<T, float><<<grid, 256, 0, (hipStream_t)stream>>>((const T*)q, (const T*)k, (const T*)v, g, beta, state_in,
                                                            state_out, (float*)out, (int)Hk, (int)H, (int)Dk, (int)Dv,
                                                            scale, vec_in, vec_out);
    return hip_check("kdelta_step launch");
  });
}
