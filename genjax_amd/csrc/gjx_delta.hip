// gjx_delta.hip -- the gated delta filter: the mean recursion of a Kalman filter over a dk x dv matrix of regression
// weights S that is observed along k_t with the gain beta_t k_t,
//   S_t = a_t S_{t-1} + k_t u_t^T,   u_t = beta_t (v_t - a_t S_{t-1}^T k_t),   o_t = scale S_t^T q_t,   a_t = exp(g_t),
// over whole sequences in chunks of 64 tokens, its gradient, and one token at a time.
//
// One chunk with gamma = cumsum(g), D_ij = exp(gamma_i - gamma_j) (i >= j), N_ij = D_ij k_i.k_j (i > j):
//   r = V - e^gamma K S0,   delta = (I + N beta)^-1 r,   V' = beta delta   (the rows are the u_t),
//   O = scale e^gamma Q S0 + P V',  P_ij = scale D_ij q_i.k_j (i >= j),   S1 = e^gamma_C S0 + K^T (e^(gamma_C - gamma) V').
// Everything but the three products with S0 is known before the recursion: k_delta_prepare forms That = (I + N beta)^-1
// and P for all chunks at once; k_delta_scan walks the chunks with S in registers.
// Gradient (e = T^T dV', T = (I + beta N)^-1 = I - beta That N):
//   dV' = P^T dO + e^(gamma_C - gamma) K dS1,  dV = beta e,  dbeta_i = e_i.delta_i,
//   dS0 = e^gamma_C dS1 + Q^T (scale e^gamma dO) - K^T (beta e^gamma e)            (k_delta_scan_back),
//   E = scale D (dO V'^T), F = -beta_i D_ij (e_i.V'_j)  (i > j),
//   dQ = scale e^gamma dO S0^T + E K,  dK as what is read = -beta e^gamma e S0^T + F K,
//   dK as what is written = E^T Q + F^T K + e^(gamma_C - gamma) V' dS1^T,
//   dg_t = sum of what the decay of token t stands in, each term with it as a factor (k_delta_back, all chunks at once):
//     q_i.(scale e^gamma dO S0^T)_i - k_i.(beta e^gamma e S0^T)_i  (i >= t)    what later tokens read of S0,
//     X_ij = E_ij q_i.k_j + F_ij k_i.k_j  (i >= t > j)                         what they read of earlier tokens,
//     k_j.(e^(gamma_C - gamma) V' dS1^T)_j  (j < t) and e^gamma_C <dS1, S0>    what S1 holds of earlier tokens and of S0.
//   (As a reverse cumsum of dgamma_i = q_i.dq_i + k_i.dk_i(read) - k_i.dk_i(written), terms without that factor stand in
//   the sums and cancel in exact arithmetic only: at log-decays below -10 what they leave behind was all of dg.)
//
// Arithmetic: 16x16x32 bf16 MFMA with f32 accumulators.  Whatever is not an input in bf16 is split into three bf16 planes
// (8 bits each) and multiplied in the partial products above 2^-23, so that states, gains and gradients keep f32
// accuracy; only the read-out of bf16 calls takes two planes (2^-16 before the rounding of o to 2^-8).
// Operands are laid out as matrix fragments: 64 lanes x 8 elements, lane = (index % 16) + 16 q, the eight elements of quad
// q in slab s being reduction indices 32 s + 4 q + {0..3} and 32 s + 16 + 4 q + {0..3}.  That order is the one in which the
// accumulators of two stacked 16-row tiles come out, so S, r, delta, ... go from accumulator to operand without moving.
#include "gjx_common.h"

#include <algorithm>

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int C = 64;           // tokens per chunk
constexpr int FRAG = 512;       // elements of one fragment
constexpr int LD = 68;          // row pitch of the 64 x 64 f32 matrices in LDS
constexpr float G_MIN = -100.0f;

struct Shape {
  int kheads, heads, group, dk, dv, dvp;
  float scale;
  int64_t batch, time;
  int64_t qs[3], ks[3], vs[3], gs[3], bs[3];
  int64_t chunks;
};

// element offsets (bf16) of the fragment blocks of one chunk
template <int DKP, int NPI>
struct KeyBlock {               // per key head
  static constexpr int KS = DKP / 32, MT = DKP / 16;
  static constexpr int KA = 0, QA = NPI * 4 * KS * FRAG, KT = 2 * QA, QT = KT + NPI * MT * 2 * FRAG;
  static constexpr int SIZE = QT, SIZE_KEEP = QT + NPI * MT * 2 * FRAG;
};
struct GateBlock {              // per head: That, P, then (keep) T^T, P^T; three planes of six fragments each
  static constexpr int TA = 0, PA = 18 * FRAG, TT = 36 * FRAG, PT = 54 * FRAG, SIZE = 36 * FRAG, SIZE_KEEP = 72 * FRAG;
};
constexpr int ROWS = 4 * C;     // f32 per head and chunk: beta, e^gamma, e^(gamma_C - gamma), e^gamma_C (repeated)

struct Work {
  bf16 *keys, *gates;
  int64_t key_size, gate_size;
  float* rows;
  float *s0, *delta;            // keep: state before the chunk (DKP x dvp), delta (64 x dvp)
  float *ds1, *e;               // gradient scratch
  float *dq, *dk;               // gradient scratch, heads that share a key head: f32 (batch, time, heads, dk)
};

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// f32 -> bf16 planes by cutting off (8 + 8 + 8 bits: exact for P = 3; nothing can overflow).  Cutting costs two
// operations a plane where rounding takes four; what it leaves out of a product of two split values is at most 2^-21 of
// it, 2^-23 on average.
template <int P, int N>
__device__ __forceinline__ void split_planes(float (&x)[N], int p, bf16 (&h)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (p + 1 < P || P == 3) {
      const float top = __uint_as_float(__float_as_uint(x[j]) & 0xffff0000u);
      h[j] = __builtin_bit_cast(bf16, (uint16_t)(__float_as_uint(x[j]) >> 16));
      x[j] -= top;
    } else {
      h[j] = (bf16)x[j];             // the last of fewer than three planes is rounded
    }
  }
}

template <int P>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&out)[P]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    bf16 h[8];
    split_planes<P, 8>(r, p, h);
#pragma unroll
    for (int j = 0; j < 8; ++j) out[p][j] = h[j];
  }
}

// acc += sum of the partial products a_p b_r with p + r < LIM, smallest first
template <int PA, int PB, int LIM>
__device__ __forceinline__ f32x4 mma_planes(const bf16x8 (&a)[PA], const bf16x8 (&b)[PB], f32x4 acc) {
#pragma unroll
  for (int s = LIM - 1; s >= 0; --s)
#pragma unroll
    for (int p = 0; p < PA; ++p)
      if (s - p >= 0 && s - p < PB) acc = mma(a[p], b[s - p], acc);
  return acc;
}

// the same with one accumulator per order of magnitude: chains of dependent products a third as long
template <int LIM>
struct Orders {
  f32x4 v[LIM];
  __device__ __forceinline__ Orders() {
#pragma unroll
    for (int s = 0; s < LIM; ++s) v[s] = f32x4{0, 0, 0, 0};
  }
  template <int PA, int PB>
  __device__ __forceinline__ void add(const bf16x8 (&a)[PA], const bf16x8 (&b)[PB]) {
#pragma unroll
    for (int s = LIM - 1; s >= 0; --s)
#pragma unroll
      for (int p = 0; p < PA; ++p)
        if (s - p >= 0 && s - p < PB) v[s] = mma(a[p], b[s - p], v[s]);
  }
  __device__ __forceinline__ f32x4 sum() const {
    f32x4 t = v[LIM - 1];
#pragma unroll
    for (int s = LIM - 2; s >= 0; --s) t += v[s];
    return t;
  }
};

// uniform base + 32-bit lane offset in bytes: one address register
template <typename V>
__device__ __forceinline__ V load_at(const void* base, uint32_t offset) { return *(const V*)((const char*)base + offset); }
template <typename V>
__device__ __forceinline__ void store_at(void* base, uint32_t offset, V v) { *(V*)((char*)base + offset) = v; }

template <int P>
__device__ __forceinline__ void load_frag(const bf16* base, int index, int plane, int lane, bf16x8 (&out)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p) out[p] = load_at<bf16x8>(base + p * plane + index * FRAG, (uint32_t)lane * 16);
}

// two accumulator tiles (rows 16 (2 s) .. 16 (2 s + 2)) as the operand of slab s
template <int P>
__device__ __forceinline__ void tiles_to_frag(f32x4 lo, f32x4 hi, bf16x8 (&out)[P]) {
  const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  split<P>(x, out);
}

// fragments of a lower triangular 64 x 64 matrix: row tile i needs slabs 0 .. i / 2; of its transpose: slabs i / 2 .. 1
__device__ __forceinline__ constexpr int lower(int i, int s) { return i < 2 ? i : 2 + 2 * (i - 2) + s; }
__device__ __forceinline__ constexpr int upper(int i, int s) { return i < 2 ? 2 * i + s : 4 + (i - 2); }

__device__ __forceinline__ int perm(int s, int q, int j) { return 32 * s + (j < 4 ? 4 * q + j : 12 + 4 * q + j); }

__device__ __forceinline__ int64_t length_of(const int32_t* lengths, int64_t b, int64_t time) {
  return lengths ? std::min<int64_t>(std::max<int64_t>(lengths[b], 0), time) : time;
}

// ---------------------------------------------------------------------------
// all chunks at once: fragments of K, Q and their transposes, That, P (keep: T^T, P^T), the row factors.  Bound by memory
// (bf16, dk = 128: 33 KB read and 84 KB written a chunk): 2048 chunks in 59 us, 4.0 TB/s
// ---------------------------------------------------------------------------
// 64 rows of K or Q: into registers (all loads in flight at once), then split and into LDS
template <typename T, int DKP, int NPI>
struct RowLoader {
  static constexpr int PIECES = C * (DKP / 8) / 256, PITCH = DKP + 8, PLANE = C * PITCH;
  typedef T vec8 __attribute__((ext_vector_type(8)));
  vec8 x[PIECES];
  __device__ __forceinline__ void load(const T* src, int64_t token_stride, int tokens, int dk, bool vec, int tid) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int u = i * 256 + tid, t = min(u / (DKP / 8), tokens - 1), c0 = (u % (DKP / 8)) * 8;
      const T* p = src + t * token_stride;
      if (vec) {
        x[i] = *(const vec8*)(p + min(c0, dk - 8));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = p[min(c0 + j, dk - 1)];
      }
    }
  }
  __device__ __forceinline__ void store(int tokens, int dk, bf16* lds, int tid) const {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int u = i * 256 + tid, t = u / (DKP / 8), c0 = (u % (DKP / 8)) * 8;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = t < tokens && c0 + j < dk ? (float)x[i][j] : 0.0f;
      bf16x8 out[NPI];
      split<NPI>(f, out);
#pragma unroll
      for (int p = 0; p < NPI; ++p) *(bf16x8*)(lds + p * PLANE + t * PITCH + c0) = out[p];
    }
  }
};

template <int DKP, int NPI>
__device__ __forceinline__ void store_row_frags(const bf16* lds, bf16* dst, int tid) {   // rows are tokens
  constexpr int PITCH = DKP + 8, PLANE = C * PITCH, KS = DKP / 32;
  for (int i = tid; i < NPI * 4 * KS * 64; i += 256) {
    const int lane = i & 63, f = i >> 6, s = f % KS, m = (f / KS) % 4, p = f / (KS * 4), q = lane >> 4;
    const bf16* row = lds + p * PLANE + (16 * m + (lane & 15)) * PITCH + 32 * s + 4 * q;
    const bf16x4 lo = *(const bf16x4*)row, hi = *(const bf16x4*)(row + 16);
    *(bf16x8*)(dst + (int64_t)i * 8) = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

template <int DKP, int NPI>
__device__ __forceinline__ void store_col_frags(const bf16* lds, bf16* dst, int tid) {   // rows are the dk axis
  constexpr int PITCH = DKP + 8, PLANE = C * PITCH, MT = DKP / 16;
  for (int i = tid; i < NPI * MT * 2 * 64; i += 256) {
    const int lane = i & 63, f = i >> 6, s = f % 2, m = (f / 2) % MT, p = f / (2 * MT), q = lane >> 4;
    bf16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = lds[p * PLANE + perm(s, q, j) * PITCH + 16 * m + (lane & 15)];
    *(bf16x8*)(dst + (int64_t)i * 8) = v;
  }
}

// 64 x 64 f32 in LDS -> three planes of the six fragments of a triangle (of its transpose: TRANS)
template <bool TRANS>
__device__ __forceinline__ void store_triangle(const float* m, bf16* dst, int tid) {
  for (int i = tid; i < 6 * 64; i += 256) {
    const int lane = i & 63, f = i >> 6, q = lane >> 4;
    int t, s;
    if (TRANS) {
      t = f < 4 ? f / 2 : f - 2;
      s = f < 4 ? f % 2 : 1;
    } else {
      t = f < 2 ? f : 2 + (f - 2) / 2;
      s = f < 2 ? 0 : (f - 2) % 2;
    }
    const int a = 16 * t + (lane & 15);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = TRANS ? m[perm(s, q, j) * LD + a] : m[a * LD + perm(s, q, j)];
    bf16x8 out[3];
    split<3>(x, out);
#pragma unroll
    for (int p = 0; p < 3; ++p) *(bf16x8*)(dst + ((int64_t)p * 6 + f) * FRAG + lane * 8) = out[p];
  }
}

// acc += X(rows i, cols l) Y(rows l, cols j) of 16 x 16 f32 blocks in LDS; X's columns times col_scale (or 1)
__device__ __forceinline__ f32x4 block_product(const float* x, const float* col_scale, const float* y, int i, int l, int j,
                                               int lane, f32x4 acc) {
  const int q = lane >> 4, c = lane & 15;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int kk = 16 * l + 4 * k + q;
    const float a = x[(16 * i + c) * LD + kk] * (col_scale ? col_scale[kk] : 1.0f);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a, y[kk * LD + 16 * j + c], acc, 0, 0, 0);
  }
  return acc;
}

template <typename T, int DKP, int NPI, bool KEEP>
__global__ void __launch_bounds__(256)
    k_delta_prepare(Shape sh, const T* __restrict__ q, const T* __restrict__ k, const float* __restrict__ g,
                    const float* __restrict__ beta, const int32_t* __restrict__ lengths, Work w, int vec) {
  constexpr int KS = DKP / 32, PITCH = DKP + 8, PLANE = C * PITCH;
  extern __shared__ char smem[];
  // the rows of K and Q; N and That take their place once the products and the fragments are out, so that three
  // workgroups fit a CU in bf16 (dk = 128; one at a time: 140 us for 2048 chunks)
  float* s_gh = (float*)smem;
  float *s_gl = s_gh + C, *s_beta = s_gl + C;
  float* sp = s_beta + C;                       // P, then T
  bf16* sk = (bf16*)(sp + C * LD);
  bf16* sq = sk + NPI * PLANE;
  float* sn = (float*)sk;                       // N
  float* st = sn + C * LD;                      // That
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, quad = lane >> 4, c = lane & 15;
  const int64_t chunk = gjx_block() % sh.chunks, bh = gjx_block() / sh.chunks, b = bh / sh.heads;
  if (b >= sh.batch) return;
  const int h = (int)(bh % sh.heads), kh = h / sh.group;
  const int64_t len = length_of(lengths, b, sh.time), t0 = chunk * C;
  if (t0 >= len) return;
  const int tokens = (int)std::min<int64_t>(C, len - t0);
  bf16* keys = w.keys + ((b * sh.kheads + kh) * sh.chunks + chunk) * w.key_size;
  bf16* gates = w.gates + (bh * sh.chunks + chunk) * w.gate_size;
  float* rows = w.rows + (bh * sh.chunks + chunk) * ROWS;

  RowLoader<T, DKP, NPI> lk, lq;
  lk.load(k + b * sh.ks[0] + t0 * sh.ks[1] + kh * sh.ks[2], sh.ks[1], tokens, sh.dk, vec, tid);
  lq.load(q + b * sh.qs[0] + t0 * sh.qs[1] + kh * sh.qs[2], sh.qs[1], tokens, sh.dk, vec, tid);
  if (wave == 0) {
    const bool in = lane < tokens;
    // differences of the cumulative decay keep f32 accuracy whatever its size: 64-bit sum, kept as two floats
    double gam = in ? (double)fmaxf(g[b * sh.gs[0] + (t0 + lane) * sh.gs[1] + h * sh.gs[2]], G_MIN) : 0.0;
    if (in && __builtin_isnan(g[b * sh.gs[0] + (t0 + lane) * sh.gs[1] + h * sh.gs[2]])) gam = __builtin_nan("");
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(gam, o);
      if (lane >= o) gam += up;
    }
    const double last = __shfl(gam, 63);
    const float be = in ? beta[b * sh.bs[0] + (t0 + lane) * sh.bs[1] + h * sh.bs[2]] : 0.0f;
    s_gh[lane] = (float)gam;
    s_gl[lane] = (float)(gam - (double)(float)gam);
    s_beta[lane] = be;
    rows[lane] = be;
    rows[C + lane] = expf((float)gam);
    rows[2 * C + lane] = expf((float)(last - gam));
    rows[3 * C + lane] = expf((float)last);
  }
  lk.store(tokens, sh.dk, sk, tid);
  lq.store(tokens, sh.dk, sq, tid);
  __syncthreads();

  // K K^T and Q K^T, row tile = wave
  f32x4 nn[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
    if (j <= wave) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf16x8 a[NPI], x[NPI], bq[NPI];
#pragma unroll
        for (int p = 0; p < NPI; ++p) {
          a[p] = *(const bf16x8*)(sk + p * PLANE + (16 * j + c) * PITCH + 32 * s + 8 * quad);
          x[p] = *(const bf16x8*)(sk + p * PLANE + (16 * wave + c) * PITCH + 32 * s + 8 * quad);
          bq[p] = *(const bf16x8*)(sq + p * PLANE + (16 * wave + c) * PITCH + 32 * s + 8 * quad);
        }
        kk = mma_planes<NPI, NPI, NPI>(x, a, kk);
        qk = mma_planes<NPI, NPI, NPI>(bq, a, qk);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * quad + r, jj = 16 * j + c;
      const float d = jj <= i ? expf((s_gh[i] - s_gh[jj]) + (s_gl[i] - s_gl[jj])) : 0.0f;
      nn[j][r] = jj < i ? d * kk[r] : 0.0f;
      sp[i * LD + jj] = jj <= i ? sh.scale * d * qk[r] : 0.0f;
    }
  }
  if (h % sh.group == 0) {
    typedef KeyBlock<DKP, NPI> KB;
    store_row_frags<DKP, NPI>(sk, keys + KB::KA, tid);
    store_row_frags<DKP, NPI>(sq, keys + KB::QA, tid);
    store_col_frags<DKP, NPI>(sk, keys + KB::KT, tid);
    if (KEEP) store_col_frags<DKP, NPI>(sq, keys + KB::QT, tid);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) sn[(16 * wave + 4 * quad + r) * LD + 16 * j + c] = nn[j][r];
  for (int i = tid; i < C * LD; i += 256) st[i] = 0.0f;
  __syncthreads();
  store_triangle<false>(sp, gates + GateBlock::PA, tid);
  if (KEEP) store_triangle<true>(sp, gates + GateBlock::PT, tid);

  // That = (I + N beta)^-1: the diagonal 16 x 16 blocks by forward substitution, one column per lane ...
  {
    float x[16];
    const float* n = sn + 16 * wave * LD + 16 * wave;
    f32x4 bt[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bt[j] = *(const f32x4*)(s_beta + 16 * wave + 4 * j);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == c ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; j += 4) {         // N is zero on and above the diagonal: whole groups of four
        const f32x4 row = *(const f32x4*)(n + i * LD + j) * bt[j / 4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < i) v -= row[e] * x[j + e];
      }
      x[i] = v;
    }
    if (quad == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[(16 * wave + i) * LD + 16 * wave + c] = x[i];
  }
  __syncthreads();
  // ... the others by block diagonals: That_ij = -That_ii sum_{j <= l < i} (N beta)_il That_lj
  for (int d = 1; d < 4; ++d) {
    const int j = wave, i = wave + d;
    f32x4 out = {0, 0, 0, 0};
    if (i < 4) {
      f32x4 tmp = {0, 0, 0, 0};
      for (int l = j; l < i; ++l) tmp = block_product(sn, s_beta, st, i, l, j, lane, tmp);
#pragma unroll
      for (int r = 0; r < 4; ++r)      // the accumulator's register r holds rows 4 q + r: take those columns of That_ii
        out = __builtin_amdgcn_mfma_f32_16x16x4f32(st[(16 * i + c) * LD + 16 * i + 4 * quad + r], tmp[r], out, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) st[(16 * i + 4 * quad + r) * LD + 16 * j + c] = -out[r];
    }
    __syncthreads();
  }
  store_triangle<false>(st, gates + GateBlock::TA, tid);
  if (KEEP) {                          // T = I - beta That N, transposed (the barriers above end all reads of P)
    for (int j = 0; j < 4; ++j) {
      f32x4 acc = {0, 0, 0, 0};
      for (int l = j; l <= wave; ++l) acc = block_product(st, nullptr, sn, wave, l, j, lane, acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * quad + r, jj = 16 * j + c;
        sp[i * LD + jj] = (i == jj ? 1.0f : 0.0f) - s_beta[i] * acc[r];
      }
    }
    __syncthreads();
    store_triangle<true>(sp, gates + GateBlock::TT, tid);
  }
}

// ---------------------------------------------------------------------------
// the recursion: eight waves share NC x 16 columns of S
// ---------------------------------------------------------------------------
// Four waves carry the state, four take what hangs off the chain.  State wave w owns the dk rows [w DKP / 4, (w + 1)
// DKP / 4) of S and the tokens [16 w, 16 w + 16) of a chunk; read-out wave w forms the outputs of the same tokens (in the
// gradient: the products with dO alone, one chunk ahead).  What one wave computes and others multiply by (S, r, V', ...)
// goes through LDS in fragment order, three barriers a chunk; what a wave takes from memory (its rows of K, Q, That, P,
// its rows of K^T) is used by no other wave, so it is loaded straight into registers, each fragment for the next chunk as
// soon as it has been used for this one.
// Bound by the chain: 1.7 us a chunk at 2.3 GHz (bf16, dk = 128; 8192 tokens in 218 us), of which the products are 0.3 us
// and the rest is the way of S, r and V' through LDS.  With kept states 2.8 us, the gradient's scan 3.0 us a chunk (2048
// tokens, all CUs taken: 88 and 96 us).  Tried and no faster: two chunks of operands in flight (239 against 230 us),
// K S split along its reduction so that S stays in registers (241 against 225).
constexpr int TEAM = 512;
// vmcnt(0) alone: with nothing in flight at the loop's entry, the waits inside it count the loop's own loads only
constexpr int WAIT_VM = 0x0f70;

// the workgroups of one head go to one XCD (workgroups go round the eight of them): they read the same fragments
__device__ __forceinline__ bool scan_place(int64_t block, int tiles, int64_t heads, int64_t& bh, int& tile) {
  bh = block / (8 * tiles) * 8 + block % 8;
  tile = (int)(block / 8 % tiles);
  return bh < heads;
}

// barrier for LDS traffic only: loads and stores of global memory stay in flight
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// four elements per lane of a 16-row tile -> its half of a slab's fragment planes
template <int P>
__device__ __forceinline__ void put_half(bf16* frag, int half, int lane, f32x4 x) {
  float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int p = 0; p < P; ++p) {
    bf16 h[4];
    split_planes<P, 4>(r, p, h);
    *(bf16x4*)(frag + p * FRAG + lane * 8 + half * 4) = bf16x4{h[0], h[1], h[2], h[3]};
  }
}

template <int P>
__device__ __forceinline__ void get_frag(const bf16* frag, int lane, bf16x8 (&out)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p) out[p] = *(const bf16x8*)(frag + p * FRAG + lane * 8);
}

// what every wave of a scan knows of its place
struct Place {
  int64_t bh, b, len, n_chunks;
  int h, kh, tile, lane, wave, quad, c, col0, tok;
  bool reads;                    // a read-out wave
};

template <int NC>
__device__ __forceinline__ bool place_of(const Shape& sh, const int32_t* lengths, Place& p) {
  p.lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  p.wave = w & 3;
  p.reads = w >= 4;
  p.quad = p.lane >> 4;
  p.c = p.lane & 15;
  if (!scan_place(gjx_block(), (sh.dvp / 16 + NC - 1) / NC, sh.batch * sh.heads, p.bh, p.tile)) return false;
  p.b = p.bh / sh.heads;
  p.h = (int)(p.bh % sh.heads);
  p.kh = p.h / sh.group;
  p.col0 = p.tile * 16 * NC + p.c;
  p.tok = 16 * p.wave + 4 * p.quad;
  p.len = length_of(lengths, p.b, sh.time);
  p.n_chunks = (p.len + C - 1) / C;
  return true;
}

// where a chunk's operands lie; step() stays inside the sequence
struct Cursor {
  const bf16 *keys, *gates;
  const float* rows;
  int64_t ch;
  __device__ __forceinline__ Cursor(const bf16* k, const bf16* g, const float* r, const Work& w, int64_t c)
      : keys(k + c * w.key_size), gates(g + c * w.gate_size), rows(r + c * ROWS), ch(c) {}
  __device__ __forceinline__ int left(const Place& p) const { return (int)std::min<int64_t>(C, p.len - ch * C); }
  __device__ __forceinline__ Cursor step(const Work& w, int d, const Place& p) const {
    Cursor n = *this;
    if (d > 0 ? ch + 1 < p.n_chunks : ch > 0) {
      n.keys += d * w.key_size;
      n.gates += d * w.gate_size;
      n.rows += d * ROWS;
      n.ch += d;
    }
    return n;
  }
};

// Touch a chunk's operands, one load of four bytes per 128-byte line, so that they are in this XCD's L2 when the waves load
// them a chunk later.  The workgroups of a head share the lines out: `first` of `waves` waves.  The loads go to LDS that
// nobody reads.
__device__ __forceinline__ void touch(const void* block, int bytes, int first, int waves, int lane, char* sink) {
  for (int i = first; i * 8192 < bytes; i += waves)
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)((const char*)block + min(i * 8192 + lane * 128, bytes - 4)),
                                     (__attribute__((address_space(3))) void*)sink, 4, 0, 0);
}

// this lane's four tokens of a (batch, time, head, dv) column block: raw values, converted and masked where they are used
template <typename T, int NC>
struct Columns {
  uint32_t step, row[4], col[NC];
  T raw[NC][4];
  __device__ __forceinline__ Columns(const Shape& sh, const Place& p, int64_t token_stride) : step((uint32_t)token_stride * sizeof(T)) {
#pragma unroll
    for (int n = 0; n < NC; ++n) col[n] = (uint32_t)min(p.col0 + 16 * n, sh.dv - 1) * sizeof(T);
  }
  __device__ __forceinline__ void load(const T* chunk, const Place& p, int left) {
#pragma unroll
    for (int e = 0; e < 4; ++e) row[e] = (uint32_t)(left < C ? min(p.tok + e, left - 1) : p.tok + e) * step;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[n][e] = load_at<T>(chunk, row[e] + col[n]);
  }
  __device__ __forceinline__ f32x4 get(const Shape& sh, const Place& p, int n, int left) const {
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = p.col0 + 16 * n < sh.dv && p.tok + e < left ? (float)raw[n][e] : 0.0f;
    return x;
  }
};

// What is kept for the gradient lies in blocks of 16 columns, rows of 64 bytes one behind the other: a workgroup of the scans
// then fills whole lines (as rows of dvp columns, which neighbours fill piece by piece, the gradient scan took 104 us instead of
// 96 for 32 chunks on all CUs).
__device__ __forceinline__ void store_rows(float* block, int row, int c, f32x4 x) {
#pragma unroll
  for (int r = 0; r < 4; ++r) store_at(block, (uint32_t)((row + r) * 16 + c) * 4, x[r]);
}

// a slab of S from its three planes (their sum is exact) to its rows of a block
__device__ __forceinline__ void store_slab(const bf16* frag, float* block, int s, const Place& p) {
  bf16x8 f[3];
  get_frag<3>(frag, p.lane, f);
  f32x4 lo, hi;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    lo[j] = (float)f[0][j] + ((float)f[1][j] + (float)f[2][j]);
    hi[j] = (float)f[0][4 + j] + ((float)f[1][4 + j] + (float)f[2][4 + j]);
  }
  store_rows(block, 32 * s + 4 * p.quad, p.c, lo);
  store_rows(block, 32 * s + 16 + 4 * p.quad, p.c, hi);
}

template <typename T>
__device__ __forceinline__ void store_tokens(T* chunk, const Place& p, int col, uint32_t step, bool all, int dv, int left, f32x4 x) {
  const uint32_t at = (uint32_t)p.tok * step + (uint32_t)col * sizeof(T);
  if (all) {
#pragma unroll
    for (int e = 0; e < 4; ++e) store_at(chunk, at + e * step, (T)x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col < dv && p.tok + e < left) store_at(chunk, at + e * step, (T)x[e]);
  }
}

template <typename T, int DKP, int NPI, bool KEEP, int NC>
__global__ void __launch_bounds__(TEAM, 2)
    k_delta_scan(Shape sh, const T* __restrict__ v, const float* __restrict__ state0, const int32_t* __restrict__ lengths,
                 T* __restrict__ o, float* __restrict__ state, Work w) {
  typedef KeyBlock<DKP, NPI> KB;
  constexpr int KS = DKP / 32, MT = DKP / 64;     // slabs of S; 16-row tiles of S per wave
  constexpr int NPO = NPI == 1 ? 2 : 3;           // planes of what only the read-out takes
  __shared__ bf16 x_s[KS * NC * 3 * FRAG], x_r[2 * NC * 3 * FRAG], x_v[2][2 * NC * NPO * FRAG], x_w[2 * NC * 3 * FRAG];
  __shared__ f32x4 x_d[KEEP ? 2 * 4 * NC * 64 : 1];        // delta, for the read-out waves to keep
  __shared__ char sink[4][256];
  const int tiles = (sh.dvp / 16 + NC - 1) / NC;
  Place p;
  if (!place_of<NC>(sh, lengths, p)) return;
  const int lane = p.lane, wave = p.wave, tok = p.tok;
  const bf16* keys = w.keys + (p.b * sh.kheads + p.kh) * sh.chunks * w.key_size;
  const bf16* gates = w.gates + p.bh * sh.chunks * w.gate_size;
  const float* rows = w.rows + p.bh * sh.chunks * ROWS;
  const int lo = wave / 2;                        // last slab of this wave's rows of That and P

  if (p.reads) {
    T* op = o + (p.b * sh.time * sh.heads + p.h) * sh.dv;
    const int64_t o_stride = (int64_t)sh.heads * sh.dv;
    const bool all_cols = p.tile * 16 * NC + 16 * NC <= sh.dv;
    bf16x8 qa[KS][NPI], pa[2][NPO];
    f32x4 f_eg;
    auto load_q = [&](const Cursor& at) {
#pragma unroll
      for (int s = 0; s < KS; ++s) load_frag<NPI>(at.keys + KB::QA, wave * KS + s, 4 * KS * FRAG, lane, qa[s]);
      f_eg = load_at<f32x4>(at.rows + C, (uint32_t)tok * 4);
    };
    auto load_p = [&](const Cursor& at) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        load_frag<NPO>(at.gates + GateBlock::PA, lower(wave, min(s, lo)), 6 * FRAG, lane, pa[s]);
    };
    Cursor next(keys, gates, rows, w, 0);
    if (p.n_chunks > 0) {
      load_q(next);
      load_p(next);
      __builtin_amdgcn_s_waitcnt(WAIT_VM);
    }
    // a chunk's outputs are finished while the state waves are at the next chunk's That r: nobody waits for them
    f32x4 qs[NC];
    auto finish = [&](int64_t ch) {
      const int left = (int)std::min<int64_t>(C, sh.time - ch * C);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        if (KEEP && p.col0 + 16 * n < sh.dvp)
          store_rows(w.delta + ((p.bh * sh.chunks + ch) * sh.dvp + (p.tile * NC + n) * 16) * C, tok, p.c,
                     x_d[(((int)(ch & 1) * 4 + wave) * NC + n) * 64 + lane]);
        Orders<NPO> acc;
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (s <= lo) {
            bf16x8 vf[NPO];
            get_frag<NPO>(x_v[ch & 1] + (s * NC + n) * NPO * FRAG, lane, vf);
            acc.add(pa[s], vf);
          }
        store_tokens(op + ch * C * o_stride, p, p.col0 + 16 * n, (uint32_t)o_stride * sizeof(T), all_cols && left == C, sh.dv, left,
                     qs[n] + acc.sum());
      }
    };
    for (int64_t ch = 0; ch < p.n_chunks; ++ch) {
      const Cursor here = next;
      next = next.step(w, 1, p);
      const Cursor later = next.step(w, 1, p);
      if (KEEP) {              // (without the stores of what is kept the loads are fast enough)
        touch(later.keys, KB::SIZE * 2, p.tile * 4 + wave, tiles * 4, lane, sink[wave]);
        touch(later.gates, (18 + 6 * NPO) * FRAG * 2, tiles * 4 - 1 - p.tile * 4 - wave, tiles * 4, lane, sink[wave]);
      }
      lds_barrier();
      f32x4 now[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        Orders<NPO> acc;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          bf16x8 sf[NPO];
          get_frag<NPO>(x_s + (s * NC + n) * 3 * FRAG, lane, sf);
          acc.add(qa[s], sf);
        }
        now[n] = acc.sum() * f_eg * sh.scale;
        // what the gradient needs is stored from here: loads of the state waves would wait behind their own stores
        if (KEEP && wave < KS && p.col0 + 16 * n < sh.dvp)
          store_slab(x_s + (wave * NC + n) * 3 * FRAG, w.s0 + ((p.bh * sh.chunks + ch) * sh.dvp + (p.tile * NC + n) * 16) * DKP, wave, p);
      }
      load_q(next);
      lds_barrier();
      if (ch > 0) {
        finish(ch - 1);
        load_p(here);
      }
#pragma unroll
      for (int n = 0; n < NC; ++n) qs[n] = now[n];
      lds_barrier();
    }
    if (p.n_chunks > 0) finish(p.n_chunks - 1);
#pragma unroll
    for (int n = 0; n < NC; ++n)
      if (p.col0 + 16 * n < sh.dv)
        for (int64_t t = p.n_chunks * C + wave * 4 + p.quad; t < sh.time; t += 16) op[t * o_stride + p.col0 + 16 * n] = (T)0.0f;
    return;
  }

  __builtin_amdgcn_s_setprio(3);                  // ahead of the read-out wave on the same SIMD
  const T* vp = v + p.b * sh.vs[0] + p.h * sh.vs[2];
  const int row0 = 16 * MT * wave + 4 * p.quad;   // first of this lane's rows of S
  f32x4 S[NC][MT];
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row0 + 16 * t + r, col = p.col0 + 16 * n;
        S[n][t][r] = state0 && col < sh.dv && row < sh.dk ? state0[(p.bh * sh.dk + row) * sh.dv + col] : 0.0f;
      }
  bf16x8 ka[KS][NPI], kt[MT][2][NPI], ta[2][3];
  f32x4 f_beta, f_eg, f_rest, whole;
  Columns<T, NC> vals(sh, p, sh.vs[1]);
  auto load_k = [&](const Cursor& at) {
#pragma unroll
    for (int s = 0; s < KS; ++s) load_frag<NPI>(at.keys + KB::KA, wave * KS + s, 4 * KS * FRAG, lane, ka[s]);
    vals.load(vp + at.ch * C * sh.vs[1], p, at.left(p));
    f_eg = load_at<f32x4>(at.rows + C, (uint32_t)tok * 4);
  };
  auto load_t = [&](const Cursor& at) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
      load_frag<3>(at.gates + GateBlock::TA, lower(wave, min(s, lo)), 6 * FRAG, lane, ta[s]);
    f_beta = load_at<f32x4>(at.rows, (uint32_t)tok * 4);
    f_rest = load_at<f32x4>(at.rows + 2 * C, (uint32_t)tok * 4);
  };
  auto load_kt = [&](const Cursor& at) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        load_frag<NPI>(at.keys + KB::KT, (wave * MT + t) * 2 + s, 2 * KS * 2 * FRAG, lane, kt[t][s]);
    whole = load_at<f32x4>(at.rows + 3 * C, (uint32_t)tok * 4);     // a vector load: the scalar kind shares the LDS counter
  };
  Cursor next(keys, gates, rows, w, 0);
  if (p.n_chunks > 0) {
    load_k(next);
    load_t(next);
    load_kt(next);
    __builtin_amdgcn_s_waitcnt(WAIT_VM);
  }
  for (int64_t ch = 0; ch < p.n_chunks; ++ch) {
    const int left = (int)std::min<int64_t>(C, p.len - ch * C);
    next = next.step(w, 1, p);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        put_half<3>(x_s + (((wave * MT + t) / 2) * NC + n) * 3 * FRAG, (wave * MT + t) & 1, lane, S[n][t]);
    lds_barrier();
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      Orders<3> acc;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf16x8 sf[3];
        get_frag<3>(x_s + (s * NC + n) * 3 * FRAG, lane, sf);
        acc.add(ka[s], sf);
      }
      put_half<3>(x_r + (lo * NC + n) * 3 * FRAG, wave & 1, lane, vals.get(sh, p, n, left) - f_eg * acc.sum());
    }
    lds_barrier();
    load_k(next);                // behind the barrier: issued while the first LDS reads are on their way
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      Orders<3> acc;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= lo) {
          bf16x8 rf[3];
          get_frag<3>(x_r + (s * NC + n) * 3 * FRAG, lane, rf);
          acc.add(ta[s], rf);
        }
      const f32x4 delta = acc.sum(), vn = delta * f_beta;
      put_half<3>(x_w + (lo * NC + n) * 3 * FRAG, wave & 1, lane, vn * f_rest);
      put_half<NPO>(x_v[ch & 1] + (lo * NC + n) * NPO * FRAG, wave & 1, lane, vn);
      if (KEEP) x_d[(((int)(ch & 1) * 4 + wave) * NC + n) * 64 + lane] = delta;
    }
    lds_barrier();
    load_t(next);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      Orders<3> acc[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t].v[0] = S[n][t] * whole;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 wf[3];
        get_frag<3>(x_w + (s * NC + n) * 3 * FRAG, lane, wf);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t].add(kt[t][s], wf);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) S[n][t] = acc[t].sum();
    }
    load_kt(next);
  }
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row0 + 16 * t + r, col = p.col0 + 16 * n;
        if (col < sh.dv && row < sh.dk) state[(p.bh * sh.dk + row) * sh.dv + col] = S[n][t][r];
      }
}

template <typename T, int DKP, int NPI, int NC>
__global__ void __launch_bounds__(TEAM, 2)
    k_delta_scan_back(Shape sh, const T* __restrict__ d_o, const float* __restrict__ d_state, const int32_t* __restrict__ lengths,
                      T* __restrict__ dv, float* __restrict__ d_state0, Work w) {
  typedef KeyBlock<DKP, NPI> KB;
  constexpr int KS = DKP / 32, MT = DKP / 64;
  // the read-out waves' P^T dO (x_p) and Q^T (scale e^gamma dO) (x_q) as accumulators of the state waves, in f32
  __shared__ bf16 x_s[KS * NC * 3 * FRAG], x_d[2 * NC * NPI * FRAG], x_g[2 * NC * 3 * FRAG], x_x[2 * NC * 3 * FRAG], x_e[2 * NC * 3 * FRAG];
  __shared__ f32x4 x_p[4 * NC * 64], x_q[4 * MT * NC * 64], x_l[4 * NC * 64];      // x_l: e, for the read-out waves to store
  __shared__ char sink[4][256];
  const int tiles = (sh.dvp / 16 + NC - 1) / NC;
  Place p;
  if (!place_of<NC>(sh, lengths, p)) return;
  const int lane = p.lane, wave = p.wave, tok = p.tok;
  const bf16* keys = w.keys + (p.b * sh.kheads + p.kh) * sh.chunks * w.key_size;
  const bf16* gates = w.gates + p.bh * sh.chunks * w.gate_size;
  const float* rows = w.rows + p.bh * sh.chunks * ROWS;
  const int64_t stride = (int64_t)sh.heads * sh.dv, base = (p.b * sh.time * sh.heads + p.h) * sh.dv;
  const int half = wave / 2;                      // first slab of this wave's rows of T^T and P^T

  if (p.reads) {
    const bool all_cols = p.tile * 16 * NC + 16 * NC <= sh.dv;
    bf16x8 qt[MT][2][NPI], pt[2][3];
    f32x4 f_eg;
    Columns<T, NC> vals(sh, p, stride);
    auto load_o = [&](const Cursor& at) {
      vals.load(d_o + base + at.ch * C * stride, p, at.left(p));
      f_eg = load_at<f32x4>(at.rows + C, (uint32_t)tok * 4);
    };
    auto load_qp = [&](const Cursor& at) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        load_frag<3>(at.gates + GateBlock::PT, upper(wave, max(s, half)), 6 * FRAG, lane, pt[s]);
#pragma unroll
        for (int t = 0; t < MT; ++t)
          load_frag<NPI>(at.keys + KB::QT, (wave * MT + t) * 2 + s, 2 * KS * 2 * FRAG, lane, qt[t][s]);
      }
    };
    // a chunk's dO into fragments, then the two products: step `ch` runs between the state waves' barriers of chunk ch + 1
    auto put_o = [&](const Cursor& at) {
      const int left = at.left(p);
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const f32x4 d = vals.get(sh, p, n, left);
        put_half<NPI>(x_d + (half * NC + n) * NPI * FRAG, wave & 1, lane, d);       // bf16 gradients are one plane
        put_half<3>(x_g + (half * NC + n) * 3 * FRAG, wave & 1, lane, d * f_eg * sh.scale);
      }
      load_o(at.step(w, -1, p));
    };
    f32x4 rp[NC], rq[NC][MT];
    auto products = [&](const Cursor& at) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        Orders<3> acc, aq[MT];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          bf16x8 df[NPI], gf[3];
          get_frag<NPI>(x_d + (s * NC + n) * NPI * FRAG, lane, df);
          get_frag<3>(x_g + (s * NC + n) * 3 * FRAG, lane, gf);
          if (s >= half) acc.add(pt[s], df);
#pragma unroll
          for (int t = 0; t < MT; ++t) aq[t].add(qt[t][s], gf);
        }
        rp[n] = acc.sum();
#pragma unroll
        for (int t = 0; t < MT; ++t) rq[n][t] = aq[t].sum();
      }
      load_qp(at.step(w, -1, p));
    };
    auto hand_over = [&]() {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        x_p[(wave * NC + n) * 64 + lane] = rp[n];
#pragma unroll
        for (int t = 0; t < MT; ++t) x_q[((wave * MT + t) * NC + n) * 64 + lane] = rq[n][t];
      }
    };
    Cursor now(keys, gates, rows, w, std::max<int64_t>(p.n_chunks, 1) - 1);
    if (p.n_chunks > 0) {
      load_o(now);
      load_qp(now);
      __builtin_amdgcn_s_waitcnt(WAIT_VM);
      put_o(now);
    }
    lds_barrier();
    if (p.n_chunks > 0) products(now);
    for (int64_t ch = p.n_chunks - 1; ch >= 0; --ch) {
      hand_over();               // read by the state waves between barriers one and two (x_p) and behind three (x_q)
      const int64_t at = p.bh * sh.chunks + ch;
      const int left = now.left(p), left_o = (int)std::min<int64_t>(C, sh.time - ch * C);
      const f32x4 f_beta = load_at<f32x4>(now.rows, (uint32_t)tok * 4);
      now = now.step(w, -1, p);
      const Cursor later = now.step(w, -1, p);
      touch(later.keys, KB::SIZE_KEEP * 2, p.tile * 4 + wave, tiles * 4, lane, sink[wave]);
      touch(later.gates + GateBlock::TT, 36 * FRAG * 2, tiles * 4 - 1 - p.tile * 4 - wave, tiles * 4, lane, sink[wave]);
      lds_barrier();
      if (wave < KS)
#pragma unroll
        for (int n = 0; n < NC; ++n)
          if (p.col0 + 16 * n < sh.dvp)
            store_slab(x_s + (wave * NC + n) * 3 * FRAG, w.ds1 + (at * sh.dvp + (p.tile * NC + n) * 16) * DKP, wave, p);
      if (ch > 0) put_o(now);
      lds_barrier();
      if (ch > 0) products(now);
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const f32x4 e = x_l[(wave * NC + n) * 64 + lane];
        if (p.col0 + 16 * n < sh.dvp) store_rows(w.e + (at * sh.dvp + (p.tile * NC + n) * 16) * C, tok, p.c, e);
        f32x4 out = e * f_beta;
        if (left < C)
#pragma unroll
          for (int r = 0; r < 4; ++r) out[r] = tok + r < left ? out[r] : 0.0f;
        store_tokens(dv + base + ch * C * stride, p, p.col0 + 16 * n, (uint32_t)stride * sizeof(T), all_cols && left_o == C, sh.dv, left_o, out);
      }
      lds_barrier();
    }
    return;
  }

  __builtin_amdgcn_s_setprio(3);
  const int row0 = 16 * MT * wave + 4 * p.quad;
  f32x4 S[NC][MT];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int col = p.col0 + 16 * n;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = row0 + 16 * t + r;
        S[n][t][r] = d_state && col < sh.dv && row < sh.dk ? d_state[(p.bh * sh.dk + row) * sh.dv + col] : 0.0f;
      }
    if (col < sh.dv)
      for (int64_t t = p.n_chunks * C + wave * 4 + p.quad; t < sh.time; t += 16) dv[base + t * stride + col] = (T)0.0f;
  }
  bf16x8 ka[KS][NPI], kt[MT][2][NPI], tt[2][3];
  f32x4 f_beta, f_eg, f_rest, whole;
  auto load_k = [&](const Cursor& at) {
#pragma unroll
    for (int s = 0; s < KS; ++s) load_frag<NPI>(at.keys + KB::KA, wave * KS + s, 4 * KS * FRAG, lane, ka[s]);
    f_rest = load_at<f32x4>(at.rows + 2 * C, (uint32_t)tok * 4);
  };
  auto load_t = [&](const Cursor& at) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
      load_frag<3>(at.gates + GateBlock::TT, upper(wave, max(s, half)), 6 * FRAG, lane, tt[s]);
    f_beta = load_at<f32x4>(at.rows, (uint32_t)tok * 4);
    f_eg = load_at<f32x4>(at.rows + C, (uint32_t)tok * 4);
  };
  auto load_kt = [&](const Cursor& at) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        load_frag<NPI>(at.keys + KB::KT, (wave * MT + t) * 2 + s, 2 * KS * 2 * FRAG, lane, kt[t][s]);
    whole = load_at<f32x4>(at.rows + 3 * C, (uint32_t)tok * 4);
  };
  Cursor next(keys, gates, rows, w, std::max<int64_t>(p.n_chunks, 1) - 1);
  if (p.n_chunks > 0) {
    load_k(next);
    load_t(next);
    load_kt(next);
    __builtin_amdgcn_s_waitcnt(WAIT_VM);
  }
  lds_barrier();
  for (int64_t ch = p.n_chunks - 1; ch >= 0; --ch) {
    next = next.step(w, -1, p);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        put_half<3>(x_s + (((wave * MT + t) / 2) * NC + n) * 3 * FRAG, (wave * MT + t) & 1, lane, S[n][t]);
    lds_barrier();
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      Orders<3> acc;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        bf16x8 sf[3];
        get_frag<3>(x_s + (s * NC + n) * 3 * FRAG, lane, sf);
        acc.add(ka[s], sf);
      }
      put_half<3>(x_x + (half * NC + n) * 3 * FRAG, wave & 1, lane, acc.sum() * f_rest + x_p[(wave * NC + n) * 64 + lane]);
    }
    lds_barrier();
    load_k(next);                // behind the barrier: issued while the first LDS reads are on their way
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      Orders<3> acc;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s >= half) {
          bf16x8 xf[3];
          get_frag<3>(x_x + (s * NC + n) * 3 * FRAG, lane, xf);
          acc.add(tt[s], xf);
        }
      const f32x4 e = acc.sum(), be = e * f_beta;
      put_half<3>(x_e + (half * NC + n) * 3 * FRAG, wave & 1, lane, -(be * f_eg));
      x_l[(wave * NC + n) * 64 + lane] = e;
    }
    lds_barrier();
    load_t(next);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      Orders<3> acc[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t].v[0] = S[n][t] * whole + x_q[((wave * MT + t) * NC + n) * 64 + lane];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bf16x8 ef[3];
        get_frag<3>(x_e + (s * NC + n) * 3 * FRAG, lane, ef);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t].add(kt[t][s], ef);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) S[n][t] = acc[t].sum();
    }
    load_kt(next);
    lds_barrier();               // x_p and x_q are written again in front of the next chunk's first barrier
  }
  if (d_state0)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = row0 + 16 * t + r, col = p.col0 + 16 * n;
          if (col < sh.dv && row < sh.dk) d_state0[(p.bh * sh.dk + row) * sh.dv + col] = S[n][t][r];
        }
}

// ---------------------------------------------------------------------------
// gradients of q, k and the gates, all chunks at once
// ---------------------------------------------------------------------------
// Sixteen waves: wave w forms the rows of tokens [16 (w % 4), + 16) and the dk quarter w / 4.  Per 32 columns of dv, S0, dS1,
// e, delta and dO become fragment planes in LDS once, for all waves (each wave splitting its own operands: 380 us for 1024
// chunks of 64 x 128 x 128), while the next columns are on their way to registers; the row sums <dS1, S0> and e.delta
// fall out of the same registers.  1024 chunks in 119 to 128 us, 320 MB at 2.6 TB/s: memory, splitting and products of the one
// workgroup that a CU holds take turns (8 us of them are the products q.k and k.k that the decays' gradient takes).  E and F go
// to LDS as fragments of themselves and of their transposes, split once.  (Eight waves of twice the work, 194 registers, before
// those products: 129 us against 113; the phases of one workgroup hardly overlapped.)
constexpr int BACK = 1024;

// eight values from LDS to a row, in vectors of 16 bytes where it is whole and aligned
template <typename T>
__device__ __forceinline__ void store8(T* to, const float* x, int n, int vec) {
  if (vec) {
    constexpr int N = 16 / sizeof(T);
    typedef T vec16 __attribute__((ext_vector_type(N)));
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      vec16 v;
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = (T)x[i + j];
      *(vec16*)(to + i) = v;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) to[j] = (T)x[j];
  }
}

template <typename T, int DKP, int NPI>
__global__ void __launch_bounds__(BACK)
    k_delta_back(Shape sh, const T* __restrict__ d_o, const float* __restrict__ g, const int32_t* __restrict__ lengths,
                 T* __restrict__ dq, T* __restrict__ dk, float* __restrict__ dg, float* __restrict__ dbeta, Work w, int vec_o, int vec_out) {
  typedef KeyBlock<DKP, NPI> KB;
  constexpr int MT = DKP / 16, MH = MT / 4;               // tiles of dk; of one wave
  constexpr int F_S0 = 0, F_S1 = MT * 3 * FRAG, F_E = 2 * F_S1, F_D = F_E + 12 * FRAG, F_O = F_D + 12 * FRAG, F_ALL = F_O + 4 * NPI * FRAG;
  constexpr int E_ROW = 0, F_ROW = 24 * FRAG, E_COL = 48 * FRAG, F_COL = 72 * FRAG, EF_ALL = 96 * FRAG;     // [tile][slab][plane]
  constexpr int KS = DKP / 32, SLABS = NPI == 1 ? KS : 1, TURNS = NPI == 1 ? 2 : 1;       // f32: registers for one slab at a time
  constexpr int LO = DKP + 4;                             // row of dq or dk in LDS: the four quads of a wave miss each other's banks
  constexpr int RESULTS = 2 * C * LO * 4;
  __shared__ __attribute__((aligned(16))) char buffer[std::max(std::max(F_ALL, EF_ALL) * 2, RESULTS)];
  __shared__ float s_gh[C], s_gl[C], s_db[C];
  __shared__ float s_x[C * LD], s_pair[16][C];            // X; its sums over i >= t > j, a wave's rows i
  __shared__ float s_read[4][C], s_put[4][C];             // a token's terms that read S0 and that write S1, by dk quarter
  __shared__ double s_sum[16];
  bf16* frag = (bf16*)buffer;
  float *sq = (float*)buffer, *sk = sq + C * LO;          // dq and dk, once E and F are
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4, c = lane & 15;
  const int wt = wave & 3, wh = wave >> 2;
  const int64_t chunk = gjx_block() % sh.chunks, bh = gjx_block() / sh.chunks, b = bh / sh.heads;
  if (b >= sh.batch) return;
  const int h = (int)(bh % sh.heads), kh = h / sh.group;
  const int64_t len = length_of(lengths, b, sh.time), t0 = chunk * C, at = bh * sh.chunks + chunk;
  const bool shared = sh.group > 1;
  const int64_t g_at = (b * sh.time + t0) * sh.heads + h;
  const int left_o = (int)std::min<int64_t>(C, sh.time - t0), left = (int)std::min<int64_t>(C, len - t0);
  if (left <= 0) {
    for (int i = tid; i < left_o; i += BACK) {
      dg[g_at + (int64_t)i * sh.heads] = 0.0f;
      dbeta[g_at + (int64_t)i * sh.heads] = 0.0f;
    }
    for (int i = tid; i < left_o * sh.dk; i += BACK) {
      const int64_t p = ((b * sh.time + t0 + i / sh.dk) * sh.heads + h) * sh.dk + i % sh.dk;
      if (shared) {
        w.dq[p] = 0.0f;
        w.dk[p] = 0.0f;
      } else {
        dq[p] = (T)0.0f;
        dk[p] = (T)0.0f;
      }
    }
    return;
  }
  const float* rb = w.rows + at * ROWS;
  const bf16* kb = w.keys + ((b * sh.kheads + kh) * sh.chunks + chunk) * w.key_size;
  if (wave == 0) {
    double gam = lane < left ? (double)fmaxf(g[b * sh.gs[0] + (t0 + lane) * sh.gs[1] + h * sh.gs[2]], G_MIN) : 0.0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(gam, o);
      if (lane >= o) gam += up;
    }
    s_gh[lane] = (float)gam;
    s_gl[lane] = (float)(gam - (double)(float)gam);
  }

  // this thread's pieces of a slab: four columns of one row of S0 and dS1, and of e and delta (first half) or dO
  const int row = tid >> 3, sub = tid & 7;                // 128 rows
  const bool has_state = row < DKP;
  const bool first = tid < 512;
  const int trow = row & 63;
  const int64_t in_s = (int64_t)(sub >> 2) * 16 * DKP + min(row, DKP - 1) * 16 + 4 * (sub & 3), in_c = (sub >> 2) * 16 * C + trow * 16 + 4 * (sub & 3);
  const float *p_s0 = w.s0 + at * sh.dvp * DKP + in_s, *p_s1 = w.ds1 + at * sh.dvp * DKP + in_s;
  const float *p_e = w.e + at * sh.dvp * C + in_c, *p_d = w.delta + at * sh.dvp * C + in_c;
  const T* p_o = d_o + ((b * sh.time + t0 + min(trow, left - 1)) * sh.heads + h) * sh.dv;
  f32x4 x0, x1, x2, x3;
  auto load = [&](int s) {
    x0 = *(const f32x4*)(p_s0 + 32 * DKP * s);
    x1 = *(const f32x4*)(p_s1 + 32 * DKP * s);
    if (first) {
      x2 = *(const f32x4*)(p_e + 32 * C * s);
      x3 = *(const f32x4*)(p_d + 32 * C * s);
    } else {
      const int c0 = 32 * s + 4 * sub;
      if (vec_o && c0 + 4 <= sh.dv) {
        typedef T vec4 __attribute__((ext_vector_type(4)));
        const vec4 v = *(const vec4*)(p_o + c0);
#pragma unroll
        for (int j = 0; j < 4; ++j) x2[j] = (float)v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x2[j] = c0 + j < sh.dv ? (float)p_o[c0 + j] : 0.0f;
      }
    }
  };
  auto put4 = [&](int base, int planes, int r, f32x4 v) {
    bf16* f = frag + base + (r >> 4) * planes * FRAG + ((r & 15) + 16 * (sub >> 1)) * 8 + (sub & 1) * 4;
    float x[4] = {v[0], v[1], v[2], v[3]};
    bf16 h[4];
#pragma unroll
    for (int p = 0; p < 3; ++p)
      if (p < planes) {
        if (planes == 3) split_planes<3, 4>(x, p, h);
        else split_planes<1, 4>(x, p, h);
        *(bf16x4*)(f + p * FRAG) = bf16x4{h[0], h[1], h[2], h[3]};
      }
  };

  f32x4 m1[MH], m2[MH], m3[MH], pe = {0, 0, 0, 0}, pf = {0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < MH; ++t) m1[t] = m2[t] = m3[t] = f32x4{0, 0, 0, 0};
  float dot = 0.0f, db = 0.0f;
  const int slabs = sh.dvp / 32;
  load(0);
  for (int s = 0; s < slabs; ++s) {
    if (has_state) {
      put4(F_S0, 3, row, x0);
      put4(F_S1, 3, row, x1);
#pragma unroll
      for (int j = 0; j < 4; ++j) dot += x0[j] * x1[j];
    }
    if (first) {
      put4(F_E, 3, trow, x2);
      put4(F_D, 3, trow, x3);
#pragma unroll
      for (int j = 0; j < 4; ++j) db += x2[j] * x3[j];
    } else {
      if (trow >= left) x2 = f32x4{0, 0, 0, 0};
      put4(F_O, NPI, trow, x2);
    }
    __syncthreads();
    if (s + 1 < slabs) load(s + 1);
    bf16x8 fo[NPI], fe[3], fd[3];
    get_frag<NPI>(frag + F_O + wt * NPI * FRAG, lane, fo);
    get_frag<3>(frag + F_E + wt * 3 * FRAG, lane, fe);
    get_frag<3>(frag + F_D + wt * 3 * FRAG, lane, fd);
#pragma unroll
    for (int t = 0; t < MH; ++t) {
      bf16x8 f0[3], f1[3];
      get_frag<3>(frag + F_S0 + (wh * MH + t) * 3 * FRAG, lane, f0);
      get_frag<3>(frag + F_S1 + (wh * MH + t) * 3 * FRAG, lane, f1);
      m1[t] = mma_planes<NPI, 3, 3>(fo, f0, m1[t]);
      m2[t] = mma_planes<3, 3, 3>(fe, f0, m2[t]);
      m3[t] = mma_planes<3, 3, 3>(fd, f1, m3[t]);
    }
    if (wh <= wt) {
      bf16x8 fj[3];
      get_frag<3>(frag + F_D + wh * 3 * FRAG, lane, fj);
      pe = mma_planes<NPI, 3, 3>(fo, fj, pe);
      pf = mma_planes<3, 3, 3>(fe, fj, pf);
    }
    __syncthreads();
  }
  {
    double d = has_state ? (double)dot : 0.0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) d += __shfl_xor(d, o);
    if (lane == 0) s_sum[wave] = d;
    db += __shfl_xor(db, 1);
    db += __shfl_xor(db, 2);
    db += __shfl_xor(db, 4);
    if (first && sub == 0) s_db[trow] = db;
  }
  {
    f32x4 ev, fv;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wt + 4 * quad + r, jj = 16 * wh + c;
      const float d = jj <= i ? expf((s_gh[i] - s_gh[jj]) + (s_gl[i] - s_gl[jj])) * rb[jj] : 0.0f;
      ev[r] = jj <= i ? sh.scale * d * pe[r] : 0.0f;
      fv[r] = jj < i ? -rb[i] * d * pf[r] : 0.0f;
    }
    f32x4 qk = {0, 0, 0, 0}, kk = {0, 0, 0, 0};
    if (wh <= wt)
#pragma unroll SLABS
      for (int s = 0; s < KS; ++s) {
        bf16x8 fq[NPI], fi[NPI], fj[NPI];
        load_frag<NPI>(kb + KB::QA, wt * KS + s, 4 * KS * FRAG, lane, fq);
        load_frag<NPI>(kb + KB::KA, wt * KS + s, 4 * KS * FRAG, lane, fi);
        load_frag<NPI>(kb + KB::KA, wh * KS + s, 4 * KS * FRAG, lane, fj);
        qk = mma_planes<NPI, NPI, NPI>(fq, fj, qk);
        kk = mma_planes<NPI, NPI, NPI>(fi, fj, kk);
      }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wt + 4 * quad + r, jj = 16 * wh + c;
      s_x[i * LD + jj] = jj < i ? ev[r] * qk[r] + fv[r] * kk[r] : 0.0f;      // (E_ii does not hang on the decay)
    }
    // their transposes (rows of the operand: jj; reduction: i) as they lie in the registers; themselves entry by entry
    put_half<3>(frag + E_COL + (wh * 2 + (wt >> 1)) * 3 * FRAG, wt & 1, lane, ev);
    put_half<3>(frag + F_COL + (wh * 2 + (wt >> 1)) * 3 * FRAG, wt & 1, lane, fv);
    bf16* at_row = frag + (wt * 2 + (wh >> 1)) * 3 * FRAG + (4 * quad + 16 * (c >> 2)) * 8 + 4 * (wh & 1) + (c & 3);
    float xe[4] = {ev[0], ev[1], ev[2], ev[3]}, xf[4] = {fv[0], fv[1], fv[2], fv[3]};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      bf16 he[4], hf[4];
      split_planes<3, 4>(xe, p, he);
      split_planes<3, 4>(xf, p, hf);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        at_row[E_ROW + p * FRAG + r * 8] = he[r];
        at_row[F_ROW + p * FRAG + r * 8] = hf[r];
      }
    }
  }
  const f32x4 be = *(const f32x4*)(rb + 16 * wt + 4 * quad), eg = *(const f32x4*)(rb + C + 16 * wt + 4 * quad);
  const f32x4 rest = *(const f32x4*)(rb + 2 * C + 16 * wt + 4 * quad);
  __syncthreads();

#pragma unroll
  for (int t = 0; t < MH; ++t) {
    m1[t] *= eg * sh.scale;
    m2[t] *= -(be * eg);
    m3[t] *= be * rest;
  }
  f32x4 sum = {0, 0, 0, 0}, put = {0, 0, 0, 0};
#pragma unroll TURNS
  for (int u = 0; u < 2; ++u) {                           // the slab of this wave's tokens, then the other
    const int s = u ^ (wt >> 1);
    bf16x8 kt[MH][NPI], qt[MH][NPI];
#pragma unroll
    for (int t = 0; t < MH; ++t) {
      load_frag<NPI>(kb + KB::KT, (wh * MH + t) * 2 + s, MT * 2 * FRAG, lane, kt[t]);
      load_frag<NPI>(kb + KB::QT, (wh * MH + t) * 2 + s, MT * 2 * FRAG, lane, qt[t]);
    }
    if (u == 0)                                           // q and k where dq and dk are: entries of the fragments at hand
#pragma unroll
      for (int t = 0; t < MH; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {                     // (tokens behind the end and columns behind dk: q and k are 0)
          float qv = 0.0f, kv = 0.0f;
#pragma unroll
          for (int p = NPI - 1; p >= 0; --p) {
            qv += (float)(wt & 1 ? qt[t][p][4 + r] : qt[t][p][r]);
            kv += (float)(wt & 1 ? kt[t][p][4 + r] : kt[t][p][r]);
          }
          sum[r] += qv * m1[t][r] + kv * m2[t][r];
          put[r] += kv * m3[t][r];
        }
    if (s <= wt >> 1) {                                   // (E and F are lower triangular)
      bf16x8 fe[3], ff[3];
      get_frag<3>(frag + E_ROW + (wt * 2 + s) * 3 * FRAG, lane, fe);
      get_frag<3>(frag + F_ROW + (wt * 2 + s) * 3 * FRAG, lane, ff);
#pragma unroll
      for (int t = 0; t < MH; ++t) {
        m1[t] = mma_planes<3, NPI, 3>(fe, kt[t], m1[t]);
        m2[t] = mma_planes<3, NPI, 3>(ff, kt[t], m2[t]);
      }
    }
    if (s >= wt >> 1) {
      bf16x8 fe[3], ff[3];
      get_frag<3>(frag + E_COL + (wt * 2 + s) * 3 * FRAG, lane, fe);
      get_frag<3>(frag + F_COL + (wt * 2 + s) * 3 * FRAG, lane, ff);
#pragma unroll
      for (int t = 0; t < MH; ++t) {
        m3[t] = mma_planes<3, NPI, 3>(fe, qt[t], m3[t]);
        m3[t] = mma_planes<3, NPI, 3>(ff, kt[t], m3[t]);
      }
    }
  }
  float pair = 0.0f;                                      // lane t: rows i >= t of every sixteenth, columns j < t
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = 16 * u + wave;
    float x = s_x[i * LD + lane];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float before = __shfl_up(x, o);
      if (lane >= o) x += before;
    }
    x = __shfl_up(x, 1);
    pair += lane > 0 && i >= lane ? x : 0.0f;
  }
  s_pair[wave][lane] = pair;
  __syncthreads();                                        // the fragments of E and F are used up
#pragma unroll
  for (int t = 0; t < MH; ++t) {
    const int col = 16 * (wh * MH + t) + c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wt + 4 * quad + r;
      sq[i * LO + col] = i < left ? m1[t][r] : 0.0f;
      sk[i * LO + col] = i < left ? m2[t][r] + m3[t][r] : 0.0f;
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float a = sum[r], b = put[r];
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      a += __shfl_xor(a, o);
      b += __shfl_xor(b, o);
    }
    if (c == 0) {
      s_read[wh][16 * wt + 4 * quad + r] = a;
      s_put[wh][16 * wt + 4 * quad + r] = b;
    }
  }
  __syncthreads();
  // out of LDS in rows: pieces of eight columns (stored from the accumulators, two bytes a lane, the kernel took 139 us instead
  // of 129 for the 1024 chunks)
  for (int u = tid; u < 2 * left_o * (DKP / 8); u += BACK) {
    const bool is_k = u >= left_o * (DKP / 8);
    const int v = is_k ? u - left_o * (DKP / 8) : u, i = v / (DKP / 8), c0 = v % (DKP / 8) * 8;
    if (c0 >= sh.dk) continue;
    const float* x = (is_k ? sk : sq) + i * LO + c0;
    const int64_t p = ((b * sh.time + t0 + i) * sh.heads + h) * sh.dk + c0;
    const int n = min(8, sh.dk - c0);
    if (shared) store8((is_k ? w.dk : w.dq) + p, x, n, vec_out);
    else store8((is_k ? dk : dq) + p, x, n, vec_out);
  }
  if (wave == 0) {
    double reads = 0.0, puts = 0.0, s = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      reads += (double)s_read[i][lane];
      puts += (double)s_put[i][lane];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s += (double)s_pair[i][lane] + (double)rb[3 * C] * s_sum[i];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double later = __shfl_down(reads, o), earlier = __shfl_up(puts, o);
      if (lane + o < 64) reads += later;
      if (lane >= o) puts += earlier;
    }
    puts = __shfl_up(puts, 1);
    s += reads + (lane > 0 ? puts : 0.0);
    if (lane < left_o) {
      dg[g_at + (int64_t)lane * sh.heads] = lane < left ? (float)s : 0.0f;
      dbeta[g_at + (int64_t)lane * sh.heads] = lane < left ? s_db[lane] : 0.0f;
    }
  }
}

// sum over the heads that share a key head, in order
template <typename T>
__global__ void __launch_bounds__(GJX_BLOCK)
    k_delta_shared_heads(Shape sh, const float* __restrict__ a, const float* __restrict__ b, T* __restrict__ out_a, T* __restrict__ out_b) {
  const int64_t total = sh.batch * sh.time * sh.kheads * sh.dk;
  for (int64_t i = (int64_t)blockIdx.x * GJX_BLOCK + threadIdx.x; i < total; i += (int64_t)gridDim.x * GJX_BLOCK) {
    const int64_t d = i % sh.dk, row = i / sh.dk;
    const float *pa = a + row * sh.group * sh.dk + d, *pb = b + row * sh.group * sh.dk + d;
    float sa = 0.0f, sb = 0.0f;
    for (int j = 0; j < sh.group; ++j) {
      sa += pa[(int64_t)j * sh.dk];
      sb += pb[(int64_t)j * sh.dk];
    }
    out_a[i] = (T)sa;
    out_b[i] = (T)sb;
  }
}

// ---------------------------------------------------------------------------
// one token: a workgroup holds a head's state in registers, 4 columns x R rows per lane
//   u = beta (v - a S^T k), S' = a S + k u^T, o = scale (a S^T q + (q.k) u)
// Bound by memory: the states of 1000 particles x 8 heads x 128 x 128 read and written, 1.05 GB, in 164 us: 6.4 TB/s (some
// ancestors are read more than once and come from the caches)
// ---------------------------------------------------------------------------
template <typename T, int CG, int R>
__global__ void __launch_bounds__(256)
    k_delta_step(Shape sh, const float* __restrict__ state, const int32_t* __restrict__ ancestors, const T* __restrict__ q,
                 const T* __restrict__ k, const T* __restrict__ v, const float* __restrict__ g, const float* __restrict__ beta,
                 T* __restrict__ o, float* __restrict__ state_out, int col_tiles) {
  constexpr int RG = 256 / CG;
  __shared__ float s_q[128], s_k[128];
  __shared__ f32x4 s_pk[RG][CG], s_pq[RG][CG];
  const int tid = threadIdx.x, cg = tid % CG, rg = tid / CG;
  const int64_t bh = gjx_block() / col_tiles, b = bh / sh.heads;
  if (b >= sh.batch) return;
  const int h = (int)(bh % sh.heads), kh = h / sh.group;
  const int col = (int)(gjx_block() % col_tiles) * CG * 4 + cg * 4;
  if (tid < 128) {
    s_q[tid] = tid < sh.dk ? (float)q[b * sh.qs[0] + kh * sh.qs[2] + tid] : 0.0f;
    s_k[tid] = tid < sh.dk ? (float)k[b * sh.ks[0] + kh * sh.ks[2] + tid] : 0.0f;
  }
  int64_t src = b;
  if (ancestors) src = std::min<int64_t>(std::max<int64_t>(ancestors[b], 0), sh.batch - 1);
  const float* sp = state + (src * sh.heads + h) * (int64_t)sh.dk * sh.dv;
  float* op = state_out + bh * (int64_t)sh.dk * sh.dv;
  const bool vec = (sh.dv & 3) == 0;
  f32x4 S[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r * RG + rg;
    S[r] = f32x4{0, 0, 0, 0};
    if (row < sh.dk) {
      if (vec && col < sh.dv) S[r] = *(const f32x4*)(sp + (int64_t)row * sh.dv + col);
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < sh.dv) S[r][e] = sp[(int64_t)row * sh.dv + col + e];
    }
  }
  const float a = expf(g[b * sh.gs[0] + h * sh.gs[2]]), be = beta[b * sh.bs[0] + h * sh.bs[2]];
  __syncthreads();
  f32x4 pk = {0, 0, 0, 0}, pq = {0, 0, 0, 0};
  float qk = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r * RG + rg;
    S[r] *= a;
    pk += S[r] * s_k[row];
    pq += S[r] * s_q[row];
  }
  for (int i = 0; i < sh.dk; ++i) qk += s_q[i] * s_k[i];
  s_pk[rg][cg] = pk;
  s_pq[rg][cg] = pq;
  __syncthreads();
  pk = pq = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < RG; ++i) {
    pk += s_pk[i][cg];
    pq += s_pq[i][cg];
  }
  f32x4 u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    u[e] = col + e < sh.dv ? be * ((float)v[b * sh.vs[0] + h * sh.vs[2] + col + e] - pk[e]) : 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r * RG + rg;
    if (row < sh.dk) {
      S[r] += u * s_k[row];
      if (vec && col < sh.dv) *(f32x4*)(op + (int64_t)row * sh.dv + col) = S[r];
      else
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < sh.dv) op[(int64_t)row * sh.dv + col + e] = S[r][e];
    }
  }
  if (rg == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < sh.dv) o[bh * sh.dv + col + e] = (T)(sh.scale * (pq[e] + qk * u[e]));
}

// ---------------------------------------------------------------------------
// gradient of a gather of states by ancestors: out[j] = sum of d[i] over the i whose ancestor is j, in ascending order of i
// (a stable sort of the ancestors comes first).  Every sum has a fixed order and every row is written once, so equal calls give
// equal bits; adding with atomics gave other bits each time.  Bound by memory, the gradient read and the sums written once:
// 1000 states of 131072 entries in 187 us, 5.6 TB/s (214 with the sort; atomics 536); 20000 of 1024 in 32 us (73; 83).  A run of
// many short rows is read by one workgroup per 4 KB of them: a third of 20000 in one run 0.6 ms, of 2^20 rows of 16 entries 1 ms (atomics
// 0.2 and 14).
// ---------------------------------------------------------------------------
// starts[j]: the first of the sorted ancestors that is not below j; j = n: their end
__global__ void __launch_bounds__(GJX_BLOCK)
    k_delta_runs(const int32_t* __restrict__ sorted, int64_t n, int64_t* __restrict__ starts) {
  for (int64_t j = (int64_t)blockIdx.x * GJX_BLOCK + threadIdx.x; j <= n; j += (int64_t)gridDim.x * GJX_BLOCK) {
    int64_t lo = 0, hi = n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (sorted[mid] < j) lo = mid + 1;
      else hi = mid;
    }
    starts[j] = lo;
  }
}

// V entries a lane, `cols` lanes (a power of two) along a row and 256 / cols rows of the run at a time: short rows of one
// ancestor that took many children are still read by all lanes
template <typename V>
__global__ void __launch_bounds__(GJX_BLOCK)
    k_delta_run_sums(const V* __restrict__ d, const int64_t* __restrict__ order, const int64_t* __restrict__ starts, int64_t n, int64_t row,
                     int cols, int tiles, V* __restrict__ out) {
  __shared__ V s_part[GJX_BLOCK];
  const int tid = threadIdx.x, rows = GJX_BLOCK / cols;
  const int64_t j = gjx_block() / tiles;
  if (j >= n) return;
  const int64_t col = (int64_t)(gjx_block() % tiles) * cols + (tid & (cols - 1)), at = min(col, row - 1);
  const int64_t end = starts[j + 1];
  V sum = {};
  int64_t i = starts[j] + tid / cols;
  for (; i + 7 * rows < end; i += 8 * rows) {               // eight loads in flight, added in order
    V x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = d[order[i + u * rows] * row + at];
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += x[u];
  }
  for (; i < end; i += rows) sum += d[order[i] * row + at];
  s_part[tid] = sum;
  __syncthreads();
  for (int o = GJX_BLOCK / 2; o >= cols; o >>= 1) {
    if (tid < o) s_part[tid] += s_part[tid + o];
    __syncthreads();
  }
  if (tid < cols && col < row) out[j * row + col] = s_part[tid];
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

int32_t check_shape(const char* who, const gjx_delta_shape* s) {
  GJX_REQUIRE(s != nullptr, GJX_EINVAL, "%s: shape is null", who);
  GJX_REQUIRE(s->dtype == GJX_F32 || s->dtype == GJX_BF16, GJX_EINVAL, "%s: dtype %d is neither GJX_F32 nor GJX_BF16", who, s->dtype);
  GJX_REQUIRE(s->batch >= 0 && s->time >= 0 && s->kheads >= 1 && s->heads >= 1 && s->heads % s->kheads == 0, GJX_EINVAL,
              "%s: bad sizes (batch %lld, time %lld, kheads %d, heads %d)", who, (long long)s->batch, (long long)s->time, s->kheads, s->heads);
  GJX_REQUIRE(s->dk >= 1 && s->dk <= 128 && s->dv >= 1 && s->dv <= 1024, GJX_ELIMIT, "%s: dk=%d not in [1, 128] or dv=%d not in [1, 1024]",
              who, s->dk, s->dv);
  GJX_REQUIRE(s->batch <= (1 << 24) && s->heads <= 1024 && s->time <= ((int64_t)1 << 30), GJX_ELIMIT,
              "%s: batch up to 2^24, heads up to 1024, time up to 2^30", who);
  GJX_REQUIRE(s->v_stride[1] <= (1 << 22), GJX_ELIMIT, "%s: v's token stride is above 2^22 elements", who);
  const int64_t blocks = s->batch * s->heads * std::max<int64_t>(up(s->time, C) / C, up(s->dv, 32) / 16 + 8);
  GJX_REQUIRE(blocks < ((int64_t)1 << 31), GJX_ELIMIT, "%s: batch x heads x chunks is too large", who);
  return GJX_OK;
}

Shape shape_of(const gjx_delta_shape* s) {
  Shape r = {};
  r.kheads = s->kheads;
  r.heads = s->heads;
  r.group = s->heads / s->kheads;
  r.dk = s->dk;
  r.dv = s->dv;
  r.dvp = (int)up(s->dv, 32);
  r.scale = s->scale;
  r.batch = s->batch;
  r.time = s->time;
  for (int i = 0; i < 3; ++i) {
    r.qs[i] = s->q_stride[i];
    r.ks[i] = s->k_stride[i];
    r.vs[i] = s->v_stride[i];
    r.gs[i] = s->g_stride[i];
    r.bs[i] = s->b_stride[i];
  }
  r.chunks = up(s->time, C) / C;
  return r;
}

struct Layout {
  int dkp, npi;
  int64_t key_size, gate_size;
  int64_t keys, gates, rows, s0, delta, bytes;       // the filter's workspace
  int64_t ds1, e, dq, dk, grad_bytes;                // the gradient's scratch
};

Layout layout_of(const gjx_delta_shape* s, bool keep) {
  Layout l = {};
  const Shape sh = shape_of(s);
  l.dkp = s->dk <= 64 ? 64 : 128;
  l.npi = s->dtype == GJX_F32 ? 3 : 1;
  const int64_t side = (int64_t)l.npi * 4 * (l.dkp / 32) * FRAG;      // K rows = Q rows = K columns = Q columns
  l.key_size = side * (keep ? 4 : 3);
  l.gate_size = keep ? GateBlock::SIZE_KEEP : GateBlock::SIZE;
  const int64_t kc = sh.batch * sh.kheads * sh.chunks, hc = sh.batch * sh.heads * sh.chunks;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at = up(at + bytes, 256);
    return p;
  };
  l.keys = take(kc * l.key_size * 2);
  l.gates = take(hc * l.gate_size * 2);
  l.rows = take(hc * ROWS * 4);
  l.s0 = take(keep ? hc * l.dkp * sh.dvp * 4 : 0);
  l.delta = take(keep ? hc * C * sh.dvp * 4 : 0);
  l.bytes = at;
  at = 0;
  const int64_t shared = sh.group > 1 ? sh.batch * sh.time * sh.heads * sh.dk * 4 : 0;
  l.ds1 = take(hc * l.dkp * sh.dvp * 4);
  l.e = take(hc * C * sh.dvp * 4);
  l.dq = take(shared);
  l.dk = take(shared);
  l.grad_bytes = at;
  return l;
}

Work work_of(const Layout& l, char* base, char* scratch) {
  Work w = {};
  w.keys = (bf16*)(base + l.keys);
  w.gates = (bf16*)(base + l.gates);
  w.key_size = l.key_size;
  w.gate_size = l.gate_size;
  w.rows = (float*)(base + l.rows);
  w.s0 = (float*)(base + l.s0);
  w.delta = (float*)(base + l.delta);
  if (scratch) {
    w.ds1 = (float*)(scratch + l.ds1);
    w.e = (float*)(scratch + l.e);
    w.dq = (float*)(scratch + l.dq);
    w.dk = (float*)(scratch + l.dk);
  }
  return w;
}

template <typename T>
bool aligned_rows(const T* p, const int64_t (&s)[3]) {
  const int per16 = 16 / (int)sizeof(T);
  return ((uintptr_t)p & 15) == 0 && s[0] % per16 == 0 && s[1] % per16 == 0 && s[2] % per16 == 0;
}

// columns per workgroup of the scans, in tiles of 16: the walk over the chunks is a chain, so narrow workgroups are faster
// until the 256 CUs are taken; wider ones then read each fragment once for twice the columns
constexpr int wide_tiles(int dkp, int npi) { return dkp == 128 && npi == 3 ? 1 : 2; }      // f32 at dk > 64: registers for one
bool scan_wide(const Shape& sh) { return sh.batch * sh.heads * (sh.dvp / 16) > 256; }
dim3 scan_grid(const Shape& sh, int nc) { return gjx_grid_rows(up(sh.batch * sh.heads, 8) * (up(sh.dvp / 16, nc) / nc)); }

template <typename T, int DKP, bool KEEP>
int32_t run_filter(const Shape& sh, const T* q, const T* k, const T* v, const float* g, const float* beta, const float* state0,
                   const int32_t* lengths, T* o, float* state, const Work& w, hipStream_t s) {
  constexpr int NPI = sizeof(T) == 4 ? 3 : 1;
  if (sh.chunks > 0) {
    constexpr int lds = std::max(2 * NPI * C * (DKP + 8) * 2, 2 * C * LD * 4) + C * LD * 4 + 3 * C * 4;
    GJX_CHECK_HIP(hipFuncSetAttribute((const void*)k_delta_prepare<T, DKP, NPI, KEEP>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    k_delta_prepare<T, DKP, NPI, KEEP><<<gjx_grid_rows(sh.batch * sh.heads * sh.chunks), 256, lds, s>>>(
        sh, q, k, g, beta, lengths, w, aligned_rows(q, sh.qs) && aligned_rows(k, sh.ks) && sh.dk % 8 == 0);
    GJX_LAUNCH_CHECK();
  }
  constexpr int NC = wide_tiles(DKP, NPI);
  if (scan_wide(sh))
    k_delta_scan<T, DKP, NPI, KEEP, NC><<<scan_grid(sh, NC), TEAM, 0, s>>>(sh, v, state0, lengths, o, state, w);
  else
    k_delta_scan<T, DKP, NPI, KEEP, 1><<<scan_grid(sh, 1), TEAM, 0, s>>>(sh, v, state0, lengths, o, state, w);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

template <typename T, int DKP>
int32_t run_grad(const Shape& sh, const float* g, const int32_t* lengths, const T* d_o, const float* d_state,
                 T* dq, T* dk, T* dv, float* dg, float* dbeta, float* d_state0, const Work& w, hipStream_t s) {
  constexpr int NPI = sizeof(T) == 4 ? 3 : 1;
  constexpr int NC = wide_tiles(DKP, NPI);
  if (scan_wide(sh))
    k_delta_scan_back<T, DKP, NPI, NC><<<scan_grid(sh, NC), TEAM, 0, s>>>(sh, d_o, d_state, lengths, dv, d_state0, w);
  else
    k_delta_scan_back<T, DKP, NPI, 1><<<scan_grid(sh, 1), TEAM, 0, s>>>(sh, d_o, d_state, lengths, dv, d_state0, w);
  GJX_LAUNCH_CHECK();
  if (sh.chunks == 0) return GJX_OK;
  const int vec_o = ((uintptr_t)d_o & 15) == 0 && sh.dv % 8 == 0;
  const int vec_out = (((uintptr_t)dq | (uintptr_t)dk) & 15) == 0 && sh.dk % 8 == 0;
  k_delta_back<T, DKP, NPI><<<gjx_grid_rows(sh.batch * sh.heads * sh.chunks), BACK, 0, s>>>(sh, d_o, g, lengths, dq, dk, dg, dbeta, w, vec_o, vec_out);
  GJX_LAUNCH_CHECK();
  if (sh.group > 1) {
    k_delta_shared_heads<T><<<gjx_grid_for(sh.batch * sh.time * sh.kheads * sh.dk), GJX_BLOCK, 0, s>>>(sh, w.dq, w.dk, dq, dk);
    GJX_LAUNCH_CHECK();
  }
  return GJX_OK;
}

template <typename T>
int32_t run_step(const Shape& sh, const float* state, const int32_t* anc, const T* q, const T* k, const T* v, const float* g,
                 const float* beta, T* o, float* out, hipStream_t s) {
  const int64_t bh = sh.batch * sh.heads;
#define GJX_STEP(CG, R)                                                                                                       \
  k_delta_step<T, CG, R><<<gjx_grid_rows(bh * (up(sh.dv, CG * 4) / (CG * 4))), 256, 0, s>>>(sh, state, anc, q, k, v, g, beta, o, out, \
                                                                                            (int)(up(sh.dv, CG * 4) / (CG * 4)))
  if (sh.dv <= 64) {
    if (sh.dk <= 64) GJX_STEP(16, 4);
    else GJX_STEP(16, 8);
  } else {
    if (sh.dk <= 64) GJX_STEP(32, 8);
    else GJX_STEP(32, 16);
  }
#undef GJX_STEP
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

}  // namespace

GJX_API int32_t gjx_delta_filter_workspace(const gjx_delta_shape* shape, int32_t keep, int64_t* bytes) {
  const char* who = "gjx_delta_filter_workspace";
  const int32_t rc = check_shape(who, shape);
  if (rc != GJX_OK) return rc;
  GJX_REQUIRE(bytes != nullptr && keep >= 0 && keep <= 2, GJX_EINVAL, "%s: bytes is null or keep not in [0, 2]", who);
  const Layout l = layout_of(shape, keep != 0);
  *bytes = keep == 2 ? l.grad_bytes : l.bytes;
  return GJX_OK;
}

GJX_API int32_t gjx_delta_filter(const gjx_delta_shape* shape, const void* d_q, const void* d_k, const void* d_v, const float* d_g,
                                 const float* d_beta, const float* d_state0, const int32_t* d_lengths, void* d_o, float* d_state,
                                 int32_t keep, void* d_work, int64_t work_bytes, void* stream) {
  const char* who = "gjx_delta_filter";
  const int32_t rc = check_shape(who, shape);
  if (rc != GJX_OK) return rc;
  if (shape->batch == 0) return GJX_OK;
  GJX_REQUIRE(d_state && (shape->time == 0 || (d_q && d_k && d_v && d_g && d_beta && d_o)), GJX_EINVAL, "%s: null argument", who);
  const Layout l = layout_of(shape, keep != 0);
  GJX_REQUIRE(l.bytes == 0 || (d_work && ((uintptr_t)d_work & 255) == 0 && work_bytes >= l.bytes), GJX_EINVAL,
              "%s: the workspace has %lld bytes, needs %lld aligned to 256", who, (long long)work_bytes, (long long)l.bytes);
  const Shape sh = shape_of(shape);
  const Work w = work_of(l, (char*)d_work, nullptr);
  hipStream_t s = (hipStream_t)stream;
#define GJX_FILTER(T, DKP, KEEP) \
  run_filter<T, DKP, KEEP>(sh, (const T*)d_q, (const T*)d_k, (const T*)d_v, d_g, d_beta, d_state0, d_lengths, (T*)d_o, d_state, w, s)
  if (shape->dtype == GJX_F32) {
    if (l.dkp == 64) return keep ? GJX_FILTER(float, 64, true) : GJX_FILTER(float, 64, false);
    return keep ? GJX_FILTER(float, 128, true) : GJX_FILTER(float, 128, false);
  }
  if (l.dkp == 64) return keep ? GJX_FILTER(bf16, 64, true) : GJX_FILTER(bf16, 64, false);
  return keep ? GJX_FILTER(bf16, 128, true) : GJX_FILTER(bf16, 128, false);
#undef GJX_FILTER
}

GJX_API int32_t gjx_delta_filter_grad(const gjx_delta_shape* shape, const void* d_q, const void* d_k, const void* d_v, const float* d_g,
                                      const float* d_beta, const int32_t* d_lengths, const void* d_do, const float* d_dstate, void* d_dq,
                                      void* d_dk, void* d_dv, float* d_dg, float* d_dbeta, float* d_dstate0, const void* d_kept,
                                      int64_t kept_bytes, void* d_work, int64_t work_bytes, void* stream) {
  const char* who = "gjx_delta_filter_grad";
  const int32_t rc = check_shape(who, shape);
  if (rc != GJX_OK) return rc;
  if (shape->batch == 0) return GJX_OK;
  GJX_REQUIRE(shape->time == 0 || (d_q && d_k && d_v && d_g && d_beta && d_do && d_dq && d_dk && d_dv && d_dg && d_dbeta), GJX_EINVAL,
              "%s: null argument", who);
  const Layout l = layout_of(shape, true);
  GJX_REQUIRE(l.bytes == 0 || (d_kept && ((uintptr_t)d_kept & 255) == 0 && kept_bytes >= l.bytes), GJX_EINVAL,
              "%s: the kept workspace has %lld bytes, needs %lld aligned to 256", who, (long long)kept_bytes, (long long)l.bytes);
  GJX_REQUIRE(l.grad_bytes == 0 || (d_work && ((uintptr_t)d_work & 255) == 0 && work_bytes >= l.grad_bytes), GJX_EINVAL,
              "%s: the workspace has %lld bytes, needs %lld aligned to 256", who, (long long)work_bytes, (long long)l.grad_bytes);
  const Shape sh = shape_of(shape);
  const Work w = work_of(l, (char*)const_cast<void*>(d_kept), (char*)d_work);
  hipStream_t s = (hipStream_t)stream;
#define GJX_GRAD(T, DKP)                                                                                                            \
  run_grad<T, DKP>(sh, d_g, d_lengths, (const T*)d_do, d_dstate, (T*)d_dq, (T*)d_dk, (T*)d_dv, d_dg, d_dbeta, \
                   d_dstate0, w, s)
  if (shape->dtype == GJX_F32) return l.dkp == 64 ? GJX_GRAD(float, 64) : GJX_GRAD(float, 128);
  return l.dkp == 64 ? GJX_GRAD(bf16, 64) : GJX_GRAD(bf16, 128);
#undef GJX_GRAD
}

GJX_API int32_t gjx_gather_states_grad_f32(const float* d_grad, const int32_t* d_sorted, const int64_t* d_order, int64_t n, int64_t row,
                                           int64_t* d_starts, float* d_out, void* stream) {
  const char* who = "gjx_gather_states_grad_f32";
  GJX_REQUIRE(n >= 0 && row >= 1, GJX_EINVAL, "%s: bad sizes (n %lld, row %lld)", who, (long long)n, (long long)row);
  if (n == 0) return GJX_OK;
  GJX_REQUIRE(d_grad && d_sorted && d_order && d_starts && d_out, GJX_EINVAL, "%s: null argument", who);
  GJX_REQUIRE(n <= (1 << 24) && row <= ((int64_t)1 << 30), GJX_ELIMIT, "%s: n up to 2^24, rows up to 2^30", who);
  const bool vec = row % 4 == 0 && (((uintptr_t)d_grad | (uintptr_t)d_out) & 15) == 0;
  const int64_t units = vec ? row / 4 : row;
  int cols = 1;
  while (cols < GJX_BLOCK && cols < units) cols *= 2;
  const int64_t tiles = up(units, cols) / cols;
  GJX_REQUIRE(n * tiles < ((int64_t)1 << 31) - (1 << 21), GJX_ELIMIT, "%s: %lld rows of %lld entries are too many", who, (long long)n, (long long)row);
  hipStream_t s = (hipStream_t)stream;
  k_delta_runs<<<gjx_grid_for(n + 1), GJX_BLOCK, 0, s>>>(d_sorted, n, d_starts);
  GJX_LAUNCH_CHECK();
  if (vec)
    k_delta_run_sums<f32x4><<<gjx_grid_rows(n * tiles), GJX_BLOCK, 0, s>>>((const f32x4*)d_grad, d_order, d_starts, n, units, cols, (int)tiles,
                                                                           (f32x4*)d_out);
  else
    k_delta_run_sums<float><<<gjx_grid_rows(n * tiles), GJX_BLOCK, 0, s>>>(d_grad, d_order, d_starts, n, units, cols, (int)tiles, d_out);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

GJX_API int32_t gjx_delta_filter_step(const gjx_delta_shape* shape, const float* d_state, const int32_t* d_ancestors, const void* d_q,
                                      const void* d_k, const void* d_v, const float* d_g, const float* d_beta, void* d_o,
                                      float* d_state_out, void* stream) {
  const char* who = "gjx_delta_filter_step";
  const int32_t rc = check_shape(who, shape);
  if (rc != GJX_OK) return rc;
  GJX_REQUIRE(shape->time == 1, GJX_EINVAL, "%s: time must be 1", who);
  if (shape->batch == 0) return GJX_OK;
  GJX_REQUIRE(d_state && d_q && d_k && d_v && d_g && d_beta && d_o && d_state_out, GJX_EINVAL, "%s: null argument", who);
  GJX_REQUIRE(!d_ancestors || d_state != d_state_out, GJX_EINVAL, "%s: with ancestors the new state needs a buffer of its own", who);
  GJX_REQUIRE((((uintptr_t)d_state | (uintptr_t)d_state_out) & 15) == 0, GJX_EINVAL, "%s: states must be aligned to 16 bytes", who);
  const Shape sh = shape_of(shape);
  hipStream_t s = (hipStream_t)stream;
  if (shape->dtype == GJX_F32)
    return run_step<float>(sh, d_state, d_ancestors, (const float*)d_q, (const float*)d_k, (const float*)d_v, d_g, d_beta, (float*)d_o,
                           d_state_out, s);
  return run_step<bf16>(sh, d_state, d_ancestors, (const bf16*)d_q, (const bf16*)d_k, (const bf16*)d_v, d_g, d_beta, (bf16*)d_o,
                        d_state_out, s);
}
