// gjx_lincat.hip -- the categorical distribution whose logits are a linear map of a feature row,
//   l_iv = x_i . w_v + b_v,   log p(y_i) = l_{i,y_i} - log sum_v exp(l_iv),
// its gradient and its Gumbel-max draw.  The forward reduces every tile of the n x vocab logits to (max, sum exp) in the
// product's epilogue and keeps none of them.  The gradient turns d l = g (onehot(y) - exp(l - lse)) into
//   dx = dl W,   dW = dl^T x,   db = sum_i dl_i,
// piece by piece of the vocabulary; dl comes from the exponentials that a forward with a gradient to follow has kept, or,
// where those are too many or the product is short, from the logits formed again, in that product's epilogue.
// The products are 16x16x32 bf16 MFMA tiles with f32 accumulators.  f32 operands are split exactly into three bf16 planes
// (8 bits each) and the six largest partial products are summed.
//
// Where a product has few tiles and a long reduction, the reduction is cut into parts (cuts_of).  Three product kernels:
// k_lincat_rows for few rows (the weights go once from memory to the matrix unit), k_lincat_gemm for bf16
// (tiles straight into LDS), k_lincat_gemm32 for f32 (tiles split into planes on their way to LDS).
#include "gjx_common.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));       // 16 bytes at any entry of a row: one load all the same
typedef bf16x8 bf16x8_any __attribute__((aligned(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define LDS_AS __attribute__((address_space(3)))
#define GLB_AS __attribute__((address_space(1)))

namespace {

constexpr int BM = 256, BK = 64, GEMM_THREADS = 512;         // bf16 tiles: BM entries of m, 64 deep, eight waves
constexpr int BM32 = 128, GEMM32_THREADS = 256;              // f32 tiles: 32 deep, four waves
constexpr int SPLIT_BYTES = 3 * 64 * 16;                      // a slab of 16 of its rows: three planes of 64 lanes x 16 bytes

enum { EPI_SCORE = 0, EPI_DL = 1, EPI_STORE = 2, EPI_DRAW = 3, EPI_KEEP = 4 };   // KEEP: SCORE that leaves what dl is formed from

// one operand of a product: `rows` memory rows of `ld` elements.  Not transposed: a row is one output index with the
// reduction along it; transposed: a row is one reduction index with the output index along it (`cols` of them, a
// multiple of 8).  Indices beyond the end are clamped: what they add is discarded or multiplied by a zero.
struct Operand {
  const bf16* p;
  int64_t ld;
  int rows, cols;
};

// an f32 operand: `rows` memory rows of `cols` valid entries
struct OperandF {
  const float* p;
  int64_t ld;
  int rows, cols;
};

struct GemmArgs {
  Operand a, b;
  OperandF fa, fb;
  int ktiles;          // reduction length / 64 (bf16), / 32 rounded up (f32)
  int mt, nt, splits;  // tiles along m and n, parts of the reduction
  // EPI_SCORE / EPI_DL: m = vocabulary entry (v0 = first of this piece), n = row
  int64_t v0, vocab, n;
  const void* bias;
  int bias_f32;
  const int32_t* y;
  float2* part;        // [tile m][n_pad]: (max, sum exp) of a row over one tile; drawing: (largest l + Gumbel, its entry)
  float* target;       // logit of y
  void* keep;          // EPI_KEEP: [n][keep_ld] exp(l - base), f32 or f16 x 2^15, base the row's largest l of a wave's block of entries
                       // (-inf where none is left: the entries are 0, and so is their factor exp(base - lse), however small lse is)
  float* keep_base;    // [v / block][n]
  int64_t keep_ld;
  int64_t n_pad;
  int part_tile0;
  uint32_t key0, key1;
  uint64_t offset;
  const float *lse, *g;
  void* dl;            // [n_pad][dl_ld] of the operands' type
  float* resid;        // [n]: dl of the row's value less its bf16 rounding (bf16 only)
  const float* resid_in;   // EPI_STORE of dW: the same, added to the value's row
  int64_t dl_ld;
  float* db_part;      // [tile n][dl_ld]
  // EPI_STORE: out[n][m] (+ split * out_split), f32 or bf16
  void* out;
  int64_t out_ld, out_split;
  int out_m, out_n, out_bf16, accumulate;
};

// what a bf16 call keeps is f16 with 2^15 before it: 11 bits for entries down to 2^-29 of their block's largest, 2^-40 of that
// below (the bf16 rounding of dl that follows is 2^-8)
constexpr float KEEP_SCALE = 32768.0f;

__device__ __forceinline__ float load_any(const void* p, int f32, int64_t i) {
  return f32 ? ((const float*)p)[i] : (float)((const bf16*)p)[i];
}

// x = h + m + l exactly by cutting off 8 bits at a time (half the operations of rounding, and nothing can overflow):
// |m| < 2^-7 |x|, |l| < 2^-15 |x|, so the partial products left out are below 2^-21 |x| |w|, 2^-23 on average.
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&out)[3]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = __float_as_uint(x[j]);
    const float r = x[j] - __uint_as_float(u & 0xffff0000u);
    const uint32_t v = __float_as_uint(r);
    const uint32_t t = __float_as_uint(r - __uint_as_float(v & 0xffff0000u));
    out[0][j] = __builtin_bit_cast(bf16, (uint16_t)(u >> 16));
    out[1][j] = __builtin_bit_cast(bf16, (uint16_t)(v >> 16));
    out[2][j] = __builtin_bit_cast(bf16, (uint16_t)(t >> 16));
  }
}

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ f32x4 mma3(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x4 c) {
  c = mma(a[0], b[2], c);
  c = mma(a[1], b[1], c);
  c = mma(a[2], b[0], c);
  c = mma(a[0], b[1], c);
  c = mma(a[1], b[0], c);
  return mma(a[0], b[0], c);
}

__device__ __forceinline__ int tr_swizzle(int k) { return (k & 3) | (((k >> 3) & 3) << 2); }

// Two transposing reads of four reduction entries each.  `other` (unused) and the restrict qualifiers give the reads alias
// information: without any, the compiler takes them to read what the loads into LDS in flight are writing and waits for
// those first.  (What is read was loaded, waited for and fenced by a barrier a tile earlier.)
__device__ __forceinline__ bf16x8 read_transposed(LDS_AS char* __restrict__ p, LDS_AS char* __restrict__ other, int four_rows) {
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_AS bf16x4*)p);
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_AS bf16x4*)(p + four_rows));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One BK-deep tile of an operand, R output indices wide: R * 8 chunks of 16 bytes straight into LDS.  The offsets of a
// lane's chunks from the tile's first byte are kept (32 bits), so a step along the reduction costs one scalar addition;
// the fragments' LDS addresses are one or two lane addresses plus constants.
template <int R, bool T>
struct TileLoader {
  static constexpr int LOADS = R * 8 / GEMM_THREADS, WAVES = GEMM_THREADS / 64, FRAGS = T ? R / 16 : 2;
  uint32_t off[LOADS];
  uint32_t at[2];                       // lane addresses of the fragments (T: of the row, swizzle apart)
  int out0, lane, wave;
  const char* base;                     // uniform
  int64_t step;

  __device__ __forceinline__ TileLoader(const Operand& o, int out, int k0, int lane_, int wave_) : out0(out), lane(lane_), wave(wave_) {
    base = (const char*)o.p + (T ? (int64_t)k0 * o.ld : (int64_t)min(out0, o.rows - 1) * o.ld + k0) * 2;
    step = T ? BK * o.ld * 2 : BK * 2;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) off[j] = offset(o, j, BK);
    const int q = lane >> 4, i = lane & 15;
    if (T) {
      at[0] = (uint32_t)((8 * q + (i >> 2)) * (R * 2) + ((i & 3) << 3));
      at[1] = (uint32_t)tr_swizzle(8 * q + (i >> 2));
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = (uint32_t)(i * 128 + (((s * 4 + q) ^ (i >> 1)) << 4));
    }
  }
  // left: rows of the reduction left from the tile on (T), at least one
  __device__ __forceinline__ uint32_t offset(const Operand& o, int j, int left) const {
    const int c = (j * WAVES + wave) * 64 + lane;
    if (T) {
      const int row = c / (R / 8), ch = c % (R / 8);
      const int col = min(out0 + ((((ch >> 1) ^ tr_swizzle(row)) << 1) | (ch & 1)) * 8, o.cols - 8);
      return ((uint32_t)min(row, max(left, 1) - 1) * (uint32_t)o.ld + (uint32_t)col) * 2u;
    }
    const int row = c >> 3, ch = (c & 7) ^ ((row >> 1) & 7);
    return ((uint32_t)(min(out0 + row, o.rows - 1) - min(out0, o.rows - 1)) * (uint32_t)o.ld + (uint32_t)ch * 8u) * 2u;
  }
  __device__ __forceinline__ void load(const Operand& o, int k0, LDS_AS char* lds) {
    const bool ragged = T && k0 + BK > o.rows;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const uint32_t f = ragged ? offset(o, j, o.rows - k0) : off[j];
      __builtin_amdgcn_global_load_lds((const GLB_AS void*)(base + f), (LDS_AS void*)(lds + (j * WAVES + wave) * 1024), 16, 0, 0);
    }
    base += step;
  }
  // the 8 reduction elements 8 q .. 8 q + 7 of slab s (32 deep) for output index i0 + lane % 16
  __device__ __forceinline__ bf16x8 frag(LDS_AS char* lds, int i0, int s) const {
    if (T) {
      LDS_AS char* p = lds + at[0] + s * 32 * (R * 2) + (((uint32_t)(i0 >> 4) ^ at[1]) << 5);
      return read_transposed(p, lds, 4 * R * 2);
    }
    return *(LDS_AS bf16x8*)(lds + at[s] + i0 * 128);
  }
};

// (max, sum exp) of two sets of logits; (largest value, its entry), ties to the lower entry
__device__ __forceinline__ void merge_lse(float& top, float& sum, float top2, float sum2) {
  const float nt = fmaxf(top, top2), b = nt == -__builtin_inff() ? 0.0f : nt;
  sum = sum * expf(top - b) + sum2 * expf(top2 - b);
  top = nt;
}
__device__ __forceinline__ void merge_best(float& best, int& arg, float best2, int arg2) {
  if (arg2 != 0x7fffffff && (best2 > best || arg == 0x7fffffff || (best2 == best && arg2 < arg))) {
    best = best2;
    arg = arg2;
  }
}

// exp(x) for x <= 0 by the hardware's exp2: the product's rounding moves it by at most 2^-24 |x| log2 e of itself, small
// where the term is not
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// the row's value relative to this lane's first entry (first + v0 of the piece), negative where there is none
__device__ __forceinline__ int value_of(const GemmArgs& g, int64_t n, int first) {
  if (n >= g.n) return -1;
  const int64_t y = min(max((int64_t)g.y[n], (int64_t)0), g.vocab - 1) - g.v0 - first;    // outside the vocabulary: the nearest
  return y < 0 || y > (1 << 20) ? -1 : (int)y;
}

// where a workgroup's tile lies
struct Tile {
  int split, tm, tn, m0, n0;
};

// neighbouring tiles to one XCD (workgroups go round the eight of them), eight m-tiles by all n-tiles at a time
template <int BM, int BN>
__device__ __forceinline__ bool tile_of(const GemmArgs& g, Tile& t) {
  const int total = g.mt * g.nt * g.splits, per = total / 8, extra = total % 8;
  int id = (int)gjx_block();                                  // (rows of a multiple of eight workgroups)
  if (id >= total) return false;
  const int xcd = id % 8;
  id = xcd * per + min(xcd, extra) + id / 8;
  t.split = id / (g.mt * g.nt);
  id -= t.split * g.mt * g.nt;
  const int group = id / (8 * g.nt), in = id - group * 8 * g.nt, height = min(8, g.mt - group * 8);
  t.tm = group * 8 + in % height;
  t.tn = in / height;
  t.m0 = t.tm * BM;
  t.n0 = t.tn * BN;
  return true;
}

// what becomes of a tile's accumulators (rows m0 + wm + 16 i + 4 q + r, columns n0 + wn + 16 j + lane % 16); T: the operands' type
template <typename T, int BM, int BN, int WM, int WN, int MT, int NT, bool TB, int EPI>
__device__ __forceinline__ void epilogue(const GemmArgs& g, const Tile& tile, f32x4 (&acc)[MT][NT], char* smem_raw) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int split = tile.split, tm = tile.tm, tn = tile.tn, m0 = tile.m0, n0 = tile.n0;
  const int wm = (wave / WN) * (MT * 16), wn = (wave % WN) * (NT * 16);
  const int q = lane >> 4, c = lane & 15;
  if (EPI == EPI_STORE) {
    if (sizeof(T) == 2 && TB && g.resid_in) {
      // dW of the rows' own values: += resid_i x_i, in ascending i, over the rows of this part of the reduction.  Every wave
      // looks for its own columns, 512 rows at a time; a lane takes the rows of its column, so that up to sixteen are added at
      // once (one after the other, 500 rows of 300 values took 86 us)
      const int64_t end = min((int64_t)g.ktiles * (split + 1) / g.splits * BK, g.n);
      for (int64_t i8 = (int64_t)g.ktiles * split / g.splits * BK; i8 < end; i8 += 512) {
        int v8[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v8[u] = g.y[min(i8 + 64 * u + lane, g.n - 1)];
#pragma unroll 1
        for (int u = 0; u < 8; ++u) {
          const int64_t i0 = i8 + 64 * u;
          int yv = v8[0];
#pragma unroll
          for (int e = 1; e < 8; ++e) yv = u == e ? v8[e] : yv;
          const int64_t v = min(max((int64_t)yv, (int64_t)0), g.vocab - 1) - g.v0 - n0 - wn;
          const bool mine = i0 + lane < end && v >= 0 && v < NT * 16;
          if (!__ballot(mine)) continue;
          const int vl = mine ? (int)v : -1;
          const float res = g.resid_in[min(i0 + lane, g.n - 1)];
          uint64_t hits = 0;                               // the rows of this lane's column
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t rows = __ballot(vl >= 0 && (vl & 15) == e);
            hits = c == e ? rows : hits;
          }
          while (__ballot(hits != 0)) {
            const int l = hits ? __builtin_ctzll(hits) : 0;
            const int vr = __shfl(vl, l);
            const float rr = __shfl(res, l);
            const float rl = hits ? rr : 0.0f;
            hits &= hits - 1;
            const bf16* xr = g.a.p + min(i0 + l, g.n - 1) * g.a.ld;
            bf16x4 xv[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) xv[i] = *(const bf16x4*)(xr + min(m0 + wm + i * 16 + 4 * q, g.a.cols - 4));
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                const float w = (vr >> 4) == j ? rl : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] += w * (float)xv[i][r];
              }
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = n0 + wn + j * 16 + c;
      if (n >= g.out_n) continue;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + wm + i * 16 + 4 * q;
        const int64_t at = (int64_t)split * g.out_split + (int64_t)n * g.out_ld + m;
        if (g.out_bf16) {
          bf16* o = (bf16*)g.out + at;
          if (m + 4 <= g.out_m && (g.out_ld & 3) == 0) {
            bf16x4 v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = (bf16)acc[i][j][r];
            *(bf16x4*)o = v;
          } else {
            for (int r = 0; r < 4; ++r)
              if (m + r < g.out_m) o[r] = (bf16)acc[i][j][r];
          }
        } else {
          float* o = (float*)g.out + at;
          if (m + 4 <= g.out_m && (g.out_ld & 3) == 0) {
            f32x4 v = acc[i][j];
            if (g.accumulate) v += *(f32x4*)o;
            *(f32x4*)o = v;
          } else {
            for (int r = 0; r < 4; ++r)
              if (m + r < g.out_m) o[r] = g.accumulate ? o[r] + acc[i][j][r] : acc[i][j][r];
          }
        }
      }
    }
    return;
  }

  // bias of the tile's 256 entries, -inf behind the last one
  float* s_bias = (float*)smem_raw;
  float* s_red = s_bias + BM;                               // 2 * WM * BN floats (score) or WN * BM (dl)
  if (tid < BM) {
    const int64_t v = g.v0 + m0 + tid;
    s_bias[tid] = v < g.vocab ? (g.bias ? load_any(g.bias, g.bias_f32, v) : 0.0f) : -__builtin_inff();
  }
  __syncthreads();
  float bias[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) bias[i][r] = s_bias[wm + i * 16 + 4 * q + r];

  if (EPI == EPI_SCORE || EPI == EPI_KEEP) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t n = n0 + wn + j * 16 + c;
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[i][j][r] += bias[i][r];
          top = fmaxf(top, acc[i][j][r]);
        }
      // the row's value, if its logit is among this lane's (rare: one entry of the vocabulary per row)
      const int y = value_of(g, n, m0 + wm + 4 * q);
      if (__ballot(y >= 0 && y < MT * 16 && (y & 15) < 4)) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (y == i * 16 + r) g.target[n] = acc[i][j][r];
      }
      top = fmaxf(top, __shfl_xor(top, 16));              // one base for the wave's whole block of entries
      top = fmaxf(top, __shfl_xor(top, 32));
      const float base = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = exp_of(acc[i][j][r] - base);
          sum += e;
          if (EPI == EPI_KEEP) acc[i][j][r] = e;
        }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (EPI == EPI_KEEP && n < g.n) {
        const int64_t v = g.v0 + m0 + wm;
        if (q == 0) g.keep_base[v / (MT * 16) * g.n + n] = top;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (sizeof(T) == 2) {
            f16x4 h;
#pragma unroll
            for (int r = 0; r < 4; ++r) h[r] = (_Float16)(acc[i][j][r] * KEEP_SCALE);
            *(f16x4*)((_Float16*)g.keep + n * g.keep_ld + v + i * 16 + 4 * q) = h;
          } else {
            *(f32x4*)((float*)g.keep + n * g.keep_ld + v + i * 16 + 4 * q) = acc[i][j];
          }
        }
      }
      if (q == 0) {
        s_red[((wave / WN) * BN + wn + j * 16 + c) * 2] = top;
        s_red[((wave / WN) * BN + wn + j * 16 + c) * 2 + 1] = sum;
      }
    }
    __syncthreads();
    if (tid < BN) {
      float top = s_red[tid * 2], sum = s_red[tid * 2 + 1];
#pragma unroll
      for (int w = 1; w < WM; ++w) {
        merge_lse(top, sum, s_red[(w * BN + tid) * 2], s_red[(w * BN + tid) * 2 + 1]);
      }
      g.part[(int64_t)(g.part_tile0 + tm) * g.n_pad + n0 + tid] = make_float2(top, sum);
    }
    return;
  }

  if (EPI == EPI_DRAW) {
    // argmax of l + Gumbel with categorical's noise: entry v of row i on counter (offset + i) vocab + v, ties to the lowest v
#pragma unroll 1
    for (int j = 0; j < NT; ++j) {
      const int64_t n = n0 + wn + j * 16 + c;
      float best = -__builtin_inff();
      int arg = 0x7fffffff;
      if (n < g.n)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int v = (int)g.v0 + m0 + wm + i * 16 + 4 * q + r;
            const float u = gjx_uniform_at(g.key0, g.key1, (g.offset + (uint64_t)n) * (uint64_t)g.vocab + (uint64_t)v,
                                           1.17549435e-38f, 1.0f);
            float l = 0.0f;                                  // acc[i][j] with a constant index, j being a loop's
#pragma unroll
            for (int jj = 0; jj < NT; ++jj) l = jj == j ? acc[i][jj][r] : l;
            const float val = bias[i][r] == -__builtin_inff() ? bias[i][r] : l + bias[i][r] + (-logf(-logf(u)));
            if (v < g.vocab && (val > best || arg == 0x7fffffff)) {
              best = val;
              arg = v;
            }
          }
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) {
        merge_best(best, arg, __shfl_xor(best, o), __shfl_xor(arg, o));
      }
      if (q == 0) {
        s_red[((wave / WN) * BN + wn + j * 16 + c) * 2] = best;
        s_red[((wave / WN) * BN + wn + j * 16 + c) * 2 + 1] = __int_as_float(arg);
      }
    }
    __syncthreads();
    if (tid < BN) {
      float best = s_red[tid * 2];
      int arg = __float_as_int(s_red[tid * 2 + 1]);
#pragma unroll
      for (int w = 1; w < WM; ++w) {
        merge_best(best, arg, s_red[(w * BN + tid) * 2], __float_as_int(s_red[(w * BN + tid) * 2 + 1]));
      }
      g.part[(int64_t)(g.part_tile0 + tm) * g.n_pad + n0 + tid] = make_float2(best, __int_as_float(arg));
    }
    return;
  }

  // EPI_DL
  float dbs[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) dbs[i][r] = 0.0f;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t n = n0 + wn + j * 16 + c;
    const bool live = n < g.n;
    const float lse = live ? g.lse[n] : 0.0f, up = live ? g.g[n] : 0.0f;      // rows behind the last: up = 0 and finite logits
    // -up exp(l - lse); entries behind the vocabulary have the bias -inf
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][j][r] = -up * exp_of(acc[i][j][r] + bias[i][r] - lse);
    if (!live)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int y = value_of(g, n, m0 + wm + 4 * q);
    const bool here = __ballot(y >= 0 && y < MT * 16 && (y & 15) < 4) != 0;
    if (here) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (y == i * 16 + r) acc[i][j][r] += up;
    }
    T* o = (T*)g.dl + n * g.dl_ld + (m0 + wm + 4 * q);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) dbs[i][r] += acc[i][j][r];
      if (sizeof(T) == 2) {
        // rounded to bf16 (the products that follow take bf16 operands): each entry is off by at most 2^-8 of it,
        // independently of its neighbours.  The value's own entry is usually far larger than the others, so that ONE
        // rounding would show in whole rows of the gradients: what it loses is kept apart and added in f32.
        bf16x4 h;
#pragma unroll
        for (int r = 0; r < 4; ++r) h[r] = (bf16)acc[i][j][r];
        *(bf16x4*)(o + i * 16) = h;
        if (here)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (y == i * 16 + r) g.resid[n] = acc[i][j][r] - (float)h[r];
      } else {
        *(f32x4*)(o + i * 16) = acc[i][j];
      }
    }
  }
  if (g.db_part) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float s = dbs[i][r];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o);
        if (c == 0) s_red[(wave % WN) * BM + wm + i * 16 + 4 * q + r] = s;
      }
    __syncthreads();
    if (tid < BM) {
      float s = s_red[tid];
#pragma unroll
      for (int w = 1; w < WN; ++w) s += s_red[w * BM + tid];
      g.db_part[(int64_t)tn * g.dl_ld + m0 + tid] = s;
    }
  }
}

// C[m][n] = sum_k A(m, k) B(n, k) in bf16; BM x BN per workgroup of eight waves.  Bound by the matrix unit at the clock that
// it sustains: 4096 x 128000 x 4096 (log-densities) in 3.06 to 3.3 ms once the clock has settled = 1.3 to 1.4 PFLOP/s, where a
// library product of these sizes reaches 1.2 to 1.4; dx and dW of 4096 x 128000 x 2048 at 1.27 and 1.12.  Two LDS buffers of one 64-deep tile each
// and two register sets of fragments: while the products of one 32-deep slab run, the next slab is read (across the tile's
// end: the one barrier of a tile stands between its two slabs, when its last slab is in registers), and the tile after the
// next one is on its way into the buffer just emptied.
template <int BN, bool TA, bool TB, int EPI>
__global__ void __launch_bounds__(GEMM_THREADS)
    k_lincat_gemm(GemmArgs g) {
  constexpr int WN = BN == 256 ? 4 : 2, WM = 8 / WN;       // waves along n and m
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
  extern __shared__ char smem_raw[];
  LDS_AS char* smem = (LDS_AS char*)smem_raw;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile tile;
  if (!tile_of<BM, BN>(g, tile)) return;
  const int kt0 = (int)((int64_t)g.ktiles * tile.split / g.splits), kt1 = (int)((int64_t)g.ktiles * (tile.split + 1) / g.splits);

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int wm = (wave / WN) * (MT * 16), wn = (wave % WN) * (NT * 16);
  TileLoader<BM, TA> la(g.a, tile.m0, kt0 * BK, lane, wave);
  TileLoader<BN, TB> lb(g.b, tile.n0, kt0 * BK, lane, wave);
  if (kt0 < kt1) {
    la.load(g.a, kt0 * BK, smem);
    lb.load(g.b, kt0 * BK, smem + 2 * A_BYTES);
  }
  if (kt0 + 1 < kt1) {
    la.load(g.a, (kt0 + 1) * BK, smem + A_BYTES);
    lb.load(g.b, (kt0 + 1) * BK, smem + 2 * A_BYTES + B_BYTES);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(la.LOADS + lb.LOADS) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  struct Frags {
    bf16x8 a[MT], b[NT];
  } f0, f1;
  auto read = [&](int buf, int s, Frags& f) {
    LDS_AS char* sa = smem + buf * A_BYTES;
    LDS_AS char* sb = smem + 2 * A_BYTES + buf * B_BYTES;
#pragma unroll
    for (int j = 0; j < NT; ++j) f.b[j] = lb.frag(sb, wn + j * 16, s);
#pragma unroll
    for (int i = 0; i < MT; ++i) f.a[i] = la.frag(sa, wm + i * 16, s);
  };
  auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mma(f.a[i], f.b[j], acc[i][j]);
    // the reads that stand in front of the products go between them
    constexpr int READS = MT * (TA ? 2 : 1) + NT * (TB ? 2 : 1), EACH = MT * NT / READS > 0 ? MT * NT / READS : 1;
#pragma unroll
    for (int r = 0; r < READS; ++r) {
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);       // one LDS read
      __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);    // EACH matrix instructions
    }
  };
  auto step = [&](int kt, int buf) {       // buf: a constant where it is called
    read(buf, 1, f1);
    multiply(f0);
    // this wave's reads of the tile are done and its loads of the next tile have arrived; behind the barrier: everyone's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt + 2 < kt1) {
      la.load(g.a, (kt + 2) * BK, smem + buf * A_BYTES);
      lb.load(g.b, (kt + 2) * BK, smem + 2 * A_BYTES + buf * B_BYTES);
    }
    read(buf ^ 1, 0, f0);                  // behind the last tile: the other buffer's old contents, not used
    multiply(f1);
  };
  if (kt0 < kt1) read(0, 0, f0);
  for (int kt = kt0; kt < kt1; kt += 2) {
    step(kt, 0);
    if (kt + 1 < kt1) step(kt + 1, 1);
  }
  __syncthreads();
  epilogue<bf16, BM, BN, WM, WN, MT, NT, TB, EPI>(g, tile, acc, smem_raw);
}

// One 32-deep slab of an f32 operand, R output indices wide: pieces of eight reduction entries of one output index, loaded
// into registers, split and written to LDS as fragments (16 indices x 3 planes x 64 slots of 16 bytes).  Whole slabs are
// read at a uniform base plus a kept 32-bit offset; the last one entry by entry, clamped and masked.
// Slot (index, group) lies at 16 group + (index + 2 group) % 16: neither the four lanes that write a row's groups nor the
// sixteen that read a group meet in a bank (without the rotation 60 % of the LDS cycles were conflicts).
template <int R, bool T>
struct SlabLoader {
  static constexpr int PIECES = (R * 4 + GEMM32_THREADS - 1) / GEMM32_THREADS;
  float x[PIECES][8];
  uint32_t off[PIECES];
  const char* base;                    // uniform
  int out0, tid;

  __device__ __forceinline__ void where(int i, int& index, int& group) const {
    const int u = min(i * GEMM32_THREADS + tid, R * 4 - 1);
    if (T) {
      index = u % R;          // neighbouring lanes take neighbouring columns
      group = u / R;
    } else {
      index = u >> 2;         // four lanes take a row's 128 bytes
      group = u & 3;
    }
  }
  __device__ __forceinline__ SlabLoader(const OperandF& o, int out, int k0, int tid_) : out0(out), tid(tid_) {
    const int row0 = min(out0, o.rows - 1);       // a tile may lie wholly behind the last row (the vocabulary is padded)
    base = (const char*)(o.p + (T ? (int64_t)k0 * o.ld : (int64_t)row0 * o.ld + k0));
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      int index, group;
      where(i, index, group);
      off[i] = T ? ((uint32_t)(8 * group) * (uint32_t)o.ld + (uint32_t)min(out0 + index, o.cols - 1)) * 4u
                 : ((uint32_t)(min(out0 + index, o.rows - 1) - row0) * (uint32_t)o.ld + (uint32_t)(8 * group)) * 4u;
    }
  }
  __device__ __forceinline__ void load(const OperandF& o, int k0) {
    if (k0 + 32 <= (T ? o.rows : o.cols)) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        if (T) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[i][j] = *(const float*)(base + (int64_t)j * o.ld * 4 + off[i]);
        } else {
          const f32x4 lo = *(const f32x4_any*)(base + off[i]), hi = *(const f32x4_any*)(base + 16 + off[i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[i][j] = lo[j];
            x[i][4 + j] = hi[j];
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        int index, group;
        where(i, index, group);
        const int k = k0 + 8 * group;
        const float* p = T ? o.p + min(out0 + index, o.cols - 1) : o.p + (int64_t)min(out0 + index, o.rows - 1) * o.ld;
        const int64_t step = T ? o.ld : 1;
        const int end = T ? o.rows : o.cols;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = p[min(k + j, end - 1) * step];       // all eight in flight, then masked
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = k + j < end ? x[i][j] : 0.0f;
      }
    }
    base += T ? 32 * o.ld * 4 : 128;
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (R * 4 % GEMM32_THREADS && i * GEMM32_THREADS + tid >= R * 4) continue;
      int index, group;
      where(i, index, group);
      bf16x8 o[3];
      split8(x[i], o);
      char* f = lds + (index >> 4) * SPLIT_BYTES + (16 * group + ((index & 15) ^ (2 * (group & 1) | (group >> 1) * 12))) * 16;
#pragma unroll
      for (int p = 0; p < 3; ++p) *(bf16x8*)(f + p * 1024) = o[p];
    }
  }
  static __device__ __forceinline__ void frag(const char* lds, int i0, int lane, bf16x8 (&out)[3]) {
    const int q = lane >> 4;
#pragma unroll
    for (int p = 0; p < 3; ++p) out[p] = *(const bf16x8*)(lds + (i0 >> 4) * SPLIT_BYTES + p * 1024 + (16 * q + ((lane & 15) ^ (2 * (q & 1) | (q >> 1) * 12))) * 16);
  }
};

// the same product of f32 operands: six matrix instructions per fragment pair, so the splitting (once per tile) and the
// LDS traffic are small beside them and no packed copy of the operands is needed (packing to bf16 planes first: pack and
// product 328 us for 200 x 50001 x 768).  One 32-deep slab in LDS, the next one in registers; three workgroups a CU
// cover each other's splitting and barriers and leave less idle at the end than one of twice the size.  No one unit is the
// bound: the matrix unit is busy 57 % of the time, the rest goes to splitting, LDS and barriers where the workgroups of a CU
// do not cover each other, and to CUs that the last tiles leave idle: 200 x 50001 x 768 in 109 to 119 us (0.83 PFLOP/s of
// partial products), 1000 x 20011 x 512 in 112 to 150 us per product (0.82 to 1.1).
template <int BN, bool TA, bool TB, int EPI>
__global__ void __launch_bounds__(GEMM32_THREADS, BN > 128 ? 2 : 3)
    k_lincat_gemm32(GemmArgs g) {
  constexpr int BM = BM32, WN = BN > 128 ? 1 : 2, WM = 4 / WN, MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int A_BYTES = BM / 16 * SPLIT_BYTES;
  extern __shared__ char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Tile tile;
  if (!tile_of<BM, BN>(g, tile)) return;
  const int kt0 = (int)((int64_t)g.ktiles * tile.split / g.splits), kt1 = (int)((int64_t)g.ktiles * (tile.split + 1) / g.splits);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int wm = (wave / WN) * (MT * 16), wn = (wave % WN) * (NT * 16);
  SlabLoader<BM, TA> la(g.fa, tile.m0, kt0 * 32, tid);
  SlabLoader<BN, TB> lb(g.fb, tile.n0, kt0 * 32, tid);
  if (kt0 < kt1) {
    la.load(g.fa, kt0 * 32);
    lb.load(g.fb, kt0 * 32);
  }
  char *sa = smem_raw, *sb = sa + A_BYTES;
  for (int kt = kt0; kt < kt1; ++kt) {
    la.store(sa);
    lb.store(sb);
    __syncthreads();
    if (kt + 1 < kt1) {
      la.load(g.fa, (kt + 1) * 32);
      lb.load(g.fb, (kt + 1) * 32);
    }
    __builtin_amdgcn_s_setprio(1);             // products first: splitting fills the gaps they leave (3 % faster)
#pragma unroll
    for (int j = 0; j < NT; j += 2) {          // two column tiles at a time: with all four, registers spill
      bf16x8 fb[2][3];
      SlabLoader<BN, TB>::frag(sb, wn + j * 16, lane, fb[0]);
      if (j + 1 < NT) SlabLoader<BN, TB>::frag(sb, wn + j * 16 + 16, lane, fb[1]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        bf16x8 fa[3];
        SlabLoader<BM, TA>::frag(sa, wm + i * 16, lane, fa);
        acc[i][j] = mma3(fa, fb[0], acc[i][j]);
        if (j + 1 < NT) acc[i][j + 1] = mma3(fa, fb[1], acc[i][j + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();
  }
  epilogue<float, BM, BN, WM, WN, MT, NT, TB, EPI>(g, tile, acc, smem_raw);
}

// few rows (n <= 16 NT): a wave takes 16 entries of the vocabulary, the weights go from memory to the matrix unit without
// a stop, the rows of x (a few KB) come from the caches.  Partial results per 64 entries.  Bound by memory: the 66 MB of
// 32000 x 1024 bf16 weights in 15 us, 4.3 TB/s.
template <typename T, int NT, int EPI>
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_rows(GemmArgs g, const T* __restrict__ x, int64_t x_ld, const T* __restrict__ w, int64_t w_ld, int width) {
  constexpr int P = sizeof(T) == 4 ? 3 : 1, U = (sizeof(T) == 4 ? 8 : 16) / NT;      // planes; slabs in flight
  __shared__ float s_red[4][16 * NT][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, c = lane & 15;
  const int v0 = blockIdx.x * 64 + wave * 16;
  const T* wp = w + min((int64_t)v0 + c, g.vocab - 1) * w_ld;
  const T* xp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) xp[j] = x + min((int64_t)(j * 16 + c), g.n - 1) * x_ld;
  // eight entries from k (a multiple of 8) on; not whole: zeros behind the end
  auto load = [&](auto whole, const T* p, int k, float (&f)[8], bf16x8& h) {
    if (whole || k + 8 <= width) {
      if (P == 1) {
        h = *(const bf16x8_any*)(p + k);
      } else {
        const f32x4 lo = *(const f32x4_any*)(p + k), hi = *(const f32x4_any*)(p + k + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = lo[e];
          f[4 + e] = hi[e];
        }
      }
    } else {
      T t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = p[min(k + e, width - 1)];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (k + e >= width) t[e] = (T)0.0f;
        if (P == 1) h[e] = (bf16)t[e];
        else f[e] = (float)t[e];
      }
    }
  };
  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  // `count` slabs from k0 on, their loads of the weights all in flight; whole: inside the width
  auto slabs = [&](int k0, auto count, auto whole) {
    constexpr int N = decltype(count)::value;
    float fw[N][8];
    bf16x8 hw[N];
#pragma unroll
    for (int u = 0; u < N; ++u) load(whole, wp, k0 + 32 * u + 8 * q, fw[u], hw[u]);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      bf16x8 a[3];
      if (P == 3) split8(fw[u], a);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float fx[8];
        bf16x8 hx, b[3];
        load(whole, xp[j], k0 + 32 * u + 8 * q, fx, hx);
        if (P == 1) {
          acc[j] = mma(hw[u], hx, acc[j]);
        } else {
          split8(fx, b);
          acc[j] = mma3(a, b, acc[j]);
        }
      }
    }
  };
  int k0 = 0;
  for (; k0 + 32 * U <= width; k0 += 32 * U) slabs(k0, std::integral_constant<int, U>(), std::true_type());
  if constexpr (U >= 8)
    for (; k0 + 8 * U <= width; k0 += 8 * U) slabs(k0, std::integral_constant<int, U / 4>(), std::true_type());
  for (; k0 + 32 <= width; k0 += 32) slabs(k0, std::integral_constant<int, 1>(), std::true_type());
  if (k0 < width) slabs(k0, std::integral_constant<int, 1>(), std::false_type());
  float bias[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t v = v0 + 4 * q + r;
    bias[r] = v < g.vocab ? (g.bias ? load_any(g.bias, g.bias_f32, v) : 0.0f) : -__builtin_inff();
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t n = j * 16 + c;
    float top = -__builtin_inff(), sum = 0.0f;
    int arg = 0x7fffffff;
    if (EPI != EPI_DRAW) {
      const int64_t y = n < g.n ? min(max((int64_t)g.y[n], (int64_t)0), g.vocab - 1) - v0 - 4 * q : -1;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[j][r] = bias[r] == -__builtin_inff() ? bias[r] : acc[j][r] + bias[r];
        top = fmaxf(top, acc[j][r]);
        if (y == r) g.target[n] = acc[j][r];
      }
      top = fmaxf(top, __shfl_xor(top, 16));              // the wave's sixteen entries
      top = fmaxf(top, __shfl_xor(top, 32));
      const float base = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[j][r] = exp_of(acc[j][r] - base);
        sum += acc[j][r];
      }
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (EPI == EPI_KEEP && n < g.n) {
        if (q == 0) g.keep_base[(int64_t)(v0 / 16) * g.n + n] = top;
        if (sizeof(T) == 2) {
          f16x4 h;
#pragma unroll
          for (int r = 0; r < 4; ++r) h[r] = (_Float16)(acc[j][r] * KEEP_SCALE);
          *(f16x4*)((_Float16*)g.keep + n * g.keep_ld + v0 + 4 * q) = h;
        } else {
          *(f32x4*)((float*)g.keep + n * g.keep_ld + v0 + 4 * q) = acc[j];
        }
      }
    } else if (n < g.n) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int v = v0 + 4 * q + r;
        const float u = gjx_uniform_at(g.key0, g.key1, (g.offset + (uint64_t)n) * (uint64_t)g.vocab + (uint64_t)v, 1.17549435e-38f, 1.0f);
        const float val = bias[r] == -__builtin_inff() ? bias[r] : acc[j][r] + bias[r] + (-logf(-logf(u)));
        if (v < g.vocab && (val > top || arg == 0x7fffffff)) {
          top = val;
          arg = v;
        }
      }
    }
    if (EPI == EPI_DRAW)
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) merge_best(top, arg, __shfl_xor(top, o), __shfl_xor(arg, o));
    if (q == 0) {
      s_red[wave][j * 16 + c][0] = top;
      s_red[wave][j * 16 + c][1] = EPI == EPI_DRAW ? __int_as_float(arg) : sum;
    }
  }
  __syncthreads();
  if (threadIdx.x < 16 * NT) {
    float top = s_red[0][threadIdx.x][0], sum = s_red[0][threadIdx.x][1];
    int arg = __float_as_int(sum);
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      if (EPI != EPI_DRAW) merge_lse(top, sum, s_red[i][threadIdx.x][0], s_red[i][threadIdx.x][1]);
      else merge_best(top, arg, s_red[i][threadIdx.x][0], __float_as_int(s_red[i][threadIdx.x][1]));
    }
    g.part[(int64_t)blockIdx.x * g.n_pad + threadIdx.x] = make_float2(top, EPI == EPI_DRAW ? __int_as_float(arg) : sum);
  }
}

// bf16 rows of any stride and width -> rows of width_pad, zeros behind the width
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_pack(const bf16* __restrict__ src, int64_t ld, int64_t rows, int width, int width_pad, bf16* __restrict__ dst) {
  const int64_t total = rows * (width_pad / 8);
  for (int64_t i = (int64_t)blockIdx.x * GJX_BLOCK + threadIdx.x; i < total; i += (int64_t)gridDim.x * GJX_BLOCK) {
    const int64_t row = i / (width_pad / 8);
    const int c0 = (int)(i - row * (width_pad / 8)) * 8;
    bf16x8 h;
#pragma unroll
    for (int k = 0; k < 8; ++k) h[k] = c0 + k < width ? src[row * ld + c0 + k] : (bf16)0.0f;
    *(bf16x8*)(dst + row * width_pad + c0) = h;
  }
}

// (max, sum exp) of the tiles of a row -> lse, and log p(y) = l_y - lse.  `width` rows by 256 / width parts per block.
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_combine(const float2* __restrict__ part, int tiles, int64_t n_pad, int64_t n, int width,
                     const float* __restrict__ target, float* __restrict__ lp, float* __restrict__ lse, float* __restrict__ lp_kept) {
  __shared__ float2 sm[GJX_BLOCK];
  const int col = threadIdx.x % width, grp = threadIdx.x / width, groups = GJX_BLOCK / width;
  const int64_t i = (int64_t)blockIdx.x * width + col;
  float top = -__builtin_inff(), sum = 0.0f;
  auto merge = [&](float2 p) { merge_lse(top, sum, p.x, p.y); };
  if (i < n)
    for (int t = grp; t < tiles; t += groups) merge(part[(int64_t)t * n_pad + i]);
  sm[threadIdx.x] = make_float2(top, sum);
  __syncthreads();
  for (int o = groups / 2; o > 0; o >>= 1) {
    if (grp < o) {
      merge(sm[threadIdx.x + o * width]);
      sm[threadIdx.x] = make_float2(top, sum);
    }
    __syncthreads();
  }
  if (grp == 0 && i < n) {
    const float l = top + logf(sum);
    if (lse) lse[i] = l;
    const float p = target[i] - l;
    lp[i] = p;
    if (lp_kept) lp_kept[i] = p;
  }
}

// the tiles' best entries -> the row's draw (ties to the lowest entry: tiles are in order of the vocabulary)
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_pick(const float2* __restrict__ part, int tiles, int64_t n_pad, int64_t n, int32_t* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * (GJX_BLOCK / 64) + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= n) return;
  float best = -__builtin_inff();
  int arg = 0x7fffffff;
  for (int t = lane; t < tiles; t += 64) {
    const float2 p = part[(int64_t)t * n_pad + i];
    if (p.x > best || arg == 0x7fffffff) {
      best = p.x;
      arg = __float_as_int(p.y);
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float b2 = __shfl_xor(best, o);
    const int a2 = __shfl_xor(arg, o);
    if (b2 > best || (b2 == best && a2 < arg)) {
      best = b2;
      arg = a2;
    }
  }
  if (lane == 0) out[i] = arg;
}

// dl of a piece of the vocabulary from what the forward kept: dl = g (onehot - exp(base - lse) e), and its sums over strips
// of rows for db.  A thread takes eight entries of a strip's rows.  Bound by memory, one read and one
// write: 2.1 GB of 4096 x 128000 in 448 us (4.7 TB/s), 160 MB of 1000 x 20011 f32 in 36 us (4.5 TB/s).

template <typename T>
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_dl(const void* __restrict__ keep, int64_t keep_ld, const float* __restrict__ base, int block,
                const float* __restrict__ lp, const float* __restrict__ lse, const float* __restrict__ up,
                const int32_t* __restrict__ y, int64_t n, int64_t vocab, int64_t v0, int cols, int strip, T* __restrict__ dl,
                int64_t dl_ld, float* __restrict__ resid, float* __restrict__ db_part, int64_t db_ld) {
  const int col = (blockIdx.y * GJX_BLOCK + threadIdx.x) * 8;
  if (col >= cols) return;
  const int64_t i0 = (int64_t)blockIdx.x * strip;
  const int rows = (int)max(min((int64_t)strip, n - i0), (int64_t)0);
  const float* b = base + (v0 + col) / block * n + i0;
  T* out = dl + i0 * dl_ld + col;
  float db[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
  for (int i = 0; i < rows; ++i) {
    const int64_t row = i0 + i;
    float x[8];
    if constexpr (sizeof(T) == 2) {
      const f16x8 h = *(const f16x8*)((const _Float16*)keep + row * keep_ld + v0 + col);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (float)h[j];
    } else {
      const float* p = (const float*)keep + row * keep_ld + v0 + col;
      const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = lo[j];
        x[4 + j] = hi[j];
      }
    }
    const float g = up[row], f = -g * exp_of(b[i] - lse[row]) * (sizeof(T) == 2 ? 1.0f / KEEP_SCALE : 1.0f);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= f;
    const int64_t at = min(max((int64_t)y[row], (int64_t)0), vocab - 1) - v0 - col;
    const bool here = at >= 0 && at < 8;
    const float own = g - g * exp_of(lp[row]);            // the value's own entry, from its log-density
    if (here)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = j == (int)at ? own : x[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) db[j] += x[j];
    if constexpr (sizeof(T) == 2) {
      bf16x8 h;
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = (bf16)x[j];
      *(bf16x8*)(out + i * dl_ld) = h;
      if (here) resid[row] = own - (float)(bf16)own;      // (see EPI_DL)
    } else {
      *(f32x4*)(out + i * dl_ld) = f32x4{x[0], x[1], x[2], x[3]};
      *(f32x4*)(out + i * dl_ld + 4) = f32x4{x[4], x[5], x[6], x[7]};
    }
  }
  for (int i = rows; i < strip; ++i) {         // the rows behind the last that the products' tiles reach
#pragma unroll
    for (int j = 0; j < 8; ++j) out[i * dl_ld + j] = (T)0.0f;
  }
  if (db_part) {
#pragma unroll
    for (int j = 0; j < 8; ++j) db_part[(int64_t)blockIdx.x * db_ld + col + j] = db[j];
  }
}

// Few tiles and a long reduction: the product is cut along the width, and its parts [s][row][entry] (f32) are added up here.
struct Parts {
  const float* p;
  int parts;
  int64_t stride, ld;
  const void* bias;
  int bias_f32;
  __device__ __forceinline__ float logit(int64_t row, int64_t v) const {
    const float* at = p + row * ld + v;
    float l = 0.0f;
    for (int s = 0; s < parts; s += 8) {                    // eight loads in flight, added in order
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = at[min(s + j, parts - 1) * stride];
#pragma unroll
      for (int j = 0; j < 8; ++j) l += s + j < parts ? x[j] : 0.0f;
    }
    return bias ? l + load_any(bias, bias_f32, v) : l;
  }
};

// a row's log-density (and what is kept, as EPI_KEEP leaves it, with lse for every base) or draw; TPR threads a row
template <int TPR, int EPI>
__global__ void __launch_bounds__(TPR > GJX_BLOCK ? TPR : GJX_BLOCK)
    k_lincat_finish(Parts parts, float* __restrict__ sums, int64_t n, int64_t vocab, const int32_t* __restrict__ y, float* __restrict__ lp,
                    float* __restrict__ lse, void* __restrict__ keep, int keep_f32, int64_t keep_ld, float* __restrict__ base, int block,
                    float* __restrict__ lp_kept, uint32_t key0, uint32_t key1, uint64_t offset, int32_t* __restrict__ out) {
  constexpr int ROWS = TPR < GJX_BLOCK ? GJX_BLOCK / TPR : 1;
  __shared__ float s_a[TPR / 64], s_b[TPR / 64], s_c[TPR / 64];
  const int t = threadIdx.x % TPR, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / TPR;
  const bool live = row < n;
  float top = -__builtin_inff(), sum = 0.0f, own = 0.0f;
  int arg = 0x7fffffff;
  if (live) {
    const int64_t value = EPI == EPI_DRAW ? -1 : min(max((int64_t)y[row], (int64_t)0), vocab - 1);
    for (int64_t v = t; v < vocab; v += TPR) {
      const float l = parts.logit(row, v);
      if (EPI == EPI_DRAW) {
        const float u = gjx_uniform_at(key0, key1, (offset + (uint64_t)row) * (uint64_t)vocab + (uint64_t)v, 1.17549435e-38f, 1.0f);
        merge_best(top, arg, l == -__builtin_inff() ? l : l + (-logf(-logf(u))), (int)v);
      } else {
        if (v == value) own = l;
        merge_lse(top, sum, l, 1.0f);
        if (EPI == EPI_KEEP) sums[row * parts.ld + v] = l;         // (the first part: this thread alone reads and writes the entry)
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    if (EPI == EPI_DRAW) {
      merge_best(top, arg, __shfl_xor(top, o), __shfl_xor(arg, o));
    } else {
      merge_lse(top, sum, __shfl_xor(top, o), __shfl_xor(sum, o));
      own += __shfl_xor(own, o);
    }
  }
  if (TPR > 64) {
    if ((threadIdx.x & 63) == 0) {
      s_a[wave] = top;
      s_b[wave] = EPI == EPI_DRAW ? __int_as_float(arg) : sum;
      s_c[wave] = own;
    }
    __syncthreads();
    top = s_a[0];
    sum = s_b[0];
    arg = __float_as_int(s_b[0]);
    own = s_c[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) {
      if (EPI == EPI_DRAW) {
        merge_best(top, arg, s_a[w], __float_as_int(s_b[w]));
      } else {
        merge_lse(top, sum, s_a[w], s_b[w]);
        own += s_c[w];
      }
    }
  }
  if (!live) return;
  if (EPI == EPI_DRAW) {
    if (t == 0) out[row] = arg;
    return;
  }
  const float all = top + logf(sum);
  if (t == 0) {
    lp[row] = own - all;
    if (lse) lse[row] = all;
    if (EPI == EPI_KEEP) lp_kept[row] = own - all;
  }
  if (EPI == EPI_KEEP) {
    for (int64_t k = t; k < keep_ld / block; k += TPR) base[k * n + row] = all;
    for (int64_t v = t; v < keep_ld; v += TPR) {
      const float e = v < vocab ? exp_of(sums[row * parts.ld + v] - all) : 0.0f;
      if (keep_f32) ((float*)keep)[row * keep_ld + v] = e;
      else ((_Float16*)keep)[row * keep_ld + v] = (_Float16)(e * KEEP_SCALE);
    }
  }
}

// dl of the whole vocabulary from the parts of the logits: 64 entries by four rows at a time of a strip (see k_lincat_dl)
template <typename T>
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_dl_parts(Parts parts, const float* __restrict__ lse, const float* __restrict__ up, const int32_t* __restrict__ y, int64_t n,
                      int64_t vocab, int strip, T* __restrict__ dl, int64_t dl_ld, float* __restrict__ resid, float* __restrict__ db_part,
                      int64_t db_ld) {
  __shared__ float s_db[4][64];
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6, col = blockIdx.y * 64 + c;
  const int64_t i0 = (int64_t)blockIdx.x * strip;
  float db = 0.0f;
  for (int i = q; i < strip; i += 4) {
    const int64_t row = i0 + i;
    float x = 0.0f;
    if (row < n && col < vocab) {
      x = -up[row] * exp_of(parts.logit(row, col) - lse[row]);
      if (min(max((int64_t)y[row], (int64_t)0), vocab - 1) == col) {
        x += up[row];
        if (resid) resid[row] = x - (float)(T)x;             // (see EPI_DL)
      }
      db += x;
    }
    dl[row * dl_ld + col] = (T)x;
  }
  s_db[q][c] = db;
  __syncthreads();
  if (db_part && q == 0) db_part[(int64_t)blockIdx.x * db_ld + col] = (s_db[0][c] + s_db[1][c]) + (s_db[2][c] + s_db[3][c]);
}

// out[i][k] = sum over parts of part[s][i][k] in f32, stored in the output's type; rows of `width`, parts of `ld` columns.
// With resid: + resid[i] w[y_i][k] (bf16 weights)
struct Fold {
  const float* part;
  int parts;
  int64_t part_stride, rows, ld, width;
  void* out;
  int out_bf16;
  const float* resid;
  const int32_t* y;
  const bf16* w;
  int64_t w_ld, vocab;
};

// up to three such sums (those of dx, db and dW) in one launch
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_fold(Fold one, Fold two, Fold three) {
  const int64_t first = one.rows * one.width, second = first + two.rows * two.width, all = second + three.rows * three.width;
  auto entry = [](const Fold& f, int64_t i) {
    const int64_t r = i / f.width, k = i - r * f.width;
    float s = 0.0f;
    const float* at = f.part + r * f.ld + k;
    int p = 0;
    for (; p + 8 <= f.parts; p += 8, at += 8 * f.part_stride) {         // eight loads in flight, added in order
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = at[j * f.part_stride];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += x[j];
    }
    for (; p < f.parts; ++p, at += f.part_stride) s += *at;
    if (f.resid) s += f.resid[r] * (float)f.w[min(max((int64_t)f.y[r], (int64_t)0), f.vocab - 1) * f.w_ld + k];
    if (f.out_bf16) ((bf16*)f.out)[i] = (bf16)s;
    else ((float*)f.out)[i] = s;
  };
  for (int64_t u = (int64_t)blockIdx.x * GJX_BLOCK + threadIdx.x; u < all; u += (int64_t)gridDim.x * GJX_BLOCK) {
    if (u < first) entry(one, u);
    else if (u < second) entry(two, u - first);
    else entry(three, u - second);
  }
}

// ---------------------------------------------------------------------------
// host: sizes and workspace
// ---------------------------------------------------------------------------
constexpr int64_t DL_BYTES = (int64_t)512 << 20;      // dl of one piece of the vocabulary (any size is right)
constexpr int64_t PACK_BYTES = (int64_t)512 << 20;    // packed weights of one piece
constexpr int64_t MAX_LD = 1 << 22;                   // 256 rows stay within 32-bit byte offsets
// f32 density or draw of 129 to 208 rows: one tile can hold them all (208: what the accumulators of two workgroups a CU leave
// room for), so that the weights are read and split once instead of once for each of two tiles of 128.  Two such workgroups on a
// CU take the time of 3.55 of the smaller ones, one alone that of 2.8, so it depends on how the tiles fill the CUs: 200 rows of
// width 256, one tile / two tiles, at 250 tiles of the vocabulary 39 / 31 us, 321: 43 / 38, 391: 44 / 51, 508: 47 / 52,
// 625: 72 / 60, 1000: 85 / 90; 200 x 50001 x 768: 105 / 132.  The row count moves neither side (130, 150, 180, 200 and 208 rows
// within 4 %): width 256 at 391 tiles 44 / 52, 508: 48 / 56, 560: 75 / 62, 1000: 95 / 100; width 768 at 321: 104 / 100, 391:
// 109 / 133, 508: 125 / 144, 625: 191 / 169, 1000: 240 / 263.
constexpr int ALL_ROWS = 208;
bool one_row_tile(int64_t n, int64_t vocab_tiles) {
  const int64_t each = (vocab_tiles + 255) / 256, halves = (2 * vocab_tiles + 255) / 256;        // workgroups per CU
  return n > 128 && n <= ALL_ROWS && 71 * (each / 2) + 56 * (each % 2) < 20 * halves;
}
// when a reduction is cut (cuts_of), in tiles of depth and of the product
constexpr int CUT_DEPTH_F32 = 12, CUT_DEPTH_BF16 = 24, CUT_ROWS_DEPTH = 24, CUT_TILES = 64, CUT_DEEP = 32;
constexpr int ROWS_MAX = 32;                          // rows up to which k_lincat_rows is used
// What the forward of a gradient keeps (the exponentials of all logits) spares the gradient its first product and costs a
// write and a read of them; up to this size, and from the width on where the product is the dearer one; up to 32 rows
// always, since the product there takes as long as the weights.  Forward and gradient, kept against formed again, on the GPU alone:
// f32 1 x 35780 x 1386: 237 / 298 us, 8 x 128000 x 256: 133 / 160, 32 x 20011 x 512: 78 / 90, 32 x 128000 x 32: 98 / 100, 32 x 300 x 32:
// 33 / 32; bf16 1 x 32000 x 1024: 73 / 90, 8 x 128000 x 256: 96 / 107, 32 x 128000 x 512: 168 / 181, x 64: 83 / 84, 32 x 32000 x 64:
// 51 / 49, 16 x 1000 x 64: 40 / 39.  More rows: bf16 4096 x 32000 x 128: 475 / 460 us, x 256: 524 / 549, x 512: 610 / 666, x 1024: 915 / 1040;
// 300 x 8000 x 256: 62 / 57, x 512: 65 / 66; f32 1000 x 20011 x 64: 180 / 180, x 128: 191 / 200, x 512: 396 / 468.
constexpr int64_t KEEP_BYTES = (int64_t)2 << 30;
constexpr int KEEP_WIDTH_F32 = 128, KEEP_WIDTH_BF16 = 512;

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// a call's inputs
struct Call {
  const char* who;
  int dtype;
  const int32_t* y;
  const void* x;
  int64_t x_ld;
  const void* w;
  int64_t w_ld;
  const void* bias;
  int64_t n, vocab, width;
  bool f32() const { return dtype == GJX_F32; }
  const char* w_row(int64_t v) const { return (const char*)w + v * w_ld * (f32() ? 4 : 2); }
};

// rows a tile loader can take as they are: aligned to 16 bytes, whole 64-deep tiles
bool direct(const void* p, int64_t ld, int64_t width) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && width % 64 == 0; }

struct Plan {
  bool rows;                    // k_lincat_rows
  int bm, bn;                       // rows per tile
  int64_t kp, n_pad, n_tiles;
  bool pack_x, pack_w;
  int64_t piece;                // vocabulary entries per piece (multiple of 256)
  int64_t tiles;                // partial results per row
  int splits, splits_w;         // parts of the reductions of dx (over the piece) and dW (over the rows)
  int strip;                    // rows per workgroup of k_lincat_dl
  int cuts;                     // parts of the logits' reduction (1: done in the product's epilogue)
  int64_t cut_ld;
  int64_t o_x, o_w, o_part, o_target, o_dl, o_db, o_dx, o_dw, o_resid, o_cut, bytes;
};

struct Carver {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t p = at;
    at = up(at + bytes, 256);
    return p;
  }
};

// Few tiles and a long reduction: it is cut into parts of four tiles of depth or more, which a second launch adds up.
// Density, whole / cut: f32 200 x 500 x 1024 42 / 13 us, 500 x 300 x 500 27 / 14, 64 x 8000 x 512 (63 tiles) 25.6 / 24.7, 64 x 12000
// x 1024 (94 tiles, 32 deep) 42 / 34, 64 x 16000 x 1024 42 / 40; of the kernel for few rows 2 x 326 x 1024 21 / 11, 1 x 6000 x 4096
// 82 / 38; bf16 (half as deep, twice as fast a tile) 30 x 8000 x 2048 42 / 23, 1 x 3000 x 1600 31 / 13, 64 x 12000 x 2048 31 / 34
// with its gradient at 80 / 73.
int cuts_of(const Call& c, int64_t tiles, bool rows) {           // tiles: of the product, at least one
  const int64_t depth = up(c.width, c.f32() ? 32 : 64) / (c.f32() ? 32 : 64);
  if (depth < (rows ? CUT_ROWS_DEPTH : c.f32() ? CUT_DEPTH_F32 : CUT_DEPTH_BF16)) return 1;
  return tiles > (c.f32() && depth >= CUT_DEEP ? 2 * CUT_TILES : CUT_TILES) ? 1 : (int)std::min<int64_t>(512 / tiles, depth / 4);
}

// keeps: a forward whose tiles a gradient's have to match
Plan plan_of(const Call& c, bool grad, bool want_dx, bool keeps) {
  Plan p = {};
  const int64_t bm = c.f32() ? BM32 : BM, vt = up(c.vocab, bm) / bm;
  p.rows = !grad && c.n <= ROWS_MAX;
  p.bm = (int)bm;
  p.kp = c.f32() ? c.width : up(c.width, 64);
  p.pack_x = !c.f32() && !p.rows && !direct(c.x, c.x_ld, c.width);
  p.pack_w = !c.f32() && !p.rows && !direct(c.w, c.w_ld, c.width);
  // wide tiles where there are enough of them to fill the 256 CUs; f32 tiles are half as wide (three planes in LDS)
  const int wide = c.f32() ? 128 : 256;
  p.bn = (c.n > 64 && up(c.n, wide) / wide * vt >= 256) ? wide : 64;
  if (!grad && !keeps && c.f32() && one_row_tile(c.n, vt)) p.bn = ALL_ROWS;
  p.n_pad = p.rows ? up(c.n, 16) : up(c.n, p.bn);
  p.n_tiles = p.n_pad / p.bn;
  p.cuts = cuts_of(c, p.rows ? vt : vt * p.n_tiles, p.rows);
  if (p.cuts > 1 && p.rows) {                               // then tiles after all
    p.rows = false;
    p.pack_x = !c.f32() && !direct(c.x, c.x_ld, c.width);
    p.pack_w = !c.f32() && !direct(c.w, c.w_ld, c.width);
    p.n_pad = up(c.n, 64);
    p.n_tiles = 1;
  }
  p.cut_ld = up(c.vocab, 4);
  p.tiles = p.rows ? up(c.vocab, 64) / 64 : vt;
  const int64_t e = c.f32() ? 4 : 2;
  int64_t piece = up(c.vocab, BM);
  if (p.pack_w) piece = std::min(piece, std::max<int64_t>(BM, PACK_BYTES / (p.kp * 2) / BM * BM));
  if (grad) piece = std::min(piece, std::max<int64_t>(BM, DL_BYTES / (p.n_pad * e) / BM * BM));
  const int64_t pieces = up(c.vocab, piece) / piece;
  p.piece = up(up(c.vocab, pieces) / pieces, BM);           // equal pieces
  if (p.piece < c.vocab) p.cuts = 1;
  Carver k;
  p.o_x = k.take(p.pack_x ? c.n * p.kp * 2 : 0);
  p.o_w = k.take(p.pack_w ? p.piece * p.kp * 2 : 0);
  p.o_cut = k.take(p.cuts > 1 ? p.cuts * c.n * p.cut_ld * 4 : 0);
  if (grad) {
    p.o_dl = k.take(p.n_pad * p.piece * e);
    // strips of 64 rows, shorter ones where those would leave CUs without work
    p.strip = 64;
    while (p.strip > 16 && up(c.n, 64) / p.strip * (up(p.piece, GJX_BLOCK * 8) / (GJX_BLOCK * 8)) < 1024) p.strip /= 2;
    p.o_db = k.take(std::max(p.n_tiles, up(c.n, 64) / p.strip) * p.piece * 4);
    p.o_resid = k.take(c.n * 4);
    const int64_t tiles = up(c.width, bm) / bm * p.n_tiles;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>((c.f32() ? 768 : 512) / tiles, p.piece / (c.f32() ? 128 : 512)));
    // few tiles of dW: their rows are shared out (1000 x 2000 x 128: 63 us in eight workgroups)
    const int64_t tiles_w = up(c.width, bm) / bm * (up(c.vocab, c.f32() ? 128 : 256) / (c.f32() ? 128 : 256));
    p.splits_w = p.piece < c.vocab ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(256 / tiles_w, c.n / 128));
    p.o_dw = k.take(p.splits_w > 1 ? p.splits_w * c.vocab * up(c.width, 4) * 4 : 0);
    p.o_dx = k.take(want_dx ? (int64_t)p.splits * c.n * up(p.kp, 4) * 4 : 0);
  } else {
    p.o_part = k.take(p.tiles * p.n_pad * 8);
    p.o_target = k.take(c.n * 4);
  }
  p.bytes = k.at;
  return p;
}

// the buffer between a forward and its gradient
struct Kept {
  int64_t ld, o_base, o_lp, bytes;      // bytes = 0: nothing is kept
  int block;                            // entries that share a base: those of a wave
};

Kept kept_of(const Call& c, const Plan& forward) {
  Kept k = {};
  if (c.n > ROWS_MAX && c.width < (c.f32() ? KEEP_WIDTH_F32 : KEEP_WIDTH_BF16)) return k;
  k.ld = up(c.vocab, BM);
  k.block = forward.rows ? 16 : c.f32() ? BM32 / 2 : forward.bn == 256 ? BM / 2 : BM / 4;
  Carver at;
  at.take(c.n * k.ld * (c.f32() ? 4 : 2));
  k.o_base = at.take(k.ld / k.block * c.n * 4);
  k.o_lp = at.take(c.n * 4);
  k.bytes = at.at <= KEEP_BYTES ? at.at : 0;
  return k;
}

// a kernel's dynamic LDS limit, raised once per device
template <typename K>
int32_t allow_lds(K* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  GJX_CHECK_HIP(hipGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return GJX_OK;
  GJX_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
  return GJX_OK;
}

template <int BN, bool TA, bool TB, int EPI>
int32_t launch16(const GemmArgs& a, int64_t blocks, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = 2 * (BM + BN) * BK * 2;
  const int32_t rc = allow_lds(k_lincat_gemm<BN, TA, TB, EPI>, lds, done);
  if (rc != GJX_OK) return rc;
  k_lincat_gemm<BN, TA, TB, EPI><<<gjx_grid_rows(blocks), GEMM_THREADS, lds, s>>>(a);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

template <int BN, bool TA, bool TB, int EPI>
int32_t launch32(const GemmArgs& a, int64_t blocks, hipStream_t s) {
  static std::atomic<uint64_t> done{0};
  constexpr int lds = (BM32 + BN) / 16 * SPLIT_BYTES;
  const int32_t rc = allow_lds(k_lincat_gemm32<BN, TA, TB, EPI>, lds, done);
  if (rc != GJX_OK) return rc;
  k_lincat_gemm32<BN, TA, TB, EPI><<<gjx_grid_rows(blocks), GEMM32_THREADS, lds, s>>>(a);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

// wide: the larger of the two row tiles
template <bool TA, bool TB, int EPI>
int32_t launch(const Call& c, bool wide, const GemmArgs& a, hipStream_t s) {
  const int64_t blocks = (int64_t)a.mt * a.nt * a.splits;
  GJX_REQUIRE(blocks < ((int64_t)1 << 31) - (1 << 21), GJX_ELIMIT, "%s: %lld tiles", c.who, (long long)blocks);
  if constexpr (TB) {           // dW: n is the vocabulary, always wide
    return c.f32() ? launch32<128, TA, TB, EPI>(a, blocks, s) : launch16<256, TA, TB, EPI>(a, blocks, s);
  } else if constexpr (EPI == EPI_STORE && !TA) {            // the cut product of few tiles
    return c.f32() ? launch32<64, TA, TB, EPI>(a, blocks, s) : launch16<64, TA, TB, EPI>(a, blocks, s);
  } else {
    if constexpr (EPI == EPI_SCORE || EPI == EPI_DRAW)
      if (c.f32() && a.n_pad == ALL_ROWS) return launch32<ALL_ROWS, TA, TB, EPI>(a, blocks, s);
    if (c.f32()) return wide ? launch32<128, TA, TB, EPI>(a, blocks, s) : launch32<64, TA, TB, EPI>(a, blocks, s);
    return wide ? launch16<256, TA, TB, EPI>(a, blocks, s) : launch16<64, TA, TB, EPI>(a, blocks, s);
  }
}

int32_t pack(const void* src, int64_t ld, int64_t rows, int64_t width, int64_t kp, bf16* dst, hipStream_t s) {
  k_lincat_pack<<<gjx_grid_for(rows * (kp / 8)), GJX_BLOCK, 0, s>>>((const bf16*)src, ld, rows, (int)width, (int)kp, dst);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

int32_t check_args(const Call& c) {
  GJX_REQUIRE(c.dtype == GJX_F32 || c.dtype == GJX_BF16, GJX_EINVAL, "%s: dtype %d is neither GJX_F32 nor GJX_BF16", c.who, c.dtype);
  GJX_REQUIRE(c.n >= 0 && c.vocab >= 1 && c.width >= 1, GJX_EINVAL, "%s: bad sizes (n %lld, vocab %lld, width %lld)", c.who,
              (long long)c.n, (long long)c.vocab, (long long)c.width);
  GJX_REQUIRE(c.n == 0 || (c.y && c.x && c.w), GJX_EINVAL, "%s: null input", c.who);
  GJX_REQUIRE(c.x_ld >= c.width && c.w_ld >= c.width, GJX_EINVAL, "%s: a row stride is smaller than the width", c.who);
  GJX_REQUIRE(c.x_ld <= MAX_LD && c.w_ld <= MAX_LD, GJX_ELIMIT, "%s: a row stride is above 2^22 elements", c.who);
  GJX_REQUIRE(c.n <= GJX_MAX_LINCAT && c.vocab <= GJX_MAX_LINCAT && c.width <= 65536, GJX_ELIMIT,
              "%s: n and vocab go up to 2^24, width up to 65536", c.who);
  return GJX_OK;
}

int32_t check_work(const Call& c, const Plan& p, const void* work, int64_t bytes) {
  GJX_REQUIRE(work && ((uintptr_t)work & 255) == 0 && bytes >= p.bytes, GJX_EINVAL,
              "%s: the workspace has %lld bytes, needs %lld aligned to 256", c.who, (long long)bytes, (long long)p.bytes);
  return GJX_OK;
}

int32_t check_kept(const Call& c, const Kept& k, const void* kept, int64_t bytes) {
  GJX_REQUIRE(k.bytes > 0 && ((uintptr_t)kept & 255) == 0 && bytes >= k.bytes, GJX_EINVAL,
              "%s: d_kept has %lld bytes, needs %lld aligned to 256 (0: nothing is kept at these sizes)", c.who, (long long)bytes,
              (long long)k.bytes);
  return GJX_OK;
}

GemmArgs common_args(const Call& c, const Plan& p) {
  GemmArgs a = {};
  a.splits = 1;
  a.vocab = c.vocab;
  a.n = c.n;
  a.n_pad = p.n_pad;
  a.bias = c.bias;
  a.bias_f32 = c.f32();
  a.y = c.y;
  return a;
}

// x and `rows` rows of W from v0 on as operands, packed where the tile loader needs it
struct Inputs {
  Operand x, w;
  OperandF fx, fw;
};

int32_t take_x(const Call& c, const Plan& p, char* ws, Inputs& in, hipStream_t s) {
  in.fx = {(const float*)c.x, c.x_ld, (int)c.n, (int)c.width};
  in.x = {(const bf16*)c.x, c.x_ld, (int)c.n, (int)p.kp};
  if (!p.pack_x) return GJX_OK;
  in.x = {(const bf16*)(ws + p.o_x), p.kp, (int)c.n, (int)p.kp};
  return pack(c.x, c.x_ld, c.n, c.width, p.kp, (bf16*)(ws + p.o_x), s);
}

int32_t take_w(const Call& c, const Plan& p, char* ws, int64_t v0, int64_t rows, Inputs& in, hipStream_t s) {
  const char* w = c.w_row(v0);
  in.fw = {(const float*)w, c.w_ld, (int)rows, (int)c.width};
  in.w = {(const bf16*)w, c.w_ld, (int)rows, (int)p.kp};
  if (!p.pack_w) return GJX_OK;
  in.w = {(const bf16*)(ws + p.o_w), p.kp, (int)rows, (int)p.kp};
  return pack(w, c.w_ld, rows, c.width, p.kp, (bf16*)(ws + p.o_w), s);
}

int depth_tiles(const Call& c, int64_t depth) { return (int)(c.f32() ? up(depth, 32) / 32 : up(depth, BK) / BK); }

// the logits without their bias in parts, for the whole vocabulary
int32_t cut_product(const Call& c, const Plan& p, const Inputs& in, char* ws, Parts& parts, hipStream_t s) {
  float* out = (float*)(ws + p.o_cut);
  GemmArgs a = common_args(c, p);
  a.a = in.w;
  a.fa = in.fw;
  a.b = in.x;
  a.fb = in.fx;
  a.ktiles = depth_tiles(c, p.kp);
  a.mt = (int)(up(c.vocab, p.bm) / p.bm);
  a.nt = (int)p.n_tiles;
  a.splits = p.cuts;
  a.out = out;
  a.out_ld = p.cut_ld;
  a.out_split = c.n * p.cut_ld;
  a.out_m = (int)c.vocab;
  a.out_n = (int)c.n;
  parts = {out, p.cuts, c.n * p.cut_ld, p.cut_ld, c.bias, c.f32()};
  return launch<false, false, EPI_STORE>(c, false, a, s);
}

// the forward product, reduced to log-densities (EPI_SCORE) or draws (EPI_DRAW)
struct Forward {
  float *lp, *lse;
  char* kept;
  uint32_t key0, key1;
  uint64_t offset;
  int32_t* out;
};

template <typename T, int EPI>
int32_t launch_rows(const Call& c, const Plan& p, const GemmArgs& a, hipStream_t s) {
  const unsigned blocks = (unsigned)p.tiles;
  if (p.n_pad == 16) k_lincat_rows<T, 1, EPI><<<blocks, GJX_BLOCK, 0, s>>>(a, (const T*)c.x, c.x_ld, (const T*)c.w, c.w_ld, (int)c.width);
  else k_lincat_rows<T, 2, EPI><<<blocks, GJX_BLOCK, 0, s>>>(a, (const T*)c.x, c.x_ld, (const T*)c.w, c.w_ld, (int)c.width);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

template <int EPI>
int32_t forward(const Call& c, const Plan& p, const Forward& f, void* d_work, int64_t work_bytes, hipStream_t s) {
  int32_t rc = check_work(c, p, d_work, work_bytes);
  if (rc != GJX_OK) return rc;
  const Kept kept = f.kept ? kept_of(c, p) : Kept{};
  char* ws = (char*)d_work;
  GemmArgs a = common_args(c, p);
  a.key0 = f.key0;
  a.key1 = f.key1;
  a.offset = f.offset;
  a.part = (float2*)(ws + p.o_part);
  a.target = (float*)(ws + p.o_target);
  a.keep = f.kept;
  a.keep_base = (float*)(f.kept + kept.o_base);
  a.keep_ld = kept.ld;
  if (p.cuts > 1) {
    Inputs in = {};
    Parts parts = {};
    if ((rc = take_x(c, p, ws, in, s)) != GJX_OK || (rc = take_w(c, p, ws, 0, c.vocab, in, s)) != GJX_OK) return rc;
    if ((rc = cut_product(c, p, in, ws, parts, s)) != GJX_OK) return rc;
    float *base = (float*)(f.kept + kept.o_base), *lp_kept = (float*)(f.kept + kept.o_lp);
    auto finish = [&](auto* kernel, int64_t blocks, int threads) {
      kernel<<<(unsigned)blocks, threads, 0, s>>>(parts, (float*)(ws + p.o_cut), c.n, c.vocab, c.y, f.lp, f.lse, f.kept, c.f32(), kept.ld,
                                                  base, kept.block, lp_kept, f.key0, f.key1, f.offset, f.out);
    };
    if (c.vocab <= 256) finish(k_lincat_finish<64, EPI>, up(c.n, 4) / 4, GJX_BLOCK);
    else if (c.vocab <= 1024) finish(k_lincat_finish<256, EPI>, c.n, 256);
    else finish(k_lincat_finish<1024, EPI>, c.n, 1024);
    GJX_LAUNCH_CHECK();
    return GJX_OK;
  }
  if (p.rows) {
    rc = c.f32() ? launch_rows<float, EPI>(c, p, a, s) : launch_rows<bf16, EPI>(c, p, a, s);
    if (rc != GJX_OK) return rc;
  } else {
    Inputs in = {};
    if ((rc = take_x(c, p, ws, in, s)) != GJX_OK) return rc;
    a.b = in.x;
    a.fb = in.fx;
    a.ktiles = depth_tiles(c, p.kp);
    a.nt = (int)p.n_tiles;
    for (int64_t v0 = 0; v0 < c.vocab; v0 += p.piece) {
      const int64_t rows = std::min(p.piece, c.vocab - v0);
      if ((rc = take_w(c, p, ws, v0, rows, in, s)) != GJX_OK) return rc;
      a.a = in.w;
      a.fa = in.fw;
      a.v0 = v0;
      a.part_tile0 = (int)(v0 / p.bm);
      a.mt = (int)(up(rows, p.bm) / p.bm);
      if ((rc = launch<false, false, EPI>(c, p.bn > 64, a, s)) != GJX_OK) return rc;
    }
  }
  if (EPI != EPI_DRAW) {
    int cols = 16;                                           // rows per workgroup; fewer where that fills more CUs
    while (cols > 1 && up(c.n, cols) / cols < 256) cols /= 2;
    k_lincat_combine<<<(unsigned)(up(c.n, cols) / cols), GJX_BLOCK, 0, s>>>(a.part, (int)p.tiles, p.n_pad, c.n, cols, a.target, f.lp, f.lse,
                                                                               f.kept ? (float*)(f.kept + kept.o_lp) : nullptr);
  } else {
    k_lincat_pick<<<(unsigned)(up(c.n, GJX_BLOCK / 64) / (GJX_BLOCK / 64)), GJX_BLOCK, 0, s>>>(a.part, (int)p.tiles, p.n_pad, c.n, f.out);
  }
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

}  // namespace

GJX_API int32_t gjx_linear_categorical_workspace(int32_t dtype, const void* d_x, int64_t x_ld, const void* d_w, int64_t w_ld,
                                                 int64_t n, int64_t vocab, int64_t width, int32_t kind, int64_t* bytes) {
  static const int32_t some_y = 0;
  const Call c = {"gjx_linear_categorical_workspace", dtype, &some_y, d_x, x_ld, d_w, w_ld, nullptr, n, vocab, width};
  GJX_REQUIRE(bytes != nullptr && kind >= 0 && kind <= 3, GJX_EINVAL, "%s: bytes is null or kind not in [0, 3]", c.who);
  const int32_t rc = check_args(c);
  if (rc != GJX_OK) return rc;
  if (n == 0) *bytes = 0;
  else if (kind == 3) *bytes = kept_of(c, plan_of(c, false, false, true)).bytes;
  else if (kind == 0) *bytes = std::max(plan_of(c, false, false, false).bytes, plan_of(c, false, false, true).bytes);
  else *bytes = plan_of(c, true, kind == 1, false).bytes;
  return GJX_OK;
}

GJX_API int32_t gjx_linear_categorical_logpdf(int32_t dtype, const int32_t* d_y, const void* d_x, int64_t x_ld,
                                              const void* d_w, int64_t w_ld, const void* d_bias, int64_t n, int64_t vocab,
                                              int64_t width, float* d_lp, float* d_lse, void* d_kept, int64_t kept_bytes,
                                              void* d_work, int64_t work_bytes, void* stream) {
  const Call c = {"gjx_linear_categorical_logpdf", dtype, d_y, d_x, x_ld, d_w, w_ld, d_bias, n, vocab, width};
  int32_t rc = check_args(c);
  if (rc != GJX_OK || n == 0) return rc;
  GJX_REQUIRE(d_lp, GJX_EINVAL, "%s: null output", c.who);
  Forward f = {};
  f.lp = d_lp;
  f.lse = d_lse;
  const Plan p = plan_of(c, false, false, d_kept != nullptr);
  if (d_kept) {
    if ((rc = check_kept(c, kept_of(c, p), d_kept, kept_bytes)) != GJX_OK) return rc;
    f.kept = (char*)d_kept;
    return forward<EPI_KEEP>(c, p, f, d_work, work_bytes, (hipStream_t)stream);
  }
  return forward<EPI_SCORE>(c, p, f, d_work, work_bytes, (hipStream_t)stream);
}

GJX_API int32_t gjx_random_linear_categorical_i32(const uint32_t key[2], uint64_t offset, int32_t dtype, const void* d_x,
                                                  int64_t x_ld, const void* d_w, int64_t w_ld, const void* d_bias, int64_t n,
                                                  int64_t vocab, int64_t width, int32_t* d_out, void* d_work,
                                                  int64_t work_bytes, void* stream) {
  static const int32_t some_y = 0;
  const Call c = {"gjx_random_linear_categorical_i32", dtype, &some_y, d_x, x_ld, d_w, w_ld, d_bias, n, vocab, width};
  const int32_t rc = check_args(c);
  if (rc != GJX_OK || n == 0) return rc;
  GJX_REQUIRE(key && d_out, GJX_EINVAL, "%s: null key or output", c.who);
  Forward f = {};
  f.key0 = key[0];
  f.key1 = key[1];
  f.offset = offset;
  f.out = d_out;
  return forward<EPI_DRAW>(c, plan_of(c, false, false, false), f, d_work, work_bytes, (hipStream_t)stream);
}

GJX_API int32_t gjx_linear_categorical_grad(int32_t dtype, const int32_t* d_y, const void* d_x, int64_t x_ld, const void* d_w,
                                            int64_t w_ld, const void* d_bias, int64_t n, int64_t vocab, int64_t width,
                                            const float* d_lse, const float* d_upstream, const void* d_kept, int64_t kept_bytes,
                                            void* d_dx, void* d_dw, void* d_db, void* d_work, int64_t work_bytes, void* stream) {
  const Call c = {"gjx_linear_categorical_grad", dtype, d_y, d_x, x_ld, d_w, w_ld, d_bias, n, vocab, width};
  int32_t rc = check_args(c);
  if (rc != GJX_OK) return rc;
  GJX_REQUIRE(n >= 1, GJX_EINVAL, "%s: no rows (the gradients are zero; the caller fills them)", c.who);
  GJX_REQUIRE(d_lse && d_upstream, GJX_EINVAL, "%s: null input", c.who);
  const bool f32 = c.f32();
  const Plan p = plan_of(c, true, d_dx != nullptr, false);
  if ((rc = check_work(c, p, d_work, work_bytes)) != GJX_OK) return rc;
  Kept kept = {};
  if (d_kept) {
    kept = kept_of(c, plan_of(c, false, false, true));
    if ((rc = check_kept(c, kept, d_kept, kept_bytes)) != GJX_OK) return rc;
  }
  if (!d_dx && !d_dw && !d_db) return GJX_OK;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)d_work;
  Inputs in = {};
  if ((rc = take_x(c, p, ws, in, s)) != GJX_OK) return rc;
  const bool wide = p.bn > 64;
  const int mk = (int)(up(width, p.bm) / p.bm);
  const int64_t part_ld = up(p.kp, 4);
  float *dx_part = (float*)(ws + p.o_dx), *db_part = (float*)(ws + p.o_db), *resid = f32 ? nullptr : (float*)(ws + p.o_resid);
  const bool whole = p.piece >= vocab;                       // one piece
  const bool dx_direct = whole && f32 && p.splits == 1;      // nothing to add up
  const int db_parts = (int)(d_kept || p.cuts > 1 ? up(n, 64) / p.strip : p.n_tiles);
  Fold dx_fold = {}, db_fold = {}, dw_fold = {};
  auto fold = [&](const Fold& one, const Fold& two, const Fold& three) -> int32_t {
    const int64_t entries = one.rows * one.width + two.rows * two.width + three.rows * three.width;
    k_lincat_fold<<<gjx_grid_for(entries), GJX_BLOCK, 0, s>>>(one, two, three);
    GJX_LAUNCH_CHECK();
    return GJX_OK;
  };
  for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
    const int64_t rows = std::min(p.piece, vocab - v0), rows_pad = up(rows, BM);
    if ((rc = take_w(c, p, ws, v0, rows, in, s)) != GJX_OK) return rc;
    const Operand dl = {(const bf16*)(ws + p.o_dl), p.piece, (int)p.n_pad, (int)p.piece};
    const OperandF fdl = {(const float*)(ws + p.o_dl), p.piece, (int)p.n_pad, (int)rows_pad};
    if (d_kept) {
      const char* k = (const char*)d_kept;
      const dim3 grid((unsigned)(up(n, 64) / p.strip), (unsigned)(up(rows_pad, GJX_BLOCK * 8) / (GJX_BLOCK * 8)));
      if (f32)
        k_lincat_dl<float><<<grid, GJX_BLOCK, 0, s>>>(k, kept.ld, (const float*)(k + kept.o_base), kept.block,
                                                      (const float*)(k + kept.o_lp), d_lse, d_upstream, d_y, n, vocab, v0, (int)rows_pad, p.strip,
                                                      (float*)(ws + p.o_dl), p.piece, resid, d_db ? db_part : nullptr, p.piece);
      else
        k_lincat_dl<bf16><<<grid, GJX_BLOCK, 0, s>>>(k, kept.ld, (const float*)(k + kept.o_base), kept.block,
                                                     (const float*)(k + kept.o_lp), d_lse, d_upstream, d_y, n, vocab, v0, (int)rows_pad, p.strip,
                                                     (bf16*)(ws + p.o_dl), p.piece, resid, d_db ? db_part : nullptr, p.piece);
      GJX_LAUNCH_CHECK();
    } else if (p.cuts > 1) {                                 // (one piece)
      Parts parts = {};
      if ((rc = cut_product(c, p, in, ws, parts, s)) != GJX_OK) return rc;
      const dim3 grid((unsigned)(up(n, 64) / p.strip), (unsigned)(rows_pad / 64));
      if (f32)
        k_lincat_dl_parts<float><<<grid, GJX_BLOCK, 0, s>>>(parts, d_lse, d_upstream, d_y, n, vocab, p.strip,
                                                            (float*)(ws + p.o_dl), p.piece, resid, d_db ? db_part : nullptr, p.piece);
      else
        k_lincat_dl_parts<bf16><<<grid, GJX_BLOCK, 0, s>>>(parts, d_lse, d_upstream, d_y, n, vocab, p.strip,
                                                           (bf16*)(ws + p.o_dl), p.piece, resid, d_db ? db_part : nullptr, p.piece);
      GJX_LAUNCH_CHECK();
    } else {
      GemmArgs a = common_args(c, p);                        // logits of the piece -> dl
      a.a = in.w;
      a.fa = in.fw;
      a.b = in.x;
      a.fb = in.fx;
      a.ktiles = depth_tiles(c, p.kp);
      a.mt = (int)(rows_pad / p.bm);
      a.nt = (int)p.n_tiles;
      a.v0 = v0;
      a.lse = d_lse;
      a.g = d_upstream;
      a.dl = ws + p.o_dl;
      a.resid = resid;
      a.dl_ld = p.piece;
      a.db_part = d_db ? db_part : nullptr;
      if ((rc = launch<false, false, EPI_DL>(c, wide, a, s)) != GJX_OK) return rc;
    }
    if (d_db) {
      db_fold = {db_part, db_parts, p.piece, 1, rows, rows, (char*)d_db + v0 * (f32 ? 4 : 2), !f32, nullptr, nullptr, nullptr, 0, 0};
      if (!whole && (rc = fold(db_fold, Fold{}, Fold{})) != GJX_OK) return rc;
    }
    if (d_dx) {                                              // dx^T = W^T dl^T: m = feature, n = row, over the piece
      GemmArgs b = common_args(c, p);
      b.a = in.w;
      b.fa = in.fw;
      b.b = dl;
      b.fb = fdl;
      b.ktiles = depth_tiles(c, rows);                       // no tile lies wholly behind the last row of W
      b.mt = mk;
      b.nt = (int)p.n_tiles;
      b.splits = p.splits;
      b.out = dx_direct ? d_dx : (void*)dx_part;
      b.out_ld = dx_direct ? width : part_ld;
      b.out_split = n * part_ld;
      b.out_m = (int)p.kp;
      b.out_n = (int)n;
      b.accumulate = v0 > 0;
      if ((rc = launch<true, false, EPI_STORE>(c, wide, b, s)) != GJX_OK) return rc;
    }
    if (d_dw) {                                              // dW^T = x^T dl: m = feature, n = entry, over the rows
      GemmArgs b = common_args(c, p);
      b.a = in.x;
      b.fa = in.fx;
      b.b = dl;
      b.fb = fdl;
      b.ktiles = depth_tiles(c, n);
      b.mt = mk;
      b.nt = (int)(f32 ? up(rows, 128) / 128 : rows_pad / 256);
      b.out = f32 ? (void*)((float*)d_dw + v0 * width) : (void*)((bf16*)d_dw + v0 * width);
      b.out_ld = width;
      b.out_bf16 = !f32;
      if (p.splits_w > 1) {                                  // (one piece)
        float* part = (float*)(ws + p.o_dw);
        const int64_t ld = up(width, 4);
        b.splits = p.splits_w;
        b.out = part;
        b.out_ld = ld;
        b.out_split = vocab * ld;
        b.out_bf16 = 0;
        dw_fold = {part, p.splits_w, vocab * ld, vocab, ld, width, d_dw, !f32, nullptr, nullptr, nullptr, 0, 0};
      }
      b.out_m = (int)width;
      b.out_n = (int)rows;
      b.resid_in = resid;
      b.v0 = v0;
      if ((rc = launch<true, true, EPI_STORE>(c, true, b, s)) != GJX_OK) return rc;
    }
  }
  if (d_dx && !dx_direct)
    dx_fold = {dx_part, p.splits, n * part_ld, n, part_ld, width, d_dx, !f32, resid, d_y, (const bf16*)d_w, w_ld, vocab};
  if (!whole) db_fold = {};                                  // (done piece by piece)
  if (dx_fold.out || db_fold.out || dw_fold.out) return fold(dx_fold, db_fold, dw_fold);
  return GJX_OK;
}
