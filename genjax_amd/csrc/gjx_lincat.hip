// gjx_lincat.hip -- the categorical distribution whose logits are a linear map of a feature row,
//   l_iv = x_i . w_v + b_v,   log p(y_i) = l_{i,y_i} - log sum_v exp(l_iv),
// its gradient and its Gumbel-max draw.  The n x vocab logits are never kept: the forward reduces every tile of
// them to (max, sum exp) in the product's epilogue, the gradient forms them again piece by piece of the vocabulary,
// turns them into d l = g (onehot(y) - exp(l - lse)) in that product's epilogue and feeds two more products,
//   dx = dl W,   dW = dl^T x,   db = sum_i dl_i.
// The products are 16x16x32 bf16 MFMA tiles with f32 accumulators.  f32 operands are split exactly into three
// bf16 planes (8 + 8 + 8 bits) and the six partial products above 2^-24 are summed smallest first.
#include "gjx_common.h"

#include <algorithm>

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

#define LDS_AS __attribute__((address_space(3)))
#define GLB_AS __attribute__((address_space(1)))

namespace {

constexpr int BM = 256, BK = 64, GEMM_THREADS = 512;

enum { EPI_SCORE = 0, EPI_DL = 1, EPI_STORE = 2, EPI_DRAW = 3 };

// one operand of a product: `rows` memory rows of `ld` elements.  Not transposed: a row is one output index with the
// reduction along it; transposed: a row is one reduction index with the output index along it (`cols` of them, a
// multiple of 8).  Indices beyond the end are clamped: what they add is discarded or multiplied by a zero.
struct Operand {
  const bf16* p;
  int64_t ld, plane;
  int rows, cols;
};

struct GemmArgs {
  Operand a, b;
  int pairs;           // 1, or 6 partial products of three planes each
  int ktiles;          // reduction length / 64
  int mt, nt, splits;  // tiles along m and n, parts of the reduction
  // EPI_SCORE / EPI_DL: m = vocabulary entry (v0 = first of this piece), n = row
  int64_t v0, vocab, n;
  const void* bias;
  int bias_f32;
  const int32_t* y;
  float2* part;        // [tile m][n_pad]: (max, sum exp) of a row over one tile; drawing: (largest l + Gumbel, its entry)
  float* target;       // logit of y
  int64_t n_pad;
  int part_tile0;
  uint32_t key0, key1;
  uint64_t offset;
  const float *lse, *g;
  bf16* dl;            // [planes][n_pad][dl_ld]
  float* resid;        // [n]: dl of the row's value less its bf16 rounding (bf16 only)
  const float* resid_in;   // EPI_STORE of dW: the same, added to the value's row
  int64_t dl_ld, dl_plane;
  float* db_part;      // [tile n][dl_ld]
  // EPI_STORE: out[n][m] (+ split * out_split), f32 or bf16
  void* out;
  int64_t out_ld, out_split;
  int out_m, out_n, out_bf16, accumulate;
};

__device__ __forceinline__ float load_any(const void* p, int f32, int64_t i) {
  return f32 ? ((const float*)p)[i] : (float)((const bf16*)p)[i];
}

// x = h + m + l exactly, each rounded to nearest (8 bits of the 24 apiece, signed): |m| <= 2^-8 |x|, |l| <= 2^-16 |x|, so the
// partial products left out are at most 2^-23 |x| |w| each.  An h that would round to infinity is cut off instead; an
// infinite x keeps h only.
__device__ __forceinline__ void split3(float x, bf16& h, bf16& m, bf16& l) {
  h = (bf16)x;
  if (__builtin_isinf((float)h) && !__builtin_isinf(x)) h = (bf16)__uint_as_float(__float_as_uint(x) & 0xffff0000u);
  const float r = __builtin_isinf(x) ? 0.0f : x - (float)h;
  m = (bf16)r;
  l = (bf16)(r - (float)m);
}

__device__ __forceinline__ int tr_swizzle(int k) { return (k & 3) | (((k >> 3) & 3) << 2); }

template <int R, bool T>
struct TileLoader {
  // one BK-deep tile of an operand, R output indices wide: R * 8 chunks of 16 bytes straight into LDS
  static constexpr int LOADS = R * 8 / GEMM_THREADS;

  static __device__ __forceinline__ void load(const Operand& o, const bf16* plane, int out0, int k0, LDS_AS char* lds,
                                              int tid) {
    const int wave = tid >> 6;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int c = (j * (GEMM_THREADS / 64) + wave) * 64 + (tid & 63);
      const bf16* src;
      if (T) {
        const int row = c / (R / 8), ch = c % (R / 8);
        const int mem = min(k0 + row, o.rows - 1);
        const int col = min(out0 + ((((ch >> 1) ^ tr_swizzle(row)) << 1) | (ch & 1)) * 8, o.cols - 8);
        src = plane + (int64_t)mem * o.ld + col;
      } else {
        const int row = c >> 3, ch = (c & 7) ^ ((row >> 1) & 7);
        src = plane + (int64_t)min(out0 + row, o.rows - 1) * o.ld + (k0 + ch * 8);
      }
      __builtin_amdgcn_global_load_lds((const GLB_AS void*)src, (LDS_AS void*)(lds + (j * (GEMM_THREADS / 64) + wave) * 1024),
                                       16, 0, 0);
    }
  }

  // the 8 reduction elements 8 q .. 8 q + 7 of slab s (32 deep) for output index i0 + lane % 16
  static __device__ __forceinline__ bf16x8 frag(LDS_AS char* lds, int i0, int s, int lane) {
    const int q = lane >> 4, i = lane & 15;
    if (T) {
      const int k = 32 * s + 8 * q + (i >> 2);
      LDS_AS char* p = lds + k * (R * 2) + (((i0 >> 4) ^ tr_swizzle(k)) << 5) + ((i & 3) << 3);
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_AS bf16x4*)p);
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_AS bf16x4*)(p + 4 * R * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    const int row = i0 + i, ch = (s * 4 + q) ^ ((row >> 1) & 7);
    return *(LDS_AS bf16x8*)(lds + row * 128 + ch * 16);
  }
};

// C[m][n] = sum over plane pairs and k of A(m, k) B(n, k); BM x BN per workgroup of eight waves.  Two LDS buffers of
// one 64-deep tile each: the loads of tile i + 1 run under the products of tile i, one barrier per tile.
template <int BN, bool TA, bool TB, int EPI>
__global__ void __launch_bounds__(GEMM_THREADS)
    k_lincat_gemm(GemmArgs g) {
  constexpr int WN = BN == 256 ? 4 : 2, WM = 8 / WN;       // waves along n and m
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE = A_BYTES + B_BYTES;
  extern __shared__ char smem_raw[];
  LDS_AS char* smem = (LDS_AS char*)smem_raw;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // neighbouring tiles to one XCD (workgroups go round the eight of them), eight m-tiles by all n-tiles at a time
  int id = blockIdx.x;
  const int total = g.mt * g.nt * g.splits;
  {
    const int per = total / 8, extra = total % 8, xcd = id % 8;
    id = xcd * per + min(xcd, extra) + id / 8;
  }
  const int split = id / (g.mt * g.nt);
  id -= split * g.mt * g.nt;
  const int group = id / (8 * g.nt), in = id - group * 8 * g.nt, height = min(8, g.mt - group * 8);
  const int tm = group * 8 + in % height, tn = in / height;
  const int m0 = tm * BM, n0 = tn * BN;

  const int all = g.ktiles;
  const int kt0 = (int)((int64_t)all * split / g.splits), kt1 = (int)((int64_t)all * (split + 1) / g.splits);
  const int per_pair = kt1 - kt0, iters = per_pair * g.pairs;

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  auto issue = [&](int it, int buf) {
    const int pair = it / per_pair, kt = kt0 + (it - pair * per_pair);
    // (h l) (m m) (l h) (h m) (m h) (h h)
    const int pa = g.pairs == 1 ? 0 : (0x010210 >> (4 * pair)) & 3;
    const int pb = g.pairs == 1 ? 0 : (0x001012 >> (4 * pair)) & 3;
    TileLoader<BM, TA>::load(g.a, g.a.p + pa * g.a.plane, m0, kt * BK, smem + buf * STAGE, tid);
    TileLoader<BN, TB>::load(g.b, g.b.p + pb * g.b.plane, n0, kt * BK, smem + buf * STAGE + A_BYTES, tid);
  };

  const int wm = (wave / WN) * (MT * 16), wn = (wave % WN) * (NT * 16);
  if (iters > 0) issue(0, 0);
  for (int it = 0; it < iters; ++it) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (it + 1 < iters) issue(it + 1, (it + 1) & 1);
    LDS_AS char* sa = smem + (it & 1) * STAGE;
    LDS_AS char* sb = sa + A_BYTES;
#pragma unroll
    for (int s = 0; s < BK / 32; ++s) {
      bf16x8 fb[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) fb[j] = TileLoader<BN, TB>::frag(sb, wn + j * 16, s, lane);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const bf16x8 fa = TileLoader<BM, TA>::frag(sa, wm + i * 16, s, lane);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb[j], acc[i][j], 0, 0, 0);
      }
    }
  }
  __syncthreads();

  const int q = lane >> 4, c = lane & 15;
  if (EPI == EPI_STORE) {
    if (TB && g.resid_in) {
      // dW of the rows' own values: += resid_i x_i, in ascending i (every wave looks for its own columns)
      for (int64_t i0 = 0; i0 < g.n; i0 += 64) {
        const int64_t row = min(i0 + lane, g.n - 1);
        const int64_t v = min(max((int64_t)g.y[row], (int64_t)0), g.vocab - 1) - g.v0 - n0 - wn;
        const float res = g.resid_in[row];
        uint64_t hits = __ballot(i0 + lane < g.n && v >= 0 && v < NT * 16);
        while (hits) {
          const int l = __builtin_ctzll(hits);
          hits &= hits - 1;
          const int vl = __builtin_amdgcn_readlane((int)v, l);
          const float rl = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(res), l));
          if ((vl & 15) == c) {
            const bf16* xr = g.a.p + (i0 + l) * g.a.ld;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const bf16x4 xv = *(const bf16x4*)(xr + min(m0 + wm + i * 16 + 4 * q, g.a.cols - 4));
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                const float w = (vl >> 4) == j ? rl : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] += w * (float)xv[r];
              }
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

  if (EPI == EPI_SCORE) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int64_t n = n0 + wn + j * 16 + c;
      const bool live = n < g.n;
      float top = -__builtin_inff();
      // y outside [0, vocab) takes the nearest entry, as categorical does
      const int64_t y = live ? min(max((int64_t)g.y[n], (int64_t)0), g.vocab - 1) - g.v0 - m0 - wm - 4 * q : -1;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[i][j][r] += bias[i][r];
          if (s_bias[wm + i * 16 + 4 * q + r] == -__builtin_inff()) acc[i][j][r] = bias[i][r];
          top = fmaxf(top, acc[i][j][r]);
          if (y == i * 16 + r) g.target[n] = acc[i][j][r];
        }
      const float base = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += expf(acc[i][j][r] - base);
#pragma unroll
      for (int o = 16; o <= 32; o <<= 1) {
        const float t2 = __shfl_xor(top, o), s2 = __shfl_xor(sum, o), nt = fmaxf(top, t2);
        const float b2 = nt == -__builtin_inff() ? 0.0f : nt;
        sum = sum * expf(top - b2) + s2 * expf(t2 - b2);
        top = nt;
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
        const float t2 = s_red[(w * BN + tid) * 2], s2 = s_red[(w * BN + tid) * 2 + 1], nt = fmaxf(top, t2);
        const float b2 = nt == -__builtin_inff() ? 0.0f : nt;
        sum = sum * expf(top - b2) + s2 * expf(t2 - b2);
        top = nt;
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
        const float b2 = __shfl_xor(best, o);
        const int a2 = __shfl_xor(arg, o);
        if (a2 != 0x7fffffff && (b2 > best || arg == 0x7fffffff || (b2 == best && a2 < arg))) {
          best = b2;
          arg = a2;
        }
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
        const float b2 = s_red[(w * BN + tid) * 2];
        const int a2 = __float_as_int(s_red[(w * BN + tid) * 2 + 1]);
        if (a2 != 0x7fffffff && (b2 > best || arg == 0x7fffffff)) {      // later waves hold later entries
          best = b2;
          arg = a2;
        }
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
    const float lse = live ? g.lse[n] : 0.0f, up = live ? g.g[n] : 0.0f;
    const int64_t y = live ? min(max((int64_t)g.y[n], (int64_t)0), g.vocab - 1) - g.v0 - m0 - wm - 4 * q : -1;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float d[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool in = live && g.v0 + m0 + wm + i * 16 + 4 * q + r < g.vocab;
        const float l = bias[i][r] == -__builtin_inff() ? bias[i][r] : acc[i][j][r] + bias[i][r];
        d[r] = in ? up * ((y == i * 16 + r ? 1.0f : 0.0f) - expf(l - lse)) : 0.0f;
        dbs[i][r] += d[r];
      }
      bf16* o = g.dl + n * g.dl_ld + (m0 + wm + i * 16 + 4 * q);
      if (g.pairs == 1) {
        // rounded to bf16 (the products that follow take bf16 operands): each entry is off by at most 2^-9 of it,
        // independently of its neighbours.  The value's own entry is usually far larger than the others, so that ONE
        // rounding would show in whole rows of the gradients: what it loses is kept apart and added in f32.
        bf16x4 h;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          h[r] = (bf16)d[r];
          if (y == i * 16 + r) g.resid[n] = d[r] - (float)h[r];
        }
        *(bf16x4*)o = h;
      } else {
        bf16x4 h, m, l;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bf16 hh, mm, ll;
          split3(d[r], hh, mm, ll);
          h[r] = hh; m[r] = mm; l[r] = ll;
        }
        *(bf16x4*)o = h;
        *(bf16x4*)(o + g.dl_plane) = m;
        *(bf16x4*)(o + 2 * g.dl_plane) = l;
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

// rows x width of f32 or bf16 (row stride ld) -> planes of bf16 rows of width_pad, zeros behind the width
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_pack(const void* __restrict__ src, int f32, int64_t ld, int64_t rows, int width, int width_pad,
                  bf16* __restrict__ dst, int64_t plane) {
  const int64_t total = rows * (width_pad / 8);
  for (int64_t i = (int64_t)blockIdx.x * GJX_BLOCK + threadIdx.x; i < total; i += (int64_t)gridDim.x * GJX_BLOCK) {
    const int64_t row = i / (width_pad / 8);
    const int c0 = (int)(i - row * (width_pad / 8)) * 8;
    bf16x8 h, m, l;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      bf16 hh = (bf16)0.0f, mm = (bf16)0.0f, ll = (bf16)0.0f;
      if (c0 + k < width) {
        if (f32) split3(((const float*)src)[row * ld + c0 + k], hh, mm, ll);
        else hh = ((const bf16*)src)[row * ld + c0 + k];
      }
      h[k] = hh; m[k] = mm; l[k] = ll;
    }
    bf16* o = dst + row * width_pad + c0;
    *(bf16x8*)o = h;
    if (f32) {
      *(bf16x8*)(o + plane) = m;
      *(bf16x8*)(o + 2 * plane) = l;
    }
  }
}

// (max, sum exp) of the tiles of a row -> lse, and log p(y) = l_y - lse.  `width` rows by 256 / width parts per block.
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_combine(const float2* __restrict__ part, int tiles, int64_t n_pad, int64_t n, int width,
                     const float* __restrict__ target, float* __restrict__ lp, float* __restrict__ lse) {
  __shared__ float2 sm[GJX_BLOCK];
  const int col = threadIdx.x % width, grp = threadIdx.x / width, groups = GJX_BLOCK / width;
  const int64_t i = (int64_t)blockIdx.x * width + col;
  float top = -__builtin_inff(), sum = 0.0f;
  auto merge = [&](float2 p) {
    const float nt = fmaxf(top, p.x), b = nt == -__builtin_inff() ? 0.0f : nt;
    sum = sum * expf(top - b) + p.y * expf(p.x - b);
    top = nt;
  };
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
    lse[i] = l;
    lp[i] = target[i] - l;
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

// out[i][k] = sum over parts of part[s][i][k] in f32, stored in the output's type; rows of `width`, parts of `ld` columns.
// With resid: + resid[i] w[y_i][k] (bf16 weights)
__global__ void __launch_bounds__(GJX_BLOCK)
    k_lincat_fold(const float* __restrict__ part, int parts, int64_t part_stride, int64_t rows, int64_t ld, int64_t width,
                  void* __restrict__ out, int out_bf16, const float* __restrict__ resid, const int32_t* __restrict__ y,
                  const bf16* __restrict__ w, int64_t w_ld, int64_t vocab) {
  const int64_t total = rows * width;
  for (int64_t i = (int64_t)blockIdx.x * GJX_BLOCK + threadIdx.x; i < total; i += (int64_t)gridDim.x * GJX_BLOCK) {
    const int64_t r = i / width, k = i - r * width;
    float s = 0.0f;
    for (int p = 0; p < parts; ++p) s += part[p * part_stride + r * ld + k];
    if (resid) s += resid[r] * (float)w[min(max((int64_t)y[r], (int64_t)0), vocab - 1) * w_ld + k];
    if (out_bf16) ((bf16*)out)[i] = (bf16)s;
    else ((float*)out)[i] = s;
  }
}

// ---------------------------------------------------------------------------
// host: sizes and workspace
// ---------------------------------------------------------------------------
constexpr int64_t DL_BYTES = (int64_t)512 << 20;      // dl of one piece of the vocabulary (any size is right)
constexpr int64_t PACK_BYTES = (int64_t)512 << 20;    // packed weights of one piece

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

struct Plan {
  int planes, pairs;
  int bn;                       // rows per tile
  int64_t kp, n_pad, n_tiles;
  int pack_x, pack_w;
  int64_t piece;                // vocabulary entries per piece (multiple of 256)
  int64_t tiles;                // tiles of 256 over the whole vocabulary
  int splits;                   // parts of dx's reduction
  int64_t o_x, o_w, o_part, o_target, o_dl, o_db, o_dx, o_resid, bytes;
};

struct Carver {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t p = at;
    at = up(at + bytes, 256);
    return p;
  }
};

bool direct(const void* p, int64_t ld, int64_t width) {
  return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && width % 64 == 0;
}

Plan plan_of(int dtype, int64_t n, int64_t vocab, int64_t width, int pack_x, int pack_w, bool grad, bool want_dx) {
  Plan p = {};
  p.planes = dtype == GJX_F32 ? 3 : 1;
  p.pairs = dtype == GJX_F32 ? 6 : 1;
  p.kp = up(width, 64);
  p.pack_x = pack_x;
  p.pack_w = pack_w;
  p.tiles = up(vocab, BM) / BM;
  p.bn = (n > 64 && up(n, 256) / 256 * p.tiles >= 256) ? 256 : 64;
  p.n_pad = up(n, p.bn);
  p.n_tiles = p.n_pad / p.bn;
  int64_t piece = p.tiles * BM;
  if (pack_w) piece = std::min(piece, std::max<int64_t>(BM, PACK_BYTES / (p.kp * 2 * p.planes) / BM * BM));
  if (grad) piece = std::min(piece, std::max<int64_t>(BM, DL_BYTES / (p.n_pad * 2 * p.planes) / BM * BM));
  const int64_t pieces = up(p.tiles * BM, piece) / piece;
  p.piece = up(up(p.tiles, pieces) / pieces * BM, BM);      // equal pieces
  Carver c;
  p.o_x = c.take(pack_x ? n * p.kp * 2 * p.planes : 0);
  p.o_w = c.take(pack_w ? p.piece * p.kp * 2 * p.planes : 0);
  if (grad) {
    p.o_dl = c.take(p.n_pad * p.piece * 2 * p.planes);
    p.o_db = c.take(p.n_tiles * p.piece * 4);
    p.o_resid = c.take(n * 4);
    const int64_t tiles = up(width, BM) / BM * p.n_tiles;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / tiles, p.piece / BK / 8));
    p.o_dx = c.take(want_dx ? (int64_t)p.splits * n * p.kp * 4 : 0);
  } else {
    p.o_part = c.take(p.tiles * p.n_pad * 8);
    p.o_target = c.take(n * 4);
  }
  p.bytes = c.at;
  return p;
}

template <int BN, bool TA, bool TB, int EPI>
int32_t launch_gemm(const GemmArgs& a, hipStream_t s) {
  const int64_t blocks = (int64_t)a.mt * a.nt * a.splits;
  GJX_REQUIRE(blocks < ((int64_t)1 << 31), GJX_ELIMIT, "linear_categorical: %lld tiles", (long long)blocks);
  constexpr int lds = 2 * (BM + BN) * BK * 2;
  GJX_CHECK_HIP(hipFuncSetAttribute((const void*)k_lincat_gemm<BN, TA, TB, EPI>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  k_lincat_gemm<BN, TA, TB, EPI><<<(unsigned)blocks, GEMM_THREADS, lds, s>>>(a);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

int32_t pack(const void* src, int dtype, int64_t ld, int64_t rows, int64_t width, int64_t kp, bf16* dst, int64_t plane,
             hipStream_t s) {
  k_lincat_pack<<<gjx_grid_for(rows * (kp / 8)), GJX_BLOCK, 0, s>>>(src, dtype == GJX_F32, ld, rows, (int)width, (int)kp, dst, plane);
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

const char* at_row(const void* p, int dtype, int64_t elements) {
  return (const char*)p + elements * (dtype == GJX_F32 ? 4 : 2);
}

int32_t check_args(const char* who, const int32_t* y, const void* x, int64_t x_ld, const void* w, int64_t w_ld, int dtype,
                   int64_t n, int64_t vocab, int64_t width) {
  GJX_REQUIRE(dtype == GJX_F32 || dtype == GJX_BF16, GJX_EINVAL, "%s: dtype %d is neither GJX_F32 nor GJX_BF16", who, dtype);
  GJX_REQUIRE(n >= 0 && vocab >= 1 && width >= 1, GJX_EINVAL, "%s: bad sizes (n %lld, vocab %lld, width %lld)", who,
              (long long)n, (long long)vocab, (long long)width);
  GJX_REQUIRE(n == 0 || (y && x && w), GJX_EINVAL, "%s: null input", who);
  GJX_REQUIRE(x_ld >= width && w_ld >= width, GJX_EINVAL, "%s: a row stride is smaller than the width", who);
  GJX_REQUIRE(n <= GJX_MAX_LINCAT && vocab <= GJX_MAX_LINCAT && width <= 65536, GJX_ELIMIT,
              "%s: n and vocab go up to 2^24, width up to 65536", who);
  return GJX_OK;
}

}  // namespace

GJX_API int32_t gjx_linear_categorical_workspace(int32_t dtype, const void* d_x, int64_t x_ld, const void* d_w, int64_t w_ld,
                                                 int64_t n, int64_t vocab, int64_t width, int32_t grad, int64_t* bytes) {
  GJX_REQUIRE(bytes != nullptr, GJX_EINVAL, "gjx_linear_categorical_workspace: bytes is null");
  static const int32_t some_y = 0;
  int32_t rc = check_args("gjx_linear_categorical_workspace", &some_y, d_x, x_ld, d_w, w_ld, dtype, n, vocab, width);
  if (rc != GJX_OK) return rc;
  if (n == 0) {
    *bytes = 0;
    return GJX_OK;
  }
  const bool f32 = dtype == GJX_F32;
  *bytes = plan_of(dtype, n, vocab, width, f32 || !direct(d_x, x_ld, width), f32 || !direct(d_w, w_ld, width), grad != 0,
                   (grad & 1) != 0).bytes;
  return GJX_OK;
}

namespace {

// the forward product, reduced to log-densities (EPI_SCORE) or draws (EPI_DRAW)
struct Forward {
  const char* who;
  int epi;
  const int32_t* y;
  float *lp, *lse;
  uint32_t key0, key1;
  uint64_t offset;
  int32_t* out;
};

template <int EPI>
int32_t launch_rows(int bn, const GemmArgs& a, hipStream_t s) {
  return bn == 256 ? launch_gemm<256, false, false, EPI>(a, s) : launch_gemm<64, false, false, EPI>(a, s);
}

int32_t forward(const Forward& f, int dtype, const void* d_x, int64_t x_ld, const void* d_w, int64_t w_ld, const void* d_bias,
                int64_t n, int64_t vocab, int64_t width, void* d_work, int64_t work_bytes, hipStream_t s) {
  const bool f32 = dtype == GJX_F32;
  const Plan p = plan_of(dtype, n, vocab, width, f32 || !direct(d_x, x_ld, width), f32 || !direct(d_w, w_ld, width), false, false);
  GJX_REQUIRE(d_work && ((uintptr_t)d_work & 255) == 0 && work_bytes >= p.bytes, GJX_EINVAL,
              "%s: the workspace has %lld bytes, needs %lld aligned to 256", f.who, (long long)work_bytes, (long long)p.bytes);
  int32_t rc;
  char* ws = (char*)d_work;
  GemmArgs a = {};
  a.pairs = p.pairs;
  a.ktiles = (int)(p.kp / BK);
  a.splits = 1;
  a.nt = (int)p.n_tiles;
  a.b = {(const bf16*)d_x, x_ld, 0, (int)n, 0};
  if (p.pack_x) {
    if ((rc = pack(d_x, dtype, x_ld, n, width, p.kp, (bf16*)(ws + p.o_x), n * p.kp, s)) != GJX_OK) return rc;
    a.b = {(const bf16*)(ws + p.o_x), p.kp, n * p.kp, (int)n, 0};
  }
  a.vocab = vocab;
  a.n = n;
  a.n_pad = p.n_pad;
  a.bias = d_bias;
  a.bias_f32 = f32;
  a.y = f.y;
  a.key0 = f.key0;
  a.key1 = f.key1;
  a.offset = f.offset;
  a.part = (float2*)(ws + p.o_part);
  a.target = (float*)(ws + p.o_target);
  for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
    const int64_t rows = std::min(p.piece, vocab - v0);
    a.a = {(const bf16*)at_row(d_w, dtype, v0 * w_ld), w_ld, 0, (int)rows, 0};
    if (p.pack_w) {
      if ((rc = pack(at_row(d_w, dtype, v0 * w_ld), dtype, w_ld, rows, width, p.kp, (bf16*)(ws + p.o_w), p.piece * p.kp, s)) != GJX_OK)
        return rc;
      a.a = {(const bf16*)(ws + p.o_w), p.kp, p.piece * p.kp, (int)rows, 0};
    }
    a.v0 = v0;
    a.part_tile0 = (int)(v0 / BM);
    a.mt = (int)(up(rows, BM) / BM);
    rc = f.epi == EPI_SCORE ? launch_rows<EPI_SCORE>(p.bn, a, s) : launch_rows<EPI_DRAW>(p.bn, a, s);
    if (rc != GJX_OK) return rc;
  }
  if (f.epi == EPI_SCORE) {
    int cols = 1;
    while (cols < 64 && cols < n) cols *= 2;
    k_lincat_combine<<<(unsigned)(up(n, cols) / cols), GJX_BLOCK, 0, s>>>(a.part, (int)p.tiles, p.n_pad, n, cols, a.target, f.lp, f.lse);
  } else {
    k_lincat_pick<<<(unsigned)(up(n, GJX_BLOCK / 64) / (GJX_BLOCK / 64)), GJX_BLOCK, 0, s>>>(a.part, (int)p.tiles, p.n_pad, n, f.out);
  }
  GJX_LAUNCH_CHECK();
  return GJX_OK;
}

}  // namespace

GJX_API int32_t gjx_linear_categorical_logpdf(int32_t dtype, const int32_t* d_y, const void* d_x, int64_t x_ld,
                                              const void* d_w, int64_t w_ld, const void* d_bias, int64_t n, int64_t vocab,
                                              int64_t width, float* d_lp, float* d_lse, void* d_work, int64_t work_bytes,
                                              void* stream) {
  Forward f = {"gjx_linear_categorical_logpdf", EPI_SCORE, d_y, d_lp, d_lse, 0, 0, 0, nullptr};
  const int32_t rc = check_args(f.who, d_y, d_x, x_ld, d_w, w_ld, dtype, n, vocab, width);
  if (rc != GJX_OK || n == 0) return rc;
  GJX_REQUIRE(d_lp && d_lse, GJX_EINVAL, "%s: null output", f.who);
  return forward(f, dtype, d_x, x_ld, d_w, w_ld, d_bias, n, vocab, width, d_work, work_bytes, (hipStream_t)stream);
}

GJX_API int32_t gjx_random_linear_categorical_i32(const uint32_t key[2], uint64_t offset, int32_t dtype, const void* d_x,
                                                  int64_t x_ld, const void* d_w, int64_t w_ld, const void* d_bias, int64_t n,
                                                  int64_t vocab, int64_t width, int32_t* d_out, void* d_work,
                                                  int64_t work_bytes, void* stream) {
  const char* who = "gjx_random_linear_categorical_i32";
  static const int32_t some_y = 0;
  const int32_t rc = check_args(who, &some_y, d_x, x_ld, d_w, w_ld, dtype, n, vocab, width);
  if (rc != GJX_OK || n == 0) return rc;
  GJX_REQUIRE(key && d_out, GJX_EINVAL, "%s: null key or output", who);
  Forward f = {who, EPI_DRAW, nullptr, nullptr, nullptr, key[0], key[1], offset, d_out};
  return forward(f, dtype, d_x, x_ld, d_w, w_ld, d_bias, n, vocab, width, d_work, work_bytes, (hipStream_t)stream);
}

GJX_API int32_t gjx_linear_categorical_grad(int32_t dtype, const int32_t* d_y, const void* d_x, int64_t x_ld, const void* d_w,
                                            int64_t w_ld, const void* d_bias, int64_t n, int64_t vocab, int64_t width,
                                            const float* d_lse, const float* d_upstream, void* d_dx, void* d_dw, void* d_db,
                                            void* d_work, int64_t work_bytes, void* stream) {
  const char* who = "gjx_linear_categorical_grad";
  int32_t rc = check_args(who, d_y, d_x, x_ld, d_w, w_ld, dtype, n, vocab, width);
  if (rc != GJX_OK) return rc;
  GJX_REQUIRE(n >= 1, GJX_EINVAL, "%s: no rows (the gradients are zero; the caller fills them)", who);
  const bool f32 = dtype == GJX_F32;
  const Plan p = plan_of(dtype, n, vocab, width, f32 || !direct(d_x, x_ld, width), f32 || !direct(d_w, w_ld, width), true,
                         d_dx != nullptr);
  GJX_REQUIRE(d_lse && d_upstream, GJX_EINVAL, "%s: null input", who);
  GJX_REQUIRE(d_work && ((uintptr_t)d_work & 255) == 0 && work_bytes >= p.bytes, GJX_EINVAL,
              "%s: the workspace has %lld bytes, needs %lld aligned to 256", who, (long long)work_bytes, (long long)p.bytes);
  if (!d_dx && !d_dw && !d_db) return GJX_OK;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)d_work;
  Operand x = {(const bf16*)d_x, x_ld, 0, (int)n, (int)p.kp};
  if (p.pack_x) {
    if ((rc = pack(d_x, dtype, x_ld, n, width, p.kp, (bf16*)(ws + p.o_x), n * p.kp, s)) != GJX_OK) return rc;
    x = {(const bf16*)(ws + p.o_x), p.kp, n * p.kp, (int)n, (int)p.kp};
  }
  const Operand dl_rows = {(const bf16*)(ws + p.o_dl), p.piece, p.n_pad * p.piece, (int)p.n_pad, (int)p.piece};
  const int mk = (int)(up(width, BM) / BM);
  float* dx_part = (float*)(ws + p.o_dx);
  float* resid = (float*)(ws + p.o_resid);
  for (int64_t v0 = 0; v0 < vocab; v0 += p.piece) {
    const int64_t rows = std::min(p.piece, vocab - v0), rows_pad = up(rows, BM);
    Operand w = {(const bf16*)at_row(d_w, dtype, v0 * w_ld), w_ld, 0, (int)rows, (int)p.kp};
    if (p.pack_w) {
      if ((rc = pack(at_row(d_w, dtype, v0 * w_ld), dtype, w_ld, rows, width, p.kp, (bf16*)(ws + p.o_w), p.piece * p.kp, s)) != GJX_OK)
        return rc;
      w = {(const bf16*)(ws + p.o_w), p.kp, p.piece * p.kp, (int)rows, (int)p.kp};
    }
    GemmArgs a = {};                                         // logits of the piece -> dl
    a.pairs = p.pairs;
    a.splits = 1;
    a.a = w;
    a.b = x;
    a.ktiles = (int)(p.kp / BK);
    a.mt = (int)(rows_pad / BM);
    a.nt = (int)p.n_tiles;
    a.v0 = v0;
    a.vocab = vocab;
    a.n = n;
    a.n_pad = p.n_pad;
    a.bias = d_bias;
    a.bias_f32 = f32;
    a.y = d_y;
    a.lse = d_lse;
    a.g = d_upstream;
    a.dl = (bf16*)(ws + p.o_dl);
    a.resid = resid;
    a.dl_ld = p.piece;
    a.dl_plane = p.n_pad * p.piece;
    a.db_part = d_db ? (float*)(ws + p.o_db) : nullptr;
    rc = p.bn == 256 ? launch_gemm<256, false, false, EPI_DL>(a, s) : launch_gemm<64, false, false, EPI_DL>(a, s);
    if (rc != GJX_OK) return rc;
    if (d_db) {
      k_lincat_fold<<<gjx_grid_for(rows), GJX_BLOCK, 0, s>>>((const float*)(ws + p.o_db), (int)p.n_tiles, p.piece, 1, rows, rows,
                                                           f32 ? (void*)((float*)d_db + v0) : (void*)((bf16*)d_db + v0), !f32,
                                                           nullptr, nullptr, nullptr, 0, 0);
      GJX_LAUNCH_CHECK();
    }
    if (d_dx) {                                              // dx^T = W^T dl^T: m = feature, n = row, over the piece
      GemmArgs b = {};
      b.pairs = p.pairs;
      b.a = w;
      b.b = dl_rows;
      b.ktiles = (int)(rows_pad / BK);
      b.mt = mk;
      b.nt = (int)p.n_tiles;
      b.splits = p.splits;
      b.out = dx_part;
      b.out_ld = p.kp;
      b.out_split = n * p.kp;
      b.out_m = (int)p.kp;
      b.out_n = (int)n;
      b.accumulate = v0 > 0;
      rc = p.bn == 256 ? launch_gemm<256, true, false, EPI_STORE>(b, s) : launch_gemm<64, true, false, EPI_STORE>(b, s);
      if (rc != GJX_OK) return rc;
    }
    if (d_dw) {                                              // dW^T = x^T dl: m = feature, n = entry, over the rows
      GemmArgs b = {};
      b.pairs = p.pairs;
      b.a = x;
      b.b = dl_rows;
      b.ktiles = (int)(p.n_pad / BK);
      b.mt = mk;
      b.nt = (int)(rows_pad / BM);
      b.splits = 1;
      b.out = f32 ? (void*)((float*)d_dw + v0 * width) : (void*)((bf16*)d_dw + v0 * width);
      b.out_ld = width;
      b.out_m = (int)width;
      b.out_n = (int)rows;
      b.out_bf16 = !f32;
      b.resid_in = f32 ? nullptr : resid;
      b.y = d_y;
      b.n = n;
      b.v0 = v0;
      b.vocab = vocab;
      rc = launch_gemm<256, true, true, EPI_STORE>(b, s);
      if (rc != GJX_OK) return rc;
    }
  }
  if (d_dx) {
    k_lincat_fold<<<gjx_grid_for(n * width), GJX_BLOCK, 0, s>>>(dx_part, p.splits, n * p.kp, n, p.kp, width, d_dx, !f32,
                                                                    f32 ? nullptr : resid, d_y, (const bf16*)d_w, w_ld, vocab);
    GJX_LAUNCH_CHECK();
  }
  return GJX_OK;
}
