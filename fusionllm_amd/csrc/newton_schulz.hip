// newton_schulz.hip — orthogonalised updates of weight matrices by Newton-Schulz
// products, many matrices of one size at once, and the Muon step around them.
//
// For a matrix G (its smaller side first: m x n, m <= n, so a tall matrix is
// taken transposed):
//   X = G / max(|G|_F, eps);  steps times:  A = X X^T,  B = b A + c A^2,  X = a X + B X
// (an odd polynomial of G's singular values, with its singular vectors kept).
// Muon: u = momentum's combination of the gradient, p = p (1 - lr wd) - lr' X(u).
//
// Arithmetic.  The products run on v_mfma_f32_16x16x32_f16: fp16 carries 11 bits
// where bf16 carries 8 at the same rate, and the iterates' range is known: singular
// values of X stay below a bound that the host computes from the coefficients,
// so X, A and B are stored with the power-of-two factors below and neither
// overflow nor leave the normal range early.  Sums are fp32 throughout.
// A step is X = (a I + B) X: one product, whose rounded operand a I + B costs errors
// within the row space that X spans already.  A rounding of X would not: small
// singular values grow by a per step (some hundredfold over five steps), and so would
// what the rounding adds to them.  So X is kept as two numbers, hi (fp16, the
// operand) and lo = X - hi (fp8 e4m3), and a lo is added to the step's product in
// fp32 (not to the last one's, whose result grows no further).  Relative error of
// the result on gradients of full and low rank (768 x 2048, simulated in 64 bits):
// bf16 products 1e-2 .. 1.6e-1, fp16 without lo 1.2e-3 .. 4.9e-2, this form
// 6e-4 .. 1.9e-3 (half a step of a bf16 result: 3.9e-3).
// fp32 matrices take every operand as hi + lo, both fp16 (three products: hi lo, lo hi,
// hi hi; relative error 3e-6), and so do matrices of a small side up to kSplitSmall: their
// products cost little next to the launches, and a bf16 result is then as near as its
// own rounding allows (96 x 2048: 1.7e-3 off in 162 us against 2.0e-3 .. 2.4e-3 in 105).  Those of a small side up to 64 run in fp32 altogether, one launch per step,
// unless they are very long (below, ns_is_small).
//
// A and B are symmetric: only the tiles on and below the diagonal are computed
// and stored twice.  3 m^2 n + m^3 flops a step, bound by the matrix units; a
// few matrices are bound by the launches (3 per step and 2 before them).
#include <algorithm>
#include <cmath>

#include "../../include/fusiontrain.h"
#include "elements.h"
#include "fmoe_common.h"
#include "gemm_core.h"

namespace fmoe {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr int kNsCus = 256;         // CUs of the chip (a multiple of its 8 XCDs): workgroups of the persistent products
constexpr int kNsMax = FMOE_MUON_MAX_TENSORS;
constexpr int kNsPad = 64;          // both sides are padded (with zeros) to a multiple of this
constexpr int64_t kSplitSmall = 128;
constexpr int kNsParts = 64;        // partial sums of squares per matrix, at most (a wave adds them)
constexpr int kNormChunk = 8192;    // elements per partial sum, at least
// Stored values: X 2^14, A 2^13, a I + B 2^13 (singular values of X below 2.8, those of a I + B
// below 7.9), lo of X as fp8 2^4 more: |lo| <= 16 fills e4m3 to 256 of 448.
constexpr float kXScale = 16384.0f, kAScale = 8192.0f, kLoScale = 16.0f;
constexpr double kMaxSigma = 2.8, kMaxPoly = 7.9;

struct NsArgs {
  const void* src[kNsMax];  // matrix, or gradient
  void* buf[kNsMax];        // momentum (Muon)
  void* dst[kNsMax];        // result, or parameter (Muon)
  uint64_t tall;            // bit i: matrix i has more rows than columns
  int count, dtype, muon, nesterov;
  int m, n, mp, np;         // sides (m <= n) and padded sides
  int parts;                // partial sums per matrix
  float mom, om;            // momentum, 1 - momentum
  float decay;              // 1 - lr * weight_decay
  float lr_tall, lr_wide;   // step sizes with their size adjustment
  double eps;
  float ca, cb, cc;         // the polynomial's coefficients
  double* norm;             // [count][parts]
  // fp16: X [count][mp][np] twice (the step reads one and writes the other), A and B
  // [count][mp][mp].  Where operands are hi + lo, the rows are twice as long: 32 elements' hi, their lo,
  // the next 32 elements' hi, ... (ns_at), so that a K step of a product has both from one
  // 128-byte piece per row.  Elsewhere lo of X is fp8 (x8, null otherwise) and there once (each
  // tile reads and writes its own), and A and B have none.
  _Float16 *xh[2], *ah, *bh;
  uint8_t* x8;
  // small matrices: X [count][panels][64][128] fp32, partial Gram matrices [2][count][panels][10][256],
  // and the panels' exponents
  float *xs, *sparts;
  int* exps;
  int panels;
};

// Index in a row of element c's hi, and the distance of its lo, where a row holds both.
template <bool SPLIT>
__host__ __device__ __forceinline__ int ns_at(int c) {
  return SPLIT ? ((c >> 5) << 6) + (c & 31) : c;
}
constexpr int kLoAt = 32;

// lo of X as fp8 (times kLoScale), 8 elements: of values v and their hi; and back, still times kLoScale.
__device__ __forceinline__ uint2 pack_lo8(const float* v, const half8& h) {
  int d[2];
  float l[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) l[e] = fmaf(static_cast<float>(h[e]), -kLoScale, v[e] * kLoScale);  // exact
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    d[i] = __builtin_amdgcn_cvt_pk_fp8_f32(l[4 * i], l[4 * i + 1], 0, false);
    d[i] = __builtin_amdgcn_cvt_pk_fp8_f32(l[4 * i + 2], l[4 * i + 3], d[i], true);
  }
  return make_uint2(d[0], d[1]);
}
__device__ __forceinline__ void unpack_lo8(const uint2& u, float* l) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int d = static_cast<int>(i == 0 ? u.x : u.y);
    const f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8(d, false), q = __builtin_amdgcn_cvt_pk_f32_fp8(d, true);
    l[4 * i] = p[0], l[4 * i + 1] = p[1], l[4 * i + 2] = q[0], l[4 * i + 3] = q[1];
  }
}

// ---- the source: elements and the value that is orthogonalised ---------------------

// N (8, or fewer at an edge) consecutive elements from e on; the rest zero.
template <int DT>
__device__ __forceinline__ void ns_load8(const void* p, int64_t e, int n, float* v) {
  if (n >= 8) {
    unpack<DT, 8>(load_raw<DT, 8>(p, e), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = 0.0f;
      if (i < n) unpack<DT, 1>(load_raw<DT, 1>(p, e + i), v + i);
    }
  }
}
template <int DT>
__device__ __forceinline__ void ns_store8(void* p, int64_t e, int n, const float* v) {
  if (n >= 8) {
    store_chunk<DT, 8>(p, e, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store_chunk<DT, 1>(p, e + i, v + i);
  }
}

// Muon: the momentum after this step (fp32, not yet rounded to its type) and the update.
__device__ __forceinline__ float ns_momentum(const NsArgs& a, float g, float buf) { return fmaf(a.mom, buf, a.om * g); }
__device__ __forceinline__ float ns_update(const NsArgs& a, float g, float newbuf) {
  return a.nesterov ? fmaf(a.mom, newbuf, a.om * g) : newbuf;
}

// Sum of squares of each matrix in fp64 (no overflow of large values, no loss over
// millions of terms): one partial sum per workgroup, in a fixed order.
template <int DT, bool MUON>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsArgs a) {
  __shared__ double red[4];
  const int mat = blockIdx.y, part = blockIdx.x;
  const int64_t total = static_cast<int64_t>(a.m) * a.n;
  const void* g = a.src[mat];
  const void* b = a.buf[mat];
  double s = 0.0;
  for (int64_t e = (part * 256 + static_cast<int>(threadIdx.x)) * 8; e < total;
       e += static_cast<int64_t>(a.parts) * 256 * 8) {
    const int n = static_cast<int>(min(total - e, int64_t(8)));
    float u[8], v[8];
    ns_load8<DT>(g, e, n, u);
    if constexpr (MUON) {
      ns_load8<DT>(b, e, n, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = ns_update(a, u[i], ns_momentum(a, u[i], v[i]));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma(static_cast<double>(u[i]), static_cast<double>(u[i]), s);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) s = s + __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.norm[mat * a.parts + part] = ((red[0] + red[1]) + red[2]) + red[3];
}

// X = u / max(|u|, eps) as hi + lo, its smaller side first, zeros in the padding; Muon: the
// new momentum.  One 64 x 64 tile of X per workgroup, through LDS (tall matrices arrive transposed).
template <int DT, bool MUON>
__global__ __launch_bounds__(256) void ns_load_kernel(const NsArgs a) {
  __shared__ float tile[64][65];
  __shared__ double scale_s;
  const int mat = blockIdx.z;
  const bool tall = (a.tall >> mat) & 1;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;  // of X
  const int rows = tall ? a.n : a.m, cols = tall ? a.m : a.n;  // of the matrix as it lies
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  const int q = (threadIdx.x & 7) * 8;
  const void* g = a.src[mat];
  void* b = a.buf[mat];
  const int n = min(cols - (c0 + q), 8);
  float u[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = r0 + (threadIdx.x >> 3) + 32 * k;
    const int64_t e = static_cast<int64_t>(r) * cols + c0 + q;
    const int valid = r < rows ? n : 0;
    ns_load8<DT>(g, e, valid, u[k]);
    if constexpr (MUON) {
      float v[8];
      ns_load8<DT>(b, e, valid, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = ns_momentum(a, u[k][i], v[i]);
        u[k][i] = ns_update(a, u[k][i], v[i]);
      }
      ns_store8<DT>(b, e, valid, v);
    }
  }
  if (threadIdx.x < 64) {  // the partial sums, in a fixed order
    double ss = static_cast<int>(threadIdx.x) < a.parts ? a.norm[mat * a.parts + threadIdx.x] : 0.0;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) ss = ss + __shfl_xor(ss, off, 64);
    const double nrm = sqrt(ss);
    // the norm of a matrix that holds NaN or infinities is none, and its X is NaN; zeros stay zeros
    // (1 / eps need not be finite)
    if (threadIdx.x == 0) scale_s = ss == 0.0 ? 0.0 : static_cast<double>(kXScale) / (nrm < a.eps ? a.eps : nrm);
  }
  __syncthreads();
  const double scale = scale_s;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = (threadIdx.x >> 3) + 32 * k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = static_cast<float>(static_cast<double>(u[k][i]) * scale);
      if (tall) tile[q + i][r] = v;
      else tile[r][q + i] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int r = (threadIdx.x >> 3) + 32 * k;
    float v[8];
    half8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = tile[r][q + e];
      h[e] = static_cast<_Float16>(v[e]);
      l[e] = static_cast<_Float16>(v[e] - static_cast<float>(h[e]));
    }
    const int64_t row = static_cast<int64_t>(mat) * a.mp + i0 + r;
    if (a.x8) {
      const int64_t o = row * a.np + j0 + q;
      *reinterpret_cast<half8*>(a.xh[0] + o) = h;
      *reinterpret_cast<uint2*>(a.x8 + o) = pack_lo8(v, h);
    } else {
      const int64_t o = row * 2 * a.np + ns_at<true>(j0 + q);
      *reinterpret_cast<half8*>(a.xh[0] + o) = h;
      *reinterpret_cast<half8*>(a.xh[0] + o + kLoAt) = l;
    }
  }
}

// ---- the products ------------------------------------------------------------------------

enum NsMode { NS_GRAM = 0, NS_POLY = 1, NS_STEP = 2, NS_LAST = 3 };

// Tile (row, column) of a symmetric product's t-th tile on or below the diagonal, row major.
__device__ __forceinline__ void triangle(int t, int& i, int& j) {
  i = static_cast<int>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
  while (i * (i + 1) / 2 > t) --i;
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  j = t - i * (i + 1) / 2;
}

enum NsOut { NS_BF16 = 0, NS_F32 = 1, NS_MUON_BF16 = 2, NS_MUON_F32 = 3 };  // of the last product

__device__ __forceinline__ half8 ns_half8(const float* v) {
  half8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = static_cast<_Float16>(v[e]);
  return h;
}

// The last product's values, n (up to 8) consecutive elements of the matrix: its result, or the
// parameter's update (p: the parameter's elements, loaded before where all 8 are there).
template <int OUT>
__device__ __forceinline__ void ns_result8(const NsArgs& a, void* dst, int64_t o, int n, float* v, float lr,
                                           const Raw<OUT & 1, 8>& raw) {
  constexpr int DT = OUT & 1;
  if (n <= 0) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * (1.0f / kXScale);
  if constexpr (OUT >= NS_MUON_BF16) {
    float p[8];
    if (n >= 8) unpack<DT, 8>(raw, p);
    else ns_load8<DT>(dst, o, n, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf(-lr, v[e], p[e] * a.decay);
  }
  ns_store8<DT>(dst, o, n, v);
}

// Epilogue of a wave's block of 16 FM rows x 16 FN columns (FN a multiple of 4) at (row0, col0) of
// the padded result: acc[i][j] of lane l holds row 16 i + l % 16, columns 16 j + 4 (l / 16) + 0..3.
// Every global access is 16 bytes (lo of X: 8) of full lines: the block goes through
// the wave's 4 KB of LDS, 16 rows x 64 columns at a time, into registers as 8 consecutive
// elements of a row per lane, and for a transposed store (the mirrored tile of a symmetric product,
// the result of a tall matrix) once more, as fp16 hi and lo, with transposing reads that
// return 8 consecutive elements of a column.  What the epilogue reads is asked for first, so
// that its latency is not paid per slice.  (Epilogues straight from the accumulators, 8 bytes
// per lane in 16 rows at once, or with the reads slice by slice, took two thirds of a step:
// 27 matrices of 768 x 2048, 141 - 182 us against 53 for the product alone; now 92 .. 98, of which
// the stores are 32.)
//
// Pieces of 8 elements sit at a uniform address plus one offset per lane, and whether they are inside
// the padded result is uniform too (its sides, and a block's place, are multiples of 64, or of the
// block's 16 rows): the vector instructions are what an epilogue takes.
template <int MODE, bool SPLIT, int OUT, int FM, int FN>
__device__ __forceinline__ void ns_epilogue(const NsArgs& a, int cur, f32x4 (&acc)[FM][FN], uint8_t* ep, int lane,
                                               int mat, int row0, int col0, bool mirror) {
  constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
  constexpr bool LO8 = !SPLIT && MODE == NS_STEP;  // a lo, of fp8, is added
  constexpr int JH = FN / 4;                       // 64-column parts
  constexpr int SR = FM >= 2 ? 32 : 16;            // rows per transposed slice
  constexpr int W = SPLIT ? 2 : 1;                 // row length per element
  const int lim = SYM ? a.mp : a.np, ld = W * lim;
  const int64_t base = (static_cast<int64_t>(mat) * a.mp + row0) * ld + W * col0;
  const int lr = lane >> 3, lc = (lane & 7) * 8;
  const uint32_t voff = static_cast<uint32_t>(lr * ld + ns_at<SPLIT>(lc));
  const bool tall = MODE == NS_LAST && ((a.tall >> mat) & 1);
  void* const dst = MODE == NS_LAST ? a.dst[mat] : nullptr;
  static_assert(kNsPad % 64 == 0);
  if (row0 >= a.mp) return;
  // piece (i, jh, p) of this lane: row 16 i + 8 p + lr, columns 64 jh + lc .. + 7
  auto on = [&](int jh) { return col0 + 64 * jh < lim; };
  auto piece = [&](auto* array, int i, int jh, int p) {
    return array + (base + static_cast<int64_t>(16 * i + 8 * p) * ld + W * 64 * jh) + voff;
  };
  // A of this block (POLY; a part of it at a time, all would spill), lo of X (STEP)
  constexpr bool POLY = MODE == NS_POLY;
  constexpr int H = POLY ? (SPLIT ? 1 : (FM + 1) / 2) : FM;
  half8 ah[POLY ? H : 1][JH][2], al[POLY && SPLIT ? H : 1][JH][2];
  uint2 x8[LO8 ? FM : 1][JH][2];
  auto load_aux = [&](int i0) {
    if constexpr (POLY || LO8) {
#pragma unroll
      for (int i = 0; i < H; ++i)
#pragma unroll
        for (int jh = 0; jh < JH; ++jh)
#pragma unroll
          for (int p = 0; p < 2; ++p)
            if (i0 + i < FM && on(jh)) {
              if constexpr (POLY) ah[i][jh][p] = *reinterpret_cast<const half8*>(piece(a.ah, i0 + i, jh, p));
              if constexpr (POLY && SPLIT) al[i][jh][p] = *reinterpret_cast<const half8*>(piece(a.ah, i0 + i, jh, p) + kLoAt);
              if constexpr (LO8) x8[i][jh][p] = *reinterpret_cast<const uint2*>(piece(a.x8, i0 + i, jh, p));
            }
    }
  };
  load_aux(0);
  // accumulators -> 8 consecutive elements of a row (in the same registers); chunk c of row r at slot c ^ r
  auto at = [&](int r, int c) { return reinterpret_cast<f32x4*>(ep + r * 256 + ((c ^ r) & 15) * 16); };
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int jh = 0; jh < JH; ++jh) {
#pragma unroll
      for (int j = 0; j < 4; ++j) *at(lane & 15, 4 * j + (lane >> 4)) = acc[i][4 * jh + j];
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        acc[i][4 * jh + 2 * p] = *at(8 * p + lr, lc >> 2);
        acc[i][4 * jh + 2 * p + 1] = *at(8 * p + lr, (lc >> 2) + 1);
      }
      __builtin_amdgcn_wave_barrier();
    }
  auto value = [&](int i, int jh, int p, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[i][4 * jh + 2 * p][e], v[4 + e] = acc[i][4 * jh + 2 * p + 1][e];
    if constexpr (MODE == NS_GRAM) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * (kAScale / (kXScale * kXScale));
    } else if constexpr (MODE == NS_POLY) {  // a I + b A + c A^2
      const float c = a.cc * (1.0f / kAScale);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float x = static_cast<float>(ah[i % H][jh][p][e]);
        if constexpr (SPLIT) x = x + static_cast<float>(al[i % H][jh][p][e]);
        v[e] = fmaf(a.cb, x, c * v[e]);
      }
      if (!mirror) {  // the diagonal is in tiles that have no mirror
        const int d = row0 + 16 * i + 8 * p + lr - (col0 + 64 * jh + lc);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (d == e) v[e] = v[e] + a.ca * kAScale;
      }
    } else if constexpr (LO8) {
      float l[8];
      unpack_lo8(x8[i][jh][p], l);
      const float c = a.ca * (1.0f / kLoScale);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e], 1.0f / kAScale, c * l[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * (1.0f / kAScale);
    }
  };
  _Float16* const oh = MODE == NS_GRAM ? a.ah : MODE == NS_POLY ? a.bh : a.xh[1 - cur];
  const bool turn = SYM ? mirror : tall;
  constexpr bool TURN_LO = SPLIT || MODE == NS_LAST;  // the transposed values need their lo
  // hi and lo of the pieces, kept in the accumulators' registers for the transposed store
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    if (i > 0 && i % H == 0) load_aux(i);
    if constexpr (MODE == NS_LAST) {
      if (!tall) {
        Raw<OUT & 1, 8> raw[JH][2];
#pragma unroll
        for (int jh = 0; jh < JH; ++jh)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int r = row0 + 16 * i + 8 * p + lr, c = col0 + 64 * jh + lc;
            if (OUT >= NS_MUON_BF16 && r < a.m && c + 8 <= a.n)
              raw[jh][p] = load_raw<OUT & 1, 8>(dst, static_cast<int64_t>(r) * a.n + c);
          }
#pragma unroll
        for (int jh = 0; jh < JH; ++jh)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int r = row0 + 16 * i + 8 * p + lr, c = col0 + 64 * jh + lc;
            float v[8];
            value(i, jh, p, v);
            ns_result8<OUT>(a, dst, static_cast<int64_t>(r) * a.n + c, r < a.m ? min(a.n - c, 8) : 0, v, a.lr_wide,
                            raw[jh][p]);
          }
        continue;
      }
    }
#pragma unroll
    for (int jh = 0; jh < JH; ++jh)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float v[8];
        value(i, jh, p, v);
        const half8 h = ns_half8(v);
        half8 l;
        if constexpr (SPLIT || MODE == NS_LAST) {
#pragma unroll
          for (int e = 0; e < 8; ++e) l[e] = static_cast<_Float16>(v[e] - static_cast<float>(h[e]));
        }
        if constexpr (MODE != NS_LAST) {
          if (on(jh)) {
            *reinterpret_cast<half8*>(piece(oh, i, jh, p)) = h;
            if constexpr (SPLIT) *reinterpret_cast<half8*>(piece(oh, i, jh, p) + kLoAt) = l;
            else if constexpr (MODE == NS_STEP) *reinterpret_cast<uint2*>(piece(a.x8, i, jh, p)) = pack_lo8(v, h);
          }
        }
        if constexpr (MODE != NS_STEP) {
          acc[i][4 * jh + 2 * p] = __builtin_bit_cast(f32x4, h);
          if constexpr (TURN_LO) acc[i][4 * jh + 2 * p + 1] = __builtin_bit_cast(f32x4, l);
        }
      }
  }
  if constexpr (MODE != NS_STEP) {
    if (!turn) return;
    // SR rows x 64 columns of fp16: 32-byte window c of row r at window c ^ (r % 4), so that the four rows
    // of a transposing read fall into different banks; a group of 16 lanes takes 8 rows x 16 columns
    constexpr int RG = SR / 8, STEPS = RG;  // row groups; windows per group: 4 RG / 4
    const int g = lane >> 4, sj = (lane >> 2) & 3, sq = lane & 3;
    const int rg = g % RG, cw0 = g / RG;
    const uint32_t lds = core::lds_addr(ep);
    const int64_t tbase = (static_cast<int64_t>(mat) * a.mp + col0) * (W * a.mp);
    const uint32_t tvoff = static_cast<uint32_t>((16 * cw0 + (lane & 15)) * (W * a.mp) + 8 * rg);
#pragma unroll
    for (int i0 = 0; i0 < FM; i0 += SR / 16)
#pragma unroll
      for (int jh = 0; jh < JH; ++jh) {
        half8 t[TURN_LO ? 2 : 1][STEPS];
#pragma unroll
        for (int part = 0; part < (TURN_LO ? 2 : 1); ++part) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int i = 0; i < SR / 16; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              const int r = 16 * i + 8 * p + lr;
              *reinterpret_cast<f32x4*>(ep + r * 128 + ((((lane & 7) >> 1) ^ (r & 3)) << 5) + ((lane & 1) << 4)) =
                  acc[i0 + i][4 * jh + 2 * p + part];
            }
          __builtin_amdgcn_wave_barrier();
          asm volatile("" ::: "memory");
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            const int cw = cw0 + (4 / RG) * k;
            typedef __attribute__((address_space(3))) core::s16x4 lds_s16x4;
            const int r = 8 * rg + sj;
            const uint32_t x = lds + r * 128 + ((cw ^ (r & 3)) << 5) + 8 * sq;
            const core::s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)x);
            const core::s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(x + 512));
            t[part][k] = __builtin_bit_cast(half8, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
          }
          __builtin_amdgcn_wave_barrier();
          asm volatile("" ::: "memory");
        }
        Raw<OUT & 1, 8> raw[STEPS];
        const int row = row0 + 16 * i0 + 8 * rg;  // rows row .. + 7 of column col
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
          const int col = col0 + 64 * jh + 16 * (cw0 + (4 / RG) * k) + (lane & 15);
          if constexpr (SYM) {
            if (on(jh)) {
              // (the 8 rows of a group stay within 32 of a multiple of 32)
              const int64_t o = tbase + static_cast<int64_t>(64 * jh + 16 * (4 / RG) * k) * (W * a.mp) +
                                ns_at<SPLIT>(row0 + 16 * i0);
              *reinterpret_cast<half8*>(oh + o + tvoff) = t[0][k];
              if constexpr (SPLIT) *reinterpret_cast<half8*>(oh + o + tvoff + kLoAt) = t[TURN_LO ? 1 : 0][k];
            }
          } else if (OUT >= NS_MUON_BF16 && col < a.n && row + 8 <= a.m) {
            raw[k] = load_raw<OUT & 1, 8>(dst, static_cast<int64_t>(col) * a.m + row);
          }
        }
        if constexpr (MODE == NS_LAST) {
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            const int col = col0 + 64 * jh + 16 * (cw0 + (4 / RG) * k) + (lane & 15);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v[e] = static_cast<float>(t[0][k][e]) + static_cast<float>(t[TURN_LO ? 1 : 0][k][e]);
            ns_result8<OUT>(a, dst, static_cast<int64_t>(col) * a.m + row, col < a.n ? min(a.m - row, 8) : 0, v,
                            a.lr_tall, raw[k]);
          }
        }
      }
  }
}

// TM x TN outputs per workgroup of four waves, K in steps of 64 through NST LDS stages.
// A step multiplies the stage that is in registers while it reads the next one from LDS and the copies
// (global -> LDS, no registers) of the stage NST steps on go into the slot that has been read: one barrier
// a step, and no latency in its way.  (64-row tiles: three stages, Gram product of 3 of 768 x 2048
// 11.1 us against 16.8 with two; four were no faster.  128-row tiles: two, two workgroups per CU.)
// The row operand, and the column operand of the symmetric products, are K-contiguous;
// the step's column operand is X as it lies ([K, N]), read with transposing LDS reads
// (gemm_core.h has both layouts and their swizzles).  SPLIT: a stage is hi and lo of 32 k, and a step
// adds hi lo + lo hi + hi hi (three passes over K instead read each operand again: 3 matrices of 768 x
// 2048, Gram product 32 us against 21).
template <int MODE, int TM, int NST, bool SPLIT, int OUT = NS_BF16>
__global__ __launch_bounds__(256, 2) void ns_product_kernel(const NsArgs a, const int cur) {
  using namespace core;
  constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
  constexpr int TN = SYM ? TM : 128;
  // 2 x 2 waves; 4 x 1 for 64 x 64 tiles (a wave's columns: 64 for the epilogue)
  constexpr int WGN = TN / 64, WGM = 4 / WGN;
  constexpr int WTM = TM / WGM, WTN = 64, FM = WTM / 16, FN = 4;
  constexpr int A_ST = TM * RB, STAGE = A_ST + TN * RB;
  constexpr int CA = TM / 32, CB = TN / 32;  // copies per wave and stage
  __shared__ __attribute__((aligned(1024))) uint8_t smem[NST * STAGE];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / WGN, wn = w % WGN;
  const uint32_t sbase = lds_addr(smem);

  // Workgroup b runs on XCD b % 8: each takes a contiguous run of tiles.
  const int tm_n = (a.mp + TM - 1) / TM, tn_n = SYM ? tm_n : (a.np + TN - 1) / TN;
  const int per = SYM ? tm_n * (tm_n + 1) / 2 : tm_n * tn_n;
  const int total = per * a.count, run = (total + 7) / 8;
  const int item = (static_cast<int>(blockIdx.x) % 8) * run + static_cast<int>(blockIdx.x) / 8;
  if (static_cast<int>(blockIdx.x) / 8 >= run || item >= total) return;
  const int mat = __builtin_amdgcn_readfirstlane(item / per), t = item - mat * per;
  int ti, tj;
  if constexpr (SYM) triangle(t, ti, tj);
  else ti = t / tn_n, tj = t - ti * tn_n;
  ti = __builtin_amdgcn_readfirstlane(ti);
  tj = __builtin_amdgcn_readfirstlane(tj);

  constexpr int W = SPLIT ? 2 : 1;  // row length per element
  const int lda = W * (MODE == NS_GRAM ? a.np : a.mp), ldb = SYM ? lda : W * a.np;
  const int steps = lda / BK;
  const int64_t msq = static_cast<int64_t>(mat) * a.mp * W * a.mp, mx = static_cast<int64_t>(mat) * a.mp * W * a.np;
  const _Float16* p = MODE == NS_GRAM ? a.xh[cur] + mx : MODE == NS_POLY ? a.ah + msq : a.bh + msq;
  const _Float16* q = SYM ? p : a.xh[cur] + mx;

  // this lane's byte offsets from the operands' bases (rows and columns past the padded end: the last)
  uint32_t aoff[CA], boff[CB];
  const int chunk = ((lane & 7) ^ (lane >> 3)) * 8;
#pragma unroll
  for (int q = 0; q < CA; ++q)
    aoff[q] = static_cast<uint32_t>(min(ti * TM + 8 * (w + 4 * q) + (lane >> 3), a.mp - 1) * lda + chunk) * 2u;
#pragma unroll
  for (int q = 0; q < CB; ++q) {
    if constexpr (SYM) {
      boff[q] = static_cast<uint32_t>(min(tj * TN + 8 * (w + 4 * q) + (lane >> 3), a.mp - 1) * ldb + chunk) * 2u;
    } else {
      const int krow = 4 * (w + 4 * q) + (lane >> 4);  // SPLIT: rows 0 .. 31's hi, then their lo
      const int cb = ((((lane & 15) >> 1) ^ wsw(krow)) << 1) | (lane & 1);
      const int at = ns_at<SPLIT>(min(tj * TN + 8 * cb, a.np - 8));
      boff[q] = static_cast<uint32_t>((SPLIT ? krow % 32 : krow) * ldb + at + (SPLIT && krow >= 32 ? kLoAt : 0)) * 2u;
    }
  }
  const uint8_t *pa = reinterpret_cast<const uint8_t*>(p), *pb = reinterpret_cast<const uint8_t*>(q);
  const int64_t bstep = SYM ? RB : static_cast<int64_t>(BK / W) * ldb * 2;
  int left = steps;
  // the next stage's copies; past the last step the last stage again (into a slot that is free and
  // not read any more), so that every wait counts the same operations
  auto copy = [&](int st, int q) __attribute__((always_inline)) {
    const uint32_t la = sbase + st * STAGE + w * 1024;
    if (q < CA) copy16(la + q * 4096, pa, aoff[q < CA ? q : 0]);
    else copy16(la + A_ST + (q - CA) * 4096, pb, boff[q < CA ? 0 : q - CA]);
    if (q + 1 < CA + CB || --left <= 0) return;
    pa += RB;
    pb += bstep;
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t xa = frag_base(wm * WTM, lane);
  const uint32_t xb = A_ST + (SYM ? frag_base(wn * WTN, lane) : tr_base(4 * wn, lane));
  typedef __attribute__((address_space(3))) half8 lds_half8;
  struct Frags {
    half8 a[2][FM], b[2][FN];
  };
  auto read = [&](Frags& f, int slot) __attribute__((always_inline)) {
    const uint32_t src = sbase + slot * STAGE;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      // opaque, so that what is added to them goes into the reads' offsets
      uint32_t ra = src + (xa ^ (kh * 64u)), rb = src + (xb ^ (kh * 64u));
      asm volatile("" : "+v"(ra), "+v"(rb));
#pragma unroll
      for (int i = 0; i < FM; ++i) f.a[kh][i] = *(const lds_half8*)(uintptr_t)(ra + 2048u * i);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (SYM) f.b[kh][j] = *(const lds_half8*)(uintptr_t)(rb + 2048u * j);
        else f.b[kh][j] = __builtin_bit_cast(half8, tr_frag(((src + xb) ^ (j << 5)) + kh * TR_KHALF));
      }
    }
  };
#pragma unroll
  for (int st = 0; st < NST; ++st)
#pragma unroll
    for (int q = 0; q < CA + CB; ++q) copy(st, q);
  Frags f0, f1;
  wait_vm_barrier<(NST - 1) * (CA + CB)>();
  read(f0, 0);
  int slot = 0;
  // products between two copies, 0: all copies first.  (Update of 3 of 768 x 2048, hi + lo: 33 us with the
  // copies first, 30 so; fp16 alone, two thirds of the products: 22.7 and 22.6, its Gram product 19.8 and 21.5.)
  constexpr int EVERY = SPLIT && TM == 128 ? 4 : 0;
  auto step = [&](const Frags& now, Frags& next) __attribute__((always_inline)) {
    // the next stage is there, and every wave has this one in registers: its slot takes the stage NST on
    wait_vm_barrier<(NST - 2) * (CA + CB)>();
    const int free = slot;
    if constexpr (EVERY == 0) {
#pragma unroll
      for (int q = 0; q < CA + CB; ++q) copy(free, q);
    }
    slot = slot + 1 == NST ? 0 : slot + 1;
    read(next, slot);
    __builtin_amdgcn_s_setprio(1);
    // the halves of a stage: k 0 .. 31 and 32 .. 63, or hi and lo of 32 k
#pragma unroll
    for (int x = 0; x < (SPLIT ? 3 : 2); ++x)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int n = (x * FM + i) * FN + j;
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(now.b[SPLIT ? x == 0 : x][j], now.a[SPLIT ? x == 1 : x][i],
                                                             acc[i][j], 0, 0, 0);
          if constexpr (EVERY > 0) {
            if (n % EVERY == 0 && n / EVERY < CA + CB) {
              __builtin_amdgcn_sched_barrier(0);
              copy(free, n / EVERY);
              __builtin_amdgcn_sched_barrier(0);
            }
          }
        }
    __builtin_amdgcn_s_setprio(0);
  };
  // two steps without a branch between them (a branch lets the compiler move the first one's reads past
  // its products, to where they are used)
  for (int it = 0; it + 1 < steps; it += 2) {
    step(f0, f1);
    step(f1, f0);
  }
  if (steps & 1) step(f0, f1);
  wait_vm_barrier<0>();  // the copies past the end have landed: the epilogue takes their LDS
  ns_epilogue<MODE, SPLIT, OUT>(a, cur, acc, smem + w * EPI, lane, mat, ti * TM + wm * WTM, tj * TN + wn * WTN,
                                ti != tj);
}

// ---- the products in 256 x 256 tiles -------------------------------------------------------
// The main loop of gemm_core.h with fp16 operands: persistent workgroups of 8 waves (64 x 128 each)
// walk the tiles; the copies run as one ring over all K steps of all of a workgroup's tiles, so
// the next tile's first operands arrive during an epilogue.  A 256 x 256 tile reads half as
// much through L2 as four of 128 x 128, which is what bounds those.

#define FMOE_NS_MF(c, a, b) "v_mfma_f32_16x16x32_f16 " c ", " a ", " b ", " c "\n"
__device__ __forceinline__ void ns_mfma4(f32x4& c00, f32x4& c10, f32x4& c01, f32x4& c11, const bf16x8& p0,
                                         const bf16x8& p1, const bf16x8& q0, const bf16x8& q1) {
  asm volatile(FMOE_NS_MF("%[c00]", "%[p0]", "%[q0]") FMOE_NS_MF("%[c10]", "%[p0]", "%[q1]")
               FMOE_NS_MF("%[c01]", "%[p1]", "%[q0]") FMOE_NS_MF("%[c11]", "%[p1]", "%[q1]")
               : [c00] "+v"(c00), [c10] "+v"(c10), [c01] "+v"(c01), [c11] "+v"(c11)
               : [p0] "v"(p0), [p1] "v"(p1), [q0] "v"(q0), [q1] "v"(q1)
               : "memory");
}
#undef FMOE_NS_MF

// Quarter (I, J) of the wave's block (core::quarter with fp16 operands).
template <int I, int J, bool SPLIT>
__device__ __forceinline__ void ns_quarter(f32x4 (&acc)[core::FM][core::FN], const core::AFrag& a,
                                           const core::BFrag& b) {
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int x = 0; x < (SPLIT ? 6 : 4); ++x) {
    const int h = x >> 1, n = (x & 1) * 2;
    const int ka = SPLIT ? h == 1 : h, kb = SPLIT ? h == 0 : h;  // hi lo, lo hi, hi hi
    ns_mfma4(acc[2 * I][4 * J + n], acc[2 * I + 1][4 * J + n], acc[2 * I][4 * J + n + 1],
             acc[2 * I + 1][4 * J + n + 1], b[kb][n], b[kb][n + 1], a[ka][0], a[ka][1]);
  }
  __builtin_amdgcn_s_setprio(0);
  core::barrier();
}

struct NsTile {
  int mat, ti, tj;
};

template <int MODE, bool SPLIT, int OUT = NS_BF16>
__global__ __launch_bounds__(core::NT, 1) void ns_big_kernel(const NsArgs a, const int cur) {
  using namespace core;
  constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[SMEM];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / WN, wn = w % WN;
  const uint32_t sbase = lds_addr(smem);
  const int tiles_m = (a.mp + BM - 1) / BM, tiles_n = SYM ? tiles_m : (a.np + BN - 1) / BN;
  const int per = SYM ? tiles_m * (tiles_m + 1) / 2 : tiles_m * tiles_n;
  const int items = per * a.count;
  // Workgroup b runs on XCD b % 8.  Each XCD takes an eighth of the tiles, a contiguous run (few
  // matrices per L2), and its workgroups take them in turn: every XCD writes as much in every
  // round.  (With runs per round the tiles of a last, partial round fell on few XCDs.)
  const int xcd = static_cast<int>(blockIdx.x) % 8, step = static_cast<int>(gridDim.x) / 8;
  const int first = static_cast<int>(static_cast<int64_t>(items) * xcd / 8) + static_cast<int>(blockIdx.x) / 8;
  const int end = static_cast<int>(static_cast<int64_t>(items) * (xcd + 1) / 8);
  const int my_items = (end - first + step - 1) / step;
  if (my_items <= 0) return;
  constexpr int W = SPLIT ? 2 : 1;  // row length per element
  const int ld = W * (MODE == NS_GRAM ? a.np : a.mp), ldb = SYM ? ld : W * a.np;
  const int steps = ld / BK;
  const int total = my_items * steps;

  auto locate = [&](int item) __attribute__((always_inline)) {
    NsTile t;
    t.mat = item / per;
    const int q = item - t.mat * per;
    if constexpr (SYM) triangle(q, t.ti, t.tj);
    else t.ti = q / tiles_n, t.tj = q - t.ti * tiles_n;
    t.mat = __builtin_amdgcn_readfirstlane(t.mat);
    t.ti = __builtin_amdgcn_readfirstlane(t.ti);
    t.tj = __builtin_amdgcn_readfirstlane(t.tj);
    return t;
  };

  // ---- copy cursor (the units of a stage and their LDS layout as in gemm_core.h)
  const uint32_t lds_a = sbase + (64 * (w >> 2) + 8 * (w & 3)) * RB;
  const uint32_t lds_b = sbase + A_BYTES + w * 1024;
  int c_ti = 0, c_kt = 0;
  const uint8_t *c_a = nullptr, *c_b = nullptr;
  uint32_t a_off[4], b_off[4];
  const int64_t bstep = SYM ? RB : static_cast<int64_t>(BK / W) * ldb * 2;
  auto copy_tile = [&](int ti) __attribute__((always_inline)) {
    const NsTile t = locate(first + ti * step);
    const int64_t msq = static_cast<int64_t>(t.mat) * a.mp * W * a.mp, mx = static_cast<int64_t>(t.mat) * a.mp * W * a.np;
    const _Float16* p = MODE == NS_GRAM ? a.xh[cur] + mx : MODE == NS_POLY ? a.ah + msq : a.bh + msq;
    const _Float16* q = SYM ? p : a.xh[cur] + mx;
    c_a = reinterpret_cast<const uint8_t*>(p + static_cast<int64_t>(t.ti) * BM * ld);
    c_b = reinterpret_cast<const uint8_t*>(SYM ? q + static_cast<int64_t>(t.tj) * BN * ld : q);
    // the lane as an opaque value: what follows is formed here, not kept through the main loop
    int l = lane;
    asm volatile("" : "+v"(l));
    const int dchunk = (l & 7) ^ swzk(l >> 3);
    const int last_m = min(a.mp - t.ti * BM, BM) - 1, last_n = min(a.mp - t.tj * BN, BN) - 1;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = min(64 * (w >> 2) + 8 * (w & 3) + (l >> 3) + 128 * (q & 1) + 32 * (q >> 1), last_m);
      a_off[q] = static_cast<uint32_t>(r * ld + dchunk * 8) * 2u;
      if constexpr (SYM) {
        const int n = min(128 * (q & 1) + 64 * (q >> 1) + 8 * w + (l >> 3), last_n);
        b_off[q] = static_cast<uint32_t>(n * ldb + dchunk * 8) * 2u;
      } else {
        const int krow = 4 * w + (l >> 4);
        const int cb = ((((l & 15) >> 1) ^ wsw(krow)) << 1) | (l & 1);
        const int col = 128 * (cb >> 3) + 8 * (cb & 7) + 64 * (q >> 1);
        const int at = ns_at<SPLIT>(min(t.tj * BN + col, a.np - 8));
        // SPLIT: the second 32 rows of a stage are the first ones' lo
        b_off[q] = static_cast<uint32_t>((SPLIT ? krow : 32 * (q & 1) + krow) * ldb + at + (SPLIT && (q & 1) ? kLoAt : 0)) * 2u;
      }
    }
  };
  copy_tile(0);
  // A stage's units are issued in the order A0, B0, B1, A1; A1 moves the cursor on.  Past the last
  // step the last stage is copied again (into slots that are free and not read any more).
  auto issue_a = [&](int it, int u) __attribute__((always_inline)) {
    const uint32_t st = lds_a + (it & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < 2; ++i) copy16(st + (128 * i + 32 * u) * RB, c_a, a_off[2 * u + i]);
    if (u == 0) return;
    c_a += RB;
    c_b += bstep;
    if (__builtin_expect(++c_kt == steps, 0)) {
      if (c_ti + 1 < my_items) {
        c_kt = 0;
        copy_tile(++c_ti);
      } else {
        --c_kt;
        c_a -= RB;
        c_b -= bstep;
      }
    }
  };
  auto issue_b = [&](int it, int u) __attribute__((always_inline)) {
    const uint32_t st = lds_b + (it & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      copy16(SYM ? st + (128 * i + 64 * u) * RB : st + u * UNIT + i * 8192, c_b, b_off[2 * u + i]);
  };

  uint32_t xa = frag_base(wm * WTM, lane);
  uint32_t xb = A_BYTES + (SYM ? frag_base(wn * WTN, lane) : tr_base(4 * wn, lane));
  AFrag a0, a1;
  BFrag b0, b1;
  typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
  auto lds_frag = [&](uint32_t x, uint32_t src, int kh, int f) {
    return *(const lds_bf16x8*)(uintptr_t)((x ^ (kh * 64u)) + src + 2048u * f);
  };
  auto read_a = [&](AFrag& f, int u, uint32_t src, int kh, int m) { f[kh][m] = lds_frag(xa, src, kh, 2 * u + m); };
  auto read_b = [&](BFrag& f, int u, uint32_t src, int kh, int n) {
    if constexpr (SYM) f[kh][n] = lds_frag(xb, src, kh, 4 * u + n);
    else f[kh][n] = tr_frag(((src + xb) ^ (n << 5)) + u * UNIT + kh * TR_KHALF);
  };
  auto read_first = [&](uint32_t src) {
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int m = 0; m < 2; ++m) read_a(a0, 0, src, kh, m);
#pragma unroll
    for (int n = 0; n < 4; ++n) read_b(b0, 0, src, 0, n);
  };

  issue_a(0, 0);
  issue_b(0, 0);
  issue_b(0, 1);
  issue_a(0, 1);
  issue_a(1, 0);
  issue_b(1, 0);
  issue_b(1, 1);
  wait_vm_barrier<5 * LU>();
  read_first(sbase);
  const bool late = w >= 4;  // this wave's SIMD partner is one phase ahead
  if (late) barrier();

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  uint8_t* ep = smem + 2 * STAGE + w * EPI;  // this wave's staging (4 KB)
  int e_ti = 0, e_kt = 0;
  for (int it = 0; it < total; ++it) {
    // keep the per-step fragment addresses from being hoisted out of the loop
    asm volatile("" : "+v"(xa), "+v"(xb));
    const uint32_t st = sbase + (it & 1) * STAGE, nxt = sbase + ((it + 1) & 1) * STAGE;
    // (0, 0)
#pragma unroll
    for (int n = 0; n < 4; ++n) read_b(b0, 0, st, 1, n);
    issue_a(it + 1, 1);
    wait_vm_barrier<5 * LU>();  // B1 of this stage
    ns_quarter<0, 0, SPLIT>(acc, a0, b0);
    // (0, 1)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int n = 0; n < 4; ++n) read_b(b1, 1, st, kh, n);
    issue_a(it + 2, 0);
    wait_vm_barrier<5 * LU>();  // A1 of this stage
    ns_quarter<0, 1, SPLIT>(acc, a0, b1);
    // (1, 0)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int m = 0; m < 2; ++m) read_a(a1, 1, st, kh, m);
    issue_b(it + 2, 0);
    wait_vm_barrier<4 * LU>();  // A0, B0 of the next stage
    ns_quarter<1, 0, SPLIT>(acc, a1, b0);
    // (1, 1): the next step's first fragments (at a tile's end they are read again after its epilogue)
    read_first(nxt);
    issue_b(it + 2, 1);
    wait_lds_barrier();
    ns_quarter<1, 1, SPLIT>(acc, a1, b1);

    if (++e_kt < steps) continue;
    // ---- tile epilogue: this wave's 64 x 128 block (both wave groups together)
    if (!late) barrier();
    e_kt = 0;
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3\n" ::: "memory");  // MFMA results -> VALU reads
    int el = lane;
    asm volatile("" : "+v"(el));  // the address arithmetic below stays out of the main loop
    {
      const NsTile t = locate(first + e_ti * step);
      ns_epilogue<MODE, SPLIT, OUT>(a, cur, acc, ep, el, t.mat, t.ti * BM + wm * WTM, t.tj * BN + wn * WTN,
                                    t.ti != t.tj);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    asm volatile("s_nop 1" ::: "memory");  // VALU writes -> MFMA reads of the accumulators
    ++e_ti;
    // the next tile's first fragments (after the last tile a harmless re-read)
    read_first(sbase + ((it + 1) & 1) * STAGE);
    if (late && it + 1 < total) barrier();
  }
  // the copies past the end have landed before the workgroup's LDS is given back
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- matrices of a small side up to 64 ---------------------------------------------------------
// (router weights): one launch per step instead of three, fp32 operands on
// v_mfma_f32_16x16x4_f32 (rounding fp32 to fp32 only; the products are small next to the latency of
// a launch).  A workgroup has 128 columns of X.  It adds the workgroups' partial Gram
// matrices of the launch before (in a fixed order), forms a I + b A + c A^2 for itself, multiplies
// its columns and writes the partial Gram matrix of the result for the next launch.  Five steps, bf16,
// against three launches a step (most of them the Gram matrix's one tile), in a graph: 64 x 2048 64 us
// against 145, 8 of 32 x 2048 72 against 147, 27 of 64 x 768 72 against 105.  Where many long ones go
// together every workgroup's sum over the partial matrices counts: 64 of 64 x 2048 235 us
// against 215, 64 of 64 x 4096 529 against 359.  The rule leaves their number out all the same, so that a
// matrix's result is the same whatever goes with it.

constexpr int kSmallSide = 64;        // the small side, at most (and the padded one)
constexpr int kSmallPanel = 128;      // columns per workgroup
constexpr int kSmallMaxPanels = 32;   // every workgroup adds the partial matrices of all (64 x 4096: 76 us
                                      // against 228)
constexpr int kSmallBlocks = 10;      // 16 x 16 blocks of a Gram matrix on or below the diagonal
// Waves per workgroup, by the 16-row blocks of X: 8 (64 x 2048 64 us, 27 of 64 x 768 72; four waves 72 and 86), 4
// for one block, which leaves the others little (64 of 16 x 4096 152 us, with eight 184).
constexpr int small_waves(int mb) { return mb > 1 ? 8 : 4; }
constexpr int kLdA = 68, kLdX = 132;  // LDS strides

struct SmallLds {
  float a[kSmallSide * kLdA], b[kSmallSide * kLdA], x[kSmallSide * kLdX];
  double red[8];
  int e;
};

__device__ __forceinline__ f32x4 mfma_f32(float p, float q, f32x4 c) {
  // D[4 (l / 16) + 0..3][l % 16] += A[l % 16][l / 16] B[l / 16][l % 16] over the lanes l
  return __builtin_amdgcn_mfma_f32_16x16x4f32(p, q, c, 0, 0, 0);
}
// Block (row, column) of the t-th block on or below the diagonal.
__device__ __forceinline__ void small_block(int t, int& i, int& j) {
  i = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
  j = t - i * (i + 1) / 2;
}

// Partial Gram matrix of the panel in LDS: blocks w, w + 8 by wave w (of eight).  MB: 16-row blocks of X.
template <int MB>
__device__ __forceinline__ void small_gram(const NsArgs& a, const SmallLds& s, int mat, int panel, int parity) {
  constexpr int BLOCKS = MB * (MB + 1) / 2, NW = small_waves(MB), PER = (BLOCKS + NW - 1) / NW;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int cols = min(a.n - panel * kSmallPanel, kSmallPanel);  // zeros after them
  float* out = a.sparts + ((static_cast<int64_t>(parity) * a.count + mat) * a.panels + panel) * (kSmallBlocks * 256);
  const float *p[PER], *q[PER];
  f32x4 c[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    int i, j;
    small_block(min(w + NW * u, BLOCKS - 1), i, j);
    p[u] = s.x + (16 * i + (lane & 15)) * kLdX + (lane >> 4);
    q[u] = s.x + (16 * j + (lane & 15)) * kLdX + (lane >> 4);
    c[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int k0 = 0; k0 < cols; k0 += 32)
#pragma unroll
    for (int k = 0; k < 32; k += 4)
#pragma unroll
      for (int u = 0; u < PER; ++u) c[u] = mfma_f32(p[u][k0 + k], q[u][k0 + k], c[u]);
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (w + NW * u < BLOCKS) *reinterpret_cast<f32x4*>(out + (w + NW * u) * 256 + lane * 4) = c[u];
}

// A thread's share (one of NT) of the panel's elements as they lie in the matrix: chunk t of 8 (t < COUNT).
template <int NT>
struct SmallChunk {
  static constexpr int COUNT = kSmallSide * kSmallPanel / 8 / NT;
  int64_t o;       // offset in the matrix
  int n, r, c;     // valid elements; row and column of X of the first
  bool down;       // the 8 go down a column of X
  __device__ __forceinline__ SmallChunk(const NsArgs& a, int mat, int panel, int t) {
    const int c0 = panel * kSmallPanel, id = t * NT + threadIdx.x;
    down = (a.tall >> mat) & 1;
    if (down) {
      const int per = (a.m + 7) / 8;
      c = id / per;
      r = (id - c * per) * 8;
      n = c < kSmallPanel && c0 + c < a.n ? min(a.m - r, 8) : 0;
      o = static_cast<int64_t>(c0 + c) * a.m + r;
    } else {
      r = id / (kSmallPanel / 8);
      c = (id % (kSmallPanel / 8)) * 8;
      n = r < a.m ? min(a.n - (c0 + c), 8) : 0;
      o = static_cast<int64_t>(r) * a.n + c0 + c;
    }
  }
  __device__ __forceinline__ int lds(int i) const { return down ? (r + i) * kLdX + c : r * kLdX + c + i; }
};

// X of the panel, still without the norm (times a power of two that brings the panel's
// norm to 1/2 .. 1), its sum of squares in fp64 and its partial Gram matrix; Muon: the new momentum.
template <int DT, bool MUON, int MB>
__global__ __launch_bounds__(64 * small_waves(MB), 2) void ns_small_load_kernel(const NsArgs a) {
  constexpr int NW = small_waves(MB), NT = 64 * NW;
  __shared__ SmallLds s;
  const int panel = blockIdx.x, mat = blockIdx.y;
  float u[SmallChunk<NT>::COUNT][8], v[MUON ? SmallChunk<NT>::COUNT : 1][8];
#pragma unroll
  for (int t = 0; t < SmallChunk<NT>::COUNT; ++t) {
    const SmallChunk<NT> k(a, mat, panel, t);
    ns_load8<DT>(a.src[mat], k.o, k.n, u[t]);
    if constexpr (MUON) ns_load8<DT>(a.buf[mat], k.o, k.n, v[t]);
  }
  for (int t = threadIdx.x; t < kSmallSide * kLdX; t += NT) s.x[t] = 0.0f;
  double ss = 0.0;
#pragma unroll
  for (int t = 0; t < SmallChunk<NT>::COUNT; ++t) {
    const SmallChunk<NT> k(a, mat, panel, t);
    if constexpr (MUON) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[t][i] = ns_momentum(a, u[t][i], v[t][i]);
        u[t][i] = ns_update(a, u[t][i], v[t][i]);
      }
      if (k.n > 0) ns_store8<DT>(a.buf[mat], k.o, k.n, v[t]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < k.n) ss = fma(static_cast<double>(u[t][i]), static_cast<double>(u[t][i]), ss);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) ss = ss + __shfl_xor(ss, off, 64);
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = ss;
  __syncthreads();
  ss = s.red[0];
  for (int i = 1; i < NW; ++i) ss = ss + s.red[i];
  int e = 0;
  if (ss > 0.0 && ss < 1e300) {
    frexp(sqrt(ss), &e);
    e = max(-126, min(e, 126));  // 2^-e a normal fp32 number (a panel beyond that stays within 2^15 of 1)
  }
  if (threadIdx.x == 0) {
    a.norm[mat * a.panels + panel] = ss;
    a.exps[mat * a.panels + panel] = e;
  }
  const float f = fm_pow2i(-e);
#pragma unroll
  for (int t = 0; t < SmallChunk<NT>::COUNT; ++t) {
    const SmallChunk<NT> k(a, mat, panel, t);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < k.n) s.x[k.lds(i)] = u[t][i] * f;
  }
  __syncthreads();
  float* x = a.xs + (static_cast<int64_t>(mat) * a.panels + panel) * (kSmallSide * kSmallPanel);
#pragma unroll 4
  for (int t = threadIdx.x; t < 16 * MB * kSmallPanel; t += NT) x[t] = s.x[(t / kSmallPanel) * kLdX + t % kSmallPanel];
  small_gram<MB>(a, s, mat, panel, 0);
}

// One step of a panel (step k reads the partial matrices of parity k % 2 and writes the others).
template <bool LAST, int OUT, int MB>
__global__ __launch_bounds__(64 * small_waves(MB), small_waves(MB) / 2) void ns_small_step_kernel(const NsArgs a, const int k) {
  constexpr int BLOCKS = MB * (MB + 1) / 2, NW = small_waves(MB), NT = 64 * NW, PER = (BLOCKS + NW - 1) / NW;
  constexpr int XV = 16 * MB * kSmallPanel / NT;
  constexpr int BATCH = 8;  // partial matrices in flight (sixteen take the registers of a second workgroup: 64 of 64 x 2048
                            // 295 us against 235)
  __shared__ SmallLds s;
  const int panel = blockIdx.x, mat = blockIdx.y;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float* x = a.xs + (static_cast<int64_t>(mat) * a.panels + panel) * (kSmallSide * kSmallPanel);
  float xv[XV];
#pragma unroll
  for (int t = 0; t < XV; ++t) xv[t] = x[t * NT + threadIdx.x];
  // the first step's X and A still lack the norm: panel p's X the factor 2^e / |u| (lane p has it)
  float mine = 1.0f;
  if (k == 0) {
    const double own = lane < a.panels ? a.norm[mat * a.panels + lane] : 0.0;
    double ss = own;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) ss = ss + __shfl_xor(ss, off, 64);
    const double nrm = sqrt(ss);
    // (a panel of zeros, whose exponent is 0, stays zero: 1 / |u| may be beyond fp32)
    mine = own == 0.0 ? 0.0f
                      : static_cast<float>(ldexp(1.0 / (nrm < a.eps ? a.eps : nrm), a.exps[mat * a.panels + lane]));
  }
  // A: blocks w, w + NW by wave w, the panels in order
  const float* parts = a.sparts + (static_cast<int64_t>(k & 1) * a.count + mat) * a.panels * (kSmallBlocks * 256);
  f32x4 sum[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) sum[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < a.panels; p0 += BATCH) {
    f32x4 v[PER][BATCH];
#pragma unroll
    for (int p = 0; p < BATCH; ++p)
#pragma unroll
      for (int u = 0; u < PER; ++u)
        v[u][p] = *reinterpret_cast<const f32x4*>(parts + min(p0 + p, a.panels - 1) * (kSmallBlocks * 256) +
                                                  min(w + NW * u, BLOCKS - 1) * 256 + lane * 4);
    __builtin_amdgcn_sched_barrier(0);  // all of them in flight
#pragma unroll
    for (int p = 0; p < BATCH; ++p) {
      // a panel past the last adds nothing (its load repeats the last one's)
      const float g = __shfl(mine, (p0 + p) & 63, 64), f = p0 + p < a.panels ? g : 0.0f;
#pragma unroll
      for (int u = 0; u < PER; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[u][e] = sum[u][e] + (v[u][p][e] * f) * f;
    }
  }
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (w + NW * u < BLOCKS) {
      int i, j;
      small_block(w + NW * u, i, j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * i + 4 * (lane >> 4) + e, q = 16 * j + (lane & 15);
        s.a[r * kLdA + q] = sum[u][e];
        s.a[q * kLdA + r] = sum[u][e];  // (a diagonal block writes the same values twice)
      }
    }
  const float f = __shfl(mine, panel, 64);
#pragma unroll
  for (int t = 0; t < XV; ++t) {
    const int q = t * NT + threadIdx.x;
    s.x[(q / kSmallPanel) * kLdX + q % kSmallPanel] = xv[t] * f;
  }
  __syncthreads();
  // B = a I + b A + c A^2: two waves for 16 rows
  constexpr int JB = MB > 1 ? MB / 2 : 1;
  const int bi = w >> 1, bj = (w & 1) * JB;
  if (bi < MB && bj < MB) {
    f32x4 c[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) c[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* p = s.a + (lane & 15) * kLdA + (lane >> 4);  // (A is symmetric)
#pragma unroll
    for (int q = 0; q < 16 * MB; q += 4)
#pragma unroll
      for (int j = 0; j < JB; ++j) c[j] = mfma_f32(p[16 * bi * kLdA + q], p[16 * (bj + j) * kLdA + q], c[j]);
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 16 * bi + 4 * (lane >> 4) + e, q = 16 * (bj + j) + (lane & 15);
        const float v = fmaf(a.cb, s.a[r * kLdA + q], a.cc * c[j][e]);
        s.b[r * kLdA + q] = r == q ? v + a.ca : v;
      }
  }
  __syncthreads();
  // X = B X: a column block or two by each wave (in place after the last read of its own columns)
  {
    constexpr int JX = kSmallPanel / 16 / NW;
    f32x4 c[MB][JX];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < JX; ++j) c[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* p = s.b + (lane & 15) * kLdA + (lane >> 4);
    const float* y = s.x + (lane >> 4) * kLdX + 16 * JX * w + (lane & 15);
#pragma unroll
    for (int q = 0; q < 16 * MB; q += 4)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < JX; ++j) c[i][j] = mfma_f32(p[16 * i * kLdA + q], y[q * kLdX + 16 * j], c[i][j]);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < JX; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s.x[(16 * i + 4 * (lane >> 4) + e) * kLdX + 16 * (JX * w + j) + (lane & 15)] = c[i][j][e];
  }
  __syncthreads();
  if constexpr (LAST) {
    constexpr int DT = OUT & 1;
    constexpr bool MUON = OUT >= NS_MUON_BF16;
    float p[MUON ? SmallChunk<NT>::COUNT : 1][8];
    if constexpr (MUON)
#pragma unroll
      for (int t = 0; t < SmallChunk<NT>::COUNT; ++t) {
        const SmallChunk<NT> q(a, mat, panel, t);
        ns_load8<DT>(a.dst[mat], q.o, q.n, p[t]);
      }
#pragma unroll
    for (int t = 0; t < SmallChunk<NT>::COUNT; ++t) {
      const SmallChunk<NT> q(a, mat, panel, t);
      if (q.n <= 0) continue;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = i < q.n ? s.x[q.lds(i)] : 0.0f;
        if constexpr (MUON) v[i] = fmaf(q.down ? -a.lr_tall : -a.lr_wide, v[i], p[t][i] * a.decay);
      }
      ns_store8<DT>(a.dst[mat], q.o, q.n, v);
    }
  } else {
#pragma unroll 4
    for (int t = 0; t < XV; ++t) {
      const int q = t * NT + threadIdx.x;
      x[q] = s.x[(q / kSmallPanel) * kLdX + q % kSmallPanel];
    }
    small_gram<MB>(a, s, mat, panel, (k + 1) & 1);
  }
}

inline int ns_panels(int64_t n) { return static_cast<int>(ceil_div(n, kSmallPanel)); }
inline bool ns_is_small(int64_t m, int64_t n) { return m <= kSmallSide && ns_panels(n) <= kSmallMaxPanels; }

// ---- host -----------------------------------------------------------------------------------

inline int64_t ns_pad(int64_t v) { return ceil_div(v, kNsPad) * kNsPad; }
inline bool ns_split(int64_t m, int dtype) { return dtype == FMOE_F32 || m <= kSplitSmall; }

struct NsLayout {
  size_t norm, x, sq, total;  // bytes of the partial sums, of one X, of one A
  int parts;
};
inline NsLayout ns_layout(int64_t m, int64_t n, int count, bool split) {
  NsLayout l;
  l.parts = static_cast<int>(std::min<int64_t>(kNsParts, ceil_div(m * n, kNormChunk)));
  l.norm = (static_cast<size_t>(count) * l.parts * sizeof(double) + 255) / 256 * 256;
  l.x = static_cast<size_t>(count) * ns_pad(m) * ns_pad(n) * 2;
  l.sq = static_cast<size_t>(count) * ns_pad(m) * ns_pad(m) * 2;
  // X twice; lo of each where operands are hi + lo, else once and half as wide
  l.total = l.norm + 2 * l.x + (split ? 2 * l.x : l.x / 2) + (split ? 4 : 2) * l.sq;
  return l;
}

// Whether the iterates stay within the stored range: the largest singular value after each
// step, from the polynomial's extrema over [0, s], and the largest |a + b t + c t^2| over t <= s^2.
inline bool ns_bounded(double a, double b, double c, int steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double s = 1.0 + 1e-6;
  for (int k = 0; k < steps; ++k) {
    if (!(s < kMaxSigma)) return false;
    const double t1 = s * s;
    double poly = std::max(std::fabs(a), std::fabs(a + b * t1 + c * t1 * t1));
    if (c != 0.0) {
      const double t = -b / (2.0 * c);
      if (t > 0.0 && t < t1) poly = std::max(poly, std::fabs(a + b * t + c * t * t));
    }
    if (!(poly < kMaxPoly)) return false;
    auto p = [&](double v) { return std::fabs(v * (a + v * v * (b + c * v * v))); };
    double next = p(s);
    // extrema: 5 c t^2 + 3 b t + a = 0, t = v^2
    double roots[2];
    int n = 0;
    if (c != 0.0) {
      const double d = 9.0 * b * b - 20.0 * a * c;
      if (d >= 0.0) {
        roots[n++] = (-3.0 * b + std::sqrt(d)) / (10.0 * c);
        roots[n++] = (-3.0 * b - std::sqrt(d)) / (10.0 * c);
      }
    } else if (b != 0.0) {
      roots[n++] = -a / (3.0 * b);
    }
    for (int i = 0; i < n; ++i)
      if (roots[i] > 0.0 && roots[i] < t1) next = std::max(next, p(std::sqrt(roots[i])));
    s = next * (1.0 + 1e-3);  // room for the roundings
  }
  return s < kMaxSigma;
}

// Output tiles of a product of `count` matrices: their number for tiles of tm x tn.
inline int64_t ns_tiles(bool sym, int64_t mp, int64_t np, int count, int tm, int tn) {
  const int64_t r = ceil_div(mp, tm);
  return (sym ? r * (r + 1) / 2 : r * ceil_div(np, tn)) * count;
}
// Rows of the output tiles.  256 x 256 tiles, persistent, where they fill the chip and pad little (their area is at most
// 1.5 times the 128 x 128 tiles'): Gram product of 27 matrices of 768 x 2048 (162 tiles) 58 us against 63, of 22
// (132 tiles) 52 against 40, of 24 (144) 54 against 41, of 25 (150) 55 against 59, of 26 (156) 56 against 58; of 18 of
// 1001 x 1503 (180) 46 against 50, of 15 (150) 43 against 44, of 14 (140) 41 against 32; of 64 of 384 x 2048 (twice the
// area) 56 against 45.  (128 x 128 tiles win while two per CU hold all of them, up to 512 of them; from there to
// 160 of these the two are within 7 %.)  Then 128 x
// 128 tiles where there is one for most CUs: Gram product of 12 of 768 x 2048 (252 tiles) 27 us
// against 31, of 5 of 1001 x 1503 (180 tiles) 20 against 19; 48 rows would leave
// most of a 128-row tile empty.
inline int ns_tile_rows(bool sym, int64_t mp, int64_t np, int count) {
  const int64_t t256 = ns_tiles(sym, mp, np, count, 256, 256), t128 = ns_tiles(sym, mp, np, count, 128, 128);
  if (t256 >= 160 && 8 * t256 < 3 * t128) return 256;
  return t128 >= 192 && ns_tiles(sym, mp, np, count, 64, 128) > t128 ? 128 : 64;
}

template <int MODE, bool SPLIT, int OUT>
inline void ns_launch(const NsArgs& a, int cur, hipStream_t s) {
  constexpr bool sym = MODE == NS_GRAM || MODE == NS_POLY;
  const int rows = ns_tile_rows(sym, a.mp, a.np, a.count);
  const int64_t tiles = ns_tiles(sym, a.mp, a.np, a.count, rows, rows == 64 ? 128 : rows);
  // workgroups: a multiple of the XCDs
  const unsigned groups = static_cast<unsigned>(8 * ceil_div(tiles, 8));
  if (rows == 256)
    ns_big_kernel<MODE, SPLIT, OUT><<<dim3(std::min<unsigned>(groups, kNsCus)), dim3(core::NT), 0, s>>>(a, cur);
  else if (rows == 128) ns_product_kernel<MODE, 128, 2, SPLIT, OUT><<<dim3(groups), dim3(256), 0, s>>>(a, cur);
  else ns_product_kernel<MODE, 64, 3, SPLIT, OUT><<<dim3(groups), dim3(256), 0, s>>>(a, cur);
}
template <int MODE>
inline void ns_product(const NsArgs& a, int cur, bool split, hipStream_t s) {
  if constexpr (MODE == NS_LAST) {
    const int out = (a.dtype == FMOE_BF16 ? NS_BF16 : NS_F32) + (a.muon ? 2 : 0);
    if (out == NS_BF16) split ? ns_launch<MODE, true, NS_BF16>(a, cur, s) : ns_launch<MODE, false, NS_BF16>(a, cur, s);
    else if (out == NS_MUON_BF16)
      split ? ns_launch<MODE, true, NS_MUON_BF16>(a, cur, s) : ns_launch<MODE, false, NS_MUON_BF16>(a, cur, s);
    else if (out == NS_F32) ns_launch<MODE, true, NS_F32>(a, cur, s);  // fp32 matrices are always split
    else ns_launch<MODE, true, NS_MUON_F32>(a, cur, s);
  } else {
    split ? ns_launch<MODE, true, NS_BF16>(a, cur, s) : ns_launch<MODE, false, NS_BF16>(a, cur, s);
  }
}

// Sizes of a call, checked: sets m, n and the tall bits.
inline int ns_sizes(const int64_t* rows, const int64_t* cols, int count, NsArgs& a) {
  for (int i = 0; i < count; ++i) {
    if (rows[i] <= 0 || cols[i] <= 0) return FMOE_ERR_INVALID_ARG;
    const int64_t m = std::min(rows[i], cols[i]), n = std::max(rows[i], cols[i]);
    if (n > FMOE_MUON_MAX_SIDE || (i > 0 && (m != a.m || n != a.n))) return FMOE_ERR_SHAPE;
    a.m = static_cast<int>(m);
    a.n = static_cast<int>(n);
    if (rows[i] > cols[i]) a.tall |= uint64_t(1) << i;
  }
  a.mp = static_cast<int>(ns_pad(a.m));
  a.np = static_cast<int>(ns_pad(a.n));
  // 32-bit byte offsets within a matrix
  return static_cast<int64_t>(a.mp) * a.np <= FMOE_MUON_MAX_ELEMENTS ? FMOE_OK : FMOE_ERR_SHAPE;
}

struct NsSmallLayout {
  size_t norm, exps, x, parts, total;
};
inline NsSmallLayout ns_small_layout(int64_t n, int count) {
  const size_t panels = static_cast<size_t>(ns_panels(n)) * count;
  NsSmallLayout l;
  l.norm = (panels * sizeof(double) + 255) / 256 * 256;
  l.exps = (panels * sizeof(int) + 255) / 256 * 256;
  l.x = panels * kSmallSide * kSmallPanel * sizeof(float);
  l.parts = 2 * panels * kSmallBlocks * 256 * sizeof(float);
  l.total = l.norm + l.exps + l.x + l.parts;
  return l;
}

template <int DT, bool MUON, int MB>
inline int ns_run_small(NsArgs& a, int steps, void* workspace, hipStream_t s) {
  const NsSmallLayout l = ns_small_layout(a.n, a.count);
  uint8_t* p = static_cast<uint8_t*>(workspace);
  a.panels = ns_panels(a.n);
  a.norm = reinterpret_cast<double*>(p);
  a.exps = reinterpret_cast<int*>(p + l.norm);
  a.xs = reinterpret_cast<float*>(p + l.norm + l.exps);
  a.sparts = reinterpret_cast<float*>(p + l.norm + l.exps + l.x);
  const dim3 grid(a.panels, a.count), block(64 * small_waves(MB));
  constexpr int out = DT + (MUON ? 2 : 0);
  ns_small_load_kernel<DT, MUON, MB><<<grid, block, 0, s>>>(a);
  for (int k = 0; k + 1 < steps; ++k) ns_small_step_kernel<false, NS_BF16, MB><<<grid, block, 0, s>>>(a, k);
  ns_small_step_kernel<true, out, MB><<<grid, block, 0, s>>>(a, steps - 1);
  return launch_status();
}

inline size_t ns_workspace(int64_t m, int64_t n, int count, int dtype) {
  return ns_is_small(m, n) ? ns_small_layout(n, count).total : ns_layout(m, n, count, ns_split(m, dtype)).total;
}

inline int ns_run(NsArgs& a, int steps, const double* coeffs, double eps, void* workspace, size_t workspace_bytes,
                  hipStream_t s) {
  if (!workspace || workspace_bytes < ns_workspace(a.m, a.n, a.count, a.dtype)) return FMOE_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return FMOE_ERR_ALIGN;
  a.ca = static_cast<float>(coeffs[0]);
  a.cb = static_cast<float>(coeffs[1]);
  a.cc = static_cast<float>(coeffs[2]);
  a.eps = eps;
  if (ns_is_small(a.m, a.n)) {
#define FMOE_NS_SMALL(DT, MUON)                                             \
  (a.m <= 16 ? ns_run_small<DT, MUON, 1>(a, steps, workspace, s) : ns_run_small<DT, MUON, 4>(a, steps, workspace, s))
    if (a.dtype == FMOE_BF16) return a.muon ? FMOE_NS_SMALL(FMOE_BF16, true) : FMOE_NS_SMALL(FMOE_BF16, false);
    return a.muon ? FMOE_NS_SMALL(FMOE_F32, true) : FMOE_NS_SMALL(FMOE_F32, false);
#undef FMOE_NS_SMALL
  }
  const bool split = ns_split(a.m, a.dtype);
  const NsLayout l = ns_layout(a.m, a.n, a.count, split);
  a.parts = l.parts;
  uint8_t* p = static_cast<uint8_t*>(workspace);
  a.norm = reinterpret_cast<double*>(p);
  p += l.norm;
  auto take = [&](size_t n) {
    _Float16* q = reinterpret_cast<_Float16*>(p);
    p += n;
    return q;
  };
  const size_t w = split ? 2 : 1;
  for (int i = 0; i < 2; ++i) a.xh[i] = take(w * l.x);
  a.ah = take(w * l.sq);
  a.bh = take(w * l.sq);
  if (!split) a.x8 = reinterpret_cast<uint8_t*>(take(l.x / 2));
#define FMOE_NS_LOAD(DT, MUON)                                                                   \
  do {                                                                                           \
    ns_norm_kernel<DT, MUON><<<dim3(a.parts, a.count), dim3(256), 0, s>>>(a);                    \
    ns_load_kernel<DT, MUON><<<dim3(a.np / 64, a.mp / 64, a.count), dim3(256), 0, s>>>(a);       \
  } while (0)
  if (a.dtype == FMOE_BF16 && a.muon) FMOE_NS_LOAD(FMOE_BF16, true);
  else if (a.dtype == FMOE_BF16) FMOE_NS_LOAD(FMOE_BF16, false);
  else if (a.muon) FMOE_NS_LOAD(FMOE_F32, true);
  else FMOE_NS_LOAD(FMOE_F32, false);
#undef FMOE_NS_LOAD
  for (int k = 0; k < steps; ++k) {
    ns_product<NS_GRAM>(a, k & 1, split, s);
    ns_product<NS_POLY>(a, k & 1, split, s);
    if (k + 1 < steps) ns_product<NS_STEP>(a, k & 1, split, s);
    else ns_product<NS_LAST>(a, k & 1, split, s);
  }
  return launch_status();
}

inline bool ns_elem_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FMOE_BF16 ? 1u : 3u)) == 0;
}

}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_newton_schulz_check(int steps, const double* coeffs) {
  if (steps < 1 || steps > FMOE_MUON_MAX_STEPS || !coeffs) return FMOE_ERR_INVALID_ARG;
  return ns_bounded(coeffs[0], coeffs[1], coeffs[2], steps) ? FMOE_OK : FMOE_ERR_COEFFICIENTS;
}

extern "C" int fmoe_newton_schulz_tile(int64_t rows, int64_t cols, int n_tensors, int symmetric) {
  if (fmoe_orthogonalize_workspace_bytes(rows, cols, n_tensors, FMOE_BF16) == 0) return 0;
  const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
  return ns_is_small(m, n) ? 0 : ns_tile_rows(symmetric != 0, ns_pad(m), ns_pad(n), n_tensors);
}

extern "C" size_t fmoe_orthogonalize_workspace_bytes(int64_t rows, int64_t cols, int n_tensors, int dtype) {
  if (rows <= 0 || cols <= 0 || rows > FMOE_MUON_MAX_SIDE || cols > FMOE_MUON_MAX_SIDE || n_tensors <= 0 ||
      n_tensors > kNsMax)
    return 0;
  const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
  if (ns_pad(m) * ns_pad(n) > FMOE_MUON_MAX_ELEMENTS) return 0;
  return ns_workspace(m, n, n_tensors, dtype);
}

extern "C" int fmoe_orthogonalize(const void* const* src, void* const* dst, const int64_t* rows, const int64_t* cols,
                                  int n_tensors, int dtype, int steps, const double* coeffs, double eps,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (n_tensors < 0 || n_tensors > kNsMax || steps < 1 || steps > FMOE_MUON_MAX_STEPS) return FMOE_ERR_INVALID_ARG;
  if (dtype != FMOE_BF16 && dtype != FMOE_F32) return FMOE_ERR_DTYPE;
  if (n_tensors == 0) return FMOE_OK;
  if (!src || !dst || !rows || !cols || !coeffs || !(eps > 0.0)) return FMOE_ERR_INVALID_ARG;
  if (const int rc = fmoe_newton_schulz_check(steps, coeffs)) return rc;
  NsArgs a = {};
  a.count = n_tensors;
  a.dtype = dtype;
  if (const int rc = ns_sizes(rows, cols, n_tensors, a)) return rc;
  for (int i = 0; i < n_tensors; ++i) {
    if (!src[i] || !dst[i]) return FMOE_ERR_INVALID_ARG;
    if (!ns_elem_aligned(src[i], dtype) || !ns_elem_aligned(dst[i], dtype)) return FMOE_ERR_ALIGN;
    a.src[i] = src[i];
    a.dst[i] = dst[i];
  }
  return ns_run(a, steps, coeffs, eps, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int fmoe_muon_step(void* const* params, const void* const* grads, void* const* momentum_bufs,
                              const int64_t* rows, const int64_t* cols, int n_tensors, int dtype, double lr_tall,
                              double lr_wide, double decay, double momentum, int nesterov, int steps,
                              const double* coeffs, double eps, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (n_tensors < 0 || n_tensors > kNsMax || steps < 1 || steps > FMOE_MUON_MAX_STEPS) return FMOE_ERR_INVALID_ARG;
  if (dtype != FMOE_BF16 && dtype != FMOE_F32) return FMOE_ERR_DTYPE;
  if (n_tensors == 0) return FMOE_OK;
  if (!params || !grads || !momentum_bufs || !rows || !cols || !coeffs || !(eps > 0.0)) return FMOE_ERR_INVALID_ARG;
  if (const int rc = fmoe_newton_schulz_check(steps, coeffs)) return rc;
  NsArgs a = {};
  a.count = n_tensors;
  a.dtype = dtype;
  a.muon = 1;
  a.nesterov = nesterov != 0;
  a.mom = static_cast<float>(momentum);
  a.om = static_cast<float>(1.0 - momentum);
  a.decay = static_cast<float>(decay);
  a.lr_tall = static_cast<float>(lr_tall);
  a.lr_wide = static_cast<float>(lr_wide);
  if (const int rc = ns_sizes(rows, cols, n_tensors, a)) return rc;
  for (int i = 0; i < n_tensors; ++i) {
    if (!params[i] || !grads[i] || !momentum_bufs[i]) return FMOE_ERR_INVALID_ARG;
    if (!ns_elem_aligned(params[i], dtype) || !ns_elem_aligned(grads[i], dtype) ||
        !ns_elem_aligned(momentum_bufs[i], dtype))
      return FMOE_ERR_ALIGN;
    a.dst[i] = params[i];
    a.src[i] = grads[i];
    a.buf[i] = momentum_bufs[i];
  }
  return ns_run(a, steps, coeffs, eps, workspace, workspace_bytes, as_stream(stream));
}
