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
// overflow nor leave the normal range early.  Sums are fp32 throughout.  X is kept
// as two fp16 numbers (hi + lo, 22 bits) and a X is formed from both: small
// singular values are carried by that term (times a per step, some hundredfold
// over five steps), and what a rounding of X adds to it would grow with them.
// Rounding X in the other products only acts within the row space that X
// spans already.  Relative error of the result on gradients of full and low rank
// (768 x 2048, simulated in 64 bits): bf16 products 1e-2 .. 1.6e-1, fp16 without
// lo 1.3e-3 .. 1.9e-2, this form 3e-4 .. 1.5e-3 (half a step of a bf16 result: 3.9e-3).
// fp32 matrices take every operand as hi + lo (three products: hi hi, hi lo, lo hi;
// relative error 2e-6), and so do matrices of a small side up to kSplitSmall, whose
// few rounding errors average out less and whose products cost nothing next to
// the launches.
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

constexpr int kNsCus = 256;         // CUs of the chip: workgroups of the persistent products
constexpr int kNsMax = FMOE_MUON_MAX_TENSORS;
constexpr int kNsPad = 64;          // both sides are padded (with zeros) to a multiple of this
constexpr int64_t kSplitSmall = 128;
constexpr int kNsParts = 64;        // partial sums of squares per matrix, at most (a wave adds them)
constexpr int kNormChunk = 8192;    // elements per partial sum, at least
// Stored values: X 2^14, A 2^13, B 2^13 (singular values of X below 2.8, |B| below 7.9).
constexpr float kXScale = 16384.0f, kAScale = 8192.0f;
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
  // fp16, hi and lo: X [count][mp][np] twice (the step reads one and writes the other; lo of
  // the second only where the products take it), A and B [count][mp][mp]
  _Float16 *xh[2], *xl[2], *ah, *al, *bh, *bl;
};

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
    // the norm of a matrix that holds NaN or infinities is none, and its X is NaN
    if (threadIdx.x == 0) scale_s = static_cast<double>(kXScale) / (nrm < a.eps ? a.eps : nrm);
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
    half8 h, l;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = tile[r][q + e];
      h[e] = static_cast<_Float16>(v);
      l[e] = static_cast<_Float16>(v - static_cast<float>(h[e]));
    }
    const int64_t o = (static_cast<int64_t>(mat) * a.mp + i0 + r) * a.np + j0 + q;
    *reinterpret_cast<half8*>(a.xh[0] + o) = h;
    *reinterpret_cast<half8*>(a.xl[0] + o) = l;
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

// The values to store from sums of 8 consecutive elements of a row (offset o in A or X).
__device__ __forceinline__ void ns_gram8(float* v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * (kAScale / (kXScale * kXScale));
}
template <bool SPLIT>
__device__ __forceinline__ void ns_poly8(const NsArgs& a, int64_t o, float* v) {  // b A + c A^2
  const half8 h = *reinterpret_cast<const half8*>(a.ah + o);
  half8 l = {0, 0, 0, 0, 0, 0, 0, 0};
  if constexpr (SPLIT) l = *reinterpret_cast<const half8*>(a.al + o);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    v[e] = fmaf(a.cb, static_cast<float>(h[e]) + static_cast<float>(l[e]), a.cc * (v[e] * (1.0f / kAScale)));
}
__device__ __forceinline__ void ns_step8(const NsArgs& a, int cur, int64_t o, float* v) {  // a X + B X
  const half8 h = *reinterpret_cast<const half8*>(a.xh[cur] + o);
  const half8 l = *reinterpret_cast<const half8*>(a.xl[cur] + o);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    v[e] = fmaf(a.ca, static_cast<float>(h[e]) + static_cast<float>(l[e]), v[e] * (1.0f / kAScale));
}
__device__ __forceinline__ void ns_put_parts(_Float16* hi, _Float16* lo, int64_t o, const float* v, bool with_lo) {
  half8 h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = static_cast<_Float16>(v[e]);
    l[e] = static_cast<_Float16>(v[e] - static_cast<float>(h[e]));
  }
  *reinterpret_cast<half8*>(hi + o) = h;
  if (with_lo) *reinterpret_cast<half8*>(lo + o) = l;
}
// The result: n (up to 8) consecutive elements of the matrix, or of the parameter's update.
template <int DT>
__device__ __forceinline__ void ns_finish(const NsArgs& a, void* dst, int64_t o, int n, float* v, float lr) {
  if (n <= 0) return;
  if (a.muon) {
    float p[8];
    ns_load8<DT>(dst, o, n, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaf(-lr, v[e], p[e] * a.decay);
  }
  ns_store8<DT>(dst, o, n, v);
}

__device__ __forceinline__ void ns_result8(const NsArgs& a, void* dst, int64_t o, int n, float* v, float lr) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = v[e] * (1.0f / kXScale);
  if (a.dtype == FMOE_BF16) ns_finish<FMOE_BF16>(a, dst, o, n, v, lr);
  else ns_finish<FMOE_F32>(a, dst, o, n, v, lr);
}

// TM x TN outputs per workgroup of four waves (2 x 2), K in steps of 64 through two LDS stages.
// A step reads its whole stage into registers, and the copies (global -> LDS, no registers) of the
// stage after the next go into its slot while it is multiplied: one to two stages are in
// flight, and of the two workgroups of a CU one reads LDS while the other multiplies.
// The row operand, and the column operand of the symmetric products, are K-contiguous;
// the step's column operand is X as it lies ([K, N]), read with transposing LDS reads
// (gemm_core.h has both layouts and their swizzles).  SPLIT: hi lo + lo hi + hi hi.
template <int MODE, int TM, bool SPLIT>
__global__ __launch_bounds__(256, 2) void ns_product_kernel(const NsArgs a, const int cur) {
  using namespace core;
  constexpr bool SYM = MODE == NS_GRAM || MODE == NS_POLY;
  constexpr int TN = SYM ? TM : 128;
  constexpr int WTM = TM / 2, WTN = TN / 2, FM = WTM / 16, FN = WTN / 16;
  constexpr int A_ST = TM * RB, STAGE = A_ST + TN * RB;
  constexpr int CA = TM / 32, CB = TN / 32;  // copies per wave and stage
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w >> 1, wn = w & 1;
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

  const int K = MODE == NS_GRAM ? a.np : a.mp;
  const int lda = K, ldb = SYM ? K : a.np;
  const int nk = K / BK, steps = nk * (SPLIT ? 3 : 1);
  const int64_t msq = static_cast<int64_t>(mat) * a.mp * a.mp, mx = static_cast<int64_t>(mat) * a.mp * a.np;
  const _Float16* ph = MODE == NS_GRAM ? a.xh[cur] + mx : MODE == NS_POLY ? a.ah + msq : a.bh + msq;
  const _Float16* pl = MODE == NS_GRAM ? a.xl[cur] + mx : MODE == NS_POLY ? a.al + msq : a.bl + msq;
  const _Float16* qh = SYM ? ph : a.xh[cur] + mx;
  const _Float16* ql = SYM ? pl : a.xl[cur] + mx;

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
      const int krow = 4 * (w + 4 * q) + (lane >> 4);
      const int cb = ((((lane & 15) >> 1) ^ wsw(krow)) << 1) | (lane & 1);
      boff[q] = static_cast<uint32_t>(krow * ldb + min(tj * TN + 8 * cb, a.np - 8)) * 2u;
    }
  }
  // SPLIT: hi lo, lo hi, then hi hi, so that the small terms are summed while the sum is small
  const uint8_t *pa = reinterpret_cast<const uint8_t*>(ph), *pb = reinterpret_cast<const uint8_t*>(SPLIT ? ql : qh);
  const int64_t bstep = SYM ? RB : static_cast<int64_t>(BK) * ldb * 2;
  int kt = 0, seg = 0;
  auto issue = [&](int st) __attribute__((always_inline)) {
    const uint32_t la = sbase + st * STAGE + w * 1024, lb = la + A_ST;
#pragma unroll
    for (int q = 0; q < CA; ++q) copy16(la + q * 4096, pa, aoff[q]);
#pragma unroll
    for (int q = 0; q < CB; ++q) copy16(lb + q * 4096, pb, boff[q]);
    pa += RB;
    pb += bstep;
    if (SPLIT && ++kt == nk) {
      kt = 0;
      ++seg;
      pa = reinterpret_cast<const uint8_t*>(seg == 1 ? pl : ph);
      pb = reinterpret_cast<const uint8_t*>(qh);
    }
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t xa = frag_base(wm * WTM, lane);
  const uint32_t xb = A_ST + (SYM ? frag_base(wn * WTN, lane) : tr_base(4 * wn, lane));
  typedef __attribute__((address_space(3))) half8 lds_half8;
  issue(0);
  if (steps > 1) issue(1);
  for (int it = 0; it < steps; ++it) {
    // this stage is there (the next may be in flight)
    if (it + 1 < steps) wait_vm_barrier<CA + CB>();
    else wait_vm_barrier<0>();
    const uint32_t src = sbase + (it & 1) * STAGE;
    half8 fa[2][FM], fb[2][FN];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[kh][i] = *(const lds_half8*)(uintptr_t)(src + (xa ^ (kh * 64u)) + 2048u * i);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        if constexpr (SYM) fb[kh][j] = *(const lds_half8*)(uintptr_t)(src + (xb ^ (kh * 64u)) + 2048u * j);
        else fb[kh][j] = __builtin_bit_cast(half8, tr_frag(((src + xb) ^ (j << 5)) + kh * TR_KHALF));
      }
    }
    wait_lds_barrier();  // every wave has this stage in registers: its slot takes the stage after the next
    if (it + 2 < steps) issue(it & 1);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[kh][j], fa[kh][i], acc[i][j], 0, 0, 0);
    __builtin_amdgcn_s_setprio(0);
  }

  // Epilogue: the wave's block goes through its part of LDS as fp32 (16-byte chunk c of row r at
  // slot c ^ f(r): no bank conflicts by rows or by columns) and comes back as 8 consecutive elements
  // of a row, or of a column for a transposed store, so that global memory sees 16-byte accesses of
  // full lines.  (Storing from the accumulators' layout, 8 bytes or less per lane in
  // 16 rows at once, took as long as the multiplication.)
  constexpr int MASK = WTN / 4 - 1;
  static_assert(4 * WTM * WTN * 4 <= 2 * STAGE);
  float* ep = reinterpret_cast<float*>(smem) + w * (WTM * WTN);
  auto slot = [](int r, int c) { return r * WTN + ((c ^ ((r & 15) ^ ((r >> 3) & 7))) & MASK) * 4; };
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<f32x4*>(ep + slot(16 * i + (lane & 15), 4 * j + (lane >> 4))) = acc[i][j];
  __builtin_amdgcn_wave_barrier();
  const int row0 = ti * TM + wm * WTM, col0 = tj * TN + wn * WTN;  // of the wave's block
  auto by_row = [&](int r, int c, float* v) {  // elements c .. c + 7 of row r
    const f32x4 lo = *reinterpret_cast<const f32x4*>(ep + slot(r, c >> 2));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(ep + slot(r, (c >> 2) + 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
  };
  constexpr int LPR = WTN / 8, RPP = 64 / LPR;  // lanes per row, rows per pass
  constexpr int LPC = WTM / 8, CPP = 64 / LPC;  // the same by columns
  const int lc = (lane % LPR) * 8, lr = lane / LPR;
  const int tr = (lane % LPC) * 8, tc = lane / LPC;

  if constexpr (SYM) {
    _Float16* oh = MODE == NS_GRAM ? a.ah : a.bh;
    _Float16* ol = MODE == NS_GRAM ? a.al : a.bl;
    // the value to store, for the element that the wave's sum at this place belongs to
#pragma unroll
    for (int p = 0; p < WTM / RPP; ++p) {
      const int r = p * RPP + lr;
      float v[8];
      by_row(r, lc, v);
      const bool on = row0 + r < a.mp && col0 + lc < a.mp;
      const int64_t o = msq + static_cast<int64_t>(on ? row0 + r : 0) * a.mp + (on ? col0 + lc : 0);
      if constexpr (MODE == NS_GRAM) ns_gram8(v);
      else ns_poly8<SPLIT>(a, o, v);
      if (on) ns_put_parts(oh, ol, o, v, SPLIT);
      if (ti != tj) {  // back into LDS for the mirrored tile
        *reinterpret_cast<f32x4*>(ep + slot(r, lc >> 2)) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(ep + slot(r, (lc >> 2) + 1)) = f32x4{v[4], v[5], v[6], v[7]};
      }
    }
    if (ti == tj) return;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < WTN / CPP; ++p) {
      const int c = p * CPP + tc;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ep[slot(tr + e, c >> 2) + (c & 3)];
      if (row0 + tr < a.mp && col0 + c < a.mp)
        ns_put_parts(oh, ol, msq + static_cast<int64_t>(col0 + c) * a.mp + row0 + tr, v, SPLIT);
    }
  } else {
    // X' = a X + B X, X from hi and lo
#pragma unroll
    for (int p = 0; p < WTM / RPP; ++p) {
      const int r = p * RPP + lr;
      float v[8];
      by_row(r, lc, v);
      const bool on = row0 + r < a.mp && col0 + lc < a.np;
      const int64_t o = mx + static_cast<int64_t>(on ? row0 + r : 0) * a.np + (on ? col0 + lc : 0);
      ns_step8(a, cur, o, v);
      if constexpr (MODE == NS_STEP) {
        if (on) ns_put_parts(a.xh[1 - cur], a.xl[1 - cur], o, v, true);
      } else {
        *reinterpret_cast<f32x4*>(ep + slot(r, lc >> 2)) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(ep + slot(r, (lc >> 2) + 1)) = f32x4{v[4], v[5], v[6], v[7]};
      }
    }
    if constexpr (MODE == NS_LAST) {
      __builtin_amdgcn_wave_barrier();
      void* const dst = a.dst[mat];
      if ((a.tall >> mat) & 1) {
#pragma unroll 2
        for (int p = 0; p < WTN / CPP; ++p) {
          const int c = p * CPP + tc;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = ep[slot(tr + e, c >> 2) + (c & 3)];
          const int n = col0 + c < a.n ? min(a.m - (row0 + tr), 8) : 0;
          ns_result8(a, dst, static_cast<int64_t>(col0 + c) * a.m + row0 + tr, n, v, a.lr_tall);
        }
      } else {
#pragma unroll 2
        for (int p = 0; p < WTM / RPP; ++p) {
          const int r = p * RPP + lr;
          float v[8];
          by_row(r, lc, v);
          const int n = row0 + r < a.m ? min(a.n - (col0 + lc), 8) : 0;
          ns_result8(a, dst, static_cast<int64_t>(row0 + r) * a.n + col0 + lc, n, v, a.lr_wide);
        }
      }
    }
  }
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
template <int I, int J>
__device__ __forceinline__ void ns_quarter(f32x4 (&acc)[core::FM][core::FN], const core::AFrag& a,
                                           const core::BFrag& b) {
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int kh = x >> 1, n = (x & 1) * 2;
    ns_mfma4(acc[2 * I][4 * J + n], acc[2 * I + 1][4 * J + n], acc[2 * I][4 * J + n + 1],
             acc[2 * I + 1][4 * J + n + 1], b[kh][n], b[kh][n + 1], a[kh][0], a[kh][1]);
  }
  __builtin_amdgcn_s_setprio(0);
  core::barrier();
}

struct NsTile {
  int mat, ti, tj;
};

template <int MODE, bool SPLIT>
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
  // Workgroup b runs on XCD b % 8: its XCD takes a contiguous run of each round's tiles.
  const int NP = static_cast<int>(gridDim.x), bid = static_cast<int>(blockIdx.x);
  const int b = NP % 8 == 0 ? (bid % 8) * (NP / 8) + bid / 8 : bid;
  const int my_items = (items - b + NP - 1) / NP;
  if (my_items <= 0) return;
  const int K = MODE == NS_GRAM ? a.np : a.mp;
  const int ld = K, ldb = SYM ? K : a.np;
  const int nk = K / BK, steps = SPLIT ? 3 * nk : nk;
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
  int c_ti = 0, c_kt = 0, c_seg = 0;
  const uint8_t *c_a = nullptr, *c_b = nullptr;
  uint32_t a_off[4], b_off[4];
  const int64_t bstep = SYM ? RB : static_cast<int64_t>(2) * BK * ldb;
  // operand bases of the tile being copied, for segment c_seg (SPLIT: hi lo, lo hi, hi hi)
  auto bases = [&](const NsTile& t) __attribute__((always_inline)) {
    const int64_t msq = static_cast<int64_t>(t.mat) * a.mp * a.mp, mx = static_cast<int64_t>(t.mat) * a.mp * a.np;
    const bool alo = SPLIT && c_seg == 1, blo = SPLIT && c_seg == 0;
    const _Float16 *p, *q;
    if constexpr (MODE == NS_GRAM) {
      p = (alo ? a.xl[cur] : a.xh[cur]) + mx;
      q = (blo ? a.xl[cur] : a.xh[cur]) + mx;
    } else if constexpr (MODE == NS_POLY) {
      p = (alo ? a.al : a.ah) + msq;
      q = (blo ? a.al : a.ah) + msq;
    } else {
      p = (alo ? a.bl : a.bh) + msq;
      q = (blo ? a.xl[cur] : a.xh[cur]) + mx;
    }
    c_a = reinterpret_cast<const uint8_t*>(p + static_cast<int64_t>(t.ti) * BM * ld);
    c_b = reinterpret_cast<const uint8_t*>(SYM ? q + static_cast<int64_t>(t.tj) * BN * ld : q);
  };
  auto copy_tile = [&](int ti) __attribute__((always_inline)) {
    const NsTile t = locate(b + ti * NP);
    c_seg = 0;
    bases(t);
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
        b_off[q] = static_cast<uint32_t>((32 * (q & 1) + krow) * ldb + min(t.tj * BN + col, a.np - 8)) * 2u;
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
    if (__builtin_expect(++c_kt == nk, 0)) {
      if (SPLIT && c_seg < 2) {
        c_kt = 0;
        ++c_seg;
        bases(locate(b + c_ti * NP));
      } else if (c_ti + 1 < my_items) {
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
  float* ep = reinterpret_cast<float*>(smem + 2 * STAGE + w * EPI);  // this wave's staging (4 KB)
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
    ns_quarter<0, 0>(acc, a0, b0);
    // (0, 1)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int n = 0; n < 4; ++n) read_b(b1, 1, st, kh, n);
    issue_a(it + 2, 0);
    wait_vm_barrier<5 * LU>();  // A1 of this stage
    ns_quarter<0, 1>(acc, a0, b1);
    // (1, 0)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int m = 0; m < 2; ++m) read_a(a1, 1, st, kh, m);
    issue_b(it + 2, 0);
    wait_vm_barrier<4 * LU>();  // A0, B0 of the next stage
    ns_quarter<1, 0>(acc, a1, b0);
    // (1, 1): the next step's first fragments (at a tile's end they are read again after its epilogue)
    read_first(nxt);
    issue_b(it + 2, 1);
    wait_lds_barrier();
    ns_quarter<1, 1>(acc, a1, b1);

    if (++e_kt < steps) continue;
    // ---- tile epilogue: this wave's 64 x 128 block (both wave groups together)
    if (!late) barrier();
    e_kt = 0;
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3\n" ::: "memory");  // MFMA results -> VALU reads
    int el = lane;
    asm volatile("" : "+v"(el));  // the address arithmetic below stays out of the main loop
    {
      const NsTile t = locate(b + e_ti * NP);
      const int row0 = t.ti * BM + wm * WTM, col0 = t.tj * BN + wn * WTN;
      const int64_t msq = static_cast<int64_t>(t.mat) * a.mp * a.mp, mx = static_cast<int64_t>(t.mat) * a.mp * a.np;
      const bool tall = (a.tall >> t.mat) & 1;
      const bool by_columns = SYM ? t.ti != t.tj : (MODE == NS_LAST && tall);
      void* const dst = MODE == NS_LAST ? a.dst[t.mat] : nullptr;
      const int lr = el >> 3, lc = (el & 7) * 8;
      // Rows: 16 x 64 values at a time (chunk c of row r at slot c ^ r)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int jh = 0; jh < 2; ++jh) {
          auto at = [&](int r, int c) { return reinterpret_cast<f32x4*>(ep + r * 64 + ((c ^ r) & 15) * 4); };
#pragma unroll
          for (int j = 0; j < 4; ++j) *at(el & 15, 4 * j + (el >> 4)) = acc[i][4 * jh + j];
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int r = 8 * p + lr, row = row0 + 16 * i + r, col = col0 + 64 * jh + lc;
            f32x4 lo4 = *at(r, lc >> 2), hi4 = *at(r, (lc >> 2) + 1);
            float v[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = lo4[e], v[4 + e] = hi4[e];
            const bool on = row < a.mp && col < (SYM ? a.mp : a.np);
            const int64_t o = SYM ? msq + static_cast<int64_t>(on ? row : 0) * a.mp + (on ? col : 0)
                                  : mx + static_cast<int64_t>(on ? row : 0) * a.np + (on ? col : 0);
            if constexpr (MODE == NS_GRAM) ns_gram8(v);
            else if constexpr (MODE == NS_POLY) ns_poly8<SPLIT>(a, o, v);
            else ns_step8(a, cur, o, v);
            if constexpr (SYM) {
              if (on) ns_put_parts(MODE == NS_GRAM ? a.ah : a.bh, MODE == NS_GRAM ? a.al : a.bl, o, v, SPLIT);
            } else if constexpr (MODE == NS_STEP) {
              if (on) ns_put_parts(a.xh[1 - cur], a.xl[1 - cur], o, v, true);
            } else if (!tall) {
              const int n = row < a.m ? min(a.n - col, 8) : 0;
              ns_result8(a, dst, static_cast<int64_t>(row) * a.n + col, n, v, a.lr_wide);
            }
            if (by_columns) {
              *at(r, lc >> 2) = f32x4{v[0], v[1], v[2], v[3]};
              *at(r, (lc >> 2) + 1) = f32x4{v[4], v[5], v[6], v[7]};
            }
          }
          __builtin_amdgcn_wave_barrier();
          if (by_columns)  // the finished values, back in the accumulators' layout
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][4 * jh + j] = *at(el & 15, 4 * j + (el >> 4));
          __builtin_amdgcn_wave_barrier();
        }
      }
      // Columns: 64 x 16 values at a time (chunk c of row r at slot c ^ (r / 2) ^ (r / 8))
      if (by_columns) {
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          auto at = [&](int r, int c) { return ep + r * 16 + ((c ^ (r >> 1) ^ (r >> 3)) & 3) * 4; };
#pragma unroll
          for (int i = 0; i < FM; ++i)
            *reinterpret_cast<f32x4*>(at(16 * i + (el & 15), el >> 4)) = acc[i][j];
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int c = 8 * p + lr, col = col0 + 16 * j + c, row = row0 + lc;  // rows row .. row + 7
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = at(lc + e, c >> 2)[c & 3];
            if constexpr (SYM) {
              if (row < a.mp && col < a.mp)
                ns_put_parts(MODE == NS_GRAM ? a.ah : a.bh, MODE == NS_GRAM ? a.al : a.bl,
                             msq + static_cast<int64_t>(col) * a.mp + row, v, SPLIT);
            } else if constexpr (MODE == NS_LAST) {
              const int n = col < a.n ? min(a.m - row, 8) : 0;
              ns_result8(a, dst, static_cast<int64_t>(col) * a.m + row, n, v, a.lr_tall);
            }
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
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
  l.total = l.norm + 4 * l.x + (split ? 4 : 2) * l.sq;
  return l;
}

// Whether the iterates stay within the stored range: the largest singular value after each
// step, from the polynomial's extrema over [0, s], and the largest |b t + c t^2| over t <= s^2.
inline bool ns_bounded(double a, double b, double c, int steps) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  double s = 1.0 + 1e-6;
  for (int k = 0; k < steps; ++k) {
    if (!(s < kMaxSigma)) return false;
    const double t1 = s * s;
    double poly = std::fabs(b * t1 + c * t1 * t1);
    if (c != 0.0) {
      const double t = -b / (2.0 * c);
      if (t > 0.0 && t < t1) poly = std::max(poly, std::fabs(b * t + c * t * t));
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

template <int MODE>
inline void ns_product(const NsArgs& a, int cur, bool split, hipStream_t s) {
  constexpr bool sym = MODE == NS_GRAM || MODE == NS_POLY;
  auto tiles = [&](int tm) {
    const int64_t r = ceil_div(a.mp, tm);
    return (sym ? r * (r + 1) / 2 : r * ceil_div(a.np, 128)) * a.count;
  };
  const int64_t t256 = sym ? ceil_div(a.mp, 256) * (ceil_div(a.mp, 256) + 1) / 2 * a.count
                           : ceil_div(a.mp, 256) * ceil_div(a.np, 256) * a.count;
  if (t256 >= 128) {
    const dim3 g(static_cast<unsigned>(std::min<int64_t>(t256, kNsCus))), blk(core::NT);
    if (split) ns_big_kernel<MODE, true><<<g, blk, 0, s>>>(a, cur);
    else ns_big_kernel<MODE, false><<<g, blk, 0, s>>>(a, cur);
    return;
  }
  const bool big = tiles(128) >= 256;
  const dim3 grid(static_cast<unsigned>(8 * ceil_div(tiles(big ? 128 : 64), 8))), block(256);
  if (big) {
    if (split) ns_product_kernel<MODE, 128, true><<<grid, block, 0, s>>>(a, cur);
    else ns_product_kernel<MODE, 128, false><<<grid, block, 0, s>>>(a, cur);
  } else {
    if (split) ns_product_kernel<MODE, 64, true><<<grid, block, 0, s>>>(a, cur);
    else ns_product_kernel<MODE, 64, false><<<grid, block, 0, s>>>(a, cur);
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

inline int ns_run(NsArgs& a, int steps, const double* coeffs, double eps, void* workspace, size_t workspace_bytes,
                  hipStream_t s) {
  const bool split = ns_split(a.m, a.dtype);
  const NsLayout l = ns_layout(a.m, a.n, a.count, split);
  if (!workspace || workspace_bytes < l.total) return FMOE_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return FMOE_ERR_ALIGN;
  a.ca = static_cast<float>(coeffs[0]);
  a.cb = static_cast<float>(coeffs[1]);
  a.cc = static_cast<float>(coeffs[2]);
  a.eps = eps;
  a.parts = l.parts;
  uint8_t* p = static_cast<uint8_t*>(workspace);
  a.norm = reinterpret_cast<double*>(p);
  p += l.norm;
  auto take = [&](size_t n) {
    _Float16* q = reinterpret_cast<_Float16*>(p);
    p += n;
    return q;
  };
  for (int i = 0; i < 2; ++i) a.xh[i] = take(l.x);
  for (int i = 0; i < 2; ++i) a.xl[i] = take(l.x);
  a.ah = take(l.sq);
  a.bh = take(l.sq);
  if (split) a.al = take(l.sq), a.bl = take(l.sq);
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

extern "C" size_t fmoe_orthogonalize_workspace_bytes(int64_t rows, int64_t cols, int n_tensors, int dtype) {
  if (rows <= 0 || cols <= 0 || rows > FMOE_MUON_MAX_SIDE || cols > FMOE_MUON_MAX_SIDE || n_tensors <= 0 ||
      n_tensors > kNsMax)
    return 0;
  const int64_t m = std::min(rows, cols), n = std::max(rows, cols);
  if (ns_pad(m) * ns_pad(n) > FMOE_MUON_MAX_ELEMENTS) return 0;
  return ns_layout(m, n, n_tensors, ns_split(m, dtype)).total;
}

extern "C" int fmoe_orthogonalize(const void* const* src, void* const* dst, const int64_t* rows, const int64_t* cols,
                                  int n_tensors, int dtype, int steps, const double* coeffs, double eps,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (n_tensors < 0 || n_tensors > kNsMax || steps < 1 || steps > FMOE_MUON_MAX_STEPS) return FMOE_ERR_INVALID_ARG;
  if (dtype != FMOE_BF16 && dtype != FMOE_F32) return FMOE_ERR_DTYPE;
  if (n_tensors == 0) return FMOE_OK;
  if (!src || !dst || !rows || !cols || !coeffs || !(eps > 0.0)) return FMOE_ERR_INVALID_ARG;
  if (!ns_bounded(coeffs[0], coeffs[1], coeffs[2], steps)) return FMOE_ERR_COEFFICIENTS;
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
  if (!ns_bounded(coeffs[0], coeffs[1], coeffs[2], steps)) return FMOE_ERR_COEFFICIENTS;
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
