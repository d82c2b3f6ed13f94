// vocab_loss.hip — cross entropy over a vocabulary, and distillation from a teacher's
// listed logits, straight from the hidden states and the vocabulary's weight.
//
//   t[r, v] = c * sum_k H[r, k] W[v, k],  c = logit_scale / temperature * log2(e)
//   (logits in units of log 2, so that exponentials are v_exp_f32 = 2^x)
//   m[r] = max_v t[r, v],  l[r] = log2 sum_v 2^(t[r, v] - m[r])
//   log p[r, v] = ln 2 * ((t[r, v] - m[r]) - l[r])
//   G[r, v] = w[r] * (p[r, v] - q[r, v]),  dH = G W,  dW = G^T H
// with q the row's target distribution: 1 at the target, or the teacher's softmax over its list.
//
// The logits [rows, vocab] are not kept (long lists of a distillation read them from a piece of at most 256 MB,
// vl_stores_logits below).  A call whose loss is one value (mean or sum), for training, forms
// its gradients at once (below): a piece of the rows at a time, whose exponentials 2^(t - o) are G
// up to a factor per row, which is known when the piece's logits are done.  A call with a loss per row, whose weights
// only the backward brings, reduces a tile's logits to a maximum and a sum of exponentials per row, and forms
// them again in the backward, a piece of the vocabulary at a time: one product more (8 instead of
// 6 T V d flops).  The extra memory is that of a piece and what goes by the rows: the packed rows, dH's sums between pieces, and
// without gradients at once the partial maxima and sums, 8 bytes per row and 128 columns (T V / 16 in all).  All products are bound by the matrix units and run on
// the main loop of gemm_core.h: 256 x 256 tiles, persistent workgroups, copies in one ring over all
// of a workgroup's tiles.
//
// Rows without a target (prompt tokens, padding) are left out first: the rows with one are packed, in
// order, with zeros up to a multiple of 64 rows and columns, so that they cost nothing and what is in
// them (also NaN) stays out of the products.
//
// Operands are bf16 (planes = 1) or fp32 (planes = 3).  The logits of fp32 operands are products of rows that are scaled
// by a power of two each (their largest element to 2^13 .. 2^14) and held as two fp16 numbers, hi + lo: 22 bits of every
// element down to 2^-17 of its row's largest, and 2^-39 of that below.  lo hi + hi lo + hi hi are added, as three passes
// over K in one ring.  G spans more: a row's gradient is as precise in its smallest elements, which make up whole rows of dW, so
// the products with it take three bf16 numbers, hi + mid + lo: 24 bits of every element down to 2^-109 (bf16 ends at 2^-133).  Of the nine products of
// such numbers the six largest are added, the smallest first; what is left out is below 2^-22 of the largest.  G is rounded the same way: half a step of bf16,
// 2^-8 of an element at most, before the elements of a row or column are summed in fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/fusionvocab.h"
#include "elements.h"
#include "fmoe_common.h"
#include "gemm_core.h"

namespace fmoe {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kVlCus = 256;        // workgroups of the persistent products: one per CU
constexpr int kRowBlock = 32;      // rows of a mask
constexpr int kGroup = 4;          // row tiles that are walked together, column by column (8: 0.5 % slower, 16: 4 %)
// index of a listed entry: none, or outside the vocabulary
constexpr int kNone = -1, kBad = -2;

inline int64_t pad64(int64_t n) { return (n + 63) / 64 * 64; }
__host__ __device__ inline int pad_rows(int n) { return (n + 63) / 64 * 64 > 64 ? (n + 63) / 64 * 64 : 64; }

// What a forward call keeps for its backward (and uses itself).
struct VlState {
  int* head;      // [0]: rows with entries
  int* perm;      // [T] packed row -> row
  int* inv;       // [T] row -> packed row, or -1
  int* index;     // [T][top] of packed rows; of equal ones all but the first are kNone
  float* q;       // [T][top] target distribution, equal entries added (distillation)
  float* picked;  // [T][top] t of the listed entries; cross entropy: p - 1 of the target
  float2* stat;   // [T] m, l
  uint16_t* h;    // [planes][Tp][Dp] packed rows
  uint16_t* h16;  // planes = 3: [2][Tp][Dp] them as fp16, hi and lo of the scaled rows,
  float* h_scale; // [Tp] and what undoes the scaling
  int64_t Tp, Dp, plane;
  size_t bytes;
  VlState(uint8_t* base, int64_t T, int64_t D, int64_t top, int planes) {
    bytes = 0;
    auto take = [&](size_t n) {
      uint8_t* p = base + bytes;
      bytes += (n + 255) & ~size_t(255);
      return p;
    };
    Tp = std::max<int64_t>(pad64(T), 64), Dp = pad64(D), plane = Tp * Dp;
    head = reinterpret_cast<int*>(take(4));
    perm = reinterpret_cast<int*>(take(T * 4));
    inv = reinterpret_cast<int*>(take(T * 4));
    index = reinterpret_cast<int*>(take(T * top * 4));
    q = reinterpret_cast<float*>(take(T * top * 4));
    picked = reinterpret_cast<float*>(take(T * top * 4));
    stat = reinterpret_cast<float2*>(take(T * 8));
    h = reinterpret_cast<uint16_t*>(take(planes * plane * 2));
    h16 = reinterpret_cast<uint16_t*>(take(planes == 3 ? 2 * plane * 2 : 0));
    h_scale = reinterpret_cast<float*>(take(planes == 3 ? Tp * 4 : 0));
  }
};

// ---- packing ---------------------------------------------------------------------------------

struct RowsArgs {
  const void *hidden, *index, *teacher;
  int64_t ldh, ignore;
  int index64, t_dtype;  // t_dtype -1: no teacher
  int T, D, Dp, V, top;
  int64_t plane;
  float inv_temp;
  uint32_t* masks;       // rows with entries, 32 per word; nullptr: every workgroup finds them itself
  int *head, *perm, *inv, *out_index;
  float* loss;           // zeros in rows without entries, where it is [T] (else nullptr)
  uint16_t *h, *h16;
  float* h_scale;
};
constexpr int kFewEntries = 4096;  // entries of all rows that a workgroup looks at itself: 4 per thread

// Entry e = row * top + k: kNone, kBad or an index; z: its teacher logit over the temperature.
__device__ __forceinline__ int vl_entry(const RowsArgs& a, int64_t e, float& z) {
  const int64_t id = a.index64 ? static_cast<const int64_t*>(a.index)[e] : static_cast<const int32_t*>(a.index)[e];
  z = 0.0f;
  float raw = 0.0f;
  if (a.t_dtype >= 0)
    raw = a.t_dtype == FMOE_BF16 ? bf2f(static_cast<const uint16_t*>(a.teacher)[e])
                                 : static_cast<const float*>(a.teacher)[e];
  z = raw * a.inv_temp;
  if (id == a.ignore || raw == -__builtin_inff()) return kNone;
  return id < 0 || id >= a.V ? kBad : static_cast<int>(id);
}

// Sets in LDS the bits of the rows row0 .. row1 - 1 that have an entry (1024 threads).
__device__ __forceinline__ void vl_mark_rows(const RowsArgs& a, int row0, int row1, uint32_t* bits) {
  const int words = (row1 - row0 + 31) / 32;
  for (int i = threadIdx.x; i < words; i += 1024) bits[i] = 0;
  __syncthreads();
  const int64_t e0 = static_cast<int64_t>(row0) * a.top, e1 = static_cast<int64_t>(row1) * a.top;
  constexpr int U = 8;
  for (int64_t e = e0 + threadIdx.x; e < e1; e += 1024 * U) {
    bool has[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float z;
      const int64_t at = e + 1024 * u;
      has[u] = vl_entry(a, min(at, e1 - 1), z) != kNone && at < e1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (has[u]) {
        const int r = static_cast<int>(e - e0 + 1024 * u) / a.top;
        atomicOr(&bits[r >> 5], 1u << (r & 31));
      }
  }
  __syncthreads();
}

__global__ __launch_bounds__(1024) void vl_mark_kernel(const RowsArgs a) {
  __shared__ uint32_t bits[1];
  vl_mark_rows(a, blockIdx.x * kRowBlock, min(static_cast<int>(blockIdx.x + 1) * kRowBlock, a.T), bits);
  if (threadIdx.x == 0) a.masks[blockIdx.x] = bits[0];
}

// hi, mid and lo of fp32 values (planes = 3), or their bf16 rounding alone.
template <int PLANES>
__device__ __forceinline__ void vl_split8(const float* v, uint4* out) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    out[p] = pack8(r);
    if (p + 1 == PLANES) break;
    float h[8];
    unpack8(out[p], h);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = r[e] - h[e];  // exact
  }
}

// A row of n elements into padded planes (zeros past n).
template <int DT, int PLANES>
__device__ __forceinline__ void vl_copy_row(const void* src, int64_t row, int n, int np, uint16_t* dst, int64_t plane,
                                            int lane, int lanes) {
  for (int c = lane * 8; c < np; c += lanes * 8) {
    float v[8];
    load_upto8<DT>(src, row + c, n - c, v);
    uint4 o[PLANES];
    vl_split8<PLANES>(v, o);
#pragma unroll
    for (int p = 0; p < PLANES; ++p) *reinterpret_cast<uint4*>(dst + p * plane + c) = o[p];
  }
}

// An fp32 row of n elements as fp16 hi and lo, scaled so that its largest element lies in 2^13 .. 2^14 (infinities
// and NaN: as they are); *undo: the inverse of the scale.
__device__ __forceinline__ void vl_half_row(const float* src, int n, int np, uint16_t* dst, int64_t plane, float* undo,
                                            int lane) {
  float most = 0.0f;
  for (int c = lane * 8; c < n; c += 512) {
    float v[8];
    load_upto8<FMOE_F32>(src, c, n - c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
  // 2^shift, shift = 13 - floor(log2(most)), up to 126 (subnormal rows are not scaled up further)
  const int exponent = static_cast<int>(__float_as_uint(most) >> 23) - 127;
  const int shift = most == 0.0f || exponent == 128 ? 0 : min(13 - exponent, 126);
  const float scale = fm_pow2i(shift);
  if (lane == 0) *undo = fm_pow2i(-shift);
  typedef _Float16 half8 __attribute__((ext_vector_type(8)));
  for (int c = lane * 8; c < np; c += 512) {
    float v[8];
    load_upto8<FMOE_F32>(src, c, n - c, v);
    half8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = v[e] * scale;
      hi[e] = static_cast<_Float16>(x);
      lo[e] = static_cast<_Float16>(x - static_cast<float>(hi[e]));
    }
    *reinterpret_cast<half8*>(dst + c) = hi;
    *reinterpret_cast<half8*>(dst + plane + c) = lo;
  }
}

// RB rows per workgroup: 32, two a wave; or 4, four waves each, where that leaves few workgroups.  The zeros up to the next
// multiple of 64 rows are shared out (5 rows x 3832 in fp32: 31 us by one workgroup of 32 rows, 7 us by 16 of 4).
template <int DT, int PLANES, int RB>
__global__ __launch_bounds__(1024) void vl_rows_kernel(const RowsArgs a) {
  constexpr int WAVES = RB < 16 ? 16 / RB : 1;  // per row
  __shared__ uint32_t bits[kFewEntries / 32];
  __shared__ int2 before_s[16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int block0 = static_cast<int>(blockIdx.x) * RB, word = block0 / 32;
  if (a.masks == nullptr) vl_mark_rows(a, 0, a.T, bits);
  const uint32_t* masks = a.masks ? a.masks : bits;
  int before = 0, all = 0;
  for (int i = threadIdx.x; i < (a.T + 31) / 32; i += 1024) {
    const int c = __popc(masks[i]);
    all += c;
    if (i < word) before += c;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off, 64), all += __shfl_xor(all, off, 64);
  if (lane == 0) before_s[w] = make_int2(before, all);
  const uint32_t mask = block0 < a.T ? masks[word] : 0;
  __syncthreads();
  int base = 0, n = 0;
#pragma unroll
  for (int q = 0; q < 16; ++q) base += before_s[q].x, n += before_s[q].y;
  if (block0 == 0 && threadIdx.x == 0) a.head[0] = n;
  for (int r = n + static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) * w; r < pad_rows(n); r += gridDim.x * 16) {
    for (int c = lane * 8; c < a.Dp; c += 512)
#pragma unroll
      for (int p = 0; p < PLANES; ++p)
        *reinterpret_cast<uint4*>(a.h + p * a.plane + static_cast<int64_t>(r) * a.Dp + c) = make_uint4(0, 0, 0, 0);
    if (PLANES == 3 && a.h16) {
      if (lane == 0) a.h_scale[r] = 1.0f;
      for (int c = lane * 8; c < a.Dp; c += 512)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          *reinterpret_cast<uint4*>(a.h16 + p * a.plane + static_cast<int64_t>(r) * a.Dp + c) = make_uint4(0, 0, 0, 0);
    }
  }
  for (int i = w / WAVES; i < RB && block0 + i < a.T; i += 16 / WAVES) {
    const int64_t t = block0 + i;
    const int bit = t & 31;
    const bool first = lane == 0 && w % WAVES == 0;
    if (!((mask >> bit) & 1)) {
      if (first) {
        a.inv[t] = -1;
        if (a.loss) a.loss[t] = 0.0f;
      }
      continue;
    }
    const int r = base + __popc(mask & ((1u << bit) - 1));
    if (first) {
      a.inv[t] = r;
      a.perm[r] = static_cast<int>(t);
      float z;
      if (a.t_dtype < 0) a.out_index[r] = vl_entry(a, t, z);
    }
    vl_copy_row<DT, PLANES>(a.hidden, t * a.ldh, a.D, a.Dp, a.h + static_cast<int64_t>(r) * a.Dp, a.plane,
                            (w % WAVES) * 64 + lane, 64 * WAVES);
    if constexpr (PLANES == 3)
      if (a.h16 && w % WAVES == 0)
        vl_half_row(static_cast<const float*>(a.hidden) + t * a.ldh, a.D, a.Dp, a.h16 + static_cast<int64_t>(r) * a.Dp, a.plane,
                    a.h_scale + r, lane);
  }
}
template <int DT, int PLANES>
void vl_rows_launch(const RowsArgs& r, hipStream_t s) {
  if (r.T <= 1024) vl_rows_kernel<DT, PLANES, 4><<<dim3(static_cast<uint32_t>(std::max((r.T + 3) / 4, 16))), 1024, 0, s>>>(r);
  else vl_rows_kernel<DT, PLANES, 32><<<dim3(static_cast<uint32_t>((r.T + 31) / 32)), 1024, 0, s>>>(r);
}

// Rows v0 .. v0 + rows - 1 of the weight as padded planes: where its rows are not bf16 of a multiple of 64
// elements at 16-byte addresses.
template <int DT, int PLANES>
__global__ __launch_bounds__(256) void vl_pack_kernel(const void* src, int64_t ld, int64_t v0, int rows, int D, int Dp,
                                                      uint16_t* dst, int64_t plane) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  vl_copy_row<DT, PLANES>(src, (v0 + r) * ld, D, Dp, dst + static_cast<int64_t>(r) * Dp, plane, lane, 64);
}

// fp32 rows, as bf16 planes (dst, where wanted) and as scaled fp16 (dst16, where wanted).
__global__ __launch_bounds__(256) void vl_pack32_kernel(const float* src, int64_t ld, int64_t v0, int rows, int D, int Dp,
                                                        uint16_t* dst, uint16_t* dst16, float* undo, int64_t plane) {
  const int lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int64_t at = static_cast<int64_t>(r) * Dp;
  if (dst16) vl_half_row(src + (v0 + r) * ld, D, Dp, dst16 + at, plane, undo + r, lane);
  if (dst) vl_copy_row<FMOE_F32, 3>(src, (v0 + r) * ld, D, Dp, dst + at, plane, lane, 64);
}

// ---- the products ----------------------------------------------------------------------------
// STATS  t = H W^T            -> a maximum and a sum of exponentials per row and 128 columns
// GRAD   t = H W^T of a piece -> G
// DH     G W of a piece, K split in ranges -> fp32 partial sums, added to the piece's before
// DW     G^T H                -> the piece's rows of dW
// PROB   t = H W^T            -> 2^(t - o), and its sum per row and 128 columns
// LOGITS as STATS, and t of the rows
// H and G are row-major, so A is K-contiguous but for DW (G^T: read with transposing LDS reads), and B is
// K-contiguous where logits are formed, and read as it lies, transposing, for DH (W) and DW (H).
// All are bound by the matrix units.  32768 rows x 2048, vocab 131072, bf16: PROB 1.42 PFLOP/s, DH 1.43, DW 1.29 (it also
// adds 1 GB of fp32 a piece), where a library product of such sizes reaches 1.42.  At K = 768 (16384 rows, vocab 50021) PROB
// has only 12 K steps a tile to an epilogue of exponentials and stores, in which the matrix units idle: 1.07; DH 1.30, DW 1.30.
enum VlMode { VL_STATS = 0, VL_GRAD = 1, VL_DH = 2, VL_DW = 3, VL_PROB = 4, VL_LOGITS = 5 };

struct VlGemm {
  const uint16_t *a, *b;
  int64_t a_plane, b_plane;
  int lda, ldb;
  const float *a_scale, *b_scale;  // logits of fp32 operands: what undoes the scaling of the rows of a and of b
  const int* head;      // rows with entries
  int row0, rows;       // the rows of this call: row0 .. row0 + rows - 1 of them (pointers to rows start at row0)
  const int* only_if;   // nothing is done where it holds 0 (nullptr: always)
  int cols;             // logits: vocabulary rows of the piece; DH, DW: columns (Dp)
  int vocab;            // DH, DW: vocabulary rows of the piece
  int k;                // logits: K (Dp)
  int v0;               // logits: the piece's first vocabulary row
  float c;              // t = c * (H W^T)
  const int* index;     // cross entropy: the rows' targets (else nullptr)
  float* picked;        // their t; GRAD: p - 1
  // STATS
  float2* part;         // [2 * column tiles][Tp]
  float* logits;        // LOGITS: t, [rows][ldt]; few rows: as well, where it is not null
  int ldt;              // a multiple of 256
  int64_t Tp;
  const float* off;     // PROB: o
  // GRAD
  const float2* stat;
  const float* d_loss;  // (nullptr: 1)
  const int* perm;      // (and DH)
  float factor;
  int reduction;
  uint16_t* g;
  int64_t g_plane;
  int ldg;              // a multiple of 256
  // DH, DW: the result, out [.][D] of out_dtype; DH: in rows perm
  void* out;
  int D, out_dtype;
  float* sum;           // DH: [Tp][Dp], DW: [vocab][Dp], the sum over the pieces before (add) and for those after (more)
  int add, more;
  const float* row_factor;  // DH: the rows' factors (nullptr: 1)
  const float* all_factor;  // DW: the product's (nullptr: 1)
  float* split;         // fp32 partial tiles
};

// Planes of a pass, the smallest products first: (0, 2), (1, 1), (2, 0), (0, 1), (1, 0), (0, 0); of two planes the last
// three.
__device__ __forceinline__ void vl_planes(int passes, int pass, int& pa, int& pb) {
  const int i = 2 * (pass + 6 - passes);
  pa = (0x124 >> i) & 3;
  pb = (0x046 >> i) & 3;
}

// core::quarter of fp16 operands.
template <int I, int J>
__device__ __forceinline__ void vl_half_quarter(f32x4 (&acc)[core::FM][core::FN], const core::AFrag& a, const core::BFrag& b) {
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int k = x >> 1, n = (x & 1) * 2;
    asm volatile(
        "v_mfma_f32_16x16x32_f16 %[c00], %[p0], %[q0], %[c00]\n"
        "v_mfma_f32_16x16x32_f16 %[c10], %[p0], %[q1], %[c10]\n"
        "v_mfma_f32_16x16x32_f16 %[c01], %[p1], %[q0], %[c01]\n"
        "v_mfma_f32_16x16x32_f16 %[c11], %[p1], %[q1], %[c11]\n"
        : [c00] "+v"(acc[2 * I][4 * J + n]), [c10] "+v"(acc[2 * I + 1][4 * J + n]), [c01] "+v"(acc[2 * I][4 * J + n + 1]),
          [c11] "+v"(acc[2 * I + 1][4 * J + n + 1])
        : [p0] "v"(b[k][n]), [p1] "v"(b[k][n + 1]), [q0] "v"(a[k][0]), [q1] "v"(a[k][1])
        : "memory");
  }
  __builtin_amdgcn_s_setprio(0);
  core::barrier();
}

// Split of DH's and DW's K: with T tiles, the T mod 256 ones of the last, partial round are cut into S ranges
// of K, which leave fp32 partial tiles that a second launch adds in order.  S fills one to four rounds of
// workgroups, whichever takes the fewest steps: a round costs its steps and an epilogue, a partial tile its traffic
// (256 KB written and read), the second launch its own.  (The ranges are walked range by range, so that the
// workgroups of an XCD read the same operand rows at a time.)
struct VlSplit {
  int whole, rest, ranges;  // tiles computed whole, tiles split, ranges of each
};
constexpr int kSplitSlots = 1024;  // partial tiles, at most
__device__ __forceinline__ VlSplit vl_split(int tiles, int units) {
  const int rest = tiles % kVlCus;
  VlSplit best{tiles, 0, 1};
  if (rest == 0) return best;
  float least = static_cast<float>(units) + 2.0f;
#pragma unroll
  for (int rounds = 1; rounds <= 4; ++rounds) {
    const int s = min(rounds * kVlCus / rest, min(units / 8, kSplitSlots / rest));
    const float cost = static_cast<float>(rounds) * (static_cast<float>(units) / static_cast<float>(max(s, 1)) + 2.0f) +
                       0.055f * static_cast<float>(s * rest) + 4.0f;
    if (s >= 2 && cost < least) least = cost, best = VlSplit{tiles - rest, rest, s};
  }
  return best;
}

// Packed rows among the call's row0 .. row0 + rows - 1.
__device__ __forceinline__ int vl_rows_here(const int* head, int row0, int rows) {
  return __builtin_amdgcn_readfirstlane(max(0, min(head[0] - row0, rows)));
}

struct VlItem {
  int tm, tn, u0, un, slot;  // tile, K steps (of all passes), partial tile (-1: the tile is whole)
};

// Tile t: groups of kGroup row tiles, in a group column by column.  The 32 workgroups of an XCD
// share 4 + 8 operand panels instead of 1 + 32.
__device__ __forceinline__ void vl_tile(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int per = kGroup * tiles_n, g = t / per, rem = t - g * per, rows = min(tiles_m - g * kGroup, kGroup);
  const int col = rem / rows;
  tm = __builtin_amdgcn_readfirstlane(g * kGroup + rem - col * rows);
  tn = __builtin_amdgcn_readfirstlane(col);
}

// 8 consecutive values of a row of the result; of several pieces: with the sum so far, or into it.
template <int MODE>
__device__ __forceinline__ void vl_result8(const VlGemm& a, int n, int row, int col, float* v) {
  {
    if (row >= (MODE == VL_DW ? a.vocab : n) || col >= a.D) return;
    float* const s = a.sum + static_cast<int64_t>(row) * a.cols + col;
    if (MODE == VL_DH && a.row_factor) {
      const float f = a.row_factor[row];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * f;
    }
    if (MODE == VL_DW && a.all_factor) {
      const float f = a.all_factor[0];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * f;
    }
    if (a.add) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(s), hi = *reinterpret_cast<const f32x4*>(s + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = lo[e] + v[e], v[4 + e] = hi[e] + v[4 + e];
    }
    if (a.more) {
      *reinterpret_cast<f32x4*>(s) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(s + 4) = f32x4{v[4], v[5], v[6], v[7]};
      return;
    }
    const int64_t o = static_cast<int64_t>(MODE == VL_DW ? row : a.perm[row]) * a.D + col;
    if (a.out_dtype == FMOE_BF16) store_upto8<FMOE_BF16>(a.out, o, a.D - col, v);
    else store_upto8<FMOE_F32>(a.out, o, a.D - col, v);
  }
}

// What a row's p - q are multiplied with.
__device__ __forceinline__ float vl_row_weight(const float* d_loss, const int* perm, int reduction, int n, int row, float factor) {
  const float up = d_loss == nullptr ? 1.0f : reduction == FMOE_REDUCE_NONE ? d_loss[perm[row]] : d_loss[0];
  return (reduction == FMOE_REDUCE_MEAN ? up / static_cast<float>(n) : up) * factor;
}

// (written out: the compiler puts an instruction for quiet NaNs before each operand of its own maximum; a NaN
// among the logits reaches the sum of exponentials whatever the maximum is)
__device__ __forceinline__ float vl_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Epilogue of STATS: maximum and sum of exponentials of each row's 128 columns.  c >= 0 here, so that the
// maximum is taken of the accumulators; the exponent of an element is one multiply-add.  FULL: all columns
// are inside the vocabulary (128 v_exp_f32 and 320 other instructions a lane; with the bounds and a
// product of its own 640).
template <bool FULL>
__device__ __forceinline__ void vl_stats_epilogue(const VlGemm& a, f32x4 (&acc)[core::FM][core::FN], float c, int n,
                                                  int row0, int col0, int piece, int el) {
  using namespace core;
  const int er = el & 15, eg = el >> 4;
  float2 mine = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int row = row0 + 16 * i + er;
    // columns of this lane inside: 16 j + e < lim (opaque, or the comparisons are kept in registers for all rows)
    int lim = a.cols - col0 - 4 * eg;
    asm volatile("" : "+v"(lim));
    if constexpr (!FULL) {
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = 16 * j + e < lim ? acc[i][j][e] : -__builtin_inff();
    }
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < FN; ++j) m = vl_max3(vl_max3(m, acc[i][j][0], acc[i][j][1]), acc[i][j][2], acc[i][j][3]);
    m = fmaxf(m, __shfl_xor(m, 16, 64));
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    // (columns outside, or c = 0: no infinity may meet it)
    if constexpr (!FULL) {
      if (m == -__builtin_inff()) m = 0.0f;
    }
    m = m * c;
    const float peak = m == -__builtin_inff() ? 0.0f : m;  // a sum of zero; NaN stays NaN
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -peak));
        if constexpr (!FULL) x = 16 * j + e < lim ? x : 0.0f;
        s = s + x;
      }
    s = s + __shfl_xor(s, 16, 64);
    s = s + __shfl_xor(s, 32, 64);
    if (eg == i) mine = make_float2(!FULL && s == 0.0f ? -__builtin_inff() : m, s);
    if (a.index) {  // the target's column, where it is in this block
      const int rel = row < n ? a.index[row] - (a.v0 + col0) : -1;
      const bool here = rel >= 0 && rel < WTN && col0 + rel < a.cols;
      if (__ballot(here) != 0) {
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) t = rel == 16 * j + 4 * eg + e ? acc[i][j][e] : t;
        if (here && ((rel >> 2) & 3) == eg) a.picked[row] = t * c;
      }
    }
  }
  const int row = row0 + el;  // lane group eg kept block eg
  if (row < n) a.part[static_cast<int64_t>(piece) * a.Tp + row] = mine;
}

// 16 rows of G (block i of the accumulators) through the wave's LDS into 16-byte stores, plane by plane.
template <int PLANES, bool FULL>
__device__ __forceinline__ void vl_store_g(const VlGemm& a, f32x4 (&acc)[core::FN], uint8_t* ep, int np, int row, int col0,
                                           int el) {
  using namespace core;
  const int er = el & 15, eg = el >> 4;
#pragma unroll 1  // (three at once would spill)
  for (int p = 0; p < PLANES; ++p) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int col = j * 16 + eg * 4;
      uint2 u;
      u.x = pack2(acc[j][0], acc[j][1]);
      u.y = pack2(acc[j][2], acc[j][3]);
      *reinterpret_cast<uint2*>(ep + er * 256 + ((((col >> 3) ^ er)) << 4) + (col & 7) * 2) = u;
      if constexpr (PLANES > 1) {
        acc[j][0] = acc[j][0] - __uint_as_float(u.x << 16);
        acc[j][1] = acc[j][1] - __uint_as_float(u.x & 0xffff0000u);
        acc[j][2] = acc[j][2] - __uint_as_float(u.y << 16);
        acc[j][3] = acc[j][3] - __uint_as_float(u.y & 0xffff0000u);
      }
    }
    __builtin_amdgcn_wave_barrier();
    // uniform addresses, one offset per lane
    uint8_t* const base = reinterpret_cast<uint8_t*>(a.g + p * a.g_plane + static_cast<int64_t>(row) * a.ldg + col0);
    const uint32_t voff = static_cast<uint32_t>(eg * a.ldg + er * 8) * 2u;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int r = t * 4 + eg;
      const uint4 v = *reinterpret_cast<const uint4*>(ep + r * 256 + ((er ^ r) << 4));
      if (FULL || row + r < np)
        *reinterpret_cast<uint4*>(base + static_cast<int64_t>(8 * t) * a.ldg + voff) = v;
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
}

// Epilogue of GRAD.  With one plane, 2^(t - m - l) takes one multiply-add (m + l rounded: 2^-24 of some tens in
// the exponent, far below G's own half step of 2^-8); with three, m is subtracted first.
template <int PLANES, bool FULL>
__device__ __forceinline__ void vl_grad_epilogue(const VlGemm& a, f32x4 (&acc)[core::FM][core::FN], uint8_t* ep, int n,
                                                 int np, int row0, int col0, int el) {
  using namespace core;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    asm volatile("" ::: "memory");  // (the rows' values of all blocks at once would spill)
    asm volatile("" : "+v"(el));
    const int er = el & 15, eg = el >> 4;
    const int row = row0 + 16 * i + er;
    float2 ml = make_float2(0.0f, 0.0f);
    float up = 0.0f;
    int rel = -1;
    if (row < n) {
      ml = a.stat[row];
      up = vl_row_weight(a.d_loss, a.perm, a.reduction, n, row, a.factor);
      if (a.index) rel = a.index[row] - (a.v0 + col0);
    }
    const float off = PLANES == 1 ? -(ml.x + ml.y) : -ml.x;
    int lim = row < n ? a.cols - col0 - 4 * eg : 0;  // as above; none in rows that are padding
    asm volatile("" : "+v"(lim));
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = fmaf(acc[i][j][e], a.c, off);
        if constexpr (PLANES > 1) x = x - ml.y;
        x = __builtin_amdgcn_exp2f(x) * up;
        if constexpr (!FULL) x = 16 * j + e < lim ? x : 0.0f;
        acc[i][j][e] = x;
      }
    const bool here = rel >= 0 && rel < WTN && col0 + rel < a.cols;
    if (__ballot(here) != 0) {  // the target
      const float v = here ? a.picked[row] * up : 0.0f;
      const int at = here ? rel : -1;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = at == 16 * j + 4 * eg + e ? v : acc[i][j][e];
    }
    vl_store_g<PLANES, FULL>(a, acc[i], ep, np, row0 + 16 * i, col0, el);
  }
}

// Epilogue of PROB: 2^(t - o), one multiply-add and one exponential an element, and its sum over the row's 128
// columns (in fp32, before the elements are rounded).
template <int PLANES, bool FULL>
__device__ __forceinline__ void vl_prob_epilogue(const VlGemm& a, f32x4 (&acc)[core::FM][core::FN], uint8_t* ep, int n,
                                                 int np, int row0, int col0, int piece, int el) {
  using namespace core;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    asm volatile("" ::: "memory");  // (as in GRAD's)
    asm volatile("" : "+v"(el));
    const int er = el & 15, eg = el >> 4;
    const int row = row0 + 16 * i + er;
    const float off = row < n ? a.off[row] : 0.0f;
    const int rel = row < n && a.index ? a.index[row] - (a.v0 + col0) : -1;
    const bool here = rel >= 0 && rel < WTN && col0 + rel < a.cols;
    if (__ballot(here) != 0) {  // the target's t
      float t = 0.0f;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) t = rel == 16 * j + 4 * eg + e ? acc[i][j][e] : t;
      if (here && ((rel >> 2) & 3) == eg) a.picked[row] = t * a.c;
    }
    int lim = row < n ? a.cols - col0 - 4 * eg : 0;
    asm volatile("" : "+v"(lim));
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], a.c, -off));
        if constexpr (!FULL) x = 16 * j + e < lim ? x : 0.0f;
        s = s + x;
        acc[i][j][e] = x;
      }
    s = s + __shfl_xor(s, 16, 64);
    s = s + __shfl_xor(s, 32, 64);
    if (eg == 0 && row < n) a.part[static_cast<int64_t>(piece) * a.Tp + row] = make_float2(off, s);
    vl_store_g<PLANES, FULL>(a, acc[i], ep, np, row0 + 16 * i, col0, el);
  }
}

template <int MODE, int PLANES>
__global__ __launch_bounds__(core::NT, 1) void vl_gemm_kernel(const VlGemm a) {
  using namespace core;
  constexpr bool ATR = MODE == VL_DW, BTR = MODE == VL_DH || MODE == VL_DW, SPLIT = MODE == VL_DH || MODE == VL_DW;
  constexpr bool HALF = PLANES == 3 && !BTR;  // logits of fp32 operands: fp16 hi and lo
  constexpr int PASSES = PLANES == 1 ? 1 : HALF ? 3 : 6;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[SMEM];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / WN, wn = w % WN;
  const uint32_t sbase = lds_addr(smem);
  if (a.only_if && a.only_if[0] == 0) return;
  const int n = vl_rows_here(a.head, a.row0, a.rows);
  if (a.row0 > 0 && n == 0) return;
  const int np = pad_rows(n);
  const int m_rows = MODE == VL_DW ? a.vocab : np;
  const int tiles_m = (m_rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN;
  const int nk = MODE == VL_DH ? (a.vocab + BK - 1) / BK : MODE == VL_DW ? np / BK : a.k / BK;
  const int units = nk * PASSES, tiles = tiles_m * tiles_n;
  const VlSplit sp = SPLIT ? vl_split(tiles, units) : VlSplit{tiles, 0, 1};
  // Workgroup b runs on XCD b % 8.  Each XCD takes a contiguous eighth of the whole tiles, then of the ranges.
  const int xcd = static_cast<int>(blockIdx.x) % 8, slot = static_cast<int>(blockIdx.x) / 8, step = static_cast<int>(gridDim.x) / 8;
  auto share = [&](int items, int& first) {
    const int lo = static_cast<int>(static_cast<int64_t>(items) * xcd / 8), hi = static_cast<int>(static_cast<int64_t>(items) * (xcd + 1) / 8);
    first = lo + slot;
    return max(hi - first + step - 1, 0) / step;
  };
  int first_whole, first_range = 0;
  const int my_whole = share(sp.whole, first_whole);
  const int my_items = my_whole + (SPLIT ? share(sp.rest * sp.ranges, first_range) : 0);
  if (my_items <= 0) return;

  auto locate = [&](int i) __attribute__((always_inline)) {
    VlItem t{0, 0, 0, units, -1};
    int tile = first_whole + i * step;
    if (SPLIT && i >= my_whole) {
      const int q = first_range + (i - my_whole) * step, range = q / sp.rest;
      tile = sp.whole + q - range * sp.rest;
      t.u0 = static_cast<int>(static_cast<int64_t>(units) * range / sp.ranges);
      t.un = static_cast<int>(static_cast<int64_t>(units) * (range + 1) / sp.ranges) - t.u0;
      t.slot = q;
    }
    vl_tile(tile, tiles_m, tiles_n, t.tm, t.tn);
    t.u0 = __builtin_amdgcn_readfirstlane(t.u0);
    t.un = __builtin_amdgcn_readfirstlane(t.un);
    t.slot = __builtin_amdgcn_readfirstlane(t.slot);
    return t;
  };

  // ---- copy cursor (the units of a stage and their LDS layout as in gemm_core.h)
  const uint32_t lds_a = ATR ? sbase + w * 1024 : sbase + (64 * (w >> 2) + 8 * (w & 3)) * RB;
  const uint32_t lds_b = sbase + A_BYTES + w * 1024;
  const int lda = a.lda, ldb = a.ldb;
  int c_ti = 0, c_tm, c_tn, c_u, c_end, c_left = 0, c_run;  // item, its tile, the next call's K step and its last one
  const uint8_t *c_a = nullptr, *c_b = nullptr;
  int64_t astep = ATR ? static_cast<int64_t>(2 * BK) * lda : RB, bstep = BTR ? static_cast<int64_t>(2 * BK) * ldb : RB;
  uint32_t a_off[4], b_off[4];
  // this lane's offsets from c_a and c_b; k: the step's first K
  auto form_offsets = [&](int k) __attribute__((always_inline)) {
    // the lane as an opaque value: what follows is formed here, not kept through the main loop
    int l = lane;
    asm volatile("" : "+v"(l));
    const int dchunk = (l & 7) ^ swzk(l >> 3);
    const int krow = 4 * w + (l >> 4);
    const int cb = ((((l & 15) >> 1) ^ wsw(krow)) << 1) | (l & 1);
    if constexpr (ATR) {
      // unit u: rows (of C) 32 u .. + 31 of every wave's 64
      const int m0 = c_tm * BM;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        a_off[q] = static_cast<uint32_t>((32 * (q & 1) + krow) * lda +
                                         min(m0 + 64 * (cb >> 2) + 32 * (q >> 1) + 8 * (cb & 3), lda - 8)) * 2u;
    } else {
      const int last_m = min(m_rows - c_tm * BM, BM) - 1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = min(64 * (w >> 2) + 8 * (w & 3) + (l >> 3) + 128 * (q & 1) + 32 * (q >> 1), last_m);
        a_off[q] = static_cast<uint32_t>(r * lda + dchunk * 8) * 2u;
      }
    }
    if constexpr (BTR) {
      const int n0 = c_tn * BN, last_k = MODE == VL_DH ? a.vocab - 1 - k : BK;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        b_off[q] = static_cast<uint32_t>(min(32 * (q & 1) + krow, last_k) * ldb +
                                         min(n0 + 128 * (cb >> 3) + 8 * (cb & 7) + 64 * (q >> 1), a.cols - 8)) * 2u;
    } else {
      const int last_n = min(a.cols - c_tn * BN, BN) - 1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = min(128 * (q & 1) + 64 * (q >> 1) + 8 * w + (l >> 3), last_n);
        b_off[q] = static_cast<uint32_t>(r * ldb + dchunk * 8) * 2u;
      }
    }
  };
  // pointers and offsets of K step c_u of the item, and the steps until the next call
  auto place = [&]() __attribute__((always_inline)) {
    int pa = 0, pb = 0, ku = c_u;
    if constexpr (PASSES > 1) {
      const int pass = c_u / nk;
      ku = c_u - pass * nk;
      vl_planes(PASSES, pass, pa, pb);
    }
    const int k = ku * BK;
    const uint16_t* p = a.a + pa * a.a_plane + (ATR ? static_cast<int64_t>(k) * lda : static_cast<int64_t>(c_tm) * BM * lda + k);
    const uint16_t* q = a.b + pb * a.b_plane + (BTR ? static_cast<int64_t>(k) * ldb : static_cast<int64_t>(c_tn) * BN * ldb + k);
    c_a = reinterpret_cast<const uint8_t*>(p);
    c_b = reinterpret_cast<const uint8_t*>(q);
    c_run = min(c_end - c_u, nk - ku);
    // the last step of a vocabulary that is no multiple of 64 has clamped rows of its own
    if (MODE == VL_DH && (a.vocab & (BK - 1)) && ku + c_run == nk && c_run > 1) --c_run;
    c_left = c_run;
    form_offsets(k);
  };
  auto take = [&](int i) __attribute__((always_inline)) {
    const VlItem t = locate(i);
    c_tm = t.tm, c_tn = t.tn, c_u = t.u0, c_end = t.u0 + t.un;
  };
  take(0);
  place();
  // A stage's units are issued in the order A0, B0, B1, A1; A1 moves the cursor on.  Past the last
  // step the last stage is copied again (into slots that are free and not read any more).
  auto advance = [&]() __attribute__((always_inline)) {
    c_u += c_run;
    if (c_u == c_end) {
      if (++c_ti == my_items) {
        c_a -= astep;
        c_b -= bstep;
        astep = bstep = 0;
        c_left = INT32_MAX;
        return;
      }
      take(c_ti);
    }
    place();
  };
  auto issue_a = [&](int it, int u) __attribute__((always_inline)) {
    const uint32_t st = lds_a + (it & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      copy16(ATR ? st + u * UNIT + i * 8192 : st + (128 * i + 32 * u) * RB, c_a, a_off[2 * u + i]);
    if (u == 0) return;
    c_a += astep;
    c_b += bstep;
    if (__builtin_expect(--c_left == 0, 0)) advance();
  };
  auto issue_b = [&](int it, int u) __attribute__((always_inline)) {
    const uint32_t st = lds_b + (it & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      copy16(BTR ? st + u * UNIT + i * 8192 : st + (128 * i + 64 * u) * RB, c_b, b_off[2 * u + i]);
  };

  uint32_t xa = ATR ? tr_base(2 * wm, lane) : frag_base(wm * WTM, lane);
  uint32_t xb = A_BYTES + (BTR ? tr_base(4 * wn, lane) : frag_base(wn * WTN, lane));
  AFrag a0, a1;
  BFrag b0, b1;
  typedef __attribute__((address_space(3))) bf16x8 lds_bf16x8;
  auto lds_frag = [&](uint32_t x, uint32_t src, int kh, int f) {
    return *(const lds_bf16x8*)(uintptr_t)((x ^ (kh * 64u)) + src + 2048u * f);
  };
  auto read_a = [&](AFrag& f, int u, uint32_t src, int kh, int m) {
    if constexpr (ATR) f[kh][m] = tr_frag(((src + xa) ^ (m << 5)) + u * UNIT + kh * TR_KHALF);
    else f[kh][m] = lds_frag(xa, src, kh, 2 * u + m);
  };
  auto read_b = [&](BFrag& f, int u, uint32_t src, int kh, int q) {
    if constexpr (BTR) f[kh][q] = tr_frag(((src + xb) ^ (q << 5)) + u * UNIT + kh * TR_KHALF);
    else f[kh][q] = lds_frag(xb, src, kh, 4 * u + q);
  };
  auto read_first = [&](uint32_t src) {
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int m = 0; m < 2; ++m) read_a(a0, 0, src, kh, m);
#pragma unroll
    for (int q = 0; q < 4; ++q) read_b(b0, 0, src, 0, q);
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
  auto step_quarter = [&](auto i, auto j, const AFrag& x, const BFrag& y) __attribute__((always_inline)) {
    if constexpr (HALF) vl_half_quarter<decltype(i)::value, decltype(j)::value>(acc, x, y);
    else quarter<decltype(i)::value, decltype(j)::value>(acc, x, y);
  };
  uint8_t* ep = smem + 2 * STAGE + w * EPI;  // this wave's staging (4 KB)
  int e_ti = 0, e_left = locate(0).un;
  for (int it = 0;; ++it) {
    // keep the per-step fragment addresses from being hoisted out of the loop
    asm volatile("" : "+v"(xa), "+v"(xb));
    const uint32_t st = sbase + (it & 1) * STAGE, nxt = sbase + ((it + 1) & 1) * STAGE;
    // (0, 0)
#pragma unroll
    for (int q = 0; q < 4; ++q) read_b(b0, 0, st, 1, q);
    issue_a(it + 1, 1);
    wait_vm_barrier<5 * LU>();  // B1 of this stage
    step_quarter(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{}, a0, b0);
    // (0, 1)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int q = 0; q < 4; ++q) read_b(b1, 1, st, kh, q);
    issue_a(it + 2, 0);
    wait_vm_barrier<5 * LU>();  // A1 of this stage
    step_quarter(std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{}, a0, b1);
    // (1, 0)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int m = 0; m < 2; ++m) read_a(a1, 1, st, kh, m);
    issue_b(it + 2, 0);
    wait_vm_barrier<4 * LU>();  // A0, B0 of the next stage
    step_quarter(std::integral_constant<int, 1>{}, std::integral_constant<int, 0>{}, a1, b0);
    // (1, 1): the next step's first fragments (at a tile's end they are read again after its epilogue)
    read_first(nxt);
    issue_b(it + 2, 1);
    wait_lds_barrier();
    step_quarter(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, a1, b1);

    if (--e_left > 0) continue;
    // ---- tile epilogue: this wave's 64 x 128 block (both wave groups together)
    if (!late) barrier();
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3\n" ::: "memory");  // MFMA results -> VALU reads
    int el = lane;
    asm volatile("" : "+v"(el));  // the address arithmetic below stays out of the main loop
    const VlItem t = locate(e_ti);
    const int row0 = t.tm * BM + wm * WTM, col0 = t.tn * BN + wn * WTN;
    const int er = el & 15, eg = el >> 4;  // acc[i][j]: row 16 i + er, columns 16 j + 4 eg + 0..3

    if constexpr (HALF) {
      // the scales together first: powers of two, whose product is exact; with one of them alone a large row against a small
      // one would leave fp32's range
      float rs[FM];
#pragma unroll
      for (int i = 0; i < FM; ++i) rs[i] = a.a_scale[min(row0 + 16 * i + er, np - 1)];
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float cs = a.b_scale[min(col0 + 16 * j + 4 * eg + e, a.cols - 1)];
#pragma unroll
          for (int i = 0; i < FM; ++i) acc[i][j][e] = acc[i][j][e] * (rs[i] * cs);
        }
      }
    }
    if constexpr (MODE == VL_STATS || MODE == VL_LOGITS) {
      float c = a.c;
      if (c < 0.0f) {
        c = -c;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = -acc[i][j];
      }
      if constexpr (MODE == VL_LOGITS) {
        // 16 bytes a lane, 64 of a row; the next store takes the other half of its 128
        float* const out = a.logits + static_cast<int64_t>(row0) * a.ldt + col0;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          int l = el;
          asm volatile("" : "+v"(l));
          const int r = 16 * i + (l & 15);
          if (row0 + r >= n) continue;
          float* const p = out + r * a.ldt + 4 * (l >> 4);
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            asm volatile("" ::: "memory");
            *reinterpret_cast<f32x4*>(p + 16 * j) = acc[i][j] * c;
          }
        }
      }
      const int piece = (a.v0 / BN + t.tn) * WN + wn;
      if (col0 + WTN <= a.cols) vl_stats_epilogue<true>(a, acc, c, n, row0, col0, piece, el);
      else vl_stats_epilogue<false>(a, acc, c, n, row0, col0, piece, el);
    } else if constexpr (MODE == VL_PROB) {
      const int piece = (a.v0 / BN + t.tn) * WN + wn;
      if (row0 + WTM <= n && col0 + WTN <= a.cols) vl_prob_epilogue<PLANES, true>(a, acc, ep, n, np, row0, col0, piece, el);
      else vl_prob_epilogue<PLANES, false>(a, acc, ep, n, np, row0, col0, piece, el);
    } else if constexpr (MODE == VL_GRAD) {
      if (row0 + WTM <= n && col0 + WTN <= a.cols) vl_grad_epilogue<PLANES, true>(a, acc, ep, n, np, row0, col0, el);
      else vl_grad_epilogue<PLANES, false>(a, acc, ep, n, np, row0, col0, el);
    } else if (t.slot >= 0) {
      // a range's partial tile, as it lies in the accumulators; 16-row slices without valid rows left out
      float* part = a.split + static_cast<int64_t>(t.slot) * (BM * BN);
      const int valid = (MODE == VL_DW ? a.vocab : n) - t.tm * BM;
#pragma unroll
      for (int i = 0; i < FM; ++i)
        if (wm * WTM + 16 * i < valid)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            *reinterpret_cast<f32x4*>(part + (wm * WTM + 16 * i + er) * BN + wn * WTN + 16 * j + 4 * eg) = acc[i][j];
    } else {
      // 16 rows x 64 columns of fp32 at a time through LDS (chunk c of row r at slot c ^ r), 8 consecutive values
      // of a row per lane
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int jh = 0; jh < FN / 4; ++jh) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f32x4*>(ep + er * 256 + (((4 * j + eg) ^ er) << 4)) = acc[i][4 * jh + j];
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int r = 8 * p + (el >> 3), c = (el & 7) * 8;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(ep + r * 256 + (((c >> 2) ^ r) << 4));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(ep + r * 256 + ((((c >> 2) + 1) ^ r) << 4));
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            vl_result8<MODE>(a, n, row0 + 16 * i + r, col0 + 64 * jh + c, v);
          }
          __builtin_amdgcn_wave_barrier();
        }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    asm volatile("s_nop 1" ::: "memory");  // VALU writes -> MFMA reads of the accumulators
    if (++e_ti == my_items) break;
    e_left = locate(e_ti).un;
    if constexpr (MODE == VL_GRAD || MODE == VL_PROB || MODE == VL_LOGITS) {
      // formed again: kept across the epilogue they made it spill
      form_offsets(0);
      xa = frag_base(wm * WTM, el);
      xb = A_BYTES + frag_base(wn * WTN, el);
    }
    // the next tile's first fragments
    read_first(sbase + ((it + 1) & 1) * STAGE);
    if (late) barrier();
  }
  // the copies past the end have landed before the workgroup's LDS is given back
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Joins the maximum and sum of exponentials of other columns.
__device__ __forceinline__ void vl_join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), peak = top == -__builtin_inff() ? 0.0f : top;
  s = s * __builtin_amdgcn_exp2f(m - peak) + s2 * __builtin_amdgcn_exp2f(m2 - peak);
  m = top;
}

// ---- logits of few rows ------------------------------------------------------------------------------
// Up to 64 rows (T, which the host knows): bound by the read of the weight, which a 256-row tile would stream through
// few workgroups (37 rows, vocab 32768, dim 768: 128 tiles).  A workgroup takes 128 columns, a wave 16 of them and all
// rows; the wave's part of the weight goes from memory straight into the fragments, as it lies (any dtype, stride and
// alignment: no packed copy), the rows' K piece through LDS.  The loads of 8 steps (4 of 64 rows, for registers) are issued at a
// time, 512 bytes of each weight row: issued one by one, 64 bytes of 32768 rows all over the chip, they reach half of
// the memory's rate (5 rows x 2048, vocab 131072: 164 us, in groups 116, 4.6 TB/s; 37 x 768 x 32768: 26 and 23).
// planes = 3: the products are v_mfma_f32_16x16x4_f32 on fp32 operands, which are done as the weight arrives up to 32 rows;
// 49 rows x 3832, vocab 24448, are bound by them (200 us; 5 rows 97).
constexpr int kThinRows = 64;
constexpr int kThinBytes = 1024;             // of a row's K piece in LDS
constexpr int kThinRow = kThinBytes + 16;    // (the 16 rows of a fragment in different banks)

struct ThinWeight {
  const void* p;
  int64_t ld;
  int D;
};

// One lane's operand of a step: E consecutive elements of its weight row.
template <int WT, int PLANES>
struct ThinFrag {
  uint32_t u[WT == FMOE_F32 && PLANES == 1 ? 8 : 4];
};
// 16 bytes of a packed row's K piece: bf16, or the three parts of four fp32 numbers.
// (or, read as they lie, 16 bytes)
template <int PLANES, bool DIRECT>
struct ThinRow {
  uint2 u[PLANES == 3 && !DIRECT ? 3 : 2];
};

// DIRECT (cross entropy's STATS): the rows are read as they lie, by the targets that every wave looks at itself, and this kernel
// packs them for the backward, instead of a launch before it (37 rows x 768, vocab 32768: 23.6 and 20.7 us of a call without
// gradients; fp32, 20 x 1024 x 50021: 69 and 57).
template <int MODE, int WT, int PLANES, int MB, bool DIRECT>
__global__ __launch_bounds__(512, 4) void vl_thin_kernel(const VlGemm a, const ThinWeight wt, const RowsArgs ra) {
  constexpr bool F = PLANES == 3;
  constexpr int E = F ? 4 : 8;               // elements per lane and step; a step is 4 E of K
  // (RING steps' loads are issued while RING others are multiplied)
  constexpr int KC = kThinBytes / (F ? 4 : 2), STEPS = KC / (4 * E), RING = (WT == FMOE_F32 && PLANES == 1 ? 4 : 8) / (MB == 4 ? 2 : 1);
  constexpr int HV = MB * 2;                 // 16-byte pieces of the rows per thread
  static_assert(STEPS == 16 && HV * 512 == 16 * MB * 64);
  __shared__ __attribute__((aligned(16))) uint8_t hs[16 * MB * kThinRow];
  __shared__ float2 red[8][16 * MB];
  __shared__ int rows_s[DIRECT ? kThinRows : 1], target_s[DIRECT ? kThinRows : 1];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int er = lane & 15, eg = lane >> 4;
  const int D = wt.D;
  const int full = D / (4 * E), total = (D + 4 * E - 1) / (4 * E);
  const int col0 = blockIdx.x * 128 + 16 * w;  // of the piece
  const int64_t row_at = static_cast<int64_t>(a.v0 + min(col0 + er, a.cols - 1)) * wt.ld;

  typedef ThinFrag<WT, PLANES> Frag;
  auto load = [&](int g) __attribute__((always_inline)) {
    Frag f;
    const int64_t at = row_at + (g * 4 * E + eg * E);
    if constexpr (WT == FMOE_BF16) {
      f = __builtin_bit_cast(Frag, load_raw<FMOE_BF16, 8>(wt.p, at));
    } else {
      const f32x4_e4* p = reinterpret_cast<const f32x4_e4*>(static_cast<const float*>(wt.p) + at);
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        const f32x4 x = p[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) f.u[4 * q + i] = __float_as_uint(x[i]);
      }
    }
    return f;
  };
  Frag ring[2][RING];
#pragma unroll
  for (int g = 0; g < RING; ++g)
    if (g < full) ring[0][g] = load(g);
  int count = 0;
  if constexpr (DIRECT) {
    float z;
    const int target = lane < ra.T ? vl_entry(ra, lane, z) : kNone;
    const uint64_t has = __ballot(target != kNone);
    count = __popcll(has);
    const int r = __popcll(has & ((uint64_t(1) << lane) - 1));
    if (w == 0) {
      if (target != kNone) rows_s[r] = lane, target_s[r] = target;
      if (blockIdx.x == 0) {
        if (lane == 0) ra.head[0] = count;
        if (lane < ra.T) ra.inv[lane] = target != kNone ? r : -1;
        if (target != kNone) ra.perm[r] = lane, ra.out_index[r] = target;
        else if (lane < ra.T && ra.loss) ra.loss[lane] = 0.0f;
      }
    }
    __syncthreads();
  }
  // the rows' K piece from step g0 on (zeros up to Dp, a multiple of 64; what is past that is not read)
  ThinRow<PLANES, DIRECT> hv[HV];
  auto load_rows = [&](int g0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HV; ++i) {
      const int r = 8 * i + w, k = g0 * 4 * E + lane * E;
      if constexpr (DIRECT) {
        hv[i].u[0] = hv[i].u[1] = make_uint2(0, 0);
        if (r < count && k < D) {
          const int64_t at = __builtin_amdgcn_readfirstlane(rows_s[r]) * ra.ldh + k;
          if constexpr (F) {
            const f32x4 x = *reinterpret_cast<const f32x4_e4*>(static_cast<const float*>(ra.hidden) + at);
            hv[i].u[0] = make_uint2(__float_as_uint(x[0]), __float_as_uint(x[1]));
            hv[i].u[1] = make_uint2(__float_as_uint(x[2]), __float_as_uint(x[3]));
          } else {
            const Raw<FMOE_BF16, 8> x = load_raw<FMOE_BF16, 8>(ra.hidden, at);
            hv[i].u[0] = make_uint2(x.u[0], x.u[1]), hv[i].u[1] = make_uint2(x.u[2], x.u[3]);
          }
        }
      } else if (k < a.lda) {
        const uint16_t* p = a.a + static_cast<int64_t>(r) * a.lda + k;
        if constexpr (F) {
#pragma unroll
          for (int q = 0; q < 3; ++q) hv[i].u[q] = *reinterpret_cast<const uint2*>(p + q * a.a_plane);
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(p);
          hv[i].u[0] = make_uint2(x.x, x.y), hv[i].u[1] = make_uint2(x.z, x.w);
        }
      }
    }
  };
  load_rows(0);

  f32x4 acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Frag& f, int s) __attribute__((always_inline)) {
    const uint8_t* hp = hs + er * kThinRow + s * 64 + eg * 16;
    if constexpr (F) {
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(hp + m * 16 * kThinRow);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          acc[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f.u[i]), x[i], acc[m], 0, 0, 0);
      }
    } else {
      bf16x8 b;
      if constexpr (WT == FMOE_F32) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(f.u[i]);
        b = __builtin_bit_cast(bf16x8, pack8(v));
      } else {
        b = __builtin_bit_cast(bf16x8, f);
      }
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const bf16x8 x = *reinterpret_cast<const bf16x8*>(hp + m * 16 * kThinRow);
        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, x, acc[m], 0, 0, 0);
      }
    }
  };
  for (int g0 = 0; g0 < total; g0 += STEPS) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HV; ++i) {
      uint4 v;
      if constexpr (F && !DIRECT) {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 2; q >= 0; --q) {  // exact: the parts of one fp32 number
          const uint2 u = hv[i].u[q];
          x[0] += __uint_as_float(u.x << 16), x[1] += __uint_as_float(u.x & 0xffff0000u);
          x[2] += __uint_as_float(u.y << 16), x[3] += __uint_as_float(u.y & 0xffff0000u);
        }
        v = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      } else {
        v = make_uint4(hv[i].u[0].x, hv[i].u[0].y, hv[i].u[1].x, hv[i].u[1].y);
      }
      *reinterpret_cast<uint4*>(hs + (8 * i + w) * kThinRow + lane * 16) = v;
    }
    __syncthreads();
    if (g0 + STEPS < total) load_rows(g0 + STEPS);  // under this piece's products
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s % RING == 0) {
#pragma unroll
        for (int g = 0; g < RING; ++g)
          if (g0 + s + RING + g < full) ring[(s / RING + 1) & 1][g] = load(g0 + s + RING + g);
      }
      if (g0 + s < full) multiply(ring[(s / RING) & 1][s % RING], s);
    }
  }
  if (full < total) {  // the end of rows whose length is no multiple of a step's
    const int k = full * 4 * E + eg * E;
    float v[8];
    load_upto8<WT>(wt.p, row_at + k, min(max(D - k, 0), E), v);
    Frag f;
    if constexpr (WT == FMOE_BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f.u[i] = pack2(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) f.u[i] = __float_as_uint(v[i]);
    }
    multiply(f, full % STEPS);
  }
  const int n = DIRECT ? count : vl_rows_here(a.head, 0, kThinRows);

  // acc[m] of lane l: row 16 m + l % 16, columns col0 + 4 (l / 16) + 0..3
  const int lim = a.cols - col0 - 4 * eg;
  if constexpr (MODE == VL_STATS) {
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int row = 16 * m + er;
      float t[4], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t[e] = e < lim ? acc[m][e] * a.c : -__builtin_inff();
        top = fmaxf(top, t[e]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float peak = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = sum + __builtin_amdgcn_exp2f(t[e] - peak);
      sum = sum + __shfl_xor(sum, 16, 64);
      sum = sum + __shfl_xor(sum, 32, 64);
      if (eg == 0) red[w][row] = make_float2(top, sum);
      if (a.logits && row < n)
        *reinterpret_cast<f32x4*>(a.logits + static_cast<int64_t>(row) * a.ldt + (col0 + 4 * eg)) = f32x4{t[0], t[1], t[2], t[3]};
      if (a.index && row < n) {
        const int rel = (DIRECT ? target_s[row] : a.index[row]) - (a.v0 + col0) - 4 * eg;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (rel == e && e < lim) a.picked[row] = t[e];
      }
    }
    __syncthreads();
    if (tid < 16 * MB && tid < n) {
      float2 ms = red[0][tid];
#pragma unroll
      for (int q = 1; q < 8; ++q) vl_join(ms.x, ms.y, red[q][tid].x, red[q][tid].y);
      a.part[static_cast<int64_t>(a.v0 / 128 + blockIdx.x) * a.Tp + tid] = ms;
    }
    if constexpr (DIRECT) {  // the packed rows, and zeros up to 64, a wave each
      for (int r = blockIdx.x * 8 + w; r < kThinRows; r += gridDim.x * 8) {
        uint16_t* const h = ra.h + static_cast<int64_t>(r) * ra.Dp;
        if (r < count)
          vl_copy_row<F ? FMOE_F32 : FMOE_BF16, PLANES>(ra.hidden, rows_s[r] * ra.ldh, D, ra.Dp, h, ra.plane, lane, 64);
        else
          for (int c = lane * 8; c < ra.Dp; c += 512)
#pragma unroll
            for (int p = 0; p < PLANES; ++p) *reinterpret_cast<uint4*>(h + p * ra.plane + c) = make_uint4(0, 0, 0, 0);
      }
    }
  } else {
    // 128 columns of G per row, a plane at a time through LDS into whole lines
    constexpr int LD = 128 * 2 + 16;
    float v[MB][4];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      const int row = 16 * m + er;
      float2 ml = make_float2(0.0f, 0.0f);
      float up = 0.0f;
      int rel = -1;
      if (row < n) {
        ml = a.stat[row];
        up = vl_row_weight(a.d_loss, a.perm, a.reduction, n, row, a.factor);
        if (a.index) rel = a.index[row] - (a.v0 + col0) - 4 * eg;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f((acc[m][e] * a.c - ml.x) - ml.y);
        v[m][e] = row < n && e < lim ? (rel == e ? a.picked[row] : p) * up : 0.0f;
      }
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const uint2 u = make_uint2(pack2(v[m][0], v[m][1]), pack2(v[m][2], v[m][3]));
        *reinterpret_cast<uint2*>(hs + (16 * m + er) * LD + 32 * w + 8 * eg) = u;
        v[m][0] = v[m][0] - __uint_as_float(u.x << 16);
        v[m][1] = v[m][1] - __uint_as_float(u.x & 0xffff0000u);
        v[m][2] = v[m][2] - __uint_as_float(u.y << 16);
        v[m][3] = v[m][3] - __uint_as_float(u.y & 0xffff0000u);
      }
      __syncthreads();
      for (int i = tid; i < kThinRows * 16; i += 512) {
        const int r = i >> 4, c = i & 15;
        const uint4 x = r < 16 * MB ? *reinterpret_cast<const uint4*>(hs + r * LD + c * 16) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(a.g + p * a.g_plane + static_cast<int64_t>(r) * a.ldg + blockIdx.x * 128 + c * 8) = x;
      }
    }
  }
}

template <int MODE, int WT, int PLANES, bool DIRECT = false>
void vl_thin_launch(const VlGemm& a, const ThinWeight& w, int64_t T, dim3 grid, hipStream_t s, const RowsArgs& r = {}) {
  if (T <= 16) vl_thin_kernel<MODE, WT, PLANES, 1, DIRECT><<<grid, 512, 0, s>>>(a, w, r);
  else if (T <= 32) vl_thin_kernel<MODE, WT, PLANES, 2, DIRECT><<<grid, 512, 0, s>>>(a, w, r);
  else vl_thin_kernel<MODE, WT, PLANES, 4, DIRECT><<<grid, 512, 0, s>>>(a, w, r);
}
// Rows that the kernel may read itself: whole 16-byte pieces, and not rounded on the way.
bool vl_is_direct(int h_dtype, int planes, int64_t D) {
  return planes == 3 ? D % 4 == 0 : h_dtype == FMOE_BF16 && D % 8 == 0;
}
// Where it is the faster form: T <= kThinRows, but for more than 32 rows against a bf16 weight whose 256-row tiles
// fill two rounds of workgroups (37 rows, 131072 x 4096: 275 us in tiles against 318; 32768 x 768 21 against 15; one
// row, 131072 x 768: 40 against 34).
bool vl_is_thin(int64_t T, int64_t V, bool packs) {
  return T <= kThinRows && (T <= 32 || packs || ceil_div(V, 256) < 2 * kVlCus);
}
// Logits of T <= kThinRows rows: STATS (two workgroups per 256 columns: each writes its partial sums, also of no
// columns) or GRAD.
template <int MODE>
void vl_thin(const VlGemm& a, const void* weight, int w_dtype, int64_t ldw, int64_t D, int planes, int64_t T, hipStream_t s) {
  const ThinWeight w{weight, ldw, static_cast<int>(D)};
  const dim3 grid(static_cast<uint32_t>(2 * ceil_div(a.cols, 256)));
  if (planes == 3) vl_thin_launch<MODE, FMOE_F32, 3>(a, w, T, grid, s);
  else if (w_dtype == FMOE_BF16) vl_thin_launch<MODE, FMOE_BF16, 1>(a, w, T, grid, s);
  else vl_thin_launch<MODE, FMOE_F32, 1>(a, w, T, grid, s);
}
void vl_thin_direct(const VlGemm& a, const RowsArgs& r, const void* weight, int w_dtype, int64_t ldw, int64_t D, int planes,
                    int64_t T, hipStream_t s) {
  const ThinWeight w{weight, ldw, static_cast<int>(D)};
  const dim3 grid(static_cast<uint32_t>(2 * ceil_div(a.cols, 256)));
  if (planes == 3) vl_thin_launch<VL_STATS, FMOE_F32, 3, true>(a, w, T, grid, s, r);
  else if (w_dtype == FMOE_BF16) vl_thin_launch<VL_STATS, FMOE_BF16, 1, true>(a, w, T, grid, s, r);
  else vl_thin_launch<VL_STATS, FMOE_F32, 1, true>(a, w, T, grid, s, r);
}

// ---- dH of few rows, fp32 ----------------------------------------------------------------------------
// G W of up to 64 rows on the weight as it lies, with v_mfma_f32_16x16x4_f32 on fp32 numbers (G: the sum of its three
// parts, exact), instead of a packed copy and six products.  Bound by the weight's read up to 32 rows.  A wave takes
// 64 columns and all rows, 32 vocabulary rows a step: a lane's load is 4 elements of a weight row, which are the A operands
// of four products (column d0 + 4 m + i is row m of product i, so that a lane ends with 16 consecutive columns), and the
// step's G comes from LDS, four vocabulary rows a lane at a time.  The vocabulary is split over workgroups, and where the
// rows are short over the waves of one; vl_thin_join_kernel adds their partial rows in order.  Training, vocab 50021 x 1024:
// 20 rows 457 us with the packed copy, 307; 60 rows 507 and 408.  (bf16 rows of odd lengths this way: 5 rows x 1001 x 50021
// 195 and 187 us, 20 rows 197 and 211: not taken.)  One workgroup a CU above 16 rows: two would spill.
constexpr int kDhRows = 256;  // vocabulary rows whose G is in LDS
struct ThinDh {
  int across, ranges;  // waves side by side; parts of the vocabulary
  int64_t T;
  ThinDh(int64_t T, int64_t D, int64_t V) : T(T) {
    across = D > 256 ? 8 : D > 128 ? 4 : D > 64 ? 2 : 1;
    ranges = static_cast<int>(std::max<int64_t>(1, std::min(ceil_div(V, kDhRows), 512 / ceil_div(D, 64 * across))));
  }
  int slots() const { return ranges * (8 / across); }
  size_t bytes(int64_t Dp) const { return static_cast<size_t>(slots()) * T * Dp * 4; }
};

template <int MB>
__global__ __launch_bounds__(512, MB == 1 ? 4 : 2) void vl_thin_dh_kernel(const VlGemm a, const ThinWeight wt, const ThinDh sh) {
  constexpr int GS = kDhRows + 4;  // (16 rows' reads of 16 bytes in different banks)
  __shared__ __attribute__((aligned(16))) float gs[16 * MB * GS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int er = lane & 15, eg = lane >> 4;
  const int n = vl_rows_here(a.head, 0, kThinRows);
  const int kw = w / sh.across, parts = 8 / sh.across;
  const int d0 = (blockIdx.x * sh.across + w % sh.across) * 64, d = d0 + 4 * er, left = wt.D - d;
  const bool active = d0 < wt.D;
  const int chunks = (a.vocab + kDhRows - 1) / kDhRows;
  const int c0 = static_cast<int>(static_cast<int64_t>(chunks) * blockIdx.y / sh.ranges);
  const int c1 = static_cast<int>(static_cast<int64_t>(chunks) * (blockIdx.y + 1) / sh.ranges);

  struct Step {
    float v[2][4][4];  // [half][vocabulary row 4 eg + s of its 16][column]
  };
  auto load = [&](int v0) __attribute__((always_inline)) {
    Step f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t at = static_cast<int64_t>(a.v0 + min(v0 + 16 * h + 4 * eg + q, a.vocab - 1)) * wt.ld + d;
        if (left >= 4) {
          const f32x4 x = *reinterpret_cast<const f32x4_e4*>(static_cast<const float*>(wt.p) + at);
#pragma unroll
          for (int i = 0; i < 4; ++i) f.v[h][q][i] = x[i];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) f.v[h][q][i] = i < left ? static_cast<const float*>(wt.p)[at + i] : 0.0f;
        }
      }
    return f;
  };

  f32x4 acc[4][MB];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[i][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  Step cur;
  if (active) cur = load(c0 * kDhRows + 32 * kw);
  for (int c = c0; c < c1; ++c) {
    __syncthreads();
    for (int i = tid; i < 16 * MB * 32; i += 512) {
      const int r = i >> 5, k = (i & 31) * 8;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = 0.0f;
#pragma unroll
      for (int p = 2; p >= 0; --p) {
        float y[8];
        unpack8(*reinterpret_cast<const uint4*>(a.g + p * a.g_plane + static_cast<int64_t>(r) * a.ldg + c * kDhRows + k), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] + y[e];
      }
      *reinterpret_cast<f32x4*>(gs + r * GS + k) = f32x4{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<f32x4*>(gs + r * GS + k + 4) = f32x4{x[4], x[5], x[6], x[7]};
    }
    __syncthreads();
    if (!active) continue;
    for (int st = kw; st < kDhRows / 32; st += parts) {
      const int v = c * kDhRows + 32 * st;
      const bool same = st + parts < kDhRows / 32;
      Step next;
      if (same || c + 1 < c1) next = load(same ? v + 32 * parts : (c + 1) * kDhRows + 32 * kw);
      if (v + 32 > a.vocab) {  // (what is read again there may be infinite)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) cur.v[h][q][i] = v + 16 * h + 4 * eg + q < a.vocab ? cur.v[h][q][i] : 0.0f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(gs + (16 * m + er) * GS + 32 * st + 16 * h + 4 * eg);
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.v[h][q][i], x[q], acc[i][m], 0, 0, 0);
        }
      }
      cur = next;
    }
  }
  if (!active) return;
  // acc[i][m][e] of a lane: column d0 + 16 eg + 4 e + i, row 16 m + er
  float* const part = a.split + static_cast<int64_t>(blockIdx.y * parts + kw) * sh.T * a.cols;
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    if (16 * m + er >= n) continue;
    float* const p = part + static_cast<int64_t>(16 * m + er) * a.cols + d0 + 16 * eg;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<f32x4*>(p + 4 * e) = f32x4{acc[0][m][e], acc[1][m][e], acc[2][m][e], acc[3][m][e]};
  }
}

// A row's partial rows added, 512 columns a workgroup: each wave every fourth, in order; then the waves.
__global__ __launch_bounds__(256) void vl_thin_join_kernel(const VlGemm a, const int* inv, int T, int slots) {
  __shared__ float sums[4][512];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = blockIdx.x, col = blockIdx.y * 512 + lane * 8;
  const int row = inv[t];
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.0f;
  if (row < 0) {
    if (w > 0 || a.more || col >= a.D) return;
    const int64_t o = static_cast<int64_t>(t) * a.D + col;
    if (a.out_dtype == FMOE_BF16) store_upto8<FMOE_BF16>(a.out, o, a.D - col, v);
    else store_upto8<FMOE_F32>(a.out, o, a.D - col, v);
    return;
  }
  constexpr int U = 8;
  if (col < a.cols)
    for (int s0 = w; s0 < slots; s0 += 4 * U) {
      f32x4 x[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* p = a.split + (static_cast<int64_t>(min(s0 + 4 * u, slots - 1)) * T + row) * a.cols + col;
        x[u][0] = *reinterpret_cast<const f32x4*>(p);
        x[u][1] = *reinterpret_cast<const f32x4*>(p + 4);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s0 + 4 * u < slots)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = v[e] + x[u][0][e], v[4 + e] = v[4 + e] + x[u][1][e];
    }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[w][lane + 64 * e] = v[e];
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int q = 1; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] + sums[q][lane + 64 * e];
  vl_result8<VL_DH>(a, kThinRows, row, col, v);
}

void vl_thin_dh(const VlGemm& a, const void* weight, int64_t ldw, const int* inv, const ThinDh& sh, hipStream_t s) {
  if (sh.T == 0) return;
  const ThinWeight w{weight, ldw, a.D};
  const dim3 grid(static_cast<uint32_t>(ceil_div(a.D, 64 * sh.across)), static_cast<uint32_t>(sh.ranges));
  if (sh.T <= 16) vl_thin_dh_kernel<1><<<grid, 512, 0, s>>>(a, w, sh);
  else if (sh.T <= 32) vl_thin_dh_kernel<2><<<grid, 512, 0, s>>>(a, w, sh);
  else vl_thin_dh_kernel<4><<<grid, 512, 0, s>>>(a, w, sh);
  const dim3 join(static_cast<uint32_t>(sh.T), static_cast<uint32_t>(ceil_div(a.D, 512)));
  vl_thin_join_kernel<<<join, 256, 0, s>>>(a, inv, static_cast<int>(sh.T), sh.slots());
}

// The split tiles: their ranges' partial tiles added in order, by the first `blocks` workgroups (32 for every tile
// that can be split).  DH's last piece: and zeros in the rows of the result without entries, 64 rows a workgroup
// behind those.
template <int MODE, int PLANES>
__global__ __launch_bounds__(256) void vl_split_kernel(const VlGemm a, const int* inv, int T, int blocks) {
  using namespace core;
  const int n = vl_rows_here(a.head, a.row0, a.rows);
  if (MODE == VL_DH && static_cast<int>(blockIdx.x) >= blocks) {
    const int t0 = (blockIdx.x - blocks) * 64;
    float zero[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) zero[e] = 0.0f;
    for (int i = threadIdx.x >> 6; i < 64 && t0 + i < T; i += 4) {
      if (inv[t0 + i] >= 0) continue;
      for (int c = (threadIdx.x & 63) * 8; c < a.D; c += 512) {
        const int64_t o = static_cast<int64_t>(t0 + i) * a.D + c;
        if (a.out_dtype == FMOE_BF16) store_upto8<FMOE_BF16>(a.out, o, a.D - c, zero);
        else store_upto8<FMOE_F32>(a.out, o, a.D - c, zero);
      }
    }
    return;
  }
  if (a.row0 > 0 && n == 0) return;
  const int np = pad_rows(n);
  const int m_rows = MODE == VL_DW ? a.vocab : np;
  const int tiles_m = (m_rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN;
  const int nk = MODE == VL_DH ? (a.vocab + BK - 1) / BK : np / BK;
  const VlSplit sp = vl_split(tiles_m * tiles_n, nk * (PLANES == 1 ? 1 : 6));
  const int64_t range = static_cast<int64_t>(sp.rest) * (BM * BN);
  const int limit = MODE == VL_DW ? a.vocab : n;
  constexpr int U = 8;
  // ranges first, first + step, ... of 8 columns, added in order
  auto add = [&](const float* src, int first, int step, float* v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    for (int s0 = first; s0 < sp.ranges; s0 += U * step) {
      f32x4 u[U][2];
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const float* p = src + min(s0 + s * step, sp.ranges - 1) * range;
        u[s][0] = *reinterpret_cast<const f32x4*>(p);
        u[s][1] = *reinterpret_cast<const f32x4*>(p + 4);
      }
#pragma unroll
      for (int s = 0; s < U; ++s)
        if (s0 + s * step < sp.ranges)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = v[e] + u[s][0][e], v[4 + e] = v[4 + e] + u[s][1][e];
    }
  };
  const int col = (threadIdx.x & 31) * 8, sub = threadIdx.x >> 5;
  int tm, tn;
  float v[8];
  if (sp.ranges < 2 * U) {  // 8 rows of a tile per workgroup
    const int r = blockIdx.x / 32, row = (blockIdx.x % 32) * 8 + sub;
    if (r >= sp.rest) return;
    vl_tile(sp.whole + r, tiles_m, tiles_n, tm, tn);
    if (tm * BM + (blockIdx.x % 32) * 8 >= limit) return;
    add(a.split + static_cast<int64_t>(r) * (BM * BN) + row * BN + col, 0, 1, v);
    vl_result8<MODE>(a, n, tm * BM + row, tn * BN + col, v);
    return;
  }
  // many ranges of few tiles: a row per workgroup, eight parts of its ranges side by side
  __shared__ float sums[8][BN];
  for (int q = blockIdx.x; q < sp.rest * BM; q += blocks) {
    const int r = q / BM, row = q % BM;
    vl_tile(sp.whole + r, tiles_m, tiles_n, tm, tn);
    if (tm * BM + row >= limit) continue;
    add(a.split + static_cast<int64_t>(r) * (BM * BN) + row * BN + col, sub, 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[sub][(threadIdx.x & 31) + 32 * e] = v[e];
    __syncthreads();
    if (sub == 0) {
      for (int p = 1; p < 8; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] + sums[p][threadIdx.x + 32 * e];
      vl_result8<MODE>(a, n, tm * BM + row, tn * BN + col, v);
    }
    __syncthreads();
  }
}

// ---- the rows' statistics and losses -------------------------------------------------------------

struct LossArgs {
  const int *head, *perm, *index;
  const float2* part;
  int64_t Tp;
  int pieces;         // partial sums per row
  float2* stat;
  float* picked;
  float* row_loss;    // of packed rows (reductions), or
  float* loss;        // of rows
  // distillation
  const uint16_t* h;
  int64_t h_plane;
  const void* weight;
  int64_t ldw;
  float c, factor;    // factor: temperature^2
  int top, planes;    // top 0: cross entropy
  int *out_index;     // distillation: of the packed rows
  const float* logits;  // t of the rows, [n_rows][ldt] (nullptr: the listed ones are formed here)
  int ldt;
  float* out_q;
  RowsArgs rows;
  int row0, n_rows;   // as in VlGemm
  // gradients at once: o of the rows; distillation: the loss without ln 2 (m - o + l), over the temperature's square;
  // set where a row's sum is not one that 2^(t - o) can stand for
  float *off, *row_part;
  int* flag;
  const int* only_if;
};

__device__ __forceinline__ void vl_store_loss(const LossArgs& a, int row, float v) {
  if (a.loss) a.loss[a.perm[row]] = v;
  else a.row_loss[row] = v;
}

// Gradients at once: the sum of a row's 2^(t - o) beyond which, and beyond whose inverse, its piece is formed in the ordinary
// way (a loss of 41.6).  Up to it 2^-l H has all of its bits where |h| >= 2^-49 (2^-66 as one bf16 number), and G' W is in
// range where |w| < 2^66.
constexpr float kFarSum = 0x1p60f;

// m and l of R rows per workgroup: each of its 1024 / R threads per row joins every so many of the partial
// sums, in order; then lanes, then waves.
template <int R>
__global__ __launch_bounds__(1024) void vl_stat_kernel(const LossArgs a) {
  __shared__ float2 red[16][R];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (a.only_if && a.only_if[0] == 0) return;
  const int n = vl_rows_here(a.head, a.row0, a.n_rows);
  const int row0 = blockIdx.x * R;
  if (row0 >= n) return;
  const int row = row0 + lane % R;
  constexpr int G = 1024 / R, U = 8;
  const int g = w * (64 / R) + lane / R;
  float m = -__builtin_inff(), s = 0.0f;
  for (int p0 = g; p0 < a.pieces; p0 += G * U) {
    float2 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = a.part[static_cast<int64_t>(min(p0 + u * G, a.pieces - 1)) * a.Tp + min(row, n - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p0 + u * G < a.pieces) vl_join(m, s, v[u].x, v[u].y);
  }
#pragma unroll
  for (int off = R; off < 64; off <<= 1) {
    const float m2 = __shfl_xor(m, off, 64), s2 = __shfl_xor(s, off, 64);
    vl_join(m, s, m2, s2);
  }
  if (lane < R) red[w][lane] = make_float2(m, s);
  __syncthreads();
  if (w > 0 || lane >= R || row >= n) return;
#pragma unroll
  for (int q = 1; q < 16; ++q) vl_join(m, s, red[q][lane].x, red[q][lane].y);
  float l = log2f(s);
  if (a.top == 0) {  // cross entropy
    if (a.index[row] == kBad) {
      l = __builtin_nanf("");
      vl_store_loss(a, row, l);
    } else {
      const float loss = ((m - a.picked[row]) + l) * kLn2;
      vl_store_loss(a, row, loss);
      a.picked[row] = expm1f(-loss);  // p - 1 (exact to its own size where p is near 1), for the backward
    }
  } else if (a.row_part) {  // distillation whose lists were read before
    const float part = a.row_part[row];
    if (part != part) l = part;
    vl_store_loss(a, row, fmaf((m - a.off[row]) + l, kLn2, part) * a.factor);
  }
  a.stat[row] = make_float2(m, l);
  if (a.flag && !(s < kFarSum && s > 1.0f / kFarSum)) a.flag[0] = 1;
}

// Distillation, a workgroup per packed row: the teacher's softmax over its list, t of the listed entries (a dot
// product of length D each, in fp32, four entries of a wave at a time; or read from the stored logits) and the loss.
// Bound by the gathered rows of the weight: 4096 rows x 2048, 64 listed of 65536: 250 us, 4.3 TB/s.
__device__ __forceinline__ float vl_block_max(float v, float* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
__device__ __forceinline__ float vl_block_sum(float v, float* red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = v + __shfl_xor(v, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

template <int DT>
__global__ __launch_bounds__(256) void vl_list_kernel(const LossArgs a) {
  __shared__ float red[4], tq[FMOE_VOCAB_MAX_TOP];
  __shared__ int ti[FMOE_VOCAB_MAX_TOP];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, row = blockIdx.y * gridDim.x + blockIdx.x;
  const bool early = a.row_part != nullptr;  // before the logits' statistics: o of the row, and its part of the loss
  if (early && row == 0 && threadIdx.x == 0) a.flag[0] = 0;
  if (row >= vl_rows_here(a.head, a.row0, a.n_rows)) return;
  const int D = a.rows.D, top = a.top;
  const uint16_t* h = a.h + static_cast<int64_t>(row) * a.rows.Dp;
  const bool round = DT == FMOE_F32 && a.planes == 1;
  // the list: thread i has entries i, i + 256, ...
  constexpr int E = FMOE_VOCAB_MAX_TOP / 256;
  const int64_t list = static_cast<int64_t>(a.perm[row]) * top, out = static_cast<int64_t>(row) * top;
  float z[E], peak = -__builtin_inff(), any_nan = 0.0f, bad = 0.0f;
  int id[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = threadIdx.x + 256 * i;
    id[i] = kNone;
    z[i] = 0.0f;
    if (k < top) id[i] = vl_entry(a.rows, list + k, z[i]);
    if (id[i] != kNone) peak = fmaxf(peak, z[i]), any_nan = z[i] != z[i] ? 1.0f : any_nan;
    if (id[i] == kBad) bad = 1.0f;
  }
  peak = vl_block_max(peak, red);
  if (vl_block_max(any_nan, red) != 0.0f) peak = __builtin_nanf("");
  const bool row_bad = vl_block_max(bad, red) != 0.0f;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) sum = id[i] == kNone ? sum : sum + expf(z[i] - peak);
  const float log_sum = logf(vl_block_sum(sum, red));
  float ent = 0.0f;  // sum of q ln q
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float lq = (z[i] - peak) - log_sum, q = id[i] == kNone ? 0.0f : expf(lq);
    if (!(q == 0.0f)) ent = fmaf(q, lq, ent);
    z[i] = q;
    const int k = threadIdx.x + 256 * i;
    if (k < top) tq[k] = q, ti[k] = id[i];
  }
  ent = vl_block_sum(ent, red);
  // entries of one index are added to the first of them
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = threadIdx.x + 256 * i;
    if (id[i] < 0) continue;
    float q = 0.0f;
    bool first = true;
    for (int j = 0; j < top; ++j)
      if (ti[j] == id[i]) first = first && j >= k, q = q + tq[j];
    id[i] = first ? id[i] : kNone;
    z[i] = first ? q : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int k = threadIdx.x + 256 * i;
    if (k < top) {
      tq[k] = z[i], ti[k] = id[i];
      a.out_index[out + k] = id[i];
      a.out_q[out + k] = z[i];
    }
  }
  __syncthreads();
  const float2 ml = early ? make_float2(0.0f, 0.0f) : a.stat[row];
  float cross = 0.0f, most = -__builtin_inff();
  if (a.logits) {
    const float* t_row = a.logits + static_cast<int64_t>(row) * a.ldt;
    for (int k = threadIdx.x; k < top; k += 256) {
      if (ti[k] < 0) continue;
      const float t = t_row[ti[k]], q = tq[k];
      most = fmaxf(most, t);
      a.picked[out + k] = t;
      if (!(q == 0.0f)) cross = fmaf(q, (ml.x - t) + ml.y, cross);
    }
  }
  constexpr int U = 4;
  for (int k0 = w * U; k0 < (a.logits ? 0 : top); k0 += 4 * U) {
    float acc[U][4];
    int64_t at[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = __builtin_amdgcn_readfirstlane(ti[min(k0 + u, top - 1)]);
      on[u] = k0 + u < top && v >= 0;
      at[u] = static_cast<int64_t>(max(v, 0)) * a.ldw;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[u][e] = 0.0f;
    }
    for (int c = lane * 8; c < D; c += 512) {
      float hv[8], v[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) load_upto8<DT>(a.weight, at[u] + c, on[u] ? D - c : 0, v[u]);
      unpack8(*reinterpret_cast<const uint4*>(h + c), hv);
      for (int q = 1; q < a.planes; ++q) {
        float x[8];
        unpack8(*reinterpret_cast<const uint4*>(h + q * a.h_plane + c), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) hv[e] = hv[e] + x[e];  // exact: the parts of one fp32 number
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[u][e & 3] = fmaf(round ? bf_round(v[u][e]) : v[u][e], hv[e], acc[u][e & 3]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s = (acc[u][0] + acc[u][1]) + (acc[u][2] + acc[u][3]);
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) s = s + __shfl_xor(s, off, 64);
      if (!on[u]) continue;
      const float t = s * a.c, q = tq[k0 + u];
      most = fmaxf(most, t);
      if (lane == 0) a.picked[out + k0 + u] = t;
      if (lane == 0 && !(q == 0.0f)) cross = fmaf(q, (ml.x - t) + ml.y, cross);
    }
  }
  if (early) {
    // o: the largest listed t.  Sum of q (o - t), with o known only now
    most = vl_block_max(most, red);
    if (most == -__builtin_inff()) most = 0.0f;
    __syncthreads();  // (picked, written by this workgroup)
    cross = 0.0f;
    for (int k = threadIdx.x; k < top; k += 256)
      if (ti[k] >= 0 && !(tq[k] == 0.0f)) cross = fmaf(tq[k], most - a.picked[out + k], cross);
    cross = vl_block_sum(cross, red);
    if (threadIdx.x == 0) {
      a.off[row] = most;
      a.row_part[row] = row_bad ? __builtin_nanf("") : fmaf(cross, kLn2, ent);
    }
    return;
  }
  cross = vl_block_sum(cross, red);
  if (threadIdx.x == 0) {
    float v = fmaf(cross, kLn2, ent) * a.factor;
    if (row_bad) {
      v = __builtin_nanf("");
      a.stat[row] = make_float2(ml.x, v);
    }
    vl_store_loss(a, row, v);
  }
}

// Sum or mean of the packed rows' losses, in fp64 and a fixed order.
__global__ __launch_bounds__(1024) void vl_sum_kernel(const int* head, const float* row_loss, int reduction, float* loss) {
  __shared__ double red[16];
  const int n = head[0];
  double s = 0.0;
  constexpr int U = 8;
  for (int i = threadIdx.x; i < n; i += 1024 * U) {
    float v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = row_loss[min(i + 1024 * u, n - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) s = i + 1024 * u < n ? s + static_cast<double>(v[u]) : s;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) s = s + __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
#pragma unroll
    for (int q = 0; q < 16; ++q) t = t + red[q];
    loss[0] = static_cast<float>(reduction == FMOE_REDUCE_MEAN ? t / static_cast<double>(n) : t);
  }
}

// ---- the listed entries of G -----------------------------------------------

struct FixArgs {
  const int *head, *perm, *index;
  const float *q, *picked;
  const float2* stat;
  const float* d_loss;
  int top, v0, v1, reduction, planes, ldg;
  float factor;
  uint16_t* g;
  int64_t g_plane;
  // gradients at once: p - q times 2^l, or by itself where flag is set; q nullptr: picked is p - 1
  int row0, rows;
  const int* flag;
};

// G at the entries that lie in this piece of the vocabulary: the row's weight times p - q in fp32, rounded once.
__global__ __launch_bounds__(256) void vl_fix_kernel(const FixArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int n = vl_rows_here(a.head, a.row0, a.rows), row = static_cast<int>(i / a.top);
  if (row >= n) return;
  const int id = a.index[i];
  if (id < a.v0 || id >= a.v1) return;
  const float2 ml = a.stat[row];
  float v = a.q ? __builtin_amdgcn_exp2f((a.picked[i] - ml.x) - ml.y) - a.q[i] : a.picked[i];
  if (a.flag) v = a.flag[0] ? v : v * __builtin_amdgcn_exp2f(ml.y);
  else v = v * vl_row_weight(a.d_loss, a.perm, a.reduction, n, row, a.factor);
  uint16_t* p = a.g + static_cast<int64_t>(row) * a.ldg + (id - a.v0);
  for (int k = 0; k < a.planes; ++k) {
    const uint16_t b = f2bf(v);
    p[k * a.g_plane] = b;
    v = v - bf2f(b);
  }
}

// ---- gradients at once ---------------------------------------------------------------------------------
// For a piece of the rows:  G' = 2^(t - o) (PROB, o: the target's t, or the largest listed one),  l = log2 of its
// sum per row,  G'[r, listed] = 2^l (p - q),  dH = w 2^-l (G' W),  dW += w (G'^T (2^-l H)).  (w, the weight of every row, stays
// out of the operands: with a small one 2^-l H would lose bits sooner.)
// bf16 has the exponents of fp32, so o need not be the maximum.  Where a row's sum leaves 2^-60 .. 2^60 all the
// same (kFarSum), or is no number, the piece's flag is set, and STATS and GRAD form its statistics and G in
// the ordinary way (with H itself in place of 2^-l H); else those launches end at once.
// 2^-l H is rounded once more (planes = 1: half a step of bf16 an element, as G).  32768 rows x 2048, vocab 131072: 51.8 ms with
// the logits formed twice, 39.4 at once.

// o of cross entropy's rows, a wave each.
template <int DT>
__global__ __launch_bounds__(256) void vl_off_kernel(const LossArgs a) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.flag[0] = 0;
  if (row >= vl_rows_here(a.head, a.row0, a.n_rows)) return;
  const int id = __builtin_amdgcn_readfirstlane(a.index[row]);
  const int D = a.rows.D;
  const bool round = DT == FMOE_F32 && a.planes == 1;
  const uint16_t* h = a.h + static_cast<int64_t>(row) * a.rows.Dp;
  float acc = 0.0f;
  for (int c = lane * 8; c < D; c += 512) {
    float hv[8], v[8];
    load_upto8<DT>(a.weight, static_cast<int64_t>(max(id, 0)) * a.ldw + c, D - c, v);
    unpack8(*reinterpret_cast<const uint4*>(h + c), hv);
    for (int q = 1; q < a.planes; ++q) {
      float x[8];
      unpack8(*reinterpret_cast<const uint4*>(h + q * a.h_plane + c), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) hv[e] = hv[e] + x[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = fmaf(round ? bf_round(v[e]) : v[e], hv[e], acc);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) acc = acc + __shfl_xor(acc, off, 64);
  if (lane == 0) a.off[row] = id < 0 ? 0.0f : acc * a.c;
}

// The weight of the rows (all_factor), the factors of the piece's rows of dH, and their 2^-l H (zeros in the padding), a wave
// each.
template <int PLANES>
__global__ __launch_bounds__(256) void vl_factor_kernel(const int* head, int row0, int rows, const float2* stat,
                                                        const int* flag, float factor, int mean, const uint16_t* h,
                                                        int64_t h_plane, int Dp, float* all_factor, float* row_factor,
                                                        uint16_t* out, int64_t out_plane) {
  const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int n = vl_rows_here(head, row0, rows);
  const float weight = head[0] == 0 ? 0.0f : mean ? factor / static_cast<float>(head[0]) : factor;
  if (blockIdx.x == 0 && threadIdx.x == 0) all_factor[0] = weight;
  if (row >= pad_rows(n)) return;
  float f = 1.0f;
  if (row < n) {
    if (flag[0] == 0) f = __builtin_amdgcn_exp2f(-stat[row].y);
    if (lane == 0) row_factor[row] = weight * f;
  }
  for (int c = lane * 8; c < Dp; c += 512) {
    const int64_t at = static_cast<int64_t>(row) * Dp + c;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < n) {
      unpack8(*reinterpret_cast<const uint4*>(h + at), v);
#pragma unroll
      for (int q = 1; q < PLANES; ++q) {
        float x[8];
        unpack8(*reinterpret_cast<const uint4*>(h + q * h_plane + at), x);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = v[e] + x[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * f;
    }
    uint4 o[PLANES];
    vl_split8<PLANES>(v, o);
#pragma unroll
    for (int p = 0; p < PLANES; ++p) *reinterpret_cast<uint4*>(out + p * out_plane + at) = o[p];
  }
}

// dW from the sum over the pieces.
template <int DT>
__global__ __launch_bounds__(256) void vl_dw_kernel(const float* sum, int64_t vocab, int D, int Dp, void* out) {
  const int lane = threadIdx.x & 63;
  const int64_t v = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (v >= vocab) return;
  for (int c = lane * 8; c < D; c += 512) {
    float x[8];
    load_upto8<FMOE_F32>(sum, v * Dp + c, 8, x);
    store_upto8<DT>(out, v * D + c, D - c, x);
  }
}

// dst = scale[0] * src of up to kScaleMax tensors (blockIdx.y); nothing where they are the same and scale[0] is 1.
constexpr int kScaleMax = FMOE_SCALE_MAX_TENSORS;
struct ScaleArgs {
  const float* scale;
  const void* src[kScaleMax];
  void* dst[kScaleMax];
  int64_t n[kScaleMax];
  int dtype[kScaleMax];
};
template <int DT>
__device__ __forceinline__ void vl_scale(float f, const void* src, void* dst, int64_t n) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256 * 8;
  for (int64_t e = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; e < n; e += stride) {
    const int k = static_cast<int>(min(n - e, int64_t(8)));
    float v[8];
    load_upto8<DT>(src, e, k, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * f;
    store_upto8<DT>(dst, e, k, v);
  }
}
__global__ __launch_bounds__(256) void vl_scale_kernel(const ScaleArgs a) {
  const float f = a.scale[0];
  const int i = blockIdx.y;
  if (a.src[i] == a.dst[i] && f == 1.0f) return;
  if (a.dtype[i] == FMOE_BF16) vl_scale<FMOE_BF16>(f, a.src[i], a.dst[i], a.n[i]);
  else vl_scale<FMOE_F32>(f, a.src[i], a.dst[i], a.n[i]);
}

// ---- host ------------------------------------------------------------------------------------------

// Vocabulary rows of a piece of the backward, a multiple of 256: as many as G's bound (kPieceBytes) allows, in
// pieces of one size.
constexpr int64_t kPieceBytes = int64_t(1) << 31;
constexpr int64_t kPackBytes = int64_t(1) << 28;

int64_t vl_bwd_piece(int64_t T, int64_t V, int planes) {
  const int64_t Tp = std::max<int64_t>(pad64(T), 64), vt = ceil_div(V, 256);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>({vt, kPieceBytes / (Tp * 512 * planes), 4096}));
  return ceil_div(vt, ceil_div(vt, most)) * 256;
}

// Partial tiles of a product of at most so many tiles: the rows that turn out to have entries may be fewer.
int64_t vl_split_slots(int64_t tiles, int64_t units) {
  if (units < 16) return 0;
  const int64_t rest = std::min<int64_t>(tiles, kVlCus - 1);
  return std::min<int64_t>(kSplitSlots, rest * (units / 8));
}

// Vocabulary rows of a piece of the forward: all of them, or as many as a packed copy may have.
int64_t vl_fwd_piece(int64_t D, int64_t V, int planes, bool packs) {
  if (!packs) return V;
  return std::min(V, std::max<int64_t>(kPackBytes / (pad64(D) * (planes == 3 ? 4 : 2)) / 256, 1) * 256);
}

// Listed logits of a distillation: dot products, which read top * D elements of the weight a row (4 .. 9 TB/s out of the
// caches), or their product with all of the vocabulary, stored a piece of the rows at a time (4 V bytes a row written,
// a line read for each listed one).  Where the statistics come first the product is there anyhow (8192 rows x 2944, vocab
// 1664, 156 listed: 993 us with dot products, 205 stored; 4096 x 768 x 32768: 64 listed 301 and 321, 256 listed 591 and
// 386); gradients at once need the lists before their product, and so one more (8192 x 2944 x 1664, 156 listed: 1243 and
// 526; 4096 x 2048 x 32768: 64 listed 1543 and 1954, 256 listed 2075 and 1970; fp32, 2000 x 1024 x 8192, 128 listed: 689
// and 673).
constexpr int64_t kLogitBytes = int64_t(1) << 28;
bool vl_stores_logits(int64_t T, int64_t D, int64_t V, int64_t top, int planes, bool once_more) {
  const int64_t read = top * D * (planes == 3 ? 4 : 2);
  if (top == 1 || T <= kThinRows || V * 4 * 1024 > kLogitBytes) return false;  // (top 1: also cross entropy)
  return once_more ? T >= 1024 && read > 5 * V + planes * V * D / 80 : read > 5 * V;
}
// Rows whose logits are stored at a time, where vl_stores_logits says so: whole row tiles, 1024 rows and more of the
// vocabularies that it takes.
int64_t vl_logit_rows(int64_t T, int64_t V) {
  return std::min(ceil_div(T, 256), kLogitBytes / (ceil_div(V, 256) * 1024) / 256) * 256;
}
// Rows whose logits the forward stores at a time (0: none).  The thin form's few rows have few workgroups for their lists,
// and it stores those of lists of more than four, all rows at once, where 64 rows would fit kLogitBytes (3 rows x 1690,
// vocab 9699, 150 listed, in fp32: 57 us, with dot products 122; 8 rows x 768 x 32768, 8 listed: 25 and 29; 64 x 256 x 65536,
// 5 listed: 27 both).  Up to 64 rows that take tiles (vl_is_thin) do not store.
int64_t vl_fwd_logit_rows(int64_t T, int64_t D, int64_t V, int64_t top, int planes, bool packs) {
  if (vl_is_thin(T, V, packs)) return top > 4 && ceil_div(V, 256) * 1024 * kThinRows <= kLogitBytes ? T : 0;
  const bool stored = vl_fwd_piece(D, V, planes, packs) >= V && vl_stores_logits(T, D, V, top, planes, false);
  return stored ? std::min(vl_logit_rows(T, V), T) : 0;
}

// Copies of weight rows: bf16 planes, and for fp32 scaled fp16 with its scales.
struct VlPackSpace {
  size_t planes = 0, half = 0, scale = 0;
  template <typename Take>
  VlPackSpace(Take take, int64_t rows, int64_t Dp, int n_planes, bool bf16) {
    planes = take(bf16 ? rows * Dp * 2 * n_planes : 0);
    half = take(n_planes == 3 ? rows * Dp * 4 : 0);
    scale = take(n_planes == 3 ? rows * 4 : 0);
  }
  VlPackSpace() = default;
};

struct VlFwdSpace {
  size_t masks, part, row_loss, logits, bytes = 0;
  int64_t logit_rows;  // whose logits are stored at a time (0: none)
  VlPackSpace pack;
  VlFwdSpace(int64_t T, int64_t D, int64_t V, int64_t top, int planes, bool packs)
      : logit_rows(vl_fwd_logit_rows(T, D, V, top, planes, packs)) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    const int64_t Tp = std::max<int64_t>(pad64(T), 64);
    masks = take(ceil_div(T, kRowBlock) * 4);
    part = take(2 * ceil_div(V, 256) * Tp * 8);
    row_loss = take(T * 4);
    logits = take(logit_rows * ceil_div(V, 256) * 1024);
    if (packs && !vl_is_thin(T, V, packs)) pack = VlPackSpace(take, vl_fwd_piece(D, V, planes, true), pad64(D), planes, planes == 1);
  }
};

struct VlBwdSpace {
  int64_t piece;
  size_t g, sum, split, bytes = 0;
  bool as_it_lies;  // fp32, few rows: no product reads a packed weight
  VlPackSpace pack;
  VlBwdSpace(int64_t T, int64_t D, int64_t V, int planes, bool packs) : piece(vl_bwd_piece(T, V, planes)) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    const int64_t Tp = std::max<int64_t>(pad64(T), 64), Dp = pad64(D), dt = ceil_div(Dp, 256);
    const int64_t passes = planes == 3 ? 6 : 1, tile = core::BM * core::BN * 4;
    as_it_lies = planes == 3 && vl_is_thin(T, V, packs);
    g = take(Tp * piece * 2 * planes);
    sum = take(V > piece ? Tp * Dp * 4 : 0);
    const int64_t dh = as_it_lies ? ThinDh(T, D, std::min(V, piece)).bytes(Dp)
                                  : vl_split_slots(ceil_div(Tp, 256) * dt, ceil_div(std::min(V, piece), 64) * passes) * tile;
    split = take(std::max<int64_t>(dh, vl_split_slots(ceil_div(std::min(V, piece), 256) * dt, Tp / 64 * passes) * tile));
    if (packs && !as_it_lies) pack = VlPackSpace(take, std::min(pad64(V), piece), Dp, planes, true);
  }
};

bool vl_sizes_ok(int64_t T, int64_t dim, int64_t vocab, int64_t top, int planes) {
  return T >= 0 && dim > 0 && vocab > 0 && top > 0 && dim <= FMOE_VOCAB_MAX_DIM && T <= FMOE_VOCAB_MAX_TOKENS &&
         vocab <= FMOE_VOCAB_MAX_VOCAB && top <= FMOE_VOCAB_MAX_TOP && T * dim <= FMOE_VOCAB_MAX_ELEMENTS &&
         vocab * dim <= FMOE_VOCAB_MAX_ELEMENTS && T * top < (int64_t(1) << 31) && (planes == 1 || planes == 3);
}

// Factors that the kernels hold in fp32: logit_scale / temperature * log2(e), logit_scale * temperature, temperature^2 and
// 1 / temperature are in range.
bool vl_factors_ok(double logit_scale, double temperature) {
  return temperature >= 0x1p-63 && temperature <= 0x1p63 &&
         std::fabs(logit_scale) * std::max(temperature, 1.0 / temperature) < 0x1p126;
}

bool vl_packs(const void* weight, int w_dtype, int64_t ldw, int64_t dim, int planes) {
  return planes != 1 || w_dtype != FMOE_BF16 || dim % 64 != 0 || ldw % 8 != 0 || !aligned16(weight);
}

// A copy of rows v0 .. v0 + rows - 1 of the weight: planes at dst, for fp32 (planes = 3) fp16 at half and its scales
// (each where it is not null); plane: elements of a plane of either.
struct VlPacked {
  uint16_t *dst, *half;
  float* scale;
  VlPacked(uint8_t* ws, const VlPackSpace& p)
      : dst(reinterpret_cast<uint16_t*>(ws + p.planes)), half(reinterpret_cast<uint16_t*>(ws + p.half)),
        scale(reinterpret_cast<float*>(ws + p.scale)) {}
};
int vl_pack(const void* weight, int w_dtype, int64_t ldw, int64_t v0, int64_t rows, int64_t D, int planes, VlPacked p,
            int64_t plane, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(ceil_div(rows, 4)));
  const int Dp = static_cast<int>(pad64(D)), r = static_cast<int>(rows), d = static_cast<int>(D);
  uint16_t* const dst = p.dst;
  if (w_dtype == FMOE_BF16) vl_pack_kernel<FMOE_BF16, 1><<<grid, 256, 0, s>>>(weight, ldw, v0, r, d, Dp, dst, plane);
  else if (planes == 1) vl_pack_kernel<FMOE_F32, 1><<<grid, 256, 0, s>>>(weight, ldw, v0, r, d, Dp, dst, plane);
  else vl_pack32_kernel<<<grid, 256, 0, s>>>(static_cast<const float*>(weight), ldw, v0, r, d, Dp, dst, p.half, p.scale, plane);
  return launch_status();
}

bool vl_elem_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FMOE_BF16 ? 1u : 3u)) == 0;
}
bool vl_ws_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }
bool vl_dtype(int d) { return d == FMOE_BF16 || d == FMOE_F32; }

// Workgroups of a product of so many tiles: one per CU, fewer only in eighths.
dim3 vl_grid(int64_t items) { return dim3(static_cast<uint32_t>(std::min<int64_t>(kVlCus, ceil_div(items, 8) * 8))); }

// The forward call's arguments.
struct VlCall {
  const void *hidden, *weight, *index, *teacher;
  int h_dtype, w_dtype, index64, t_dtype;
  int64_t ldh, ldw, T, dim, vocab, top, ignore_index;
  double logit_scale, temperature;
  int planes, reduction;
  float* loss;
  bool distill() const { return teacher != nullptr || top != 1; }
};

int vl_check(const VlCall& a, const void* state, const void* workspace) {
  const bool distill = a.distill();
  if (a.T < 0 || a.dim <= 0 || a.vocab <= 0 || a.top <= 0 || a.index64 < 0 || a.index64 > 1 || a.reduction < 0 ||
      a.reduction > 2 || (a.planes != 1 && a.planes != 3) || !vl_factors_ok(a.logit_scale, a.temperature) ||
      (!distill && a.T > 0 && a.temperature != 1.0))  // (without rows there may be no address to tell them apart)
    return FMOE_ERR_INVALID_ARG;
  if (!vl_sizes_ok(a.T, a.dim, a.vocab, a.top, a.planes)) return FMOE_ERR_SHAPE;
  if ((a.T > 1 && (a.ldh < a.dim || a.ldh > (int64_t(1) << 38))) ||
      (a.vocab > 1 && (a.ldw < a.dim || a.ldw >= (int64_t(1) << 22))))
    return FMOE_ERR_SHAPE;
  if (!vl_dtype(a.h_dtype) || !vl_dtype(a.w_dtype) || (a.teacher && !vl_dtype(a.t_dtype)) ||
      (a.planes == 3 && (a.h_dtype != FMOE_F32 || a.w_dtype != FMOE_F32)))
    return FMOE_ERR_DTYPE;
  if (a.weight == nullptr || a.loss == nullptr ||
      (a.T > 0 && (a.hidden == nullptr || a.index == nullptr || (distill && a.teacher == nullptr))))
    return FMOE_ERR_INVALID_ARG;
  if (!vl_elem_aligned(a.hidden, a.h_dtype) || !vl_elem_aligned(a.weight, a.w_dtype) || !vl_elem_aligned(a.loss, FMOE_F32) ||
      (a.teacher && !vl_elem_aligned(a.teacher, a.t_dtype)) ||
      (reinterpret_cast<uintptr_t>(a.index) & (a.index64 ? 7u : 3u)) != 0 || !vl_ws_aligned(state) || !vl_ws_aligned(workspace))
    return FMOE_ERR_ALIGN;
  return FMOE_OK;
}

// Packs the rows with entries; the arguments for those that read lists later.
RowsArgs vl_pack_rows(const VlCall& a, const VlState& st, uint32_t* masks, bool half, bool direct, hipStream_t s) {
  RowsArgs r{};
  r.hidden = a.hidden, r.index = a.index, r.teacher = a.teacher, r.ldh = a.ldh, r.ignore = a.ignore_index;
  r.index64 = a.index64, r.t_dtype = a.distill() ? a.t_dtype : -1;
  r.T = static_cast<int>(a.T), r.D = static_cast<int>(a.dim), r.Dp = static_cast<int>(st.Dp), r.V = static_cast<int>(a.vocab);
  r.top = static_cast<int>(a.top), r.plane = st.plane;
  r.inv_temp = static_cast<float>(1.0 / a.temperature);
  r.masks = a.T * a.top <= kFewEntries ? nullptr : masks;
  r.head = st.head, r.perm = st.perm, r.inv = st.inv, r.out_index = st.index, r.h = st.h;
  r.h16 = half ? st.h16 : nullptr, r.h_scale = st.h_scale;
  r.loss = a.reduction == FMOE_REDUCE_NONE ? a.loss : nullptr;
  if (direct) return r;  // (the first product does it)
  if (r.masks) vl_mark_kernel<<<dim3(static_cast<uint32_t>(ceil_div(a.T, kRowBlock))), 1024, 0, s>>>(r);
  if (a.h_dtype == FMOE_BF16) vl_rows_launch<FMOE_BF16, 1>(r, s);
  else if (a.planes == 1) vl_rows_launch<FMOE_F32, 1>(r, s);
  else vl_rows_launch<FMOE_F32, 3>(r, s);
  return r;
}

// The statistics (and losses) of `rows` rows.
void vl_stat(const LossArgs& l, int64_t rows, hipStream_t s) {
  if (rows >= 8192) vl_stat_kernel<64><<<dim3(static_cast<uint32_t>(ceil_div(rows, 64))), 1024, 0, s>>>(l);
  else if (rows >= 1024) vl_stat_kernel<16><<<dim3(static_cast<uint32_t>(ceil_div(rows, 16))), 1024, 0, s>>>(l);
  else vl_stat_kernel<4><<<dim3(static_cast<uint32_t>(ceil_div(rows, 4))), 1024, 0, s>>>(l);
}

void vl_lists(const LossArgs& l, int w_dtype, int64_t rows, hipStream_t s) {
  // (a side of the grid stays below 2^32 threads)
  constexpr int64_t kSide = int64_t(1) << 23;
  const dim3 grid(static_cast<uint32_t>(std::min(rows, kSide)), static_cast<uint32_t>(ceil_div(rows, kSide)));
  if (w_dtype == FMOE_BF16) vl_list_kernel<FMOE_BF16><<<grid, 256, 0, s>>>(l);
  else vl_list_kernel<FMOE_F32><<<grid, 256, 0, s>>>(l);
}

// STATS or LOGITS of up to so many rows.
template <int MODE>
void vl_stats(const VlGemm& g, int planes, int64_t rows, hipStream_t s) {
  const dim3 grid = vl_grid(ceil_div(rows, 256) * ceil_div(g.cols, 256));
  if (planes == 1) vl_gemm_kernel<MODE, 1><<<grid, core::NT, 0, s>>>(g);
  else vl_gemm_kernel<MODE, 3><<<grid, core::NT, 0, s>>>(g);
}

// The lists of g's and l's `rows` rows from stored logits, `most` rows at a time; stat: with the rows' statistics between.
void vl_stored_lists(const VlGemm& g, const LossArgs& l, int w_dtype, int64_t rows, int64_t most, int64_t Dp, int top,
                     bool stat, hipStream_t s) {
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t here = std::min(most, rows - r0);
    VlGemm q = g;
    q.row0 += static_cast<int>(r0), q.rows = static_cast<int>(here);
    q.a += r0 * Dp, q.part += r0;
    if (l.planes == 3) q.a_scale += r0;
    vl_stats<VL_LOGITS>(q, l.planes, here, s);
    LossArgs m = l;
    m.row0 = q.row0, m.n_rows = q.rows, m.perm += r0, m.part += r0, m.stat += r0, m.index += r0, m.h += r0 * Dp;
    m.picked += r0 * top, m.out_index += r0 * top, m.out_q += r0 * top;
    if (m.row_loss) m.row_loss += r0;
    if (m.off) m.off += r0;
    if (m.row_part) m.row_part += r0;
    m.logits = g.logits, m.ldt = g.ldt;
    if (stat) vl_stat(m, here, s);
    vl_lists(m, w_dtype, here, s);
  }
}

// DH and DW with their split tiles; rest of DH's result (rows without entries) with its last piece.
template <int MODE>
void vl_product(const VlGemm& g, int planes, int64_t mt, int64_t nt, int64_t units, const int* inv, int64_t T, hipStream_t s) {
  if (planes == 1) vl_gemm_kernel<MODE, 1><<<dim3(kVlCus), core::NT, 0, s>>>(g);
  else vl_gemm_kernel<MODE, 3><<<dim3(kVlCus), core::NT, 0, s>>>(g);
  // the split tiles' number depends on the rows with entries, which the host does not know
  const int64_t passes = planes == 3 ? 6 : 1;
  const int64_t blocks = units * passes < 16 ? 0 : std::min<int64_t>(mt * nt, kVlCus - 1) * 32;
  const int64_t clear = MODE == VL_DH && inv ? ceil_div(T, 64) : 0;
  if (blocks + clear == 0) return;
  const dim3 grid(static_cast<uint32_t>(blocks + clear));
  if (planes == 1) vl_split_kernel<MODE, 1><<<grid, 256, 0, s>>>(g, inv, static_cast<int>(T), static_cast<int>(blocks));
  else vl_split_kernel<MODE, 3><<<grid, 256, 0, s>>>(g, inv, static_cast<int>(T), static_cast<int>(blocks));
}

// Gradients at once: rows of a piece, or 0 where that form is not taken.  It needs G of at least kFusedRows rows (or
// all) within kPieceBytes, since every piece adds to all of dW (fp32: written and read once more a piece), a packed copy of
// the whole weight where one is needed, and rows enough for the tiles.
constexpr int64_t kFusedRows = 2048, kFusedBytes = int64_t(1) << 31;
int64_t vl_fused_piece(int64_t T, int64_t D, int64_t V, int planes, bool packs) {
  const int64_t Vp = ceil_div(V, 256) * 256, Tp = ceil_div(std::max<int64_t>(T, 1), 256) * 256;
  if (T <= kThinRows || V > (int64_t(1) << 22) || (packs && Vp * pad64(D) * (planes == 3 ? 10 : 2) > kFusedBytes)) return 0;
  const int64_t most = std::min(Tp, kPieceBytes / (Vp * 2 * planes) / 256 * 256);
  if (most < std::min(Tp, kFusedRows) || (most < Tp && V * pad64(D) * 4 > kFusedBytes)) return 0;
  const int64_t pieces = ceil_div(Tp, most);
  return ceil_div(Tp / 256, pieces) * 256;
}

struct VlFusedSpace {
  int64_t piece;
  size_t state, masks, part, row_loss, row_part, off, factor, all_factor, flag, logits, g, fh, split, sum, bytes = 0;
  bool stored;  // the logits, for the lists: of a part of the piece at a time
  VlPackSpace pack;
  VlFusedSpace(int64_t T, int64_t D, int64_t V, int64_t top, int planes, bool packs)
      : piece(vl_fused_piece(T, D, V, planes, packs)) {
    if (piece == 0) return;
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    const int64_t Dp = pad64(D), dt = ceil_div(Dp, 256), vt = ceil_div(V, 256), passes = planes == 3 ? 6 : 1;
    state = take(VlState(nullptr, T, D, top, planes).bytes);
    masks = take(ceil_div(T, kRowBlock) * 4);
    part = take(2 * vt * piece * 8);
    row_loss = take(T * 4);
    row_part = take(piece * 4);
    off = take(piece * 4);
    factor = take(piece * 4);
    all_factor = take(4);
    flag = take(4);
    stored = vl_stores_logits(T, D, V, top, planes, true);
    logits = take(stored ? vl_logit_rows(piece, V) * vt * 1024 : 0);
    g = take(piece * vt * 512 * planes);
    fh = take(piece * Dp * 2 * planes);
    split = take(std::max(vl_split_slots(piece / 256 * dt, ceil_div(V, 64) * passes),
                          vl_split_slots(vt * dt, piece / 64 * passes)) * (core::BM * core::BN * 4));
    sum = take(piece < T ? V * Dp * 4 : 0);
    if (packs) pack = VlPackSpace(take, V, Dp, planes, true);
  }
};

}  // namespace fmoe

using namespace fmoe;

extern "C" size_t fmoe_vocab_loss_state_bytes(int64_t T, int64_t dim, int64_t top, int planes) {
  return vl_sizes_ok(T, dim, 1, top, planes) ? VlState(nullptr, T, dim, top, planes).bytes : 0;
}

extern "C" int fmoe_vocab_loss_packs(const void* weight, int w_dtype, int64_t ldw, int64_t dim, int planes) {
  return vl_packs(weight, w_dtype, ldw, dim, planes);
}

extern "C" size_t fmoe_vocab_loss_fwd_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int64_t top, int planes,
                                                      int packs) {
  return vl_sizes_ok(T, dim, vocab, top, planes) ? VlFwdSpace(T, dim, vocab, top, planes, packs).bytes : 0;
}

extern "C" size_t fmoe_vocab_loss_bwd_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int planes, int packs) {
  return vl_sizes_ok(T, dim, vocab, 1, planes) ? VlBwdSpace(T, dim, vocab, planes, packs).bytes : 0;
}

extern "C" int fmoe_vocab_loss_fwd(const void* hidden, int h_dtype, int64_t ldh, const void* weight, int w_dtype,
                                   int64_t ldw, const void* index, int index64, const void* teacher, int t_dtype,
                                   int64_t T, int64_t dim, int64_t vocab, int64_t top, int64_t ignore_index,
                                   double logit_scale, double temperature, int planes, int reduction, float* loss,
                                   void* state, size_t state_bytes, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const VlCall call{hidden, weight, index, teacher, h_dtype, w_dtype, index64, t_dtype, ldh, ldw, T, dim, vocab, top,
                    ignore_index, logit_scale, temperature, planes, reduction, loss};
  const bool distill = call.distill();
  if (const int rc = vl_check(call, state, workspace); rc != FMOE_OK) return rc;
  const bool packs = vl_packs(weight, w_dtype, ldw, dim, planes);
  const VlFwdSpace space(T, dim, vocab, top, planes, packs);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const VlState st(static_cast<uint8_t*>(state), T, dim, top, planes);
  if (state == nullptr || state_bytes < st.bytes || workspace == nullptr || workspace_bytes < space.bytes)
    return FMOE_ERR_WORKSPACE;
  const hipStream_t s = as_stream(stream);
  // (the tiles' operands of fp32 are fp16; the form of few rows reads the planes)
  const bool thin = vl_is_thin(T, vocab, packs), half = planes == 3 && !thin;
  const bool direct = thin && !distill && T > 0 && vl_is_direct(h_dtype, planes, dim);
  const RowsArgs r = vl_pack_rows(call, st, reinterpret_cast<uint32_t*>(ws + space.masks), half, direct, s);

  VlGemm g{};
  g.a = half ? st.h16 : st.h, g.a_plane = st.plane, g.lda = static_cast<int>(st.Dp), g.a_scale = st.h_scale;
  g.head = st.head, g.rows = static_cast<int>(T), g.k = static_cast<int>(st.Dp);
  g.c = static_cast<float>(logit_scale / temperature * static_cast<double>(kLog2e));
  g.part = reinterpret_cast<float2*>(ws + space.part), g.Tp = st.Tp;
  g.index = distill ? nullptr : st.index, g.picked = st.picked;
  LossArgs l{};
  l.head = st.head, l.perm = st.perm, l.index = st.index, l.part = g.part, l.Tp = st.Tp;
  l.pieces = static_cast<int>(2 * ceil_div(vocab, 256));
  l.stat = st.stat, l.picked = st.picked;
  l.row_loss = reinterpret_cast<float*>(ws + space.row_loss);
  l.loss = r.loss;
  l.h = st.h, l.h_plane = st.plane, l.weight = weight, l.ldw = ldw;
  l.top = distill ? static_cast<int>(top) : 0;
  l.planes = planes, l.c = g.c, l.out_index = st.index, l.out_q = st.q, l.rows = r, l.n_rows = g.rows;
  l.factor = static_cast<float>(temperature * temperature);

  if (space.logit_rows > 0) {
    g.logits = reinterpret_cast<float*>(ws + space.logits), g.ldt = static_cast<int>(ceil_div(vocab, 256) * 256);
    l.logits = g.logits, l.ldt = g.ldt;
  }
  if (thin) {
    g.cols = static_cast<int>(vocab);
    if (direct) vl_thin_direct(g, r, weight, w_dtype, ldw, dim, planes, T, s);
    else vl_thin<VL_STATS>(g, weight, w_dtype, ldw, dim, planes, T, s);
  }
  const int64_t piece = vl_fwd_piece(dim, vocab, planes, packs);
  for (int64_t v0 = 0; v0 < vocab && !thin; v0 += piece) {
    const int64_t rows = std::min(piece, vocab - v0);
    if (packs) {
      VlPacked copy(ws, space.pack);
      if (half) copy.dst = nullptr;
      const int rc = vl_pack(weight, w_dtype, ldw, v0, rows, dim, planes, copy, piece * st.Dp, s);
      if (rc != FMOE_OK) return rc;
      g.b = half ? copy.half : copy.dst, g.b_plane = piece * st.Dp, g.ldb = static_cast<int>(st.Dp), g.b_scale = copy.scale;
    } else {
      g.b = static_cast<const uint16_t*>(weight) + v0 * ldw, g.ldb = static_cast<int>(ldw);
    }
    g.cols = static_cast<int>(rows), g.v0 = static_cast<int>(v0);
    if (space.logit_rows > 0) break;  // (one piece of the vocabulary)
    vl_stats<VL_STATS>(g, planes, st.Tp, s);
  }
  if (space.logit_rows > 0 && !thin) {
    vl_stored_lists(g, l, w_dtype, T, space.logit_rows, st.Dp, static_cast<int>(top), true, s);
  } else if (T > 0) {
    vl_stat(l, T, s);
    if (distill) vl_lists(l, w_dtype, T, s);
  }
  if (reduction != FMOE_REDUCE_NONE) vl_sum_kernel<<<1, 1024, 0, s>>>(st.head, l.row_loss, reduction, loss);
  return launch_status();
}

extern "C" int fmoe_vocab_loss_bwd(const float* d_loss, const void* weight, int w_dtype, int64_t ldw, int64_t T,
                                   int64_t dim, int64_t vocab, int64_t top, int distill, double logit_scale,
                                   double temperature, int planes, int reduction, const void* state, size_t state_bytes,
                                   void* d_hidden, int dh_dtype, void* d_weight, int dw_dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (T < 0 || dim <= 0 || vocab <= 0 || top <= 0 || distill < 0 || distill > 1 || (!distill && top != 1) ||
      reduction < 0 || reduction > 2 || (planes != 1 && planes != 3) || !vl_factors_ok(logit_scale, temperature) ||
      (!distill && temperature != 1.0))
    return FMOE_ERR_INVALID_ARG;
  if (!vl_sizes_ok(T, dim, vocab, top, planes)) return FMOE_ERR_SHAPE;
  if (vocab > 1 && (ldw < dim || ldw >= (int64_t(1) << 22))) return FMOE_ERR_SHAPE;
  if (!vl_dtype(w_dtype) || !vl_dtype(dh_dtype) || !vl_dtype(dw_dtype) || (planes == 3 && w_dtype != FMOE_F32))
    return FMOE_ERR_DTYPE;
  if (weight == nullptr || d_loss == nullptr) return FMOE_ERR_INVALID_ARG;
  if (!vl_elem_aligned(weight, w_dtype) || !vl_elem_aligned(d_loss, FMOE_F32) || !vl_elem_aligned(d_hidden, dh_dtype) ||
      !vl_elem_aligned(d_weight, dw_dtype) || !vl_ws_aligned(state) || !vl_ws_aligned(workspace))
    return FMOE_ERR_ALIGN;
  const bool packs = vl_packs(weight, w_dtype, ldw, dim, planes);
  const VlBwdSpace space(T, dim, vocab, planes, packs);
  const VlState st(static_cast<uint8_t*>(const_cast<void*>(state)), T, dim, top, planes);
  if (state == nullptr || state_bytes < st.bytes || workspace == nullptr || workspace_bytes < space.bytes)
    return FMOE_ERR_WORKSPACE;
  if (d_hidden == nullptr && d_weight == nullptr) return FMOE_OK;
  const hipStream_t s = as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint16_t* const gbuf = reinterpret_cast<uint16_t*>(ws + space.g);
  const int64_t piece = space.piece, g_plane = st.Tp * piece;
  const int64_t pack_plane = std::min(pad64(vocab), piece) * st.Dp;
  const int Dp = static_cast<int>(st.Dp);
  const int64_t mt = ceil_div(st.Tp, 256), dt = ceil_div(st.Dp, 256);
  const bool thin = vl_is_thin(T, vocab, packs), half = planes == 3 && !thin;
  for (int64_t v0 = 0; v0 < vocab; v0 += piece) {
    const int64_t rows = std::min(piece, vocab - v0), vt = ceil_div(rows, 256);
    VlGemm g{};
    g.head = st.head, g.rows = static_cast<int>(T), g.Tp = st.Tp, g.perm = st.perm, g.D = static_cast<int>(dim);
    g.split = reinterpret_cast<float*>(ws + space.split);
    const uint16_t* w = static_cast<const uint16_t*>(weight) + v0 * ldw;
    int64_t w_plane = 0;
    int w_ld = static_cast<int>(ldw);
    if (packs && !space.as_it_lies && (!thin || d_hidden != nullptr)) {
      VlPacked copy(ws, space.pack);
      if (!half) copy.half = nullptr;
      else g.b = copy.half, g.b_scale = copy.scale;
      if (planes == 3 && d_hidden == nullptr) copy.dst = nullptr;
      const int rc = vl_pack(weight, w_dtype, ldw, v0, rows, dim, planes, copy, pack_plane, s);
      if (rc != FMOE_OK) return rc;
      w = copy.dst, w_plane = pack_plane, w_ld = Dp;
    }
    g.a = half ? st.h16 : st.h, g.a_plane = st.plane, g.lda = Dp, g.k = Dp, g.a_scale = st.h_scale;
    if (!half) g.b = w;
    g.b_plane = w_plane, g.ldb = w_ld, g.cols = static_cast<int>(rows), g.v0 = static_cast<int>(v0);
    g.c = static_cast<float>(logit_scale / temperature * static_cast<double>(kLog2e));
    g.index = distill ? nullptr : st.index, g.picked = st.picked;
    g.stat = st.stat, g.d_loss = d_loss, g.reduction = reduction;
    g.factor = static_cast<float>(temperature * logit_scale);  // temperature^2 times d t / d logit
    g.g = gbuf, g.g_plane = g_plane, g.ldg = static_cast<int>(piece);
    if (thin) vl_thin<VL_GRAD>(g, weight, w_dtype, ldw, dim, planes, T, s);
    else if (planes == 1) vl_gemm_kernel<VL_GRAD, 1><<<vl_grid(mt * vt), core::NT, 0, s>>>(g);
    else vl_gemm_kernel<VL_GRAD, 3><<<vl_grid(mt * vt), core::NT, 0, s>>>(g);
    if (distill && T > 0) {
      FixArgs f{};
      f.head = st.head, f.perm = st.perm, f.index = st.index, f.q = st.q, f.picked = st.picked, f.stat = st.stat;
      f.d_loss = d_loss, f.top = static_cast<int>(top), f.rows = g.rows;
      f.v0 = static_cast<int>(v0), f.v1 = static_cast<int>(v0 + rows), f.reduction = reduction, f.planes = planes;
      f.ldg = g.ldg, f.factor = g.factor, f.g = gbuf, f.g_plane = g_plane;
      vl_fix_kernel<<<dim3(static_cast<uint32_t>(ceil_div(T * top, 256))), 256, 0, s>>>(f);
    }
    VlGemm h = g;
    h.a = gbuf, h.a_plane = g_plane, h.lda = g.ldg, h.b = w;
    h.cols = Dp, h.vocab = static_cast<int>(rows);
    if (d_hidden != nullptr) {
      h.out = d_hidden, h.out_dtype = dh_dtype, h.sum = reinterpret_cast<float*>(ws + space.sum);
      h.add = v0 > 0, h.more = v0 + rows < vocab;
      if (space.as_it_lies) vl_thin_dh(h, weight, ldw, st.inv, ThinDh(T, dim, std::min(vocab, piece)), s);
      else vl_product<VL_DH>(h, planes, mt, dt, ceil_div(rows, 64), h.more ? nullptr : st.inv, T, s);
    }
    if (d_weight != nullptr) {
      h.b = st.h, h.b_plane = st.plane, h.ldb = Dp, h.add = h.more = 0;
      h.out = static_cast<uint8_t*>(d_weight) + v0 * dim * (dw_dtype == FMOE_BF16 ? 2 : 4), h.out_dtype = dw_dtype;
      vl_product<VL_DW>(h, planes, vt, dt, st.Tp / 64, nullptr, 0, s);
    }
  }
  return launch_status();
}

extern "C" size_t fmoe_vocab_loss_grad_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int64_t top, int planes,
                                                       int packs) {
  return vl_sizes_ok(T, dim, vocab, top, planes) ? VlFusedSpace(T, dim, vocab, top, planes, packs).bytes : 0;
}

extern "C" int fmoe_vocab_loss_fwd_grad(const void* hidden, int h_dtype, int64_t ldh, const void* weight, int w_dtype,
                                        int64_t ldw, const void* index, int index64, const void* teacher, int t_dtype,
                                        int64_t T, int64_t dim, int64_t vocab, int64_t top, int64_t ignore_index,
                                        double logit_scale, double temperature, int planes, int reduction, float* loss,
                                        void* d_hidden, int dh_dtype, void* d_weight, int dw_dtype, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  const VlCall call{hidden, weight, index, teacher, h_dtype, w_dtype, index64, t_dtype, ldh, ldw, T, dim, vocab, top,
                    ignore_index, logit_scale, temperature, planes, reduction, loss};
  const bool distill = call.distill();
  if (const int rc = vl_check(call, nullptr, workspace); rc != FMOE_OK) return rc;
  if (reduction == FMOE_REDUCE_NONE) return FMOE_ERR_INVALID_ARG;
  if (!vl_dtype(dh_dtype) || !vl_dtype(dw_dtype)) return FMOE_ERR_DTYPE;
  if (!vl_elem_aligned(d_hidden, dh_dtype) || !vl_elem_aligned(d_weight, dw_dtype)) return FMOE_ERR_ALIGN;
  const bool packs = vl_packs(weight, w_dtype, ldw, dim, planes);
  const VlFusedSpace space(T, dim, vocab, top, planes, packs);
  if (space.piece == 0) return FMOE_ERR_SHAPE;
  if (workspace == nullptr || workspace_bytes < space.bytes) return FMOE_ERR_WORKSPACE;
  const hipStream_t s = as_stream(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const VlState st(ws + space.state, T, dim, top, planes);
  const RowsArgs r = vl_pack_rows(call, st, reinterpret_cast<uint32_t*>(ws + space.masks), true, false, s);

  const int Dp = static_cast<int>(st.Dp);
  const int64_t piece = space.piece, vt = ceil_div(vocab, 256), dt = ceil_div(st.Dp, 256), mt = piece / 256;
  const int64_t g_plane = piece * vt * 256, fh_plane = piece * st.Dp;
  uint16_t* const gbuf = reinterpret_cast<uint16_t*>(ws + space.g);
  uint16_t* const fh = reinterpret_cast<uint16_t*>(ws + space.fh);
  float* const factor = reinterpret_cast<float*>(ws + space.factor);
  float* const all_factor = reinterpret_cast<float*>(ws + space.all_factor);
  int* const flag = reinterpret_cast<int*>(ws + space.flag);
  const uint16_t *w = static_cast<const uint16_t*>(weight), *w16 = nullptr;
  const float* w_scale = nullptr;
  const bool half = planes == 3;
  int64_t w_plane = 0;
  int w_ld = static_cast<int>(ldw);
  if (packs) {
    VlPacked copy(ws, space.pack);
    if (!half) copy.half = nullptr;
    w16 = copy.half, w_scale = copy.scale;
    const int rc = vl_pack(weight, w_dtype, ldw, 0, vocab, dim, planes, copy, vocab * st.Dp, s);
    if (rc != FMOE_OK) return rc;
    w = copy.dst, w_plane = vocab * st.Dp, w_ld = Dp;
  }
  for (int64_t r0 = 0; r0 < std::max<int64_t>(T, 1); r0 += piece) {
    const int64_t rows = std::min(piece, T - r0);
    VlGemm g{};
    g.head = st.head, g.row0 = static_cast<int>(r0), g.rows = static_cast<int>(rows);
    const uint16_t* const rows_h = st.h + r0 * st.Dp;
    g.a = half ? st.h16 + r0 * st.Dp : rows_h, g.a_plane = st.plane, g.lda = Dp, g.k = Dp;
    if (half) g.a_scale = st.h_scale + r0, g.b_scale = w_scale;
    g.b = half ? w16 : w, g.b_plane = w_plane, g.ldb = w_ld, g.cols = static_cast<int>(vocab);
    g.c = static_cast<float>(logit_scale / temperature * static_cast<double>(kLog2e));
    g.index = distill ? nullptr : st.index + r0, g.picked = st.picked + r0 * top;
    g.part = reinterpret_cast<float2*>(ws + space.part), g.Tp = piece;
    g.off = reinterpret_cast<float*>(ws + space.off);
    g.stat = st.stat + r0, g.perm = st.perm + r0, g.factor = 1.0f, g.reduction = FMOE_REDUCE_SUM;
    g.g = gbuf, g.g_plane = g_plane, g.ldg = static_cast<int>(vt * 256);
    g.D = static_cast<int>(dim), g.split = reinterpret_cast<float*>(ws + space.split);

    LossArgs l{};
    l.head = st.head, l.row0 = g.row0, l.n_rows = g.rows, l.perm = g.perm, l.index = st.index + r0;
    l.part = g.part, l.Tp = piece, l.pieces = static_cast<int>(2 * vt), l.stat = st.stat + r0, l.picked = g.picked;
    l.row_loss = reinterpret_cast<float*>(ws + space.row_loss) + r0;
    l.h = rows_h, l.h_plane = st.plane, l.weight = weight, l.ldw = ldw;
    l.top = distill ? static_cast<int>(top) : 0;
    l.planes = planes, l.c = g.c, l.out_index = st.index + r0 * top, l.out_q = st.q + r0 * top, l.rows = r;
    l.factor = static_cast<float>(temperature * temperature);
    l.off = reinterpret_cast<float*>(ws + space.off), l.flag = flag;
    if (distill) l.row_part = reinterpret_cast<float*>(ws + space.row_part);

    const dim3 grid = vl_grid(mt * vt);
    if (space.stored) {
      VlGemm q = g;
      q.logits = reinterpret_cast<float*>(ws + space.logits), q.ldt = g.ldg;
      vl_stored_lists(q, l, w_dtype, std::max<int64_t>(rows, 1), vl_logit_rows(piece, vocab), st.Dp, static_cast<int>(top), false, s);
    } else if (distill) vl_lists(l, w_dtype, std::max<int64_t>(rows, 1), s);
    else if (w_dtype == FMOE_BF16) vl_off_kernel<FMOE_BF16><<<dim3(static_cast<uint32_t>(ceil_div(std::max<int64_t>(rows, 1), 4))), 256, 0, s>>>(l);
    else vl_off_kernel<FMOE_F32><<<dim3(static_cast<uint32_t>(ceil_div(std::max<int64_t>(rows, 1), 4))), 256, 0, s>>>(l);
    if (planes == 1) vl_gemm_kernel<VL_PROB, 1><<<grid, core::NT, 0, s>>>(g);
    else vl_gemm_kernel<VL_PROB, 3><<<grid, core::NT, 0, s>>>(g);
    vl_stat(l, std::max<int64_t>(rows, 1), s);
    // the ordinary way, where a row asks for it
    VlGemm q = g;
    LossArgs lq = l;
    q.only_if = lq.only_if = flag;
    lq.flag = nullptr;
    vl_stats<VL_STATS>(q, planes, piece, s);
    vl_stat(lq, std::max<int64_t>(rows, 1), s);
    q.index = nullptr;  // (the listed entries follow)
    if (planes == 1) vl_gemm_kernel<VL_GRAD, 1><<<grid, core::NT, 0, s>>>(q);
    else vl_gemm_kernel<VL_GRAD, 3><<<grid, core::NT, 0, s>>>(q);

    FixArgs f{};
    f.head = st.head, f.index = l.out_index, f.q = distill ? l.out_q : nullptr, f.picked = g.picked, f.stat = g.stat;
    f.top = static_cast<int>(top), f.v1 = static_cast<int>(vocab), f.planes = planes, f.ldg = g.ldg, f.g = gbuf;
    f.g_plane = g_plane, f.row0 = g.row0, f.rows = g.rows, f.flag = flag;
    if (rows > 0) vl_fix_kernel<<<dim3(static_cast<uint32_t>(ceil_div(rows * top, 256))), 256, 0, s>>>(f);
    const float fac = static_cast<float>(temperature * logit_scale);  // temperature^2 times d t / d logit
    const dim3 wave_rows(static_cast<uint32_t>(ceil_div(pad64(std::max<int64_t>(rows, 1)), 4)));
    if (planes == 1)
      vl_factor_kernel<1><<<wave_rows, 256, 0, s>>>(st.head, g.row0, g.rows, g.stat, flag, fac, reduction == FMOE_REDUCE_MEAN,
                                                   rows_h, st.plane, Dp, all_factor, factor, fh, fh_plane);
    else
      vl_factor_kernel<3><<<wave_rows, 256, 0, s>>>(st.head, g.row0, g.rows, g.stat, flag, fac, reduction == FMOE_REDUCE_MEAN,
                                                   rows_h, st.plane, Dp, all_factor, factor, fh, fh_plane);
    VlGemm h = g;
    h.a = gbuf, h.a_plane = g_plane, h.lda = g.ldg, h.b = w, h.cols = Dp, h.vocab = static_cast<int>(vocab);
    if (d_hidden != nullptr) {
      h.out = d_hidden, h.out_dtype = dh_dtype, h.row_factor = factor;
      // (rows without entries: once)
      vl_product<VL_DH>(h, planes, mt, dt, ceil_div(vocab, 64), r0 + piece >= T ? st.inv : nullptr, T, s);
    }
    if (d_weight != nullptr) {
      h.b = fh, h.b_plane = fh_plane, h.ldb = Dp, h.out = d_weight, h.out_dtype = dw_dtype, h.all_factor = all_factor;
      h.sum = reinterpret_cast<float*>(ws + space.sum), h.add = r0 > 0, h.more = piece < T;
      vl_product<VL_DW>(h, planes, vt, dt, ceil_div(rows, 64), nullptr, 0, s);
    }
  }
  if (d_weight != nullptr && piece < T) {
    const dim3 grid(static_cast<uint32_t>(ceil_div(vocab, 4)));
    const float* sum = reinterpret_cast<const float*>(ws + space.sum);
    const int d = static_cast<int>(dim);
    if (dw_dtype == FMOE_BF16) vl_dw_kernel<FMOE_BF16><<<grid, 256, 0, s>>>(sum, vocab, d, Dp, d_weight);
    else vl_dw_kernel<FMOE_F32><<<grid, 256, 0, s>>>(sum, vocab, d, Dp, d_weight);
  }
  vl_sum_kernel<<<1, 1024, 0, s>>>(st.head, reinterpret_cast<const float*>(ws + space.row_loss), reduction, loss);
  return launch_status();
}

extern "C" int fmoe_scale(const float* scale, const void* const* src, void* const* dst, const int* dtype,
                          const int64_t* n, int n_tensors, void* stream) {
  if (n_tensors < 0 || n_tensors > kScaleMax) return FMOE_ERR_INVALID_ARG;
  if (n_tensors == 0) return FMOE_OK;
  if (scale == nullptr || src == nullptr || dst == nullptr || dtype == nullptr || n == nullptr) return FMOE_ERR_INVALID_ARG;
  if (!vl_elem_aligned(scale, FMOE_F32)) return FMOE_ERR_ALIGN;
  ScaleArgs a{};
  a.scale = scale;
  int64_t most = 0;
  for (int i = 0; i < n_tensors; ++i) {
    if (n[i] < 0 || (n[i] > 0 && (src[i] == nullptr || dst[i] == nullptr))) return FMOE_ERR_INVALID_ARG;
    if (!vl_dtype(dtype[i])) return FMOE_ERR_DTYPE;
    if (!vl_elem_aligned(src[i], dtype[i]) || !vl_elem_aligned(dst[i], dtype[i])) return FMOE_ERR_ALIGN;
    a.src[i] = src[i], a.dst[i] = dst[i], a.n[i] = n[i], a.dtype[i] = dtype[i];
    most = std::max(most, n[i]);
  }
  if (most == 0) return FMOE_OK;
  const dim3 grid(static_cast<uint32_t>(std::min<int64_t>(ceil_div(most, 2048), 2048)), static_cast<uint32_t>(n_tensors));
  vl_scale_kernel<<<grid, 256, 0, as_stream(stream)>>>(a);
  return launch_status();
}
