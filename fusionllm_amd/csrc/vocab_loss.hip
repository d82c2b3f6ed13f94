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
// The logits [rows, vocab] are never stored: a tile's are reduced to a maximum and a sum of
// exponentials per row (forward), or turned into G (backward), a piece of the vocabulary at a time.
// That costs one product more than keeping them would (8 instead of 6 T V d flops), and
// bounds the extra memory by a piece.  All four products are bound by the matrix units and run on
// the main loop of gemm_core.h: 256 x 256 tiles, persistent workgroups, copies in one ring over all
// of a workgroup's tiles.
//
// Rows without a target (prompt tokens, padding) are left out first: the rows with one are packed, in
// order, with zeros up to a multiple of 64 rows and columns, so that they cost nothing and what is in
// them (also NaN) stays out of the products.
//
// Operands are bf16 (planes = 1), or fp32 as three bf16 numbers, hi + mid + lo (planes = 3): 24
// bits.  Of the nine products of such numbers the six largest are added, the smallest first, as six passes over K
// in one ring; what is left out is below 2^-22 of the largest.  G is rounded the same way: half a step of bf16,
// 2^-8 of an element at most, before the elements of a row or column are summed in fp32.
#include <algorithm>

#include "../../include/fusionvocab.h"
#include "elements.h"
#include "fmoe_common.h"
#include "gemm_core.h"

namespace fmoe {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kVlCus = 256;        // workgroups of the persistent products: one per CU
constexpr int kRowBlock = 32;      // rows per workgroup of the packing
constexpr int kGroup = 8;          // row tiles that are walked together, column by column
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
  float* entropy; // [T] sum of q ln q over the list as it was (distillation)
  float* picked;  // [T][top] t of the listed entries
  float2* stat;   // [T] m, l
  uint16_t* h;    // [planes][Tp][Dp] packed rows
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
    entropy = reinterpret_cast<float*>(take(T * 4));
    picked = reinterpret_cast<float*>(take(T * top * 4));
    stat = reinterpret_cast<float2*>(take(T * 8));
    h = reinterpret_cast<uint16_t*>(take(planes * plane * 2));
  }
};

// ---- packing ---------------------------------------------------------------------------------

struct RowsArgs {
  const void *hidden, *index, *teacher;
  int64_t ldh, ignore;
  int h_dtype, index64, t_dtype;  // t_dtype -1: no teacher
  int T, D, Dp, V, top, planes;
  int64_t plane;
  float inv_temp;
  int *counts, *head, *perm, *inv, *out_index;
  float *q, *entropy, *loss;  // loss: of rows without entries, where it is [T] (else nullptr)
  uint16_t* h;
};

// Entry k of row t: kNone, kBad or an index; z: its teacher logit over the temperature.
__device__ __forceinline__ int vl_entry(const RowsArgs& a, int64_t t, int k, float& z) {
  const int64_t e = t * a.top + k;
  const int64_t id = a.index64 ? static_cast<const int64_t*>(a.index)[e] : static_cast<const int32_t*>(a.index)[e];
  z = 0.0f;
  if (a.t_dtype >= 0) {
    const float raw = a.t_dtype == FMOE_BF16 ? bf2f(static_cast<const uint16_t*>(a.teacher)[e])
                                             : static_cast<const float*>(a.teacher)[e];
    if (raw == -__builtin_inff()) return kNone;
    z = raw * a.inv_temp;
  }
  if (id == a.ignore) return kNone;
  return id < 0 || id >= a.V ? kBad : static_cast<int>(id);
}

// Bit i: row block0 + i of the workgroup's rows has an entry (256 threads, all get the mask).
__device__ __forceinline__ uint32_t vl_rows_mask(const RowsArgs& a, int block0, uint32_t* shared_mask) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (threadIdx.x == 0) *shared_mask = 0;
  __syncthreads();
  float z;
  if (a.top == 1) {
    if (w == 0) {
      const bool has = lane < kRowBlock && block0 + lane < a.T && vl_entry(a, block0 + lane, 0, z) != kNone;
      const uint64_t m = __ballot(has);
      if (lane == 0) *shared_mask = static_cast<uint32_t>(m);
    }
  } else {
    for (int i = w; i < kRowBlock && block0 + i < a.T; i += 4) {
      bool has = false;
      for (int k = lane; k < a.top; k += 64) has = has || vl_entry(a, block0 + i, k, z) != kNone;
      if (__ballot(has) != 0 && lane == 0) atomicOr(shared_mask, 1u << i);
    }
  }
  __syncthreads();
  return *shared_mask;
}

__global__ __launch_bounds__(256) void vl_count_kernel(const RowsArgs a) {
  __shared__ uint32_t mask;
  const uint32_t m = vl_rows_mask(a, blockIdx.x * kRowBlock, &mask);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = __popc(m);
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

template <int DT, int PLANES>
__global__ __launch_bounds__(256) void vl_rows_kernel(const RowsArgs a) {
  __shared__ uint32_t mask_s;
  __shared__ int before_s[4];
  __shared__ float tz[4][FMOE_VOCAB_MAX_TOP];
  __shared__ int ti[4][FMOE_VOCAB_MAX_TOP];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int block0 = blockIdx.x * kRowBlock;
  const uint32_t mask = vl_rows_mask(a, block0, &mask_s);
  int before = 0;
  for (int i = threadIdx.x; i < static_cast<int>(blockIdx.x); i += 256) before += a.counts[i];
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off, 64);
  if (lane == 0) before_s[w] = before;
  __syncthreads();
  const int base = before_s[0] + before_s[1] + before_s[2] + before_s[3];
  const int n = base + __popc(mask);
  const bool last = blockIdx.x + 1 == gridDim.x;
  if (last) {  // zeros up to the next multiple of 64 rows
    if (threadIdx.x == 0) a.head[0] = n;
    for (int r = n + w; r < pad_rows(n); r += 4)
      for (int c = lane * 8; c < a.Dp; c += 512)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          *reinterpret_cast<uint4*>(a.h + p * a.plane + static_cast<int64_t>(r) * a.Dp + c) = make_uint4(0, 0, 0, 0);
  }
  for (int i = w; i < kRowBlock && block0 + i < a.T; i += 4) {
    const int64_t t = block0 + i;
    if (!((mask >> i) & 1)) {
      if (lane == 0) {
        a.inv[t] = -1;
        if (a.loss) a.loss[t] = 0.0f;
      }
      continue;
    }
    const int r = base + __popc(mask & ((1u << i) - 1));
    if (lane == 0) {
      a.inv[t] = r;
      a.perm[r] = static_cast<int>(t);
    }
    if (a.t_dtype < 0) {
      float z;
      if (lane == 0) a.out_index[r] = vl_entry(a, t, 0, z);
    } else {
      // softmax over the list; entries of one index are added to the first of them
      float peak = -__builtin_inff();
      bool nan = false;
      for (int k = lane; k < a.top; k += 64) {
        float z;
        const int id = vl_entry(a, t, k, z);
        ti[w][k] = id;
        tz[w][k] = z;
        if (id != kNone) peak = fmaxf(peak, z), nan = nan || z != z;
      }
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) peak = fmaxf(peak, __shfl_xor(peak, off, 64));
      if (__ballot(nan) != 0) peak = __builtin_nanf("");
      float sum = 0.0f;
      for (int k = lane; k < a.top; k += 64) {
        const float e = ti[w][k] == kNone ? 0.0f : expf(tz[w][k] - peak);
        sum = sum + e;
      }
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) sum = sum + __shfl_xor(sum, off, 64);
      const float log_sum = logf(sum);
      float ent = 0.0f;
      for (int k = lane; k < a.top; k += 64) {
        const float lq = (tz[w][k] - peak) - log_sum;
        const float q = ti[w][k] == kNone ? 0.0f : expf(lq);
        if (ti[w][k] != kNone && !(q == 0.0f)) ent = fmaf(q, lq, ent);
        tz[w][k] = q;
      }
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) ent = ent + __shfl_xor(ent, off, 64);
      if (lane == 0) a.entropy[r] = ent;
      __builtin_amdgcn_wave_barrier();
      for (int k = lane; k < a.top; k += 64) {
        const int id = ti[w][k];
        float q = tz[w][k];
        bool first = true;
        if (id >= 0) {
          q = 0.0f;
          for (int j = 0; j < a.top; ++j)
            if (ti[w][j] == id) {
              first = first && j >= k;
              q = q + tz[w][j];
            }
        }
        a.out_index[static_cast<int64_t>(r) * a.top + k] = first ? id : kNone;
        a.q[static_cast<int64_t>(r) * a.top + k] = first ? q : 0.0f;
      }
    }
    vl_copy_row<DT, PLANES>(a.hidden, t * a.ldh, a.D, a.Dp, a.h + static_cast<int64_t>(r) * a.Dp, a.plane, lane, 64);
  }
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

// ---- the products ----------------------------------------------------------------------------
// STATS  t = H W^T            -> a maximum and a sum of exponentials per row and 128 columns
// GRAD   t = H W^T of a piece -> G
// DH     G W of a piece, K split in ranges -> fp32 partial sums, added to the piece's before
// DW     G^T H                -> the piece's rows of dW
// H and G are row-major, so A is K-contiguous but for DW (G^T: read with transposing LDS reads), and B is
// K-contiguous for STATS and GRAD, and read as it lies, transposing, for DH (W) and DW (H).
enum VlMode { VL_STATS = 0, VL_GRAD = 1, VL_DH = 2, VL_DW = 3 };

struct VlGemm {
  const uint16_t *a, *b;
  int64_t a_plane, b_plane;
  int lda, ldb;
  int passes;           // 1, or 6: products of planes
  const int* head;      // rows with entries
  int cols;             // STATS, GRAD: vocabulary rows of the piece; DH, DW: columns (Dp)
  int vocab;            // DH, DW: vocabulary rows of the piece
  int k;                // STATS, GRAD: K (Dp)
  int ranges;           // DH: ranges of K
  float c;
  // STATS
  float2* part;         // [2 * column tiles][Tp]
  int64_t Tp;
  const int* index;     // cross entropy: the target's t is picked on the way (else nullptr)
  float* picked;
  int v0;               // the piece's first vocabulary row
  // GRAD
  const float2* stat;
  const float* d_loss;
  const int* perm;
  float factor;
  int reduction, planes;
  uint16_t* g;
  int64_t g_plane;
  int ldg;              // a multiple of 256
  // DH
  float* sum;           // [ranges][Tp][Dp]
  int add;              // there is a piece before
  // DW
  void* dw;
  int D, dw_dtype;
};

struct VlItem {
  int tm, tn, k0, kn, range;
};

// Planes of a pass, the smallest products first: (0, 2), (1, 1), (2, 0), (0, 1), (1, 0), (0, 0).
__device__ __forceinline__ void vl_planes(int passes, int pass, int& pa, int& pb) {
  const int i = 2 * (pass + 6 - passes);  // (a single pass: the last)
  pa = (0x124 >> i) & 3;
  pb = (0x046 >> i) & 3;
}

template <int MODE>
__global__ __launch_bounds__(core::NT, 1) void vl_gemm_kernel(const VlGemm a) {
  using namespace core;
  constexpr bool ATR = MODE == VL_DW, BTR = MODE == VL_DH || MODE == VL_DW;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[SMEM];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = w / WN, wn = w % WN;
  const uint32_t sbase = lds_addr(smem);
  const int n = __builtin_amdgcn_readfirstlane(a.head[0]);
  const int np = pad_rows(n);
  const int m_rows = MODE == VL_DW ? a.vocab : np;
  const int tiles_m = (m_rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN;
  const int nk = MODE == VL_DH ? (a.vocab + BK - 1) / BK : MODE == VL_DW ? np / BK : a.k / BK;
  const int ranges = MODE == VL_DH ? a.ranges : 1;
  const int tiles = tiles_m * tiles_n, items = tiles * ranges;
  // Workgroup b runs on XCD b % 8.  Each XCD takes a contiguous eighth of the items.
  const int xcd = static_cast<int>(blockIdx.x) % 8, step = static_cast<int>(gridDim.x) / 8;
  const int first = static_cast<int>(static_cast<int64_t>(items) * xcd / 8) + static_cast<int>(blockIdx.x) / 8;
  const int end = static_cast<int>(static_cast<int64_t>(items) * (xcd + 1) / 8);
  const int my_items = (end - first + step - 1) / step;
  if (my_items <= 0) return;

  // Items in order: K ranges, then groups of kGroup row tiles, in a group column by column: the 32
  // workgroups of an XCD share 8 + 4 operand panels instead of 1 + 32.
  auto locate = [&](int item) __attribute__((always_inline)) {
    VlItem t;
    t.range = MODE == VL_DH ? item / tiles : 0;
    const int q = item - t.range * tiles, per = kGroup * tiles_n;
    const int g = q / per, rem = q - g * per, rows = min(tiles_m - g * kGroup, kGroup);
    t.tn = rem / rows;
    t.tm = g * kGroup + rem - t.tn * rows;
    t.k0 = static_cast<int>(static_cast<int64_t>(nk) * t.range / ranges);
    t.kn = static_cast<int>(static_cast<int64_t>(nk) * (t.range + 1) / ranges) - t.k0;
    t.tm = __builtin_amdgcn_readfirstlane(t.tm);
    t.tn = __builtin_amdgcn_readfirstlane(t.tn);
    t.k0 = __builtin_amdgcn_readfirstlane(t.k0);
    t.kn = __builtin_amdgcn_readfirstlane(t.kn);
    t.range = __builtin_amdgcn_readfirstlane(t.range);
    return t;
  };

  // ---- copy cursor (the units of a stage and their LDS layout as in gemm_core.h)
  const uint32_t lds_a = ATR ? sbase + w * 1024 : sbase + (64 * (w >> 2) + 8 * (w & 3)) * RB;
  const uint32_t lds_b = sbase + A_BYTES + w * 1024;
  const int lda = a.lda, ldb = a.ldb;
  VlItem c_t = locate(first);
  int c_ti = 0, c_pass = 0, c_k = 0, c_left = 0;
  const uint8_t *c_a = nullptr, *c_b = nullptr;
  int64_t astep = ATR ? static_cast<int64_t>(2 * BK) * lda : RB, bstep = BTR ? static_cast<int64_t>(2 * BK) * ldb : RB;
  uint32_t a_off[4], b_off[4];
  // pointers and offsets of step c_k of pass c_pass, and the steps until the next call
  auto place = [&]() __attribute__((always_inline)) {
    int pa, pb;
    vl_planes(a.passes, c_pass, pa, pb);
    const int k = (c_t.k0 + c_k) * BK;
    const uint16_t* p = a.a + pa * a.a_plane + (ATR ? static_cast<int64_t>(k) * lda : static_cast<int64_t>(c_t.tm) * BM * lda + k);
    const uint16_t* q = a.b + pb * a.b_plane + (BTR ? static_cast<int64_t>(k) * ldb : static_cast<int64_t>(c_t.tn) * BN * ldb + k);
    c_a = reinterpret_cast<const uint8_t*>(p);
    c_b = reinterpret_cast<const uint8_t*>(q);
    c_left = c_t.kn - c_k;
    if (MODE == VL_DH && (a.vocab & (BK - 1)) && c_t.k0 + c_t.kn == nk && c_left > 1) --c_left;  // the last step has clamped rows
    // the lane as an opaque value: what follows is formed here, not kept through the main loop
    int l = lane;
    asm volatile("" : "+v"(l));
    const int dchunk = (l & 7) ^ swzk(l >> 3);
    const int krow = 4 * w + (l >> 4);
    const int cb = ((((l & 15) >> 1) ^ wsw(krow)) << 1) | (l & 1);
    if constexpr (ATR) {
      // unit u: rows (of C) 32 u .. + 31 of every wave's 64
      const int m0 = c_t.tm * BM;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        a_off[q] = static_cast<uint32_t>((32 * (q & 1) + krow) * lda +
                                         min(m0 + 64 * (cb >> 2) + 32 * (q >> 1) + 8 * (cb & 3), lda - 8)) * 2u;
    } else {
      const int last_m = min(m_rows - c_t.tm * BM, BM) - 1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = min(64 * (w >> 2) + 8 * (w & 3) + (l >> 3) + 128 * (q & 1) + 32 * (q >> 1), last_m);
        a_off[q] = static_cast<uint32_t>(r * lda + dchunk * 8) * 2u;
      }
    }
    if constexpr (BTR) {
      const int n0 = c_t.tn * BN, last_k = MODE == VL_DH ? a.vocab - 1 - k : BK;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        b_off[q] = static_cast<uint32_t>(min(32 * (q & 1) + krow, last_k) * ldb +
                                         min(n0 + 128 * (cb >> 3) + 8 * (cb & 7) + 64 * (q >> 1), a.cols - 8)) * 2u;
    } else {
      const int last_n = min(a.cols - c_t.tn * BN, BN) - 1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = min(128 * (q & 1) + 64 * (q >> 1) + 8 * w + (l >> 3), last_n);
        b_off[q] = static_cast<uint32_t>(r * ldb + dchunk * 8) * 2u;
      }
    }
  };
  place();
  int c_run = c_left;
  // A stage's units are issued in the order A0, B0, B1, A1; A1 moves the cursor on.  Past the last
  // step the last stage is copied again (into slots that are free and not read any more).
  auto advance = [&]() __attribute__((always_inline)) {
    c_k += c_run;
    if (c_k == c_t.kn) {
      c_k = 0;
      if (++c_pass == a.passes) {
        c_pass = 0;
        if (++c_ti == my_items) {
          c_a -= astep;
          c_b -= bstep;
          astep = bstep = 0;
          c_left = INT32_MAX;
          return;
        }
        c_t = locate(first + c_ti * step);
      }
    }
    place();
    c_run = c_left;
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
  uint8_t* ep = smem + 2 * STAGE + w * EPI;  // this wave's staging (4 KB)
  int e_ti = 0;
  VlItem e_t = locate(first);
  int e_left = e_t.kn * a.passes;
  for (int it = 0;; ++it) {
    // keep the per-step fragment addresses from being hoisted out of the loop
    asm volatile("" : "+v"(xa), "+v"(xb));
    const uint32_t st = sbase + (it & 1) * STAGE, nxt = sbase + ((it + 1) & 1) * STAGE;
    // (0, 0)
#pragma unroll
    for (int q = 0; q < 4; ++q) read_b(b0, 0, st, 1, q);
    issue_a(it + 1, 1);
    wait_vm_barrier<5 * LU>();  // B1 of this stage
    quarter<0, 0>(acc, a0, b0);
    // (0, 1)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int q = 0; q < 4; ++q) read_b(b1, 1, st, kh, q);
    issue_a(it + 2, 0);
    wait_vm_barrier<5 * LU>();  // A1 of this stage
    quarter<0, 1>(acc, a0, b1);
    // (1, 0)
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int m = 0; m < 2; ++m) read_a(a1, 1, st, kh, m);
    issue_b(it + 2, 0);
    wait_vm_barrier<4 * LU>();  // A0, B0 of the next stage
    quarter<1, 0>(acc, a1, b0);
    // (1, 1): the next step's first fragments (at a tile's end they are read again after its epilogue)
    read_first(nxt);
    issue_b(it + 2, 1);
    wait_lds_barrier();
    quarter<1, 1>(acc, a1, b1);

    if (--e_left > 0) continue;
    // ---- tile epilogue: this wave's 64 x 128 block (both wave groups together)
    if (!late) barrier();
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3\n" ::: "memory");  // MFMA results -> VALU reads
    int el = lane;
    asm volatile("" : "+v"(el));  // the address arithmetic below stays out of the main loop
    const int row0 = e_t.tm * BM + wm * WTM, col0 = e_t.tn * BN + wn * WTN;
    const int er = el & 15, eg = el >> 4;  // acc[i][j]: row 16 i + er, columns 16 j + 4 eg + 0..3

    if constexpr (MODE == VL_STATS) {
      float2 mine = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = row0 + 16 * i + er;
        float m = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float t = col0 + 16 * j + 4 * eg + e < a.cols ? acc[i][j][e] * a.c : -__builtin_inff();
            acc[i][j][e] = t;
            m = fmaxf(m, t);
          }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float peak = m == -__builtin_inff() ? 0.0f : m;  // (no columns: a sum of zero; NaN stays NaN)
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s = s + __builtin_amdgcn_exp2f(acc[i][j][e] - peak);
        s = s + __shfl_xor(s, 16, 64);
        s = s + __shfl_xor(s, 32, 64);
        if (eg == i) mine = make_float2(m, s);
        if (a.index) {  // the target's column, where it is in this block
          const int rel = row < n ? a.index[row] - (a.v0 + col0) : -1;
          const bool here = rel >= 0 && rel < WTN && col0 + rel < a.cols;
          if (__ballot(here) != 0) {
            float t = 0.0f;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) t = rel == 16 * j + 4 * eg + e ? acc[i][j][e] : t;
            if (here && ((rel >> 2) & 3) == eg) a.picked[row] = t;
          }
        }
      }
      const int row = row0 + el;  // lane group eg kept block eg
      if (row < n) a.part[((a.v0 / BN + e_t.tn) * WN + wn) * a.Tp + row] = mine;
    } else if constexpr (MODE == VL_GRAD) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = row0 + 16 * i + er;
        float2 ml = make_float2(0.0f, 0.0f);
        float up = 0.0f;
        if (row < n) {
          ml = a.stat[row];
          up = a.reduction == FMOE_REDUCE_NONE ? a.d_loss[a.perm[row]] : a.d_loss[0];
          if (a.reduction == FMOE_REDUCE_MEAN) up = up / static_cast<float>(n);
          up = up * a.factor;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = __builtin_amdgcn_exp2f((acc[i][j][e] * a.c - ml.x) - ml.y);
            acc[i][j][e] = row < n && col0 + 16 * j + 4 * eg + e < a.cols ? p * up : 0.0f;
          }
        for (int p = 0; p < a.planes; ++p) {
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            const int col = j * 16 + eg * 4;
            const uint32_t off = er * 256 + ((((col >> 3) ^ er)) << 4) + (col & 7) * 2;
            uint2 u;
            u.x = pack2(acc[i][j][0], acc[i][j][1]);
            u.y = pack2(acc[i][j][2], acc[i][j][3]);
            *reinterpret_cast<uint2*>(ep + off) = u;
            acc[i][j][0] = acc[i][j][0] - __uint_as_float(u.x << 16);
            acc[i][j][1] = acc[i][j][1] - __uint_as_float(u.x & 0xffff0000u);
            acc[i][j][2] = acc[i][j][2] - __uint_as_float(u.y << 16);
            acc[i][j][3] = acc[i][j][3] - __uint_as_float(u.y & 0xffff0000u);
          }
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int r = t * 4 + eg, c = er, grow = row0 + 16 * i + r;
            const uint4 v = *reinterpret_cast<const uint4*>(ep + r * 256 + ((c ^ r) << 4));
            if (grow < np) *reinterpret_cast<uint4*>(a.g + p * a.g_plane + static_cast<int64_t>(grow) * a.ldg + col0 + c * 8) = v;
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    } else if constexpr (MODE == VL_DH) {
      float* out = a.sum + static_cast<int64_t>(e_t.range) * a.Tp * a.cols;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int row = row0 + 16 * i + er;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int col = col0 + 16 * j + 4 * eg;
          if (row < n && col < a.cols) {
            f32x4* p = reinterpret_cast<f32x4*>(out + static_cast<int64_t>(row) * a.cols + col);
            f32x4 v = acc[i][j];
            if (a.add) {
              const f32x4 o = *p;
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = o[e] + v[e];
            }
            *p = v;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        // 16 rows x 64 columns of fp32 at a time; chunk c of row r at slot c ^ r
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
            const int row = row0 + 16 * i + r, col = col0 + 64 * jh + c;
            const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (row < a.vocab && col < a.D) {
              const int64_t o = static_cast<int64_t>(row) * a.D + col;
              if (a.dw_dtype == FMOE_BF16) store_upto8<FMOE_BF16>(a.dw, o, a.D - col, v);
              else store_upto8<FMOE_F32>(a.dw, o, a.D - col, v);
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
    if (++e_ti == my_items) break;
    e_t = locate(first + e_ti * step);
    e_left = e_t.kn * a.passes;
    // the next tile's first fragments
    read_first(sbase + ((it + 1) & 1) * STAGE);
    if (late) barrier();
  }
  // the copies past the end have landed before the workgroup's LDS is given back
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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
  const float *q, *entropy;
  const uint16_t* h;
  int64_t h_plane;
  const void* weight;
  int64_t ldw;
  int top, D, Dp, w_dtype, planes;
  float c, factor;    // factor: temperature^2
};

__device__ __forceinline__ void vl_store_loss(const LossArgs& a, int row, float v) {
  if (a.loss) a.loss[a.perm[row]] = v;
  else a.row_loss[row] = v;
}

// m and l of R rows per workgroup: each of its 1024 / R threads per row joins every so many of the partial
// sums, in order; then lanes, then waves.
__device__ __forceinline__ void vl_join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2), peak = top == -__builtin_inff() ? 0.0f : top;
  s = s * __builtin_amdgcn_exp2f(m - peak) + s2 * __builtin_amdgcn_exp2f(m2 - peak);
  m = top;
}

template <int R>
__global__ __launch_bounds__(1024) void vl_stat_kernel(const LossArgs a) {
  __shared__ float2 red[16][R];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = a.head[0];
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
    const int id = a.index[row];
    if (id == kBad) l = __builtin_nanf("");
    else vl_store_loss(a, row, ((m - a.picked[row]) + l) * kLn2);
    if (id == kBad) vl_store_loss(a, row, l);
  }
  a.stat[row] = make_float2(m, l);
}

// Distillation: t of a row's listed entries (a dot product of length D each, in fp32), and its loss.
template <int DT>
__global__ __launch_bounds__(256) void vl_list_kernel(const LossArgs a) {
  extern __shared__ float h[];
  __shared__ float red[4];
  __shared__ int bad_s;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, row = blockIdx.x;
  if (row >= a.head[0]) return;
  if (threadIdx.x == 0) bad_s = 0;
  const bool round = DT == FMOE_F32 && a.planes == 1;
  for (int c = threadIdx.x * 8; c < a.Dp; c += 2048) {
    float v[8];
    const uint16_t* p = a.h + static_cast<int64_t>(row) * a.Dp + c;
    unpack8(*reinterpret_cast<const uint4*>(p), v);
    for (int q = 1; q < a.planes; ++q) {
      float u[8];
      unpack8(*reinterpret_cast<const uint4*>(p + q * a.h_plane), u);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] + u[e];  // exact: the parts of one fp32 number
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) h[c + e] = v[e];
  }
  __syncthreads();
  const float2 ml = a.stat[row];
  float cross = 0.0f;
  for (int k = w; k < a.top; k += 4) {
    const int id = __builtin_amdgcn_readfirstlane(a.index[static_cast<int64_t>(row) * a.top + k]);
    if (id < 0) {
      if (id == kBad && lane == 0) bad_s = 1;
      continue;
    }
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    for (int c = lane * 8; c < a.D; c += 512) {
      float v[8];
      load_upto8<DT>(a.weight, static_cast<int64_t>(id) * a.ldw + c, a.D - c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(round ? bf_round(v[e]) : v[e], h[c + e], acc[e]);
    }
    float s = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s = s + __shfl_xor(s, off, 64);
    const float t = s * a.c, q = a.q[static_cast<int64_t>(row) * a.top + k];
    if (lane == 0) a.picked[static_cast<int64_t>(row) * a.top + k] = t;
    if (!(q == 0.0f)) cross = fmaf(q, (ml.x - t) + ml.y, cross);
  }
  if (lane == 0) red[w] = cross;
  __syncthreads();
  if (threadIdx.x == 0) {
    float v = fmaf((red[0] + red[1]) + (red[2] + red[3]), kLn2, a.entropy[row]) * a.factor;
    if (bad_s) {
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
  for (int i = threadIdx.x; i < n; i += 1024) s = s + static_cast<double>(row_loss[i]);
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

// ---- backward: the listed entries of G, and dH ------------------------------------------------------

struct FixArgs {
  const int *head, *perm, *index;
  const float *q, *picked;
  const float2* stat;
  const float* d_loss;
  int top, distill, v0, v1, reduction, planes, ldg;
  int64_t rows_cap;
  float factor;
  uint16_t* g;
  int64_t g_plane;
};

// G at the entries that lie in this piece of the vocabulary: factor * (p - q) in fp32, rounded once.
__global__ __launch_bounds__(256) void vl_fix_kernel(const FixArgs a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int n = a.head[0];
  const int64_t row = i / a.top;
  if (row >= n) return;
  const int id = a.index[i];
  if (id < a.v0 || id >= a.v1) return;
  const float2 ml = a.stat[row];
  const float lp = (a.picked[i] - ml.x) - ml.y;  // log2 p
  float up = a.reduction == FMOE_REDUCE_NONE ? a.d_loss[a.perm[row]] : a.d_loss[0];
  if (a.reduction == FMOE_REDUCE_MEAN) up = up / static_cast<float>(n);
  up = up * a.factor;
  // (p - 1 where p is near 1: from the logarithm)
  float v = (a.distill ? __builtin_amdgcn_exp2f(lp) - a.q[i] : expm1f(lp * kLn2)) * up;
  uint16_t* p = a.g + row * a.ldg + (id - a.v0);
  for (int k = 0; k < a.planes; ++k) {
    const uint16_t b = f2bf(v);
    p[k * a.g_plane] = b;
    v = v - bf2f(b);
  }
}

// dH of a row: its partial sums in order; zeros in rows that were not packed.
template <int DT>
__global__ __launch_bounds__(256) void vl_dh_kernel(const int* inv, const float* sum, int64_t stride, int ranges, int64_t T,
                                                    int D, int Dp, void* out) {
  const int lane = threadIdx.x & 63;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (t >= T) return;
  const int r = __builtin_amdgcn_readfirstlane(inv[t]);
  for (int c = lane * 8; c < D; c += 512) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (r >= 0) {
      const float* p = sum + static_cast<int64_t>(r) * Dp + c;
      constexpr int U = 4;
      for (int s0 = 0; s0 < ranges; s0 += U) {
        f32x4 u[U][2];
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const f32x4* q = reinterpret_cast<const f32x4*>(p + min(s0 + s, ranges - 1) * stride);
          u[s][0] = q[0], u[s][1] = q[1];
        }
#pragma unroll
        for (int s = 0; s < U; ++s)
          if (s0 + s < ranges)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = v[e] + u[s][0][e], v[4 + e] = v[4 + e] + u[s][1][e];
      }
    }
    store_upto8<DT>(out, t * D + c, D - c, v);
  }
}

// ---- host ------------------------------------------------------------------------------------------

// Pieces of the vocabulary and ranges of dH's K.  The pieces' G is bounded (kPieceBytes); within that, the
// number of pieces, and of ranges, whose tiles fill the CUs' rounds best: a launch's time is its rounds of
// tiles, each K steps and an epilogue long.
constexpr int64_t kPieceBytes = int64_t(1) << 29;
constexpr int64_t kPackBytes = int64_t(1) << 28;
constexpr int64_t kSumBytes = int64_t(1) << 30;

struct VlPlan {
  int64_t piece;  // vocabulary rows of a piece, a multiple of 256 (the last one has fewer)
  int ranges;
};

VlPlan vl_plan(int64_t T, int64_t D, int64_t V, int planes) {
  const int64_t mt = std::max<int64_t>(ceil_div(T, 256), 1), dt = ceil_div(D, 256), vt = ceil_div(V, 256);
  const int64_t Tp = std::max<int64_t>(pad64(T), 64), Dp = pad64(D);
  const int passes = planes == 3 ? 6 : 1;
  // us: a K step of a full chip, a tile's epilogue, a launch
  const double step = 1.9 * passes, tile = 4.0, launch = 6.0;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>({vt, kPieceBytes / (Tp * 512 * planes), 4096}));
  const int64_t fewest = ceil_div(vt, most);
  auto rounds = [](int64_t items) { return static_cast<double>(ceil_div(items, kVlCus)); };
  VlPlan best{};
  double best_time = 0.0;
  for (int64_t pieces = fewest; pieces <= fewest + 12 && pieces <= vt; ++pieces) {
    const int64_t pt = ceil_div(vt, pieces);
    for (int s = 1; s <= 64; ++s) {
      if (s > 1 && (pt * 4 < s * 8 || s * Tp * Dp * 4 > kSumBytes)) break;
      const double add = static_cast<double>(s) * Tp * Dp * 8.0 / 4e6;  // the partial sums' traffic, us
      const double time = ceil_div(vt, pt) * (rounds(mt * pt) * (Dp / 64 * step + tile) + rounds(pt * dt) * (Tp / 64 * step + tile) +
                                    rounds(mt * dt * s) * (4.0 * pt / s * step + tile) + add + 3 * launch);
      if (best.piece == 0 || time < best_time) best = {pt * 256, s}, best_time = time;
    }
  }
  return best;
}

// Vocabulary rows of a piece of the forward: all of them, or as many as a packed copy may have.
int64_t vl_fwd_piece(int64_t D, int64_t V, int planes, bool packs) {
  if (!packs) return V;
  return std::min(V, std::max<int64_t>(kPackBytes / (pad64(D) * 2 * planes) / 256, 1) * 256);
}

struct VlFwdSpace {
  size_t counts, part, row_loss, pack, bytes = 0;
  VlFwdSpace(int64_t T, int64_t D, int64_t V, int planes, bool packs) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    const int64_t Tp = std::max<int64_t>(pad64(T), 64);
    counts = take(ceil_div(T, kRowBlock) * 4);
    part = take(2 * ceil_div(V, 256) * Tp * 8);
    row_loss = take(T * 4);
    pack = take(packs ? vl_fwd_piece(D, V, planes, true) * pad64(D) * 2 * planes : 0);
  }
};

struct VlBwdSpace {
  VlPlan plan;
  size_t g, sum, pack, bytes = 0;
  VlBwdSpace(int64_t T, int64_t D, int64_t V, int planes, bool packs) : plan(vl_plan(T, D, V, planes)) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    const int64_t Tp = std::max<int64_t>(pad64(T), 64), Dp = pad64(D);
    g = take(Tp * plan.piece * 2 * planes);
    sum = take(plan.ranges * Tp * Dp * 4);
    pack = take(packs ? std::min(pad64(V), plan.piece) * Dp * 2 * planes : 0);
  }
};

bool vl_sizes_ok(int64_t T, int64_t dim, int64_t vocab, int64_t top, int planes) {
  return T >= 0 && dim > 0 && vocab > 0 && top > 0 && dim <= FMOE_VOCAB_MAX_DIM && T <= FMOE_VOCAB_MAX_TOKENS &&
         vocab <= FMOE_VOCAB_MAX_VOCAB && top <= FMOE_VOCAB_MAX_TOP && T * dim <= FMOE_VOCAB_MAX_ELEMENTS &&
         vocab * dim <= FMOE_VOCAB_MAX_ELEMENTS && T * top < (int64_t(1) << 31) && (planes == 1 || planes == 3);
}

bool vl_packs(const void* weight, int w_dtype, int64_t ldw, int64_t dim, int planes) {
  return planes != 1 || w_dtype != FMOE_BF16 || dim % 64 != 0 || ldw % 8 != 0 || !aligned16(weight);
}

int vl_pack(const void* weight, int w_dtype, int64_t ldw, int64_t v0, int64_t rows, int64_t D, int planes, uint16_t* dst,
            int64_t plane, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>(ceil_div(rows, 4)));
  const int Dp = static_cast<int>(pad64(D)), r = static_cast<int>(rows), d = static_cast<int>(D);
  if (w_dtype == FMOE_BF16 && planes == 1) vl_pack_kernel<FMOE_BF16, 1><<<grid, 256, 0, s>>>(weight, ldw, v0, r, d, Dp, dst, plane);
  else if (w_dtype == FMOE_BF16) vl_pack_kernel<FMOE_BF16, 3><<<grid, 256, 0, s>>>(weight, ldw, v0, r, d, Dp, dst, plane);
  else if (planes == 1) vl_pack_kernel<FMOE_F32, 1><<<grid, 256, 0, s>>>(weight, ldw, v0, r, d, Dp, dst, plane);
  else vl_pack_kernel<FMOE_F32, 3><<<grid, 256, 0, s>>>(weight, ldw, v0, r, d, Dp, dst, plane);
  return launch_status();
}

bool vl_elem_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FMOE_BF16 ? 1u : 3u)) == 0;
}
bool vl_ws_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }
bool vl_dtype(int d) { return d == FMOE_BF16 || d == FMOE_F32; }

// Workgroups of a product of so many tiles: one per CU, fewer only in eighths.
dim3 vl_grid(int64_t items) { return dim3(static_cast<uint32_t>(std::min<int64_t>(kVlCus, ceil_div(items, 8) * 8))); }

}  // namespace fmoe

using namespace fmoe;

extern "C" size_t fmoe_vocab_loss_state_bytes(int64_t T, int64_t dim, int64_t top, int planes) {
  return vl_sizes_ok(T, dim, 1, top, planes) ? VlState(nullptr, T, dim, top, planes).bytes : 0;
}

extern "C" int fmoe_vocab_loss_packs(const void* weight, int w_dtype, int64_t ldw, int64_t dim, int planes) {
  return vl_packs(weight, w_dtype, ldw, dim, planes);
}

extern "C" size_t fmoe_vocab_loss_fwd_workspace_bytes(int64_t T, int64_t dim, int64_t vocab, int planes, int packs) {
  return vl_sizes_ok(T, dim, vocab, 1, planes) ? VlFwdSpace(T, dim, vocab, planes, packs).bytes : 0;
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
  const bool distill = teacher != nullptr || top != 1;
  if (T < 0 || dim <= 0 || vocab <= 0 || top <= 0 || index64 < 0 || index64 > 1 || reduction < 0 || reduction > 2 ||
      (planes != 1 && planes != 3) || !(temperature > 0.0) || (!distill && temperature != 1.0))
    return FMOE_ERR_INVALID_ARG;
  if (!vl_sizes_ok(T, dim, vocab, top, planes)) return FMOE_ERR_SHAPE;
  if ((T > 1 && (ldh < dim || ldh > (int64_t(1) << 38))) || (vocab > 1 && (ldw < dim || ldw >= (int64_t(1) << 22))))
    return FMOE_ERR_SHAPE;
  if (!vl_dtype(h_dtype) || !vl_dtype(w_dtype) || (teacher && !vl_dtype(t_dtype))) return FMOE_ERR_DTYPE;
  if (weight == nullptr || (T > 0 && (hidden == nullptr || index == nullptr || (distill && teacher == nullptr))) ||
      loss == nullptr)
    return FMOE_ERR_INVALID_ARG;
  if (!vl_elem_aligned(hidden, h_dtype) || !vl_elem_aligned(weight, w_dtype) || !vl_elem_aligned(loss, FMOE_F32) ||
      (teacher && !vl_elem_aligned(teacher, t_dtype)) ||
      (reinterpret_cast<uintptr_t>(index) & (index64 ? 7u : 3u)) != 0 || !vl_ws_aligned(state) || !vl_ws_aligned(workspace))
    return FMOE_ERR_ALIGN;
  const bool packs = vl_packs(weight, w_dtype, ldw, dim, planes);
  const VlFwdSpace space(T, dim, vocab, planes, packs);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const VlState st(static_cast<uint8_t*>(state), T, dim, top, planes);
  if (state == nullptr || state_bytes < st.bytes || workspace == nullptr || workspace_bytes < space.bytes)
    return FMOE_ERR_WORKSPACE;
  const hipStream_t s = as_stream(stream);
  const int64_t blocks = std::max<int64_t>(ceil_div(T, kRowBlock), 1);

  RowsArgs r{};
  r.hidden = hidden, r.index = index, r.teacher = teacher, r.ldh = ldh, r.ignore = ignore_index;
  r.h_dtype = h_dtype, r.index64 = index64, r.t_dtype = distill ? t_dtype : -1;
  r.T = static_cast<int>(T), r.D = static_cast<int>(dim), r.Dp = static_cast<int>(st.Dp), r.V = static_cast<int>(vocab);
  r.top = static_cast<int>(top), r.planes = planes, r.plane = st.plane;
  r.inv_temp = static_cast<float>(1.0 / temperature);
  r.counts = reinterpret_cast<int*>(ws + space.counts);
  r.head = st.head, r.perm = st.perm, r.inv = st.inv, r.out_index = st.index, r.q = st.q, r.entropy = st.entropy, r.h = st.h;
  r.loss = reduction == FMOE_REDUCE_NONE ? loss : nullptr;
  if (blocks > 1) vl_count_kernel<<<dim3(static_cast<uint32_t>(blocks)), 256, 0, s>>>(r);
  const dim3 rows_grid(static_cast<uint32_t>(blocks));
  if (h_dtype == FMOE_BF16 && planes == 1) vl_rows_kernel<FMOE_BF16, 1><<<rows_grid, 256, 0, s>>>(r);
  else if (h_dtype == FMOE_BF16) vl_rows_kernel<FMOE_BF16, 3><<<rows_grid, 256, 0, s>>>(r);
  else if (planes == 1) vl_rows_kernel<FMOE_F32, 1><<<rows_grid, 256, 0, s>>>(r);
  else vl_rows_kernel<FMOE_F32, 3><<<rows_grid, 256, 0, s>>>(r);

  VlGemm g{};
  g.a = st.h, g.a_plane = st.plane, g.lda = static_cast<int>(st.Dp);
  g.passes = planes == 3 ? 6 : 1, g.head = st.head, g.k = static_cast<int>(st.Dp);
  g.c = static_cast<float>(logit_scale / temperature * static_cast<double>(kLog2e));
  g.part = reinterpret_cast<float2*>(ws + space.part), g.Tp = st.Tp;
  g.index = distill ? nullptr : st.index, g.picked = st.picked;
  const int64_t piece = vl_fwd_piece(dim, vocab, planes, packs);
  for (int64_t v0 = 0; v0 < vocab; v0 += piece) {
    const int64_t rows = std::min(piece, vocab - v0);
    if (packs) {
      uint16_t* dst = reinterpret_cast<uint16_t*>(ws + space.pack);
      const int rc = vl_pack(weight, w_dtype, ldw, v0, rows, dim, planes, dst, piece * st.Dp, s);
      if (rc != FMOE_OK) return rc;
      g.b = dst, g.b_plane = piece * st.Dp, g.ldb = static_cast<int>(st.Dp);
    } else {
      g.b = static_cast<const uint16_t*>(weight) + v0 * ldw, g.ldb = static_cast<int>(ldw);
    }
    g.cols = static_cast<int>(rows), g.v0 = static_cast<int>(v0);
    vl_gemm_kernel<VL_STATS><<<vl_grid(ceil_div(st.Tp, 256) * ceil_div(rows, 256)), core::NT, 0, s>>>(g);
  }

  LossArgs l{};
  l.head = st.head, l.perm = st.perm, l.index = st.index, l.part = g.part, l.Tp = st.Tp;
  l.pieces = static_cast<int>(2 * ceil_div(vocab, 256));
  l.stat = st.stat, l.picked = st.picked;
  l.row_loss = reinterpret_cast<float*>(ws + space.row_loss);
  l.loss = r.loss;
  l.q = st.q, l.entropy = st.entropy, l.h = st.h, l.h_plane = st.plane, l.weight = weight, l.ldw = ldw;
  l.top = distill ? static_cast<int>(top) : 0;
  l.D = r.D, l.Dp = r.Dp, l.w_dtype = w_dtype, l.planes = planes, l.c = g.c;
  l.factor = static_cast<float>(temperature * temperature);
  if (T > 0) {
    if (T >= 8192) vl_stat_kernel<64><<<dim3(static_cast<uint32_t>(ceil_div(T, 64))), 1024, 0, s>>>(l);
    else if (T >= 1024) vl_stat_kernel<16><<<dim3(static_cast<uint32_t>(ceil_div(T, 16))), 1024, 0, s>>>(l);
    else vl_stat_kernel<4><<<dim3(static_cast<uint32_t>(ceil_div(T, 4))), 1024, 0, s>>>(l);
    if (distill) {
      const dim3 grid(static_cast<uint32_t>(T));
      const size_t lds = st.Dp * 4;
      if (w_dtype == FMOE_BF16) vl_list_kernel<FMOE_BF16><<<grid, 256, lds, s>>>(l);
      else vl_list_kernel<FMOE_F32><<<grid, 256, lds, s>>>(l);
    }
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
      reduction < 0 || reduction > 2 || (planes != 1 && planes != 3) || !(temperature > 0.0) ||
      (!distill && temperature != 1.0))
    return FMOE_ERR_INVALID_ARG;
  if (!vl_sizes_ok(T, dim, vocab, top, planes)) return FMOE_ERR_SHAPE;
  if (vocab > 1 && (ldw < dim || ldw >= (int64_t(1) << 22))) return FMOE_ERR_SHAPE;
  if (!vl_dtype(w_dtype) || !vl_dtype(dh_dtype) || !vl_dtype(dw_dtype)) return FMOE_ERR_DTYPE;
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
  uint16_t* const pack = reinterpret_cast<uint16_t*>(ws + space.pack);
  float* const sum = reinterpret_cast<float*>(ws + space.sum);
  const int64_t piece = space.plan.piece, g_plane = st.Tp * piece;
  const int64_t pack_plane = std::min(pad64(vocab), piece) * st.Dp;
  const int passes = planes == 3 ? 6 : 1, Dp = static_cast<int>(st.Dp);
  const float factor = static_cast<float>(temperature * logit_scale);  // temperature^2 times d t / d logit
  const int64_t mt = ceil_div(st.Tp, 256), dt = ceil_div(st.Dp, 256);
  for (int64_t v0 = 0; v0 < vocab; v0 += piece) {
    const int64_t rows = std::min(piece, vocab - v0);
    VlGemm g{};
    g.passes = passes, g.head = st.head, g.Tp = st.Tp, g.planes = planes;
    const uint16_t* w = static_cast<const uint16_t*>(weight) + v0 * ldw;
    int64_t w_plane = 0;
    int w_ld = static_cast<int>(ldw);
    if (packs) {
      const int rc = vl_pack(weight, w_dtype, ldw, v0, rows, dim, planes, pack, pack_plane, s);
      if (rc != FMOE_OK) return rc;
      w = pack, w_plane = pack_plane, w_ld = Dp;
    }
    g.a = st.h, g.a_plane = st.plane, g.lda = Dp, g.k = Dp;
    g.b = w, g.b_plane = w_plane, g.ldb = w_ld, g.cols = static_cast<int>(rows), g.v0 = static_cast<int>(v0);
    g.c = static_cast<float>(logit_scale / temperature * static_cast<double>(kLog2e));
    g.stat = st.stat, g.d_loss = d_loss, g.perm = st.perm, g.factor = factor, g.reduction = reduction;
    g.g = gbuf, g.g_plane = g_plane, g.ldg = static_cast<int>(piece);
    vl_gemm_kernel<VL_GRAD><<<vl_grid(mt * ceil_div(rows, 256)), core::NT, 0, s>>>(g);
    FixArgs f{};
    f.head = st.head, f.perm = st.perm, f.index = st.index, f.q = st.q, f.picked = st.picked, f.stat = st.stat;
    f.d_loss = d_loss, f.top = static_cast<int>(top), f.distill = distill;
    f.v0 = static_cast<int>(v0), f.v1 = static_cast<int>(v0 + rows), f.reduction = reduction, f.planes = planes;
    f.ldg = g.ldg, f.factor = factor, f.g = gbuf, f.g_plane = g_plane;
    if (T > 0) vl_fix_kernel<<<dim3(static_cast<uint32_t>(ceil_div(T * top, 256))), 256, 0, s>>>(f);
    if (d_hidden != nullptr) {
      VlGemm h = g;
      h.a = gbuf, h.a_plane = g_plane, h.lda = g.ldg;
      h.cols = Dp, h.vocab = static_cast<int>(rows), h.sum = sum, h.add = v0 > 0;
      h.ranges = static_cast<int>(std::min<int64_t>(space.plan.ranges, ceil_div(rows, 64)));
      // (a short last piece may have fewer ranges: the others keep their sums)
      vl_gemm_kernel<VL_DH><<<vl_grid(mt * dt * h.ranges), core::NT, 0, s>>>(h);
    }
    if (d_weight != nullptr) {
      VlGemm d = g;
      d.a = gbuf, d.a_plane = g_plane, d.lda = g.ldg;
      d.b = st.h, d.b_plane = st.plane, d.ldb = Dp;
      d.cols = Dp, d.vocab = static_cast<int>(rows), d.D = static_cast<int>(dim), d.dw_dtype = dw_dtype;
      d.dw = static_cast<uint8_t*>(d_weight) + v0 * dim * (dw_dtype == FMOE_BF16 ? 2 : 4);
      vl_gemm_kernel<VL_DW><<<vl_grid(ceil_div(rows, 256) * dt), core::NT, 0, s>>>(d);
    }
  }
  if (d_hidden != nullptr && T > 0) {
    const dim3 grid(static_cast<uint32_t>(ceil_div(T, 4)));
    const int64_t stride = st.Tp * st.Dp;
    const int d = static_cast<int>(dim);
    if (dh_dtype == FMOE_BF16)
      vl_dh_kernel<FMOE_BF16><<<grid, 256, 0, s>>>(st.inv, sum, stride, space.plan.ranges, T, d, Dp, d_hidden);
    else
      vl_dh_kernel<FMOE_F32><<<grid, 256, 0, s>>>(st.inv, sum, stride, space.plan.ranges, T, d, Dp, d_hidden);
  }
  return launch_status();
}
