// layer_norm.hip — layer norm of the rows of a matrix and its backward pass,
// with the reduction of the weight's and bias's gradients.
//
//   mean = sum x / D,  r = 1 / sqrt(sum (x - mean)^2 / D + eps),
//   xh = (x - mean) r,  y = xh w + b
//   g = dy w,  dx = r (g - sum(g) / D - xh sum(g xh) / D) [+ d_residual]
//   dw = sum_t dy xh,  db = sum_t dy
//
// Memory bound: the forward reads x once and writes y once; the backward reads
// x and dy once and writes dx once.  A row lives in the registers of 1 to 16
// waves, so that the mean, the centred sum of squares (second pass over
// registers: no cancellation of two large sums) and the result come from one
// read.  The backward's workgroups walk the rows with the columns' sums of dy xh
// and dy in registers, write one partial row each, and a second kernel adds
// the partial rows in a fixed order (no atomics: same bits every run).
//
// A row is split into chunks of 8 elements (16-byte loads of bf16); lane l of
// the row's wave w owns chunks l + 64 (w + W i).  Where dim is no multiple of
// 8, the last chunk is the window of the row's last 8 elements: its first
// elements belong to the chunk before too, are left out of the row's sums and
// otherwise come out the same in both lanes.  The hardware takes 16-byte
// accesses at any element's address, so rows may start anywhere and odd dims
// need no path of their own.  Rows of fewer than 8 elements take chunks of one.
#include <algorithm>

#include "../../include/fusiontrain.h"
#include "elements.h"
#include "fmoe_common.h"

namespace fmoe {

constexpr int kLnMaxWaves = 16;   // waves per row
// Chunks per lane, at most: 2; up to 4 in the forward of fp32 rows that one wave then holds (no barrier
// between the waves of a row: 32768 x 2048 113 -> 102 us, 16384 x 1500 45 -> 41; longer rows over half the waves
// 8192 x 4096 57 -> 60, 4000 x 10240 75 -> 85; bf16 16384 x 2048 34 -> 36).
constexpr int kLnMaxChunks = 2, kLnMaxChunksOneWave = 4;
constexpr int kLnRowsPerGroup = 4;  // rows a workgroup works on at once where a wave holds a row
// Waves of the backward's launch: 8 for each of the 256 CUs, whose partial rows cost half as much as
// 16 (32768 x 2048 fp32 159 against 171 us with their reduction, 4099 x 1023 bf16 15 against 19); 16 for
// bf16 rows where each still gets 16 of them (65536 x 768: 62 against 66 us).
constexpr int kLnWaves = 256 * 8, kLnManyRows = 16;

static_assert(kLnMaxWaves * 64 * 8 * kLnMaxChunks == FMOE_LAYER_NORM_MAX_DIM);

// A chunk of the weight or bias (dtype known at run time), or `none` everywhere.
template <int V>
__device__ __forceinline__ void load_vector(const void* p, int dtype, int64_t e, float none, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = none;
  } else if (dtype == FMOE_BF16) {
    unpack<FMOE_BF16, V>(load_raw<FMOE_BF16, V>(p, e), v);
  } else {
    unpack<FMOE_F32, V>(load_raw<FMOE_F32, V>(p, e), v);
  }
}

// Sums of N values over the waves of a row: an xor butterfly over the lanes,
// then the waves' sums in wave order.  Called by every wave of the workgroup.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int waves, int wave, float (*red)[N]) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = v[n] + __shfl_xor(v[n], off, 64);
  if (waves == 1) return;
  __syncthreads();  // the last call's sums have been read
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) red[wave][n] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float s = red[0][n];
    for (int w = 1; w < waves; ++w) s = s + red[w][n];
    v[n] = s;
  }
}

// Chunk i of this lane: its first element, whether the lane has it, and how
// many of its leading elements belong to the chunk before.
template <int V>
struct Chunk {
  int start, skip;
  bool on;
  __device__ __forceinline__ Chunk(int c, int dim) {
    const int e = c * V;
    on = e < dim;
    start = min(e, dim - V);
    skip = e - start;
  }
};

template <int XT, int YT, int V, int NCH>
__global__ __launch_bounds__(kLnMaxWaves * 64) void layer_norm_fwd_kernel(
    const void* __restrict__ x, int64_t ldx, const void* __restrict__ wt, const void* __restrict__ bs, int w_dtype,
    int64_t T, int dim, int waves, float eps, void* __restrict__ y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out) {
  __shared__ float red[kLnMaxWaves][1];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // waves == 1: every wave has a row; otherwise the workgroup has one
  const int wave = waves == 1 ? 0 : wid;
  const int64_t t = waves == 1 ? static_cast<int64_t>(blockIdx.x) * kLnRowsPerGroup + wid : blockIdx.x;
  if (t >= T) return;  // only whole waves of a one-wave-per-row group (no barrier there)
  Raw<XT, V> raw[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
    raw[i] = load_raw<XT, V>(x, t * ldx + (c.on ? c.start : 0));
  }
  float wv[NCH][V], bv[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
    load_vector<V>(wt, w_dtype, c.on ? c.start : 0, 1.0f, wv[i]);
    load_vector<V>(bs, w_dtype, c.on ? c.start : 0, 0.0f, bv[i]);
  }
  float v[NCH][V];
  float s[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
    unpack<XT, V>(raw[i], v[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) s[0] = s[0] + (c.on && e >= c.skip ? v[i][e] : 0.0f);
  }
  row_sums<1>(s, waves, wave, red);
  const float mean = s[0] / static_cast<float>(dim);
  float q[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[i][e] = v[i][e] - mean;
      q[0] = c.on && e >= c.skip ? fmaf(v[i][e], v[i][e], q[0]) : q[0];
    }
  }
  row_sums<1>(q, waves, wave, red);
  const float r = 1.0f / sqrtf(q[0] / static_cast<float>(dim) + eps);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
    float o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = fmaf(v[i][e] * r, wv[i][e], bv[i][e]);
    if (c.on) store_chunk<YT, V>(y, t * dim + c.start, o);
  }
  if (lane == 0 && wave == 0) {
    if (mean_out) mean_out[t] = mean;
    if (rstd_out) rstd_out[t] = r;
  }
}

template <int XT, int DT, int V, int NCH>
__global__ __launch_bounds__(kLnMaxWaves * 64) void layer_norm_bwd_kernel(
    const void* __restrict__ dy, int64_t lddy, const void* __restrict__ x, int64_t ldx, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, const void* __restrict__ wt, int w_dtype, const void* __restrict__ d_res,
    int64_t T, int dim, int waves, void* __restrict__ dx, float* __restrict__ parts) {
  __shared__ float red[kLnMaxWaves][2];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = waves == 1 ? 0 : wid;
  const int rows = waves == 1 ? kLnRowsPerGroup : 1;
  float pw[NCH][V], pb[NCH][V], wv[NCH][V];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
    load_vector<V>(wt, w_dtype, c.on ? c.start : 0, 1.0f, wv[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) pw[i][e] = pb[i][e] = 0.0f;
  }
  const float inv = 1.0f / static_cast<float>(dim);
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows;
  // every wave of a workgroup that shares a row makes the same trips
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * rows + (waves == 1 ? wid : 0); t < T; t += step) {
    Raw<XT, V> rx[NCH];
    Raw<DT, V> rd[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
      rx[i] = load_raw<XT, V>(x, t * ldx + (c.on ? c.start : 0));
      rd[i] = load_raw<DT, V>(dy, t * lddy + (c.on ? c.start : 0));
    }
    const float mean = mean_in[t], r = rstd_in[t];
    float g[NCH][V], xh[NCH][V];
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
      float d[V];
      unpack<XT, V>(rx[i], xh[i]);
      unpack<DT, V>(rd[i], d);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        xh[i][e] = (xh[i][e] - mean) * r;
        g[i][e] = d[e] * wv[i][e];
        pw[i][e] = fmaf(d[e], xh[i][e], pw[i][e]);
        pb[i][e] = pb[i][e] + d[e];
        if (c.on && e >= c.skip) {
          s[0] = s[0] + g[i][e];
          s[1] = fmaf(g[i][e], xh[i][e], s[1]);
        }
      }
    }
    if (!dx) continue;
    row_sums<2>(s, waves, wave, red);
    const float m0 = s[0] * inv, m1 = s[1] * inv;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
      if (!c.on) continue;
      float o[V];
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] = r * ((g[i][e] - m0) - xh[i][e] * m1);
      if (d_res) {
        float dr[V];
        unpack<XT, V>(load_raw<XT, V>(d_res, t * dim + c.start), dr);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = o[e] + dr[e];
      }
      store_chunk<XT, V>(dx, t * dim + c.start, o);
    }
  }
  if (!parts) return;
  // The workgroup's partial rows: of dy xh, then of dy.  Where its waves have
  // rows of their own, they add into LDS one after the other.
  float* out = parts + static_cast<int64_t>(blockIdx.x) * 2 * dim;
  if (waves > 1) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const Chunk<V> c(lane + 64 * (wave + waves * i), dim);
      if (!c.on) continue;
      store_chunk<FMOE_F32, V>(out, c.start, pw[i]);
      store_chunk<FMOE_F32, V>(out, dim + c.start, pb[i]);
    }
    return;
  }
  __shared__ float acc[kLnRowsPerGroup][64][V + 1];
#pragma unroll
  for (int i = 0; i < 2 * NCH; ++i) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) acc[wid][lane][e] = i < NCH ? pw[i % NCH][e] : pb[i % NCH][e];
    __syncthreads();
    if (wid == 0) {
      const Chunk<V> c(lane + 64 * (i % NCH), dim);
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = acc[0][lane][e];
#pragma unroll
        for (int w = 1; w < kLnRowsPerGroup; ++w) v[e] = v[e] + acc[w][lane][e];
      }
      if (c.on) store_chunk<FMOE_F32, V>(out, (i < NCH ? 0 : dim) + c.start, v);
    }
  }
}

// d_weight[c], d_bias[c] = sum over the partial rows, one column per lane: a
// workgroup of 16 waves takes 64 columns; wave w adds rows w, w + 16, ... in
// order, then the waves' sums are added in wave order.
constexpr int kLnReduceWaves = 16;
__global__ __launch_bounds__(kLnReduceWaves * 64) void layer_norm_reduce_kernel(const float* __restrict__ parts, int n,
                                                                                int dim, void* __restrict__ dw,
                                                                                void* __restrict__ db, int dtype) {
  __shared__ float q[kLnReduceWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + lane;
  const bool on = col < dim;
  void* const out = blockIdx.y == 0 ? dw : db;
  if (!out) return;  // the whole workgroup
  const float* p = parts + static_cast<int64_t>(blockIdx.y) * dim + col;
  float s = 0.0f;
  constexpr int B = 8;  // loads in flight
  for (int i0 = wave; i0 < n; i0 += B * kLnReduceWaves) {
    float v[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int row = i0 + i * kLnReduceWaves;
      v[i] = on && row < n ? p[static_cast<int64_t>(row) * 2 * dim] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < B; ++i) s = s + v[i];
  }
  q[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || !on) return;
  s = q[0][lane];
#pragma unroll
  for (int w = 1; w < kLnReduceWaves; ++w) s = s + q[w][lane];
  if (dtype == FMOE_BF16) static_cast<uint16_t*>(out)[col] = f2bf(s);
  else static_cast<float*>(out)[col] = s;
}

// How a row is spread: the fewest waves that hold it with at most kLnMaxChunks
// chunks per lane (one_wave: one wave where kLnMaxChunksOneWave suffice), and the chunks that takes.
struct LnShape {
  int vec, waves, nch;
};
inline LnShape ln_shape(int64_t dim, bool one_wave = false) {
  if (dim < 8) return {1, 1, 1};
  const int64_t chunks = ceil_div(dim, 8);
  if (one_wave && chunks <= 64 * kLnMaxChunksOneWave) return {8, 1, static_cast<int>(ceil_div(chunks, 64))};
  const int waves = static_cast<int>(ceil_div(chunks, 64 * kLnMaxChunks));
  return {8, waves, static_cast<int>(ceil_div(chunks, 64 * waves))};
}
inline int ln_rows(const LnShape& s) { return s.waves == 1 ? kLnRowsPerGroup : 1; }
inline int ln_threads(const LnShape& s) { return 64 * (s.waves == 1 ? kLnRowsPerGroup : s.waves); }
inline int64_t ln_bwd_groups(int64_t T, const LnShape& s, int x_dtype) {
  const int64_t many = x_dtype == FMOE_BF16 && T * s.waves >= int64_t(kLnManyRows) * 2 * kLnWaves ? 2 : 1;
  return std::min<int64_t>(ceil_div(T, ln_rows(s)), many * kLnWaves * 64 / ln_threads(s));
}

inline bool ln_dtype(int d) { return d == FMOE_BF16 || d == FMOE_F32; }
constexpr int ln_bytes(int d) { return d == FMOE_BF16 ? 2 : 4; }
inline bool ln_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FMOE_BF16 ? 1u : 3u)) == 0;
}
// Rows of up to T start within the tensor and its offsets within 63 bits.
inline bool ln_stride(int64_t T, int64_t dim, int64_t ld) {
  return T <= 1 || (ld >= dim && ld <= (INT64_MAX / 8) / T);
}

}  // namespace fmoe

using namespace fmoe;

// The kernel's instance for a shape: F(vec, chunks per lane).
#define FMOE_LN_SHAPES(s, F)          \
  do {                                \
    if ((s).vec == 1) F(1, 1);        \
    else if ((s).nch == 1) F(8, 1);   \
    else F(8, 2);                     \
  } while (0)
#define FMOE_LN_SHAPES_F32(s, F)      \
  do {                                \
    if ((s).nch == 3) F(8, 3);        \
    else if ((s).nch == 4) F(8, 4);   \
    else FMOE_LN_SHAPES(s, F);        \
  } while (0)

extern "C" int fmoe_layer_norm_fwd(const void* x, int x_dtype, int64_t ldx, const void* weight, const void* bias,
                                   int w_dtype, int64_t T, int64_t dim, float eps, void* y, int y_dtype, float* mean,
                                   float* rstd, void* stream) {
  if (T < 0 || dim <= 0) return FMOE_ERR_INVALID_ARG;
  if (dim > FMOE_LAYER_NORM_MAX_DIM || T > INT32_MAX || !ln_stride(T, dim, ldx)) return FMOE_ERR_SHAPE;
  if (!ln_dtype(x_dtype) || !ln_dtype(y_dtype) || !ln_dtype(w_dtype)) return FMOE_ERR_DTYPE;
  if (T == 0) return FMOE_OK;
  if (!x || !y) return FMOE_ERR_INVALID_ARG;
  if (!ln_aligned(x, x_dtype) || !ln_aligned(y, y_dtype) || !ln_aligned(weight, w_dtype) ||
      !ln_aligned(bias, w_dtype) || !ln_aligned(mean, FMOE_F32) || !ln_aligned(rstd, FMOE_F32))
    return FMOE_ERR_ALIGN;
  const LnShape s = ln_shape(dim, x_dtype == FMOE_F32);
  const dim3 block(ln_threads(s));
  hipStream_t st = as_stream(stream);
  // a launch has fewer than 2^32 threads: 2^31 at once
  const int64_t most = (int64_t(1) << 31) / ln_threads(s) * ln_rows(s);
#define FMOE_LN_FWD(XT, YT, V, N)                                                                                  \
  do for (int64_t t0 = 0; t0 < T; t0 += most) {                                                                       \
    const int64_t rows = std::min(T - t0, most);                                                                   \
    layer_norm_fwd_kernel<XT, YT, V, N><<<dim3(ceil_div(rows, ln_rows(s))), block, 0, st>>>(                       \
        static_cast<const char*>(x) + t0 * ldx * ln_bytes(XT), ldx, weight, bias, w_dtype, rows, (int)dim, s.waves, eps, \
        static_cast<char*>(y) + t0 * dim * ln_bytes(YT), mean ? mean + t0 : nullptr, rstd ? rstd + t0 : nullptr);  \
  } while (0)
#define FMOE_LN_FWD_BB(V, N) FMOE_LN_FWD(FMOE_BF16, FMOE_BF16, V, N)
#define FMOE_LN_FWD_BF(V, N) FMOE_LN_FWD(FMOE_BF16, FMOE_F32, V, N)
#define FMOE_LN_FWD_FB(V, N) FMOE_LN_FWD(FMOE_F32, FMOE_BF16, V, N)
#define FMOE_LN_FWD_FF(V, N) FMOE_LN_FWD(FMOE_F32, FMOE_F32, V, N)
  if (x_dtype == FMOE_BF16 && y_dtype == FMOE_BF16) FMOE_LN_SHAPES(s, FMOE_LN_FWD_BB);
  else if (x_dtype == FMOE_BF16) FMOE_LN_SHAPES(s, FMOE_LN_FWD_BF);
  else if (y_dtype == FMOE_BF16) FMOE_LN_SHAPES_F32(s, FMOE_LN_FWD_FB);
  else FMOE_LN_SHAPES_F32(s, FMOE_LN_FWD_FF);
  return launch_status();
}

extern "C" size_t fmoe_layer_norm_bwd_workspace_bytes(int64_t T, int64_t dim) {
  if (T <= 0 || dim <= 0 || dim > FMOE_LAYER_NORM_MAX_DIM) return 0;
  return static_cast<size_t>(ln_bwd_groups(T, ln_shape(dim), FMOE_BF16)) * 2 * static_cast<size_t>(dim) * sizeof(float);
}

extern "C" int fmoe_layer_norm_bwd(const void* dy, int dy_dtype, int64_t lddy, const void* x, int x_dtype, int64_t ldx,
                                   const float* mean, const float* rstd, const void* weight, int w_dtype,
                                   const void* d_residual, int64_t T, int64_t dim, void* dx, void* d_weight,
                                   void* d_bias, void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || dim <= 0) return FMOE_ERR_INVALID_ARG;
  if (dim > FMOE_LAYER_NORM_MAX_DIM || T > INT32_MAX || !ln_stride(T, dim, ldx) || !ln_stride(T, dim, lddy))
    return FMOE_ERR_SHAPE;
  if (!ln_dtype(dy_dtype) || !ln_dtype(x_dtype) || !ln_dtype(w_dtype)) return FMOE_ERR_DTYPE;
  const bool vectors = d_weight || d_bias;
  if (!dx && !vectors) return FMOE_OK;
  if (vectors && workspace_bytes < fmoe_layer_norm_bwd_workspace_bytes(T, dim)) return FMOE_ERR_WORKSPACE;
  if (!ln_aligned(d_weight, w_dtype) || !ln_aligned(d_bias, w_dtype)) return FMOE_ERR_ALIGN;
  const LnShape s = ln_shape(dim);
  hipStream_t st = as_stream(stream);
  int groups = 0;
  if (T > 0) {
    if (!dy || !x || !mean || !rstd) return FMOE_ERR_INVALID_ARG;
    if (vectors && !workspace) return FMOE_ERR_WORKSPACE;
    if (!ln_aligned(dy, dy_dtype) || !ln_aligned(x, x_dtype) || !ln_aligned(mean, FMOE_F32) ||
        !ln_aligned(rstd, FMOE_F32) || !ln_aligned(weight, w_dtype) || !ln_aligned(d_residual, x_dtype) ||
        !ln_aligned(dx, x_dtype) || (vectors && !ln_aligned(workspace, FMOE_F32)))
      return FMOE_ERR_ALIGN;
    groups = static_cast<int>(ln_bwd_groups(T, s, x_dtype));
    const dim3 grid(groups), block(ln_threads(s));
    float* parts = vectors ? static_cast<float*>(workspace) : nullptr;
#define FMOE_LN_BWD(XT, DT, V, N)                                                                              \
  layer_norm_bwd_kernel<XT, DT, V, N><<<grid, block, 0, st>>>(dy, lddy, x, ldx, mean, rstd, weight, w_dtype,   \
                                                              d_residual, T, (int)dim, s.waves, dx, parts)
#define FMOE_LN_BWD_BB(V, N) FMOE_LN_BWD(FMOE_BF16, FMOE_BF16, V, N)
#define FMOE_LN_BWD_BF(V, N) FMOE_LN_BWD(FMOE_BF16, FMOE_F32, V, N)
#define FMOE_LN_BWD_FB(V, N) FMOE_LN_BWD(FMOE_F32, FMOE_BF16, V, N)
#define FMOE_LN_BWD_FF(V, N) FMOE_LN_BWD(FMOE_F32, FMOE_F32, V, N)
    if (x_dtype == FMOE_BF16 && dy_dtype == FMOE_BF16) FMOE_LN_SHAPES(s, FMOE_LN_BWD_BB);
    else if (x_dtype == FMOE_BF16) FMOE_LN_SHAPES(s, FMOE_LN_BWD_BF);
    else if (dy_dtype == FMOE_BF16) FMOE_LN_SHAPES(s, FMOE_LN_BWD_FB);
    else FMOE_LN_SHAPES(s, FMOE_LN_BWD_FF);
  }
  // No rows: the vectors' gradients are sums over nothing.
  if (vectors)
    layer_norm_reduce_kernel<<<dim3(ceil_div(dim, 64), 2), dim3(kLnReduceWaves * 64), 0, st>>>(
        static_cast<const float*>(workspace), groups, (int)dim, d_weight, d_bias, w_dtype);
  return launch_status();
}
