// embedding.hip — token embedding y[t] = scale * W[ids[t]] and its gradient
// dW[v] = scale * sum of dy[t] over the tokens t of v.
//
// Both are bound by memory: the forward reads and writes T rows; the backward reads
// T rows and writes the V rows of the gradient, most of them zeros.  A row is read in
// pieces of 512 columns, 8 consecutive elements per lane, one wave per piece.
//
// The gradient is summed without atomics, so that the same bits come out every run:
//   1. embed_sort_kernel sorts the tokens by id, stably, in one launch: a workgroup owns 512 ids and
//      walks all the tokens itself (T indices from L2), so that no workgroup waits for another.
//   2. embed_sum_kernel adds the rows of the sorted tokens, kTile at a time per wave: an id whose tokens
//      lie in one tile is written there; one that crosses tiles leaves an fp32 partial row per tile.
//   3. embed_rest_kernel writes the ids that cross tiles, from their partial rows in order, and zeros
//      for the ids without tokens.
#include "../../include/fusionvocab.h"
#include "elements.h"
#include "fmoe_common.h"

namespace fmoe {

constexpr int kSegment = 512;      // columns per wave: 64 lanes of 8
constexpr int kTile = 32;          // sorted tokens per wave of embed_sum_kernel
constexpr int kSortIds = 512;      // ids per workgroup of the sort
constexpr int kSortWaves = 16;
constexpr int kRestIds = 8;        // ids per wave of embed_rest_kernel
constexpr int kRestWaves = 16;
constexpr int kLongTiles = 32;     // tiles above which a workgroup adds an id's partial rows together

__device__ __forceinline__ int64_t load_index(const void* p, bool index64, int64_t i) {
  return index64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

struct EmbedArgs {
  const void* ids;
  const void* src;   // weight, or dy
  void* dst;         // y, or d_weight
  int64_t ld;        // of src
  int64_t T;
  int V, D, segments;
  int index64;
  int pad;           // -1: none
  float scale;
  int *start, *order, *key;  // backward: first sorted position of each id [V + 1], tokens and ids by position
  float* part;               // [tiles][2][D]: of the id that comes from the tile before, of the one that goes on
};

// ROWS rows per wave: their loads are in flight together.
template <int DT, int ROWS>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const EmbedArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t group = item / a.segments;
  const int c = static_cast<int>(item - group * a.segments) * kSegment + lane * 8;
  const int n = min(a.D - c, 8);
  const int64_t t0 = group * ROWS;
  if (t0 >= a.T) return;
  float v[ROWS][8];
  bool bad[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t id = load_index(a.ids, a.index64, min(t0 + r, a.T - 1));
    bad[r] = id < 0 || id >= a.V;
    load_upto8<DT>(a.src, (bad[r] ? 0 : id) * a.ld + c, bad[r] ? 0 : n, v[r]);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (t0 + r >= a.T) break;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[r][e] = bad[r] ? __builtin_nanf("") : v[r][e] * a.scale;
    store_upto8<DT>(a.dst, (t0 + r) * a.D + c, n, v[r]);
  }
}

// Sorted positions of the tokens of ids lo .. lo + 511, after the tokens of smaller ids.  Wave w walks
// its sixteenth of the tokens twice: counts per id first, then places, where a token's rank among its
// wave's earlier tokens of the same id comes from ballots over the bits of the id.
__global__ __launch_bounds__(64 * kSortWaves) void embed_sort_kernel(const EmbedArgs a) {
  __shared__ int hist[kSortWaves][kSortIds];
  __shared__ int below[kSortWaves], waves[kSortIds / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int lo = blockIdx.x * kSortIds;
  for (int i = tid; i < kSortWaves * kSortIds; i += 64 * kSortWaves) (&hist[0][0])[i] = 0;
  __syncthreads();
  const int64_t per = ((a.T + 63) / 64 + kSortWaves - 1) / kSortWaves * 64;
  const int64_t t0 = min(w * per, a.T), t1 = min(t0 + per, a.T);
  // an id as int: -1 where the token adds nothing
  auto token_id = [&](int64_t t) {
    if (t >= t1) return -1;
    const int64_t id = load_index(a.ids, a.index64, t);
    return id < 0 || id >= a.V || id == a.pad ? -1 : static_cast<int>(id);
  };
  constexpr int U = 8;
  int less = 0;
  for (int64_t t = t0; t < t1; t += 64 * U) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = token_id(t + 64 * u + lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      less += id[u] >= 0 && id[u] < lo;
      const int k = id[u] - lo;
      if (id[u] >= lo && k < kSortIds) atomicAdd(&hist[w][k], 1);  // counts: any order
    }
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) less += __shfl_xor(less, off, 64);
  if (lane == 0) below[w] = less;
  __syncthreads();
  int total = 0, incl = 0;
  if (tid < kSortIds) {
#pragma unroll
    for (int q = 0; q < kSortWaves; ++q) total += hist[q][tid];
    incl = wave_incl_scan(total, lane);
    if (lane == 63) waves[w] = incl;
  }
  __syncthreads();
  if (tid < kSortIds) {
    int at = incl - total;
#pragma unroll
    for (int q = 0; q < kSortWaves; ++q) at += below[q];
    for (int q = 0; q < w; ++q) at += waves[q];
    if (lo + tid <= a.V) a.start[lo + tid] = at;  // (of id V: where the last id ends)
    if (tid == kSortIds - 1 && lo + kSortIds == a.V) a.start[a.V] = at + total;
#pragma unroll
    for (int q = 0; q < kSortWaves; ++q) {
      const int n = hist[q][tid];
      hist[q][tid] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int64_t t = t0; t < t1; t += 64 * U) {
    int id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) id[u] = token_id(t + 64 * u + lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = id[u] - lo;
      const bool mine = id[u] >= lo && k < kSortIds;
      uint64_t same = __ballot(mine);
      if (same == 0) continue;
#pragma unroll
      for (int b = 0; b < 9; ++b) {
        const bool bit = (k >> b) & 1;
        const uint64_t on = __ballot(bit);
        same &= bit ? on : ~on;
      }
      if (mine) {
        const int rank = __popcll(same & ((uint64_t(1) << lane) - 1));
        const int base = hist[w][k];
        const int at = base + rank;
        a.order[at] = static_cast<int>(t + 64 * u + lane);
        a.key[at] = id[u];
        // (the wave's reads of base are before this: LDS operations of a wave run in order)
        if (rank == 0) hist[w][k] = base + __popcll(same);
      }
    }
  }
}

template <int DY, int DW>
__global__ __launch_bounds__(256) void embed_sum_kernel(const EmbedArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = item / a.segments;
  const int c = static_cast<int>(item - tile * a.segments) * kSegment + lane * 8;
  const int n = min(a.D - c, 8);
  const int total = a.start[a.V];
  const int64_t p0 = tile * kTile;
  if (p0 >= total) return;
  const int count = static_cast<int>(min(static_cast<int64_t>(total) - p0, int64_t(kTile)));
  // lane i: the i-th sorted token and its id; the ids before and after the tile
  const int64_t at = p0 + min(lane, count - 1);
  const int token = a.order[at], id = a.key[at];
  const int before = p0 > 0 ? a.key[p0 - 1] : -1;
  const int after = p0 + count < total ? a.key[p0 + count] : -1;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
  bool from_before = __builtin_amdgcn_readlane(id, 0) == before;
  constexpr int U = 8;
  for (int i0 = 0; i0 < count; i0 += U) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = __builtin_amdgcn_readlane(token, min(i0 + u, count - 1));
      load_upto8<DY>(a.src, t * a.ld + c, n, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= count) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = acc[e] + v[u][e];
      const int cur = __builtin_amdgcn_readlane(id, i);
      const int next = i + 1 < count ? __builtin_amdgcn_readlane(id, min(i + 1, 63)) : after;
      if (i + 1 < count && next == cur) continue;
      const bool goes_on = next == cur;
      if (from_before || goes_on) {
        store_upto8<FMOE_F32>(a.part, (2 * tile + (from_before ? 0 : 1)) * a.D + c, n, acc);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = acc[e] * a.scale;
        store_upto8<DW>(a.dst, static_cast<int64_t>(cur) * a.D + c, n, acc);
      }
      from_before = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
    }
  }
}

// Partial rows first .. last of an id's later tiles, stepping by step, added to acc.
__device__ __forceinline__ void add_partials(const EmbedArgs& a, int64_t first, int64_t last, int64_t step, int c, int n,
                                             float* acc) {
  constexpr int U = 8;
  for (int64_t q = first; q <= last; q += U * step) {
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
      load_upto8<FMOE_F32>(a.part, 2 * min(q + u * step, last) * a.D + c, n, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = q + u * step <= last ? acc[e] + v[u][e] : acc[e];
  }
}

template <int DW>
__global__ __launch_bounds__(64 * kRestWaves) void embed_rest_kernel(const EmbedArgs a) {
  __shared__ float sums[kRestWaves][kSegment];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t group = blockIdx.x / a.segments;
  const int c = static_cast<int>(blockIdx.x - group * a.segments) * kSegment + lane * 8;
  const int n = min(a.D - c, 8);
  const int block0 = static_cast<int>(group) * (kRestIds * kRestWaves);
  const int v0 = block0 + w * kRestIds;
  const int starts = a.start[min(v0 + min(lane, kRestIds), a.V)];
  float zero[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) zero[e] = 0.0f;
  uint64_t longs = 0;
#pragma unroll
  for (int i = 0; i < kRestIds; ++i) {
    if (v0 + i >= a.V) break;
    const int s = __builtin_amdgcn_readlane(starts, i), e = __builtin_amdgcn_readlane(starts, i + 1);
    const int64_t o = static_cast<int64_t>(v0 + i) * a.D + c;
    if (s == e) {
      store_upto8<DW>(a.dst, o, n, zero);
      continue;
    }
    const int64_t ta = s / kTile, tb = (e - 1) / kTile;
    if (ta == tb) continue;  // written with its tile
    if (tb - ta > kLongTiles) {
      longs |= uint64_t(1) << i;
      continue;
    }
    // first piece: the second partial of its tile, or the first one where the id begins with the tile
    // and fills it (then nothing comes from the tile before, and it is the one that goes on)
    float acc[8];
    load_upto8<FMOE_F32>(a.part, (2 * ta + 1) * a.D + c, n, acc);
    add_partials(a, ta + 1, tb, 1, c, n, acc);
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = acc[q] * a.scale;
    store_upto8<DW>(a.dst, o, n, acc);
  }
  // ids of many tiles: the whole workgroup, wave w every 16th partial row, then the waves in order
  __shared__ uint64_t long_ids[kRestWaves];
  if (lane == 0) long_ids[w] = longs;
  __syncthreads();
  for (int q = 0; q < kRestWaves; ++q)
    for (uint64_t left = long_ids[q]; left != 0; left &= left - 1) {
      const int v = block0 + q * kRestIds + __builtin_ctzll(left);
      const int64_t ta = a.start[v] / kTile, tb = (a.start[v + 1] - 1) / kTile;
      float acc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
      if (w == 0) load_upto8<FMOE_F32>(a.part, (2 * ta + 1) * a.D + c, n, acc);
      add_partials(a, ta + 1 + w, tb, kRestWaves, c, n, acc);
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[w][lane * 8 + e] = acc[e];
      __syncthreads();
      if (w == 0) {
        for (int p = 1; p < kRestWaves; ++p)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] = acc[e] + sums[p][lane * 8 + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = acc[e] * a.scale;
        store_upto8<DW>(a.dst, static_cast<int64_t>(v) * a.D + c, n, acc);
      }
      __syncthreads();
    }
}

inline bool elem_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FMOE_BF16 ? 1u : 3u)) == 0;
}

int embed_check(const void* ids, int index64, const void* src, int src_dtype, int64_t ld, int64_t src_rows, int64_t T,
                int64_t vocab, int64_t dim, const void* dst, int dst_dtype) {
  if (T < 0 || vocab <= 0 || dim <= 0 || index64 < 0 || index64 > 1) return FMOE_ERR_INVALID_ARG;
  if (dim > FMOE_VOCAB_MAX_DIM || T > FMOE_VOCAB_MAX_TOKENS || vocab > FMOE_VOCAB_MAX_VOCAB) return FMOE_ERR_SHAPE;
  // (more elements than the card's memory holds: the launches stay below 2^32 threads)
  if (T * dim > FMOE_VOCAB_MAX_ELEMENTS || vocab * dim > FMOE_VOCAB_MAX_ELEMENTS) return FMOE_ERR_SHAPE;
  if (src_rows > 1 && (ld < dim || ld > (int64_t(1) << 38))) return FMOE_ERR_SHAPE;
  for (const int d : {src_dtype, dst_dtype})
    if (d != FMOE_BF16 && d != FMOE_F32) return FMOE_ERR_DTYPE;
  if (dst == nullptr && T > 0) return FMOE_ERR_INVALID_ARG;
  if (T > 0 && (ids == nullptr || src == nullptr)) return FMOE_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(ids) & (index64 ? 7u : 3u)) != 0 || !elem_aligned(src, src_dtype) ||
      !elem_aligned(dst, dst_dtype))
    return FMOE_ERR_ALIGN;
  return FMOE_OK;
}

struct EmbedSpace {
  size_t start, order, key, part, bytes;
  EmbedSpace(int64_t T, int64_t V, int64_t D) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    bytes = 0;
    start = take((V + 1) * 4);
    order = take(T * 4);
    key = take(T * 4);
    part = take(static_cast<size_t>(ceil_div(T, kTile)) * 2 * D * 4);
  }
};

}  // namespace fmoe

using namespace fmoe;

extern "C" int fmoe_embedding_fwd(const void* ids, int index64, const void* weight, int dtype, int64_t ldw, int64_t T,
                                  int64_t vocab, int64_t dim, float scale, void* y, void* stream) {
  const int rc = embed_check(ids, index64, weight, dtype, ldw, vocab, T, vocab, dim, y, dtype);
  if (rc != FMOE_OK) return rc;
  if (T == 0) return FMOE_OK;
  EmbedArgs a{};
  a.ids = ids, a.index64 = index64, a.src = weight, a.ld = ldw, a.dst = y, a.T = T;
  a.V = static_cast<int>(vocab), a.D = static_cast<int>(dim), a.scale = scale;
  a.segments = static_cast<int>(ceil_div(dim, kSegment));
  // four rows per wave (their loads overlap) where that still fills every CU with 16 waves
  constexpr int R = 4;
  const bool many = T * a.segments >= R * 256 * 16;
  const int64_t items = ceil_div(T, many ? R : 1) * a.segments;
  const dim3 grid(static_cast<uint32_t>(ceil_div(items, 4)));
  const hipStream_t s = as_stream(stream);
  if (dtype == FMOE_BF16) {
    if (many) embed_fwd_kernel<FMOE_BF16, R><<<grid, 256, 0, s>>>(a);
    else embed_fwd_kernel<FMOE_BF16, 1><<<grid, 256, 0, s>>>(a);
  } else {
    if (many) embed_fwd_kernel<FMOE_F32, R><<<grid, 256, 0, s>>>(a);
    else embed_fwd_kernel<FMOE_F32, 1><<<grid, 256, 0, s>>>(a);
  }
  return launch_status();
}

extern "C" size_t fmoe_embedding_bwd_workspace_bytes(int64_t T, int64_t vocab, int64_t dim) {
  if (T < 0 || vocab <= 0 || dim <= 0 || T > FMOE_VOCAB_MAX_TOKENS || vocab > FMOE_VOCAB_MAX_VOCAB ||
      dim > FMOE_VOCAB_MAX_DIM || T * dim > FMOE_VOCAB_MAX_ELEMENTS || vocab * dim > FMOE_VOCAB_MAX_ELEMENTS)
    return 0;
  return EmbedSpace(T, vocab, dim).bytes;
}

extern "C" int fmoe_embedding_bwd(const void* ids, int index64, const void* dy, int dy_dtype, int64_t lddy, int64_t T,
                                  int64_t vocab, int64_t dim, float scale, int64_t padding_idx, void* d_weight,
                                  int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = embed_check(ids, index64, dy, dy_dtype, lddy, T, T, vocab, dim, d_weight, dtype);
  if (rc != FMOE_OK) return rc;
  if (d_weight == nullptr || padding_idx < -1 || padding_idx >= vocab) return FMOE_ERR_INVALID_ARG;
  const EmbedSpace space(T, vocab, dim);
  if (workspace == nullptr || workspace_bytes < space.bytes) return FMOE_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return FMOE_ERR_ALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  EmbedArgs a{};
  a.ids = ids, a.index64 = index64, a.src = dy, a.ld = lddy, a.dst = d_weight, a.T = T;
  a.V = static_cast<int>(vocab), a.D = static_cast<int>(dim), a.scale = scale, a.pad = static_cast<int>(padding_idx);
  a.segments = static_cast<int>(ceil_div(dim, kSegment));
  a.start = reinterpret_cast<int*>(ws + space.start);
  a.order = reinterpret_cast<int*>(ws + space.order);
  a.key = reinterpret_cast<int*>(ws + space.key);
  a.part = reinterpret_cast<float*>(ws + space.part);
  const hipStream_t s = as_stream(stream);
  embed_sort_kernel<<<dim3(static_cast<uint32_t>(ceil_div(vocab, kSortIds))), 64 * kSortWaves, 0, s>>>(a);
  if (T > 0) {
    const dim3 grid(static_cast<uint32_t>(ceil_div(ceil_div(T, kTile) * a.segments, 4)));
    if (dy_dtype == FMOE_BF16 && dtype == FMOE_BF16) embed_sum_kernel<FMOE_BF16, FMOE_BF16><<<grid, 256, 0, s>>>(a);
    else if (dy_dtype == FMOE_BF16) embed_sum_kernel<FMOE_BF16, FMOE_F32><<<grid, 256, 0, s>>>(a);
    else if (dtype == FMOE_BF16) embed_sum_kernel<FMOE_F32, FMOE_BF16><<<grid, 256, 0, s>>>(a);
    else embed_sum_kernel<FMOE_F32, FMOE_F32><<<grid, 256, 0, s>>>(a);
  }
  const dim3 rest(static_cast<uint32_t>(ceil_div(vocab, kRestIds * kRestWaves) * a.segments));
  if (dtype == FMOE_BF16) embed_rest_kernel<FMOE_BF16><<<rest, 64 * kRestWaves, 0, s>>>(a);
  else embed_rest_kernel<FMOE_F32><<<rest, 64 * kRestWaves, 0, s>>>(a);
  return launch_status();
}
