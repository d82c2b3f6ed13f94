// embedding.hip — token embedding y[t] = scale * W[ids[t]] and its gradient
// dW[v] = scale * sum of dy[t] over the tokens t of v.
//
// Both are bound by memory: the forward reads and writes T rows; the backward reads
// T rows and writes the V rows of the gradient, most of them zeros.  A wave takes 1 KB of a row at a time,
// 16 bytes per lane.  32768 tokens x 2048 in fp32, vocab 131072: forward 89 us (6.0 TB/s), backward 281 (the sums and zeros 244:
// 5.5 TB/s, of a copy's 4.9); 16384 x 768 in bf16, vocab 50021: 10 and 41.
//
// The gradient is summed without atomics, so that the same bits come out every run:
//   1. embed_sort_kernel sorts the tokens by id, stably, in one launch: a workgroup owns up to 512 ids and
//      walks all the tokens itself (T indices from L2), so that no workgroup waits for another.  It owns every
//      G-th id (G workgroups, a power of two): the frequent ids, which a tokenizer numbers first, fall to
//      different workgroups.  So "sorted" is by slot, (id mod G) * 512 + id / G.
//   2. embed_sum_kernel adds the rows of the sorted tokens, kTile at a time per wave: an id whose tokens
//      lie in one tile is written there; one that crosses tiles leaves an fp32 partial row per tile.  Workgroups
//      behind those write zeros for the ids without tokens.
//   3. embed_join_kernel writes the ids that cross tiles, from their partial rows in order.
// Up to 64 tokens, embed_few_kernel does all of it without a sort.
#include "../../include/fusionvocab.h"
#include "elements.h"
#include "fmoe_common.h"

namespace fmoe {

constexpr int kTile = 16;          // sorted tokens per wave of embed_sum_kernel
constexpr int kSortIds = 512;      // ids per workgroup of the sort, at most
constexpr int kSortWaves = 16;
constexpr int kZeroIds = 8;        // slots per wave that looks for ids without tokens
constexpr int kJoinWaves = 16;     // waves, and tiles, per workgroup of embed_join_kernel
constexpr int kLongTiles = 8;      // tiles above which a workgroup adds an id's partial rows together

// Consecutive elements per lane: 16 bytes.
template <int DT>
constexpr int kPer = DT == FMOE_BF16 ? 8 : 4;
constexpr int segments_of(int64_t D, int dtype) { return static_cast<int>((D + (dtype == FMOE_BF16 ? 511 : 255)) / (dtype == FMOE_BF16 ? 512 : 256)); }

// V elements at any element's address, n of them inside the row.
template <int DT, int V>
__device__ __forceinline__ void load_v(const void* base, int64_t e, int n, float* v) {
  if (n >= V && DT == FMOE_BF16 && V == 8) {
    unpack<FMOE_BF16, 8>(load_raw<FMOE_BF16, 8>(base, e), v);
  } else if (n >= V && DT == FMOE_F32 && V % 4 == 0) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const f32x4 x = reinterpret_cast<const f32x4_e4*>(static_cast<const float*>(base) + e)[q];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * q + i] = x[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[i] = 0.0f;
      if (i < n) unpack<DT, 1>(load_raw<DT, 1>(base, e + i), v + i);
    }
  }
}
template <int DT, int V>
__device__ __forceinline__ void store_v(void* base, int64_t e, int n, const float* v) {
  if (n >= V && DT == FMOE_BF16 && V == 8) {
    store_chunk<FMOE_BF16, 8>(base, e, v);
  } else if (n >= V && DT == FMOE_F32 && V % 4 == 0) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q)
      reinterpret_cast<f32x4_e4*>(static_cast<float*>(base) + e)[q] = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) store_chunk<DT, 1>(base, e + i, v + i);
  }
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
  // backward
  int shift;         // G = 1 << shift
  int slots;         // G * kSortIds
  int* start;        // first sorted position of each slot [slots + 1]
  int2* sorted;      // token and slot by position
  float* part;       // [tiles][2][D]: of the id that comes from the tile before, of the one that goes on
};

// ROWS rows per wave: their loads are in flight together.
template <int DT, int ROWS>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const EmbedArgs a) {
  constexpr int V = kPer<DT>;
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t group = item / a.segments;
  const int c = (static_cast<int>(item - group * a.segments) * 64 + lane) * V;
  const int n = min(a.D - c, V);
  const int64_t t0 = group * ROWS;
  if (t0 >= a.T) return;
  float v[ROWS][V];
  bool bad[ROWS];
  int64_t id[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t at = min(t0 + r, a.T - 1);
    id[r] = a.index64 ? static_cast<const int64_t*>(a.ids)[at] : static_cast<const int32_t*>(a.ids)[at];
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    bad[r] = id[r] < 0 || id[r] >= a.V;
    load_v<DT, V>(a.src, (bad[r] ? 0 : id[r]) * a.ld + c, bad[r] ? 0 : n, v[r]);
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (t0 + r >= a.T) break;
#pragma unroll
    for (int e = 0; e < V; ++e) v[r][e] = bad[r] ? __builtin_nanf("") : v[r][e] * a.scale;
    store_v<DT, V>(a.dst, (t0 + r) * a.D + c, n, v[r]);
  }
}

// Sorted positions of the tokens of this workgroup's ids, after the tokens of those of lower workgroups.  Wave w walks
// its sixteenth of the tokens twice: counts per id first, then places, where a token's rank among the
// 64 tokens of the same id comes from ballots.  The loads of 16 tokens
// per lane are in flight together (no branch around them).
template <bool I64>
__global__ __launch_bounds__(64 * kSortWaves) void embed_sort_kernel(const EmbedArgs a) {
  __shared__ int hist[kSortWaves][kSortIds];
  __shared__ int below[kSortWaves], waves[kSortIds / 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int mine = blockIdx.x, lo = mine * kSortIds;
  const int per = static_cast<int>(((a.T + 63) / 64 + kSortWaves - 1) / kSortWaves * 64);
  const int T = static_cast<int>(a.T), t0 = min(w * per, T), t1 = min(t0 + per, T);
  constexpr int U = 16;
  // slots of the tokens t + 64 u + lane relative to lo, -1 where a token adds nothing here; less: tokens of
  // lower workgroups
  auto load_slots = [&](int t, int (&k)[U], int& less) __attribute__((always_inline)) {
    uint32_t id[U], high[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(t + 64 * u + lane, T - 1);
      if constexpr (I64) {
        const uint2 raw = static_cast<const uint2*>(a.ids)[at];
        id[u] = raw.x, high[u] = raw.y;
      } else {
        id[u] = static_cast<const uint32_t*>(a.ids)[at], high[u] = 0;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool out = high[u] != 0 || id[u] >= static_cast<uint32_t>(a.V) || id[u] == static_cast<uint32_t>(a.pad) ||
                       t + 64 * u + lane >= t1;
      const int owner = out ? INT32_MAX : static_cast<int>(id[u]) & ((1 << a.shift) - 1);
      less += owner < mine;
      k[u] = owner == mine ? static_cast<int>(id[u]) >> a.shift : -1;
    }
  };
  int k[U], less = 0, ignored = 0;
  if (t0 < t1) load_slots(t0, k, less);
  for (int i = tid; i < kSortWaves * kSortIds / 4; i += 64 * kSortWaves)
    reinterpret_cast<int4*>(&hist[0][0])[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  for (int t = t0; t < t1; t += 64 * U) {
    if (t > t0) load_slots(t, k, less);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k[u] >= 0) atomicAdd(&hist[w][k[u]], 1);  // counts: any order
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
    a.start[lo + tid] = at;
    if (lo + tid + 1 == a.slots) a.start[a.slots] = at + total;
#pragma unroll
    for (int q = 0; q < kSortWaves; ++q) {
      const int n = hist[q][tid];
      hist[q][tid] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int t = t0; t < t1; t += 64 * U) {
    if (per > 64 * U) load_slots(t, k, ignored);  // (else they are there still)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t left = __ballot(k[u] >= 0), same = left;
      if (left == 0) continue;
      if (__popcll(left) <= 8) {  // few of this workgroup's tokens: one comparison per id among them
        while (left != 0) {
          const int first = __builtin_amdgcn_readlane(k[u], __builtin_ctzll(left));
          const uint64_t equal = __ballot(k[u] == first);
          if (k[u] == first) same = equal;
          left &= ~equal;
        }
      } else {  // one per bit of the id
#pragma unroll
        for (int b = 0; b < 9; ++b) {
          const bool bit = (k[u] >> b) & 1;
          const uint64_t on = __ballot(bit);
          same &= bit ? on : ~on;
        }
      }
      if (k[u] >= 0) {
        const int rank = __popcll(same & ((uint64_t(1) << lane) - 1));
        const int base = hist[w][k[u]];
        a.sorted[base + rank] = make_int2(t + 64 * u + lane, lo + k[u]);
        // (the wave's reads of base are before this: LDS operations of a wave run in order)
        if (rank == 0) hist[w][k[u]] = base + __popcll(same);
      }
    }
  }
}

// Row of the weight that a slot stands for.
__device__ __forceinline__ int64_t slot_id(const EmbedArgs& a, int slot) {
  return (static_cast<int64_t>(slot % kSortIds) << a.shift) + slot / kSortIds;
}

// 16 bytes of a row as they lie in memory.
template <int DT>
struct Row16 {
  typedef u32x4_e2 type;
};
template <>
struct Row16<FMOE_F32> {
  typedef f32x4_e4 type;
};

// Zeros in the rows of 8 slots without tokens, per wave.
template <int DW>
__device__ __forceinline__ void embed_zero(const EmbedArgs& a, int64_t item) {
  constexpr int V = kPer<DW>;
  const int segments = (a.D + 64 * V - 1) / (64 * V);
  const int lane = threadIdx.x & 63, group = static_cast<int>(item / segments);
  const int c = (static_cast<int>(item - static_cast<int64_t>(group) * segments) * 64 + lane) * V, n = min(a.D - c, V);
  const int s0 = group * kZeroIds;
  if (s0 >= a.slots) return;
  const int starts = a.start[min(s0 + min(lane, kZeroIds), a.slots)];
  float zero[V];
#pragma unroll
  for (int e = 0; e < V; ++e) zero[e] = 0.0f;
#pragma unroll
  for (int i = 0; i < kZeroIds; ++i) {
    const int64_t id = slot_id(a, s0 + i);
    if (id < a.V && __builtin_amdgcn_readlane(starts, i) == __builtin_amdgcn_readlane(starts, i + 1))
      store_v<DW, V>(a.dst, id * a.D + c, n, zero);
  }
}

// A tile's rows are all in flight together.  Workgroups from `blocks` on: zeros.
template <int DY, int DW>
__global__ __launch_bounds__(256) void embed_sum_kernel(const EmbedArgs a, int blocks) {
  constexpr int V = kPer<DY>;
  if (static_cast<int>(blockIdx.x) >= blocks) {
    embed_zero<DW>(a, static_cast<int64_t>(blockIdx.x - blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6));
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = item / a.segments;
  const int c = (static_cast<int>(item - tile * a.segments) * 64 + lane) * V;
  const int n = min(a.D - c, V);
  const int total = a.start[a.slots];
  const int64_t p0 = tile * kTile;
  if (p0 >= total) return;
  const int count = static_cast<int>(min(static_cast<int64_t>(total) - p0, int64_t(kTile)));
  // lane i: the i-th sorted token and its slot, then the slot after the tile; lane 63: the one before
  const int64_t at = lane == 63 ? p0 - 1 : p0 + lane;
  int2 ts = make_int2(0, -1);
  if (at >= 0 && at < total && (lane <= kTile || lane == 63)) ts = a.sorted[at];
  const int token = ts.x, slot = ts.y;
  const int before = __builtin_amdgcn_readlane(slot, 63);
  const bool whole = n >= V;  // of this lane's columns
  typedef typename Row16<DY>::type Raw16;
  Raw16 raw[kTile];
#pragma unroll
  for (int i = 0; i < kTile; ++i) {
    const int64_t t = __builtin_amdgcn_readlane(token, min(i, count - 1));
    if (whole)
      raw[i] = *reinterpret_cast<const Raw16*>(static_cast<const uint8_t*>(a.src) + (t * a.ld + c) * (16 / V));
  }
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.0f;
  bool from_before = __builtin_amdgcn_readlane(slot, 0) == before;
  auto flush = [&](int cur, bool goes_on) {
    if (from_before || goes_on) {
      store_v<FMOE_F32, V>(a.part, (2 * tile + (from_before ? 0 : 1)) * a.D + c, n, acc);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = acc[e] * a.scale;
      store_v<DW, V>(a.dst, slot_id(a, cur) * a.D + c, n, acc);
    }
    from_before = false;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
  };
#pragma unroll
  for (int i = 0; i < kTile; ++i) {
    if (i < count) {
      float v[V];
      if (!whole) {
        load_v<DY, V>(a.src, static_cast<int64_t>(__builtin_amdgcn_readlane(token, i)) * a.ld + c, n, v);
      } else if constexpr (DY == FMOE_F32) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = raw[i][e];
      } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          v[2 * e] = __uint_as_float(raw[i][e] << 16);
          v[2 * e + 1] = __uint_as_float(raw[i][e] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = acc[e] + v[e];
      // (past the last token the slot is -1)
      const int cur = __builtin_amdgcn_readlane(slot, i), next = __builtin_amdgcn_readlane(slot, i + 1);
      if (i + 1 >= count || next != cur) flush(cur, next == cur);
    }
  }
}

// Partial rows first .. last of an id's later tiles, stepping by step, added to acc.
template <int V>
__device__ __forceinline__ void add_partials(const EmbedArgs& a, int64_t first, int64_t last, int64_t step, int c, int n,
                                             float* acc) {
  constexpr int U = 8;
  for (int64_t q = first; q <= last; q += U * step) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      load_v<FMOE_F32, V>(a.part, 2 * min(q + u * step, last) * a.D + c, n, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = q + u * step <= last ? acc[e] + v[u][e] : acc[e];
  }
}

// Wave w: the id that goes on from its tile into the next one, if it begins in that tile; one of many tiles is the
// whole workgroup's.
template <int DW>
__global__ __launch_bounds__(64 * kJoinWaves) void embed_join_kernel(const EmbedArgs a) {
  constexpr int V = kPer<DW>;
  __shared__ float sums[kJoinWaves][64 * V];
  __shared__ int found[kJoinWaves];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = blockIdx.x / a.segments;
  const int c = ((static_cast<int>(blockIdx.x) - group * a.segments) * 64 + lane) * V, n = min(a.D - c, V);
  const int64_t tile = static_cast<int64_t>(group) * kJoinWaves + w, next = (tile + 1) * kTile;
  int slot = -1;
  if (next < a.start[a.slots]) {
    const int s = a.sorted[next].y;
    const int64_t ta = a.start[s] / kTile, tb = (a.start[s + 1] - 1) / kTile;
    if (ta == tile && tb - ta > kLongTiles) {
      slot = s;
    } else if (ta == tile && tb > ta) {
      float acc[V];
      load_v<FMOE_F32, V>(a.part, (2 * ta + 1) * a.D + c, n, acc);
      add_partials<V>(a, ta + 1, tb, 1, c, n, acc);
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] = acc[q] * a.scale;
      store_v<DW, V>(a.dst, slot_id(a, s) * a.D + c, n, acc);
    }
  }
  if (lane == 0) found[w] = slot;
  __syncthreads();
  for (int f = 0; f < kJoinWaves; ++f) {
    const int s = found[f];
    if (s < 0) continue;
    const int64_t ta = a.start[s] / kTile, tb = (a.start[s + 1] - 1) / kTile;
    // wave w every 16th partial row, then the waves in order
    float acc[V];
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = 0.0f;
    if (w == 0) load_v<FMOE_F32, V>(a.part, (2 * ta + 1) * a.D + c, n, acc);
    add_partials<V>(a, ta + 1 + w, tb, kJoinWaves, c, n, acc);
#pragma unroll
    for (int q = 0; q < V; ++q) sums[w][q * 64 + lane] = acc[q];
    __syncthreads();
    if (w == 0) {
      for (int p = 1; p < kJoinWaves; ++p)
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] = acc[q] + sums[p][q * 64 + lane];
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] = acc[q] * a.scale;
      store_v<DW, V>(a.dst, slot_id(a, s) * a.D + c, n, acc);
    }
    __syncthreads();
  }
}

// Up to 64 tokens, one launch and no sort: a lane holds a token's id, and a wave asks for each of its rows which lanes
// have it.  Eight rows and a segment per wave, as embed_zero (64 tokens, 32768 x 768: 11 us, sorted 20; all of one id 12
// and 21; 3 tokens, 46435 x 128 in fp32: 7 and 15).
constexpr int kFewTokens = 64;
template <int DY, int DW>
__global__ __launch_bounds__(256) void embed_few_kernel(const EmbedArgs a) {
  constexpr int V = kPer<DY>;
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = static_cast<int>(item / a.segments);
  const int c = (static_cast<int>(item - static_cast<int64_t>(group) * a.segments) * 64 + lane) * V, n = min(a.D - c, V);
  int64_t id = -1;
  if (lane < a.T)
    id = a.index64 ? static_cast<const int64_t*>(a.ids)[lane] : static_cast<const int32_t*>(a.ids)[lane];
  if (id == a.pad) id = -1;
  const bool whole = n >= V;  // of this lane's columns
  typedef typename Row16<DY>::type Raw16;
  const uint8_t* const src = static_cast<const uint8_t*>(a.src) + static_cast<int64_t>(c) * (16 / V);
#pragma unroll
  for (int i = 0; i < kZeroIds; ++i) {
    const int64_t v = static_cast<int64_t>(group) * kZeroIds + i;
    if (v >= a.V) return;
    uint64_t who = __ballot(id == v);
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    const bool any = who != 0;
    while (who != 0) {
      constexpr int U = 16;
      int t[U];
      const int count = min(__popcll(who), U);
      uint64_t rest = who;
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (past the last token it is read again: no branch between the loads)
        t[u] = who != 0 ? __builtin_ctzll(who) : t[u > 0 ? u - 1 : 0];
        who &= who - 1;
      }
      Raw16 raw[U];
      if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = *reinterpret_cast<const Raw16*>(src + t[u] * a.ld * (16 / V));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u >= count) continue;
          if constexpr (DY == FMOE_F32) {
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = acc[e] + raw[u][e];
          } else {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
              acc[2 * e] = acc[2 * e] + __uint_as_float(raw[u][e] << 16);
              acc[2 * e + 1] = acc[2 * e + 1] + __uint_as_float(raw[u][e] & 0xffff0000u);
            }
          }
        }
      } else if (n > 0) {
        for (int u = 0; u < count; ++u, rest &= rest - 1) {
          float x[V];
          load_v<DY, V>(a.src, __builtin_ctzll(rest) * a.ld + c, n, x);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] = acc[e] + x[e];
        }
      }
    }
    if (any)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] = acc[e] * a.scale;
    store_v<DW, V>(a.dst, v * a.D + c, n, acc);
  }
}

inline bool elem_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FMOE_BF16 ? 1u : 3u)) == 0;
}

int embed_check(const void* ids, int index64, const void* src, int src_dtype, int64_t ld, int64_t src_rows, int64_t T,
                int64_t vocab, int64_t dim, const void* dst, int dst_dtype) {
  if (T < 0 || vocab <= 0 || dim <= 0 || index64 < 0 || index64 > 1) return FMOE_ERR_INVALID_ARG;
  if (dim > FMOE_VOCAB_MAX_DIM || T > FMOE_VOCAB_MAX_TOKENS || vocab > FMOE_VOCAB_MAX_VOCAB) return FMOE_ERR_SHAPE;
  // (the launches stay below 2^32 threads)
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
  int shift = 0;
  int64_t slots = 0;
  size_t start = 0, sorted = 0, part = 0, bytes = 0;
  EmbedSpace(int64_t T, int64_t V, int64_t D) {
    if (T <= kFewTokens) return;
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) & ~size_t(255);
      return at;
    };
    while ((int64_t(kSortIds) << shift) < V) ++shift;
    slots = int64_t(kSortIds) << shift;
    start = take((slots + 1) * 4);
    sorted = take(T * 8);
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
  a.segments = segments_of(dim, dtype);
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
  if (workspace_bytes < space.bytes || (workspace == nullptr && space.bytes > 0)) return FMOE_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return FMOE_ERR_ALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  EmbedArgs a{};
  a.ids = ids, a.index64 = index64, a.src = dy, a.ld = lddy, a.dst = d_weight, a.T = T;
  a.V = static_cast<int>(vocab), a.D = static_cast<int>(dim), a.scale = scale, a.pad = static_cast<int>(padding_idx);
  a.shift = space.shift, a.slots = static_cast<int>(space.slots);
  a.start = reinterpret_cast<int*>(ws + space.start);
  a.sorted = reinterpret_cast<int2*>(ws + space.sorted);
  a.part = reinterpret_cast<float*>(ws + space.part);
  const hipStream_t s = as_stream(stream);
  if (T <= kFewTokens) {
    a.segments = segments_of(dim, dy_dtype);
    const dim3 grid(static_cast<uint32_t>(ceil_div(ceil_div(vocab, kZeroIds) * a.segments, 4)));
    if (dy_dtype == FMOE_BF16 && dtype == FMOE_BF16) embed_few_kernel<FMOE_BF16, FMOE_BF16><<<grid, 256, 0, s>>>(a);
    else if (dy_dtype == FMOE_BF16) embed_few_kernel<FMOE_BF16, FMOE_F32><<<grid, 256, 0, s>>>(a);
    else if (dtype == FMOE_BF16) embed_few_kernel<FMOE_F32, FMOE_BF16><<<grid, 256, 0, s>>>(a);
    else embed_few_kernel<FMOE_F32, FMOE_F32><<<grid, 256, 0, s>>>(a);
    return launch_status();
  }
  const dim3 sort(1u << space.shift);
  if (index64) embed_sort_kernel<true><<<sort, 64 * kSortWaves, 0, s>>>(a);
  else embed_sort_kernel<false><<<sort, 64 * kSortWaves, 0, s>>>(a);
  const int64_t tiles = ceil_div(T, kTile);
  a.segments = segments_of(dim, dy_dtype);
  const int64_t blocks = ceil_div(tiles * a.segments, 4);
  const int64_t zeros = ceil_div(ceil_div(space.slots, kZeroIds) * segments_of(dim, dtype), 4);
  const dim3 grid(static_cast<uint32_t>(blocks + zeros));
  const int b = static_cast<int>(blocks);
  if (dy_dtype == FMOE_BF16 && dtype == FMOE_BF16) embed_sum_kernel<FMOE_BF16, FMOE_BF16><<<grid, 256, 0, s>>>(a, b);
  else if (dy_dtype == FMOE_BF16) embed_sum_kernel<FMOE_BF16, FMOE_F32><<<grid, 256, 0, s>>>(a, b);
  else if (dtype == FMOE_BF16) embed_sum_kernel<FMOE_F32, FMOE_BF16><<<grid, 256, 0, s>>>(a, b);
  else embed_sum_kernel<FMOE_F32, FMOE_F32><<<grid, 256, 0, s>>>(a, b);
  a.segments = segments_of(dim, dtype);
  const dim3 join(static_cast<uint32_t>(ceil_div(tiles, kJoinWaves) * a.segments));
  if (dtype == FMOE_BF16) embed_join_kernel<FMOE_BF16><<<join, 64 * kJoinWaves, 0, s>>>(a);
  else embed_join_kernel<FMOE_F32><<<join, 64 * kJoinWaves, 0, s>>>(a);
  return launch_status();
}
