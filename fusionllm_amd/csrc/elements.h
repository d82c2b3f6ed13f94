// elements.h — chunks of 8 (or 1) consecutive bf16 or fp32 elements at any
// element's address: the hardware takes 16-byte accesses there, so rows and
// tensors that start anywhere need no path of their own.
#pragma once

#include "fmoe_common.h"

namespace fmoe {

typedef uint32_t u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));

template <int DT, int V>
struct Raw {  // a chunk as it lies in memory
  uint32_t u[DT == FMOE_BF16 ? (V == 8 ? 4 : 1) : V];
};

template <int DT, int V>
__device__ __forceinline__ Raw<DT, V> load_raw(const void* base, int64_t e) {
  Raw<DT, V> r;
  if constexpr (DT == FMOE_BF16) {
    const uint16_t* p = static_cast<const uint16_t*>(base) + e;
    if constexpr (V == 8) {
      const u32x4_e2 v = *reinterpret_cast<const u32x4_e2*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.u[i] = v[i];
    } else {
      r.u[0] = *p;
    }
  } else {
    const float* p = static_cast<const float*>(base) + e;
    if constexpr (V == 8) {
      const f32x4_e4 a = reinterpret_cast<const f32x4_e4*>(p)[0], b = *reinterpret_cast<const f32x4_e4*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.u[i] = __float_as_uint(a[i]), r.u[4 + i] = __float_as_uint(b[i]);
    } else {
      r.u[0] = __float_as_uint(*p);
    }
  }
  return r;
}

template <int DT, int V>
__device__ __forceinline__ void unpack(const Raw<DT, V>& r, float* v) {
  if constexpr (DT == FMOE_F32) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r.u[i]);
  } else if constexpr (V == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r.u[i] << 16);
      v[2 * i + 1] = __uint_as_float(r.u[i] & 0xffff0000u);
    }
  } else {
    v[0] = bf2f(static_cast<uint16_t>(r.u[0]));
  }
}

template <int DT, int V>
__device__ __forceinline__ void store_chunk(void* base, int64_t e, const float* v) {
  if constexpr (DT == FMOE_BF16) {
    uint16_t* p = static_cast<uint16_t*>(base) + e;
    if constexpr (V == 8) {
      u32x4_e2 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = pack2(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<u32x4_e2*>(p) = o;
    } else {
      *p = f2bf(v[0]);
    }
  } else {
    float* p = static_cast<float*>(base) + e;
    if constexpr (V == 8) {
      *reinterpret_cast<f32x4_e4*>(p) = f32x4_e4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_e4*>(p + 4) = f32x4_e4{v[4], v[5], v[6], v[7]};
    } else {
      *p = v[0];
    }
  }
}

// The same for n (up to 8) elements at the end of a row; what is past them reads as zero and is not written.
template <int DT>
__device__ __forceinline__ void load_upto8(const void* base, int64_t e, int n, float* v) {
  if (n >= 8) {
    unpack<DT, 8>(load_raw<DT, 8>(base, e), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = 0.0f;
      if (i < n) unpack<DT, 1>(load_raw<DT, 1>(base, e + i), v + i);
    }
  }
}
template <int DT>
__device__ __forceinline__ void store_upto8(void* base, int64_t e, int n, const float* v) {
  if (n >= 8) {
    store_chunk<DT, 8>(base, e, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store_chunk<DT, 1>(base, e + i, v + i);
  }
}

}  // namespace fmoe
