// What the forward and the backward kernel of the norm share: rows as 16-byte vectors, wherever in 16 bytes they begin.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common.cuh"
#include "norm_api.h"

namespace b200ep {
namespace norm {

template <typename T> constexpr int kEpv = 16 / (int)sizeof(T);      // elements of a vector

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// A vector's elements in f32, and back (rounded to nearest even).
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float* f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 4) {
      f[q] = __uint_as_float(u[q]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * q] = __uint_as_float(u[q] << 16);
      f[2 * q + 1] = __uint_as_float(u[q] & 0xffff0000u);
    } else {
      const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&u[q]));
      f[2 * q] = d.x;
      f[2 * q + 1] = d.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float* f) {
  uint32_t u[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (sizeof(T) == 4) {
      u[q] = __float_as_uint(f[q]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 d = __floats2bfloat162_rn(f[2 * q], f[2 * q + 1]);
      u[q] = *reinterpret_cast<const uint32_t*>(&d);
    } else {
      const __half2 d = __floats2half2_rn(f[2 * q], f[2 * q + 1]);
      u[q] = *reinterpret_cast<const uint32_t*>(&d);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// Vector v of a row holds the elements [e0, e0 + kEpv) with e0 = v * kEpv - shift, where shift is how many elements
// behind a 16-byte boundary the row begins: its inner vectors are aligned, the first and the last may be partial and are
// moved element by element. Nothing outside the row is touched.
template <typename T>
__device__ __forceinline__ bool whole(int e0, int H) { return e0 >= 0 && e0 + kEpv<T> <= H; }

template <typename T>
__device__ __forceinline__ uint4 load_vec(const T* row, int e0, int H) {
  if (whole<T>(e0, H)) return ld_global_nc_v4(row + e0);
  union { uint4 v; T e[kEpv<T>]; } u;
  u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < kEpv<T>; ++j)
    if (e0 + j >= 0 && e0 + j < H) u.e[j] = row[e0 + j];
  return u.v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* row, int e0, int H, const uint4& v) {
  if (whole<T>(e0, H)) { st_global_v4(row + e0, v); return; }
  union { uint4 v; T e[kEpv<T>]; } u;
  u.v = v;
#pragma unroll
  for (int j = 0; j < kEpv<T>; ++j)
    if (e0 + j >= 0 && e0 + j < H) row[e0 + j] = u.e[j];
}

// The weights of one vector of rows in T, kept as they are stored (W: T or float) so that they take few registers.
template <typename T, typename W>
struct WeightVec {
  static constexpr int N = kEpv<T> * (int)sizeof(W) / 16;
  uint4 r[N];
  __device__ __forceinline__ void load(const W* w, int e0, int H, bool aligned) {
    if (aligned && whole<T>(e0, H)) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = ld_global_nc_v4(w + e0 + i * kEpv<W>);
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      union { uint4 v; W e[kEpv<W>]; } u;
      u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < kEpv<W>; ++j) {
        const int e = e0 + i * kEpv<W> + j;
        if (e >= 0 && e < H) u.e[j] = w[e];
      }
      r[i] = u.v;
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < N; ++i) unpack<W>(r[i], f + i * kEpv<W>);
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, the same order in every thread. `slots` alternates between two rows of 32 words from one call to the
// next, so that one barrier a call is enough.
__device__ __forceinline__ float block_sum(float v, float* slots) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  const int warps = (int)blockDim.x >> 5, lane = threadIdx.x & 31;
  return warp_sum(lane < warps ? slots[lane] : 0.f);
}

// After how many rows the place of a row's first element within 16 bytes comes again.
inline int align_period(long long ld_bytes) {
  int p = 1;
  while ((ld_bytes * p) % 16) p *= 2;
  return p;
}

}  // namespace norm
}  // namespace b200ep
