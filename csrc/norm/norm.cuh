// What the forward and the backward kernel of the norm share: rows as 16-byte vectors, wherever in 16 bytes they begin.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <mutex>
#include <type_traits>
#include "../common.cuh"
#include "norm_api.h"

namespace b200ep {
namespace norm {

template <typename T> constexpr int kEpv = 16 / (int)sizeof(T);      // elements of a vector
// vectors that the longest row lies in
template <typename T, bool ALIGNED> constexpr int kMaxVecs = kNormMaxHidden / kEpv<T> + (ALIGNED ? 0 : 1);

template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{ .reg .b64 x, y, z, w; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 w, x, y, z; mov.b64 {%0, %1}, w; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A vector's elements in f32, and back (rounded to nearest even).
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float2 (&f)[kEpv<T> / 2]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(u[0]), __uint_as_float(u[1]));
    f[1] = make_float2(__uint_as_float(u[2]), __uint_as_float(u[3]));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) f[q] = make_float2(__uint_as_float(u[q] << 16), __uint_as_float(u[q] & 0xffff0000u));
      else f[q] = __half22float2(*reinterpret_cast<const __half2*>(&u[q]));
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float2 (&f)[kEpv<T> / 2]) {
  uint32_t u[4];
  if constexpr (sizeof(T) == 4) {
    u[0] = __float_as_uint(f[0].x); u[1] = __float_as_uint(f[0].y);
    u[2] = __float_as_uint(f[1].x); u[3] = __float_as_uint(f[1].y);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 d = __floats2bfloat162_rn(f[q].x, f[q].y);
        u[q] = *reinterpret_cast<const uint32_t*>(&d);
      } else {
        const __half2 d = __floats2half2_rn(f[q].x, f[q].y);
        u[q] = *reinterpret_cast<const uint32_t*>(&d);
      }
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// Vector v of a row holds the elements [e0, e0 + kEpv) with e0 = v * kEpv - shift, where shift is how many elements
// behind a 16-byte boundary the row begins. So all loads are of aligned vectors. The first of a row may begin with elements of
// the row before (or of what lies between them): they are set to zero. The last one is read up to the row's end. Both are
// stored element by element. ALIGNED: shift is 0 and H a multiple of kEpv, all vectors are whole.
template <typename T>
__device__ __forceinline__ bool whole(int e0, int H) { return e0 >= 0 && e0 + kEpv<T> <= H; }

template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 inside(uint4 v, int e0) {
  if constexpr (!ALIGNED) {
    if (e0 < 0) {
      uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < kEpv<T>; ++j) {
        if constexpr (sizeof(T) == 4) u[j] = e0 + j < 0 ? 0u : u[j];
        else u[j / 2] = e0 + j < 0 ? u[j / 2] & (j % 2 ? 0xffffu : 0xffff0000u) : u[j / 2];
      }
      v = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  return v;
}
template <typename T, bool ALIGNED>
__device__ __forceinline__ void store_vec(char* at, int e0, int H, const uint4& v) {
  if (ALIGNED ? e0 < H : whole<T>(e0, H)) {
    st_global_v4(at, v);
  } else if constexpr (!ALIGNED) {
    union { uint4 v; T e[kEpv<T>]; } u;
    u.v = v;
#pragma unroll
    for (int j = 0; j < kEpv<T>; ++j)
      if (e0 + j >= 0 && e0 + j < H) reinterpret_cast<T*>(at)[j] = u.e[j];
  }
}

// A row's vector straight from memory, zeros outside the row. (Coherent loads, as of all inputs: the kernel before, in
// stream order, may still write what this one reads when its CTAs are placed.)
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 load_vec(const T* row, int e0, int H) {
  if (ALIGNED || whole<T>(e0, H)) return ld_global_once_v4(row + e0);
  union { uint4 v; T e[kEpv<T>]; } u;
  u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < kEpv<T>; ++j)
    if (e0 + j >= 0 && e0 + j < H) u.e[j] = row[e0 + j];
  return u.v;
}

// Asynchronous copy of a vector to this thread's own place in shared memory. Where it is not whole, `bytes` of it are read
// and the rest of its place is filled with zeros.
template <bool ALIGNED>
__device__ __forceinline__ void fetch_vec(uint32_t to, const char* from, int bytes) {
  if constexpr (ALIGNED) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 lds_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
// One tensor's rows as a thread walks over them: the address of its first vector in the next row that it looks at.
template <typename T>
struct Walk {
  char* at;
  long long step;
  __device__ __forceinline__ Walk(const void* t, long long ld, long long row0, int step_rows, int e0) {
    at = const_cast<char*>(reinterpret_cast<const char*>(static_cast<const T*>(t) + row0 * ld + e0));
    step = (long long)step_rows * ld * (long long)sizeof(T);
  }
};
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest `left` groups have arrived.
__device__ __forceinline__ void fetch_wait(int left) {
  if (left <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (left == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (left == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 3;" ::: "memory");
}
constexpr int kMaxStages = 4;            // rows that a thread has under way, for fetch_wait
// Rows come by way of shared memory unless they are so long (more than 2048 vectors of 16-bit elements, 4096 of f32) that their
// tensors do not fit there: those are loads enough at a time by themselves.
template <typename T, int VPT, bool WARP> constexpr bool kStaged = WARP || VPT * kEpv<T> <= 16;

// The weights of one vector of rows in T, kept as they are stored (W: T or float) so that they take few registers.
template <typename T, typename W>
struct WeightVec {
  static constexpr int N = kEpv<T> * (int)sizeof(W) / 16;
  uint4 r[N];
  __device__ __forceinline__ void load(const W* w, int e0, int H, bool aligned) {
    if (aligned && whole<T>(e0, H)) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = ld_global_v4(w + e0 + i * kEpv<W>);
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
  __device__ __forceinline__ void get(float2 (&f)[kEpv<T> / 2]) const {
    if constexpr (N == 1) {
      unpack<W>(r[0], f);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f[2 * i] = make_float2(__uint_as_float(r[i].x), __uint_as_float(r[i].y));
        f[2 * i + 1] = make_float2(__uint_as_float(r[i].z), __uint_as_float(r[i].w));
      }
    }
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, the same order in every thread. `slots` alternates between two rows of 32 words from one call to the
// next, so that one barrier a call is enough. `width`: a power of two, the warps of the CTA or more.
__device__ __forceinline__ float block_sum(float v, float* slots, int width) {
  v = warp_sum(v);
  const int warps = (int)blockDim.x >> 5, at = threadIdx.x & (width - 1);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  v = at < warps ? slots[at] : 0.f;
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ int block_width() {
  int w = 1;
  while (w < ((int)blockDim.x >> 5)) w *= 2;
  return w;
}

// 1 / sqrt(v): the hardware's approximation and one step of Newton's iteration, off by about a unit in the last place.
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v);
  return v > 0.f && v < INFINITY ? fmaf(r * 0.5f, fmaf(-(v * r), r, 1.f), r) : r;
}
// 1 / v for 2^-126 <= v <= 2^126 likewise, without the branches of a division; 0 above (the approximation has no denormals).
__device__ __forceinline__ float inverse(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return v < INFINITY ? fmaf(r, fmaf(-v, r, 1.f), r) : r;
}

// After how many rows the place of a row's first element within 16 bytes comes again.
inline int align_period(long long ld_bytes) {
  int p = 1;
  while ((ld_bytes * p) % 16) p *= 2;
  return p;
}

// How a kernel is launched for a number of threads and bytes a row: rows under way (as many as fit beside what the
// registers allow of CTAs, at most kMaxStages) and CTAs per SM. Asked of the runtime once, kept for the last question.
class Launch {
 public:
  template <typename K>
  bool get(K kern, int threads, int row_bytes, int* stages, int* fit) {
    std::lock_guard<std::mutex> lock(m_);
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    if (dev != dev_ || threads != threads_ || row_bytes != row_bytes_) {
      int most = 0, sm = 0, ctas = 0;
      cudaFuncAttributes at{};
      if (cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev) != cudaSuccess ||
          cudaDeviceGetAttribute(&sm, cudaDevAttrMaxSharedMemoryPerMultiprocessor, dev) != cudaSuccess || cudaFuncGetAttributes(&at, kern) != cudaSuccess)
        return false;
      most -= (int)at.sharedSizeBytes;
      if (row_bytes > most || cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess ||
          cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kern, threads, row_bytes) != cudaSuccess || ctas < 1)
        return false;
      int n = kMaxStages;
      while (n > 1 && (n * row_bytes > most || (long long)ctas * (n * row_bytes + (int)at.sharedSizeBytes + 1024) > sm)) --n;
      dev_ = dev; threads_ = threads; row_bytes_ = row_bytes; stages_ = n; fit_ = ctas;
    }
    *stages = stages_;
    *fit = fit_;
    return true;
  }

 private:
  std::mutex m_;
  int dev_ = -1, threads_ = 0, row_bytes_ = 0, stages_ = 0, fit_ = 0;
};

}  // namespace norm
}  // namespace b200ep
