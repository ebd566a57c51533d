// What the choice of experts and the balance loss share. A warp has a token. In the balance loss, and where the choice is made
// exactly as it is defined, lane l has the experts l, l + 32, ...; in the quick way of the choice, a run of neighbours.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common.cuh"
#include "route_api.h"

namespace b200ep {
namespace route {

// (coherent loads, here and of all other inputs: the kernel before, in stream order, may still write what this one reads when
// its CTAs are placed, so the data is not read-only for their lifetime, as the non-coherent path requires)
__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float logit(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// (not a number stays what it is: a logit that is none shows in every score of its row)
__device__ __forceinline__ float nan_max(float a, float b) { return a > b || a != a ? a : b; }
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = nan_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

constexpr float kSumEps = 1e-20f;      // added to sums of scores that others are divided by

}  // namespace route
}  // namespace b200ep
