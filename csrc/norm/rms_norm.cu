// Root-mean-square norm with the residual's addition, rows in bf16, f16 or f32 out, or e4m3 with 1x128 scales.
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w,  scale = max(amax of 128 channels of y, 1e-4) / 448
// h, its square sum and y are held in f32 and rounded once, where they are stored: y is that of the sum before its
// rounding. Bound: memory (two tensors read and two written with a residual), for few rows latency. A row is read once
// and stays in registers; a warp has a row of up to 128 vectors of 16 bytes, a CTA a longer one; CTAs are persistent and
// keep their columns' weights in registers.
#include <cuda_fp8.h>
#include "../ep/cast.cuh"
#include "norm.cuh"

namespace b200ep {
namespace norm {

constexpr int kWarpRows = 8;             // rows of a CTA at a time where a warp has a row

template <typename T, typename W, int VPT, bool FP8, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : 1024, WARP ? 2 : 1)
rms_norm_fwd_kernel(const NormFwdParams p) {
  constexpr int EPV = kEpv<T>;
  __shared__ float s_sum[2][32];
  const int H = p.H;
  const int row0 = WARP ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int step = WARP ? gridDim.x * kWarpRows : gridDim.x;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x;
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  T* y = static_cast<T*>(p.y);
  T* ho = static_cast<T*>(p.h);
  // (the same for every row of this thread: the grid strides by a multiple of the alignment's period)
  const int shift = (int)((reinterpret_cast<uintptr_t>(x + (long long)row0 * p.x_ld) & 15) / sizeof(T));
  const bool w_aligned = shift == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15) == 0;
  WeightVec<T, W> w[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) w[i].load(static_cast<const W*>(p.w), (i * threads + tid) * EPV - shift, H, w_aligned);
  int parity = 0;
  for (long long row = row0; row < p.T; row += step, parity ^= 1) {
    uint4 xv[VPT], rv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) xv[i] = load_vec(x + row * p.x_ld, (i * threads + tid) * EPV - shift, H);
    if (res != nullptr) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) rv[i] = load_vec(res + row * p.res_ld, (i * threads + tid) * EPV - shift, H);
    }
    float h[VPT][EPV], ss = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      unpack<T>(xv[i], h[i]);
      if (res != nullptr) {
        float r[EPV];
        unpack<T>(rv[i], r);
#pragma unroll
        for (int j = 0; j < EPV; ++j) h[i][j] += r[j];
        store_vec(ho + row * H, (i * threads + tid) * EPV - shift, H, pack<T>(h[i]));
      }
#pragma unroll
      for (int j = 0; j < EPV; ++j) ss = fmaf(h[i][j], h[i][j], ss);
    }
    ss = WARP ? warp_sum(ss) : block_sum(ss, s_sum[parity]);
    const float rstd = 1.f / sqrtf(ss / (float)H + p.eps);
    if (tid == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = (i * threads + tid) * EPV - shift;
      float wf[EPV];
      w[i].get(wf);
#pragma unroll
      for (int j = 0; j < EPV; ++j) h[i][j] = h[i][j] * rstd * wf[j];
      if (y != nullptr) store_vec(y + row * H, e0, H, pack<T>(h[i]));
      if constexpr (FP8) {
        // (H is a multiple of 128 and shift 0: the 128 / EPV lanes of a block are neighbours and all in or all out)
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < EPV; ++j) amax = fmaxf(amax, fabsf(h[i][j]));
#pragma unroll
        for (int o = kNormScaleBlock / EPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        amax = fmaxf(amax, 1e-4f);
        const float inv = 448.f / amax;
        if (e0 < H) {
          uint32_t o[EPV / 4];
#pragma unroll
          for (int j = 0; j < EPV / 4; ++j)
            o[j] = cvt4_e4m3(h[i][4 * j] * inv, h[i][4 * j + 1] * inv, h[i][4 * j + 2] * inv, h[i][4 * j + 3] * inv);
          char* q = static_cast<char*>(p.q) + row * H + e0;
          if constexpr (EPV == 8) *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
          else *reinterpret_cast<uint32_t*>(q) = o[0];
          if (e0 % kNormScaleBlock == 0) p.scales[row * (H / kNormScaleBlock) + e0 / kNormScaleBlock] = amax * (1.f / 448.f);
        }
      }
    }
  }
}

template <typename T, typename W, int VPT, bool FP8, bool WARP>
int launch_fwd(const NormFwdParams& p, int threads, cudaStream_t st) {
  const auto kern = rms_norm_fwd_kernel<T, W, VPT, FP8, WARP>;
  int fit = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, threads, 0) != cudaSuccess || fit < 1) return 2;
  const int rows = WARP ? kWarpRows : 1;
  const long long need = ((long long)p.T + rows - 1) / rows;
  long long grid = (long long)fit * sm_count();
  const int period = WARP ? 1 : align_period(p.x_ld * (long long)sizeof(T));      // (8 rows at a time are a multiple of every period)
  grid -= grid % period;
  kern<<<(int)(need < grid ? need : grid), threads, 0, st>>>(p);
  return 0;
}

template <typename T, typename W, bool FP8>
int launch_fwd_sized(const NormFwdParams& p, cudaStream_t st) {
  const bool aligned = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && (p.x_ld * sizeof(T)) % 16 == 0;
  const int nvec = (p.H + (aligned ? 0 : kEpv<T> - 1) + kEpv<T> - 1) / kEpv<T>;
  if (nvec <= 32) return launch_fwd<T, W, 1, FP8, true>(p, kWarpRows * 32, st);
  if (nvec <= 64) return launch_fwd<T, W, 2, FP8, true>(p, kWarpRows * 32, st);
  if (nvec <= 128) return launch_fwd<T, W, 4, FP8, true>(p, kWarpRows * 32, st);
  const auto threads = [nvec](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
  if (nvec <= 2048) return launch_fwd<T, W, 2, FP8, false>(p, threads(2), st);
  if (nvec <= 4096) return launch_fwd<T, W, 4, FP8, false>(p, threads(4), st);
  return launch_fwd<T, W, 9, FP8, false>(p, threads(9), st);
}

template <typename T, typename W>
int launch_fwd_out(const NormFwdParams& p, cudaStream_t st) {
  return p.q != nullptr ? launch_fwd_sized<T, W, true>(p, st) : launch_fwd_sized<T, W, false>(p, st);
}

}  // namespace norm

int launch_rms_norm_fwd(const NormFwdParams& p, cudaStream_t st) {
  using namespace norm;
  if (p.T < 0 || p.H < 1 || p.H > kNormMaxHidden || !(p.eps >= 0.f)) return 1;
  if (p.wtype != p.type && p.wtype != ELEM_F32) return 1;
  const long long es = p.type == ELEM_F32 ? 4 : 2;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x);
  // every tensor that is moved in vectors has its rows where x has them within 16 bytes
  const auto alike = [&](const void* t, long long ld) {
    return t == nullptr || ((reinterpret_cast<uintptr_t>(t) ^ at) % 16 == 0 && (ld - p.x_ld) * es % 16 == 0);
  };
  if (!alike(p.y, p.H) || !alike(p.h, p.H) || !alike(p.residual, p.res_ld) || at % es || reinterpret_cast<uintptr_t>(p.w) % (p.wtype == ELEM_F32 ? 4 : 2)) return 1;
  if ((p.residual == nullptr) != (p.h == nullptr) || (p.y == nullptr && p.q == nullptr)) return 1;
  if (p.q != nullptr && (p.H % kNormScaleBlock || p.scales == nullptr || at % 16 || p.x_ld * es % 16 || reinterpret_cast<uintptr_t>(p.q) % 8)) return 1;
  if (p.T == 0) return 0;
  if (p.type == ELEM_BF16) return p.wtype == ELEM_F32 ? launch_fwd_out<__nv_bfloat16, float>(p, st) : launch_fwd_out<__nv_bfloat16, __nv_bfloat16>(p, st);
  if (p.type == ELEM_F16) return p.wtype == ELEM_F32 ? launch_fwd_out<__half, float>(p, st) : launch_fwd_out<__half, __half>(p, st);
  return launch_fwd_out<float, float>(p, st);
}

}  // namespace b200ep
