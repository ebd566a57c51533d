// Gradients of the root-mean-square norm with the residual's addition (y = h r w, h = x + residual, r from the forward):
//   a = dy w,  n = h r,  dx = dresidual = r (a - n mean(a n)) + dh,  dw = sum over the rows of dy n
// all in f32, rounded where they are stored. Bound: memory (three or four tensors read, one written). h is read as the
// forward stored it, which costs dw a relative error of one rounding of h (2^-9 for bf16, about that of storing dw in bf16);
// for weights in f32 the caller passes x and the residual instead and h is summed again: a tensor more, dw exact to 32 bits. A row is read once and stays in registers; persistent CTAs keep the weights and their part of dw there too, so
// that dw costs one row of f32 a CTA, summed in a fixed order by a second launch: the same bits from run to run.
#include "norm.cuh"

namespace b200ep {
namespace norm {

constexpr int kWarpRows = 8;

template <typename T, typename W, int VPT, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : (VPT <= 2 ? 512 : 1024), WARP ? 2 : 1)
rms_norm_bwd_kernel(const NormBwdParams p) {
  constexpr int EPV = kEpv<T>;
  __shared__ float s_sum[2][32];
  __shared__ float s_dw[WARP ? 32 * VPT * EPV : 1];
  const int H = p.H;
  const int row0 = WARP ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int step = WARP ? gridDim.x * kWarpRows : gridDim.x;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x;
  const T* dy = static_cast<const T*>(p.dy);
  const T* dh = static_cast<const T*>(p.dh);
  const T* h = static_cast<const T*>(p.h);
  const T* res = static_cast<const T*>(p.res);
  T* dx = static_cast<T*>(p.dx);
  const int shift = (int)((reinterpret_cast<uintptr_t>(h + (long long)row0 * p.h_ld) & 15) / sizeof(T));
  const bool w_aligned = shift == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15) == 0;
  const float inv_h = 1.f / (float)H;
  WeightVec<T, W> w[VPT];
  float acc[VPT][EPV];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    w[i].load(static_cast<const W*>(p.w), (i * threads + tid) * EPV - shift, H, w_aligned);
#pragma unroll
    for (int j = 0; j < EPV; ++j) acc[i][j] = 0.f;
  }
  int parity = 0;
  for (long long row = row0; row < p.T; row += step, parity ^= 1) {
    uint4 gv[VPT], hv[VPT], sv[VPT], rv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = (i * threads + tid) * EPV - shift;
      gv[i] = load_vec(dy + row * p.dy_ld, e0, H);
      hv[i] = load_vec(h + row * p.h_ld, e0, H);
      if (res != nullptr) sv[i] = load_vec(res + row * p.res_ld, e0, H);
      if (dh != nullptr) rv[i] = load_vec(dh + row * p.dh_ld, e0, H);
    }
    const float rstd = p.rstd[row];
    const auto normed = [&](int i, float* n) {
      unpack<T>(hv[i], n);
      if (res != nullptr) {
        float s[EPV];
        unpack<T>(sv[i], s);
#pragma unroll
        for (int j = 0; j < EPV; ++j) n[j] += s[j];
      }
#pragma unroll
      for (int j = 0; j < EPV; ++j) n[j] *= rstd;
    };
    float c = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float g[EPV], n[EPV], wf[EPV];
      unpack<T>(gv[i], g);
      normed(i, n);
      w[i].get(wf);
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        const float gn = g[j] * n[j];
        acc[i][j] += gn;
        c = fmaf(gn, wf[j], c);
      }
    }
    c = (WARP ? warp_sum(c) : block_sum(c, s_sum[parity])) * inv_h;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float g[EPV], n[EPV], wf[EPV], r[EPV];
      unpack<T>(gv[i], g);
      normed(i, n);
      w[i].get(wf);
      if (dh != nullptr) unpack<T>(rv[i], r);
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        const float d = rstd * (g[j] * wf[j] - n[j] * c);
        g[j] = dh != nullptr ? d + r[j] : d;
      }
      store_vec(dx + row * H, (i * threads + tid) * EPV - shift, H, pack<T>(g));
    }
  }
  if (p.part == nullptr) return;
  float* part = p.part + (long long)blockIdx.x * H;
  if constexpr (WARP) {
    // the warps add their sums one after the other (rows of one CTA may begin at different places within 16 bytes)
    for (int e = threadIdx.x; e < H; e += blockDim.x) s_dw[e] = 0.f;
    for (int k = 0; k < kWarpRows; ++k) {
      __syncthreads();
      if ((threadIdx.x >> 5) == k) {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int j = 0; j < EPV; ++j) {
            const int e = (i * 32 + tid) * EPV - shift + j;
            if (e >= 0 && e < H) s_dw[e] += acc[i][j];
          }
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < H; e += blockDim.x) part[e] = s_dw[e];
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        const int e = (i * threads + tid) * EPV - shift + j;
        if (e >= 0 && e < H) part[e] = acc[i][j];
      }
  }
}

// dw[e] = sum of the parts in ascending order, 8 strands of them side by side: 32 columns a CTA.
template <typename W>
__global__ void __launch_bounds__(256)
sum_rows_kernel(const float* __restrict__ part, int parts, int H, W* __restrict__ dw) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (e < H) {
#pragma unroll 4
    for (int g = strand; g < parts; g += 8) v += part[(long long)g * H + e];
  }
  s[strand][lane] = v;
  __syncthreads();
  if (strand == 0 && e < H) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += s[k][lane];
    dw[e] = from_f<W>(v);
  }
}

// `grid` null: launches; else only says how many CTAs the launch would have.
template <typename T, typename W, int VPT, bool WARP>
int run_bwd(const NormBwdParams& p, int threads, int* parts, cudaStream_t st) {
  const auto kern = rms_norm_bwd_kernel<T, W, VPT, WARP>;
  if (parts != nullptr) {
    int fit = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, threads, 0) != cudaSuccess || fit < 1) return 2;
    const int rows = WARP ? kWarpRows : 1;
    const long long need = ((long long)p.T + rows - 1) / rows;
    long long grid = (long long)fit * sm_count();
    const int period = WARP ? 1 : align_period(p.h_ld * (long long)sizeof(T));
    grid -= grid % period;
    *parts = (int)(need < grid ? need : grid);
    return 0;
  }
  kern<<<p.parts, threads, 0, st>>>(p);
  if (p.part != nullptr) sum_rows_kernel<W><<<(p.H + 31) / 32, 256, 0, st>>>(p.part, p.parts, p.H, static_cast<W*>(p.dw));
  return 0;
}

template <typename T, typename W>
int bwd_sized(const NormBwdParams& p, int* parts, cudaStream_t st) {
  const bool aligned = (reinterpret_cast<uintptr_t>(p.h) & 15) == 0 && (p.h_ld * sizeof(T)) % 16 == 0;
  const int nvec = (p.H + (aligned ? 0 : kEpv<T> - 1) + kEpv<T> - 1) / kEpv<T>;
  if (nvec <= 32) return run_bwd<T, W, 1, true>(p, kWarpRows * 32, parts, st);
  if (nvec <= 64) return run_bwd<T, W, 2, true>(p, kWarpRows * 32, parts, st);
  const auto threads = [nvec](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
  if (nvec <= 1024) return run_bwd<T, W, 2, false>(p, threads(2), parts, st);
  if (nvec <= 4096) return run_bwd<T, W, 4, false>(p, threads(4), parts, st);
  return run_bwd<T, W, 9, false>(p, threads(9), parts, st);
}

static int bwd(const NormBwdParams& p, int* parts, cudaStream_t st) {
  if (p.T < 0 || p.H < 1 || p.H > kNormMaxHidden) return 1;
  if (p.wtype != p.type && p.wtype != ELEM_F32) return 1;
  const long long es = p.type == ELEM_F32 ? 4 : 2;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.h);
  const auto alike = [&](const void* t, long long ld) {
    return t == nullptr || ((reinterpret_cast<uintptr_t>(t) ^ at) % 16 == 0 && (ld - p.h_ld) * es % 16 == 0);
  };
  if (!alike(p.dy, p.dy_ld) || !alike(p.dh, p.dh_ld) || !alike(p.res, p.res_ld) || !alike(p.dx, p.H) || at % es || reinterpret_cast<uintptr_t>(p.w) % (p.wtype == ELEM_F32 ? 4 : 2)) return 1;
  if (p.T == 0) { if (parts != nullptr) *parts = 0; return 0; }
  if (p.type == ELEM_BF16) return p.wtype == ELEM_F32 ? bwd_sized<__nv_bfloat16, float>(p, parts, st) : bwd_sized<__nv_bfloat16, __nv_bfloat16>(p, parts, st);
  if (p.type == ELEM_F16) return p.wtype == ELEM_F32 ? bwd_sized<__half, float>(p, parts, st) : bwd_sized<__half, __half>(p, parts, st);
  return bwd_sized<float, float>(p, parts, st);
}

}  // namespace norm

int rms_norm_bwd_parts(const NormBwdParams& p) {
  int parts = 0;
  return norm::bwd(p, &parts, nullptr) == 0 ? parts : -1;
}

int launch_rms_norm_bwd(const NormBwdParams& p, cudaStream_t st) { return norm::bwd(p, nullptr, st); }

}  // namespace b200ep
