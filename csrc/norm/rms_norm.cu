// Root-mean-square norm with the residual's addition, rows in bf16, f16 or f32 out, or e4m3 with 1x128 scales.
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w,  scale = max(amax of 128 channels of y, 1e-4) / 448
// h, its square sum and y are held in f32 and rounded once, where they are stored: y is that of the sum before its
// rounding. Bound: memory (two tensors read and two written with a residual), for few rows latency. A row is read once
// and stays in registers; a warp has a row of up to 128 vectors of 16 bytes, a CTA a longer one; CTAs are persistent, keep
// their columns' weights in registers and have the next rows under way while they are at one: every thread copies the
// vectors that it will need itself (cp.async), so that no barrier goes with them. One B200: 8191 x 7168 with a residual to fp8
// and bf16 88.6 us (6.0 TB/s, 92 % of a copy's rate; without the rows to come under way 97), 16384 x 7168 to bf16 154 to 166,
// 4095 x 4096 20.2; f16 rows of 1407 (12001 of them) 18.1, bound by instructions, of 1408 14.4; 7 x 7168 3.4.
#include <cuda_fp8.h>
#include "../ep/cast.cuh"
#include "norm.cuh"

namespace b200ep {
namespace norm {

constexpr int kWarpRows = 8;             // rows of a CTA at a time where a warp has a row

template <typename T, typename W, int VPT, bool FP8, bool WARP, bool ALIGNED>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : 1024, WARP ? 2 : 1)
rms_norm_fwd_kernel(const __grid_constant__ NormFwdParams p, int stages) {
  stream_order_wait();
  constexpr int EPV = kEpv<T>, PAIRS = EPV / 2;
  extern __shared__ __align__(16) uint4 s_rows[];           // [stage][x, residual][vector][thread]
  __shared__ float s_sum[2][32];
  const int H = p.H;
  const int row0 = WARP ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int step = WARP ? gridDim.x * kWarpRows : gridDim.x;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x;
  constexpr bool STAGED = kStaged<T, VPT, WARP>;
  const bool add = p.residual != nullptr;
  // (the same for every row of this thread: the grid strides by a multiple of the alignment's period)
  const int shift = ALIGNED ? 0 : (int)((reinterpret_cast<uintptr_t>(static_cast<const T*>(p.x) + (long long)row0 * p.x_ld) & 15) / sizeof(T));
  const int e_first = tid * EPV - shift, e_next = threads * EPV;         // the thread's first element, and to its next vector's
  Walk<T> x(p.x, p.x_ld, row0, step, e_first), res(p.residual, p.res_ld, row0, step, e_first);
  const uint32_t word = 16u * blockDim.x, plane = VPT * word, stage_bytes = plane * (add ? 2u : 1u);      // bytes of a vector of all threads, of a tensor, of a stage
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_rows) + 16u * threadIdx.x, mine_end = mine + stages * stage_bytes;
  long long ahead = row0;                                   // the next row to be fetched
  const auto fetch = [&](uint32_t to) {
    if constexpr (!STAGED) return;
    if (ahead < p.T) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (e_first + i * e_next < H) {
          const int off = i * e_next * (int)sizeof(T), bytes = min(16, (H - e_first - i * e_next) * (int)sizeof(T));
          fetch_vec<ALIGNED>(to + i * word, x.at + off, bytes);
          if (add) fetch_vec<ALIGNED>(to + plane + i * word, res.at + off, bytes);
        }
      x.at += x.step;
      res.at += res.step;
    }
    ahead += step;
    fetch_commit();
  };
  for (int k = 0; k < stages; ++k) fetch(mine + k * stage_bytes);
  const bool w_aligned = shift == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15) == 0;
  WeightVec<T, W> w[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) w[i].load(static_cast<const W*>(p.w), e_first + i * e_next, H, w_aligned);
  const float inv_h = 1.f / (float)H;
  const int width = WARP ? 32 : block_width();
  int parity = 0;
  uint32_t from = mine;
  // Where the results go: addresses that are moved along (60000 x 257 34 us, 51 with them made anew from the row's offset), but
  // in the fp8 form, whose registers that costs (8191 x 7168 94.4 us, 91.6 from the offset).
  Walk<T> y(p.y, H, row0, step, e_first), sum(p.h, H, row0, step, e_first);
  const long long out_step = (long long)step * H;
  long long out = (long long)row0 * H;
  const auto at = [&](const Walk<T>& w, void* t, int i) {
    if constexpr (FP8) return reinterpret_cast<char*>(static_cast<T*>(t) + out + e_first + i * e_next);
    else return w.at + i * e_next * (int)sizeof(T);
  };
  for (long long row = row0; row < p.T; row += step, out += out_step, y.at += y.step, sum.at += sum.step, parity ^= 1) {
    if constexpr (STAGED) fetch_wait(stages - 1);
    float2 h[VPT][PAIRS], ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * e_next;
      if (e0 < H) {
        if constexpr (STAGED) unpack<T>(inside<T, ALIGNED>(lds_v4(from + i * word), e0), h[i]);
        else unpack<T>(load_vec<T, ALIGNED>(static_cast<const T*>(p.x) + row * p.x_ld, e0, H), h[i]);
        if (add) {
          float2 r[PAIRS];
          if constexpr (STAGED) unpack<T>(inside<T, ALIGNED>(lds_v4(from + plane + i * word), e0), r);
          else unpack<T>(load_vec<T, ALIGNED>(static_cast<const T*>(p.residual) + row * p.res_ld, e0, H), r);
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) h[i][j] = add2(h[i][j], r[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) h[i][j] = make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) ss = fma2(h[i][j], h[i][j], ss);
    }
    const float total = WARP ? warp_sum(ss.x + ss.y) : block_sum(ss.x + ss.y, s_sum[parity], width);
    // (this thread's place is free: what it held is in registers, and went into the sum)
    fetch(from);
    from = from + stage_bytes == mine_end ? mine : from + stage_bytes;
    if (add) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) store_vec<T, ALIGNED>(at(sum, p.h, i), e_first + i * e_next, H, pack<T>(h[i]));
    }
    const float rstd = inverse_root(fmaf(total, inv_h, p.eps));
    if (tid == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * e_next;
      float2 wf[PAIRS];
      w[i].get(wf);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) h[i][j] = mul2(mul2(h[i][j], both(rstd)), wf[j]);
      if (!FP8 || p.y != nullptr) store_vec<T, ALIGNED>(at(y, p.y, i), e0, H, pack<T>(h[i]));
      if constexpr (FP8) {
        // (the 128 / EPV lanes of a block are neighbours and all in or all out of the row)
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) amax = fmaxf(amax, fmaxf(fabsf(h[i][j].x), fabsf(h[i][j].y)));
#pragma unroll
        for (int o = kNormScaleBlock / EPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        amax = fmaxf(amax, 1e-4f);
        const float2 inv = both(1.75f * inverse(amax * 0x1p-8f));      // 448 / amax (a power of 2 aside, so that every finite amax has one)
        if (e0 < H) {
          uint32_t o[EPV / 4];
#pragma unroll
          for (int j = 0; j < EPV / 4; ++j) {
            const float2 a = mul2(h[i][2 * j], inv), b = mul2(h[i][2 * j + 1], inv);
            o[j] = cvt4_e4m3(a.x, a.y, b.x, b.y);
          }
          char* q = static_cast<char*>(p.q) + out + e0;
          if constexpr (EPV == 8) *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
          else *reinterpret_cast<uint32_t*>(q) = o[0];
          if (e0 % kNormScaleBlock == 0) p.scales[(out + e0) / kNormScaleBlock] = amax * (1.f / 448.f);
        }
      }
    }
  }
}

template <typename T, typename W, int VPT, bool FP8, bool WARP, bool ALIGNED>
int launch_fwd(const NormFwdParams& p, int threads, cudaStream_t st) {
  const auto kern = rms_norm_fwd_kernel<T, W, VPT, FP8, WARP, ALIGNED>;
  const int row_bytes = kStaged<T, VPT, WARP> ? VPT * threads * 16 * (p.residual != nullptr ? 2 : 1) : 0;
  const int rows = WARP ? kWarpRows : 1;
  const long long need = ((long long)p.T + rows - 1) / rows;
  static Launch plan;
  int stages = 0, fit = 0;
  if (!plan.get(kern, threads, row_bytes, &stages, &fit)) return 2;
  long long grid = (long long)fit * sm_count();
  const int period = WARP ? 1 : align_period(p.x_ld * (long long)sizeof(T));      // (8 rows at a time are a multiple of every period)
  grid -= grid % period;
  if (need <= grid) { grid = need; stages = 1; }
  return launch_ordered(kern, dim3((unsigned)grid), dim3(threads), stages * row_bytes, st, 1, p, stages) == cudaSuccess ? 0 : 2;
}

template <typename T, typename W, bool FP8, bool ALIGNED>
int launch_fwd_sized(const NormFwdParams& p, cudaStream_t st) {
  const int nvec = (p.H + (ALIGNED ? 0 : kEpv<T> - 1) + kEpv<T> - 1) / kEpv<T>;
  if (nvec <= 32) return launch_fwd<T, W, 1, FP8, true, ALIGNED>(p, kWarpRows * 32, st);
  if (nvec <= 64) return launch_fwd<T, W, 2, FP8, true, ALIGNED>(p, kWarpRows * 32, st);
  if (nvec <= 128) return launch_fwd<T, W, 4, FP8, true, ALIGNED>(p, kWarpRows * 32, st);
  const auto threads = [nvec](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
  // The cast of 16-bit rows wants more warps (8191 x 7168: 95.7 us with two vectors a thread, 90.2 with one), without it, and
  // of f32 rows, fewer and longer threads are as good or better (12001 x 1408 in f16: 14.6 and 16.7; 8191 x 4096 in f32 to
  // fp8: 52.0 and 68.8).
  if constexpr (FP8 && sizeof(T) == 2) {
    if (nvec > 256 && nvec <= 1024) return launch_fwd<T, W, 1, FP8, false, ALIGNED>(p, threads(1), st);
  }
  if (nvec <= 2048) return launch_fwd<T, W, 2, FP8, false, ALIGNED>(p, threads(2), st);
  if constexpr (kMaxVecs<T, ALIGNED> > 4096) {
    if (nvec > 4096) return launch_fwd<T, W, 9, FP8, false, ALIGNED>(p, threads(9), st);
  }
  return launch_fwd<T, W, 4, FP8, false, ALIGNED>(p, threads(4), st);
}

template <typename T, typename W>
int launch_fwd_out(const NormFwdParams& p, cudaStream_t st) {
  if (p.q != nullptr) return launch_fwd_sized<T, W, true, true>(p, st);
  const bool aligned = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 && p.H % kEpv<T> == 0 && (p.T == 1 || p.x_ld % kEpv<T> == 0);
  return aligned ? launch_fwd_sized<T, W, false, true>(p, st) : launch_fwd_sized<T, W, false, false>(p, st);
}

}  // namespace norm

int launch_rms_norm_fwd(const NormFwdParams& p, cudaStream_t st) {
  using namespace norm;
  if (p.T < 0 || p.H < 1 || p.H > kNormMaxHidden || !(p.eps >= 0.f)) return 1;
  if (p.wtype != p.type && p.wtype != ELEM_F32) return 1;
  const long long es = p.type == ELEM_F32 ? 4 : 2;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x);
  // every tensor has its first row on a 16-byte boundary, and the others where x has them within 16 bytes
  const auto alike = [&](const void* t, long long ld) {
    return t == nullptr || (reinterpret_cast<uintptr_t>(t) % 16 == 0 && (ld - p.x_ld) * es % 16 == 0);
  };
  if (!alike(p.x, p.x_ld) || !alike(p.y, p.H) || !alike(p.h, p.H) || !alike(p.residual, p.res_ld) || at % 16) return 1;
  if (reinterpret_cast<uintptr_t>(p.w) % (p.wtype == ELEM_F32 ? 4 : 2)) return 1;
  if ((p.residual == nullptr) != (p.h == nullptr) || (p.y == nullptr && p.q == nullptr)) return 1;
  if (p.q != nullptr && (p.H % kNormScaleBlock || p.scales == nullptr || (p.T > 1 && p.x_ld * es % 16) || reinterpret_cast<uintptr_t>(p.q) % 8)) return 1;
  if (p.T == 0) return 0;
  if (p.type == ELEM_BF16) return p.wtype == ELEM_F32 ? launch_fwd_out<__nv_bfloat16, float>(p, st) : launch_fwd_out<__nv_bfloat16, __nv_bfloat16>(p, st);
  if (p.type == ELEM_F16) return p.wtype == ELEM_F32 ? launch_fwd_out<__half, float>(p, st) : launch_fwd_out<__half, __half>(p, st);
  return launch_fwd_out<float, float>(p, st);
}

}  // namespace b200ep
