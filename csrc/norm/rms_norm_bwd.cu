// Gradients of the root-mean-square norm with the residual's addition (y = h r w, h = x + residual, r from the forward):
//   a = dy w,  n = h r,  dx = dresidual = r (a - n mean(a n)) + dh,  dw = sum over the rows of dy n
// all in f32, rounded where they are stored. Bound: memory (three to five tensors read, one written). Of 16-bit rows with a
// residual h was rounded when the forward stored it. Where dw is wanted the caller passes x and the residual instead and h is
// summed again, a tensor more: from the stored h, dw had a second rounding's error (bf16 2.33e-3 for 1.64e-3 of its norm; dx, where h
// stands in a correction alone, 1.6574e-3 for the same, so without dw h is read: 16384 x 7168 158 for 192 us).
// Persistent CTAs have the next rows under way in shared memory while they are at one (every thread copies what it will need
// itself), and keep the weights and their part of dw in registers, so that dw costs one row of f32 a CTA, summed in a fixed
// order by a second launch: the same bits from run to run. One B200, bf16 with a residual: 16384 x 7168 188 to 201 us with f32 weights
// (5.9 TB/s or more, 91 % of a copy's rate), 192 with bf16 weights, 4095 x 4096 35.5 to 38.7, and 3 to 4 us for the second
// launch. The two-vector form spills 32 to 40 bytes a thread.
#include "norm.cuh"

namespace b200ep {
namespace norm {

constexpr int kWarpRows = 8;

template <typename T, typename W, int VPT, bool WARP, bool ALIGNED>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : 1024, 1)
rms_norm_bwd_kernel(const __grid_constant__ NormBwdParams p, int stages) {
  stream_order_wait();
  stream_order_next();
  constexpr int EPV = kEpv<T>, PAIRS = EPV / 2;
  extern __shared__ __align__(16) uint4 s_rows[];           // [stage][dy, h, other part of h, dh][vector][thread]
  __shared__ float s_sum[2][32];
  __shared__ float s_dw[WARP ? 32 * VPT * EPV : 1];
  const int H = p.H;
  const int row0 = WARP ? blockIdx.x * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  const int step = WARP ? gridDim.x * kWarpRows : gridDim.x;
  const int tid = WARP ? threadIdx.x & 31 : threadIdx.x, threads = WARP ? 32 : blockDim.x;
  constexpr bool STAGED = kStaged<T, VPT, WARP>;
  const bool two = p.res != nullptr, add = p.dh != nullptr;
  const int shift = ALIGNED ? 0 : (int)((reinterpret_cast<uintptr_t>(static_cast<const T*>(p.h) + (long long)row0 * p.h_ld) & 15) / sizeof(T));
  const int e_first = tid * EPV - shift, e_next = threads * EPV;         // the thread's first element, and to its next vector's
  Walk<T> dy(p.dy, p.dy_ld, row0, step, e_first), h(p.h, p.h_ld, row0, step, e_first);
  Walk<T> res(p.res, p.res_ld, row0, step, e_first), dh(p.dh, p.dh_ld, row0, step, e_first);
  const uint32_t word = 16u * blockDim.x, plane = VPT * word, at_dh = two ? 3 * plane : 2 * plane, stage_bytes = plane * (2u + two + add);
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(s_rows) + 16u * threadIdx.x, mine_end = mine + stages * stage_bytes;
  long long ahead = row0;                                   // the next row to be fetched
  const auto fetch = [&](uint32_t to) {
    if constexpr (!STAGED) return;
    if (ahead < p.T) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (e_first + i * e_next < H) {
          const int off = i * e_next * (int)sizeof(T), bytes = min(16, (H - e_first - i * e_next) * (int)sizeof(T));
          fetch_vec<ALIGNED>(to + i * word, dy.at + off, bytes);
          fetch_vec<ALIGNED>(to + plane + i * word, h.at + off, bytes);
          if (two) fetch_vec<ALIGNED>(to + 2 * plane + i * word, res.at + off, bytes);
          if (add) fetch_vec<ALIGNED>(to + at_dh + i * word, dh.at + off, bytes);
        }
      dy.at += dy.step;
      h.at += h.step;
      res.at += res.step;
      dh.at += dh.step;
    }
    ahead += step;
    fetch_commit();
  };
  for (int k = 0; k < stages; ++k) fetch(mine + k * stage_bytes);
  const bool w_aligned = shift == 0 && (reinterpret_cast<uintptr_t>(p.w) & 15) == 0;
  const float inv_h = 1.f / (float)H;
  WeightVec<T, W> w[VPT];
  float2 acc[VPT][PAIRS];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    w[i].load(static_cast<const W*>(p.w), e_first + i * e_next, H, w_aligned);
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) acc[i][j] = make_float2(0.f, 0.f);
  }
  // Short rows stay in registers from the sum to the result; of long ones that would cost too many, they are read again.
  constexpr bool KEEP = WARP || VPT == 1;
  const int width = WARP ? 32 : block_width();
  int parity = 0;
  uint32_t from = mine;
  const long long out_step = (long long)step * H;
  long long out = (long long)row0 * H;                      // the row in a contiguous tensor
  float next_rstd = row0 < p.T ? p.rstd[row0] : 0.f;
  for (long long row = row0; row < p.T; row += step, out += out_step, parity ^= 1) {
    const float rstd = next_rstd;
    if (row + step < p.T) next_rstd = p.rstd[row + step];
    if constexpr (STAGED) fetch_wait(stages - 1);
    const auto vec = [&](uint32_t at, int i, const void* t, long long ld, int e0) {
      if constexpr (STAGED) return inside<T, ALIGNED>(lds_v4(from + at + i * word), e0);
      else return load_vec<T, ALIGNED>(static_cast<const T*>(t) + row * ld, e0, H);
    };
    // dy and n = h r of a vector
    const auto get = [&](int i, int e0, float2 (&g)[PAIRS], float2 (&n)[PAIRS]) {
      unpack<T>(vec(0, i, p.dy, p.dy_ld, e0), g);
      unpack<T>(vec(plane, i, p.h, p.h_ld, e0), n);
      if (two) {
        float2 s[PAIRS];
        unpack<T>(vec(2 * plane, i, p.res, p.res_ld, e0), s);
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) n[j] = add2(n[j], s[j]);
      }
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) n[j] = mul2(n[j], both(rstd));
    };
    const auto result = [&](int i, int e0, float2 (&g)[PAIRS], const float2 (&n)[PAIRS], const uint4& r4, float c) {
      float2 wf[PAIRS];
      w[i].get(wf);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) g[j] = mul2(fma2(n[j], both(-c), mul2(g[j], wf[j])), both(rstd));
      if (add) {
        float2 r[PAIRS];
        unpack<T>(r4, r);
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) g[j] = add2(g[j], r[j]);
      }
      store_vec<T, ALIGNED>(reinterpret_cast<char*>(static_cast<T*>(p.dx) + out + e0), e0, H, pack<T>(g));
    };
    float2 g[KEEP ? VPT : 1][PAIRS], n[KEEP ? VPT : 1][PAIRS], c2 = make_float2(0.f, 0.f);
    uint4 r4[KEEP ? VPT : 1];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e0 = e_first + i * e_next, k = KEEP ? i : 0;
      if (e0 >= H) continue;
      float2 wf[PAIRS];
      get(i, e0, g[k], n[k]);
      if (KEEP && add) r4[k] = vec(at_dh, i, p.dh, p.dh_ld, e0);
      w[i].get(wf);
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const float2 gn = mul2(g[k][j], n[k][j]);
        acc[i][j] = add2(acc[i][j], gn);
        c2 = fma2(gn, wf[j], c2);
      }
    }
    const float c = (WARP ? warp_sum(c2.x + c2.y) : block_sum(c2.x + c2.y, s_sum[parity], width)) * inv_h;
    if constexpr (KEEP) {
      fetch(from);         // (this thread's place is free: what it held is in registers)
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e0 = e_first + i * e_next;
        if (e0 < H) result(i, e0, g[i], n[i], r4[i], c);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int e0 = e_first + i * e_next;
        if (e0 >= H) continue;
        get(i, e0, g[0], n[0]);
        if (add) r4[0] = vec(at_dh, i, p.dh, p.dh_ld, e0);
        result(i, e0, g[0], n[0], r4[0], c);
      }
      fetch(from);
    }
    from = from + stage_bytes == mine_end ? mine : from + stage_bytes;
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
            const int e = e_first + i * e_next + j;
            if (e >= 0 && e < H) s_dw[e] += j % 2 ? acc[i][j / 2].y : acc[i][j / 2].x;
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
        const int e = e_first + i * e_next + j;
        if (e >= 0 && e < H) part[e] = j % 2 ? acc[i][j / 2].y : acc[i][j / 2].x;
      }
  }
}

// dw[e] = sum of the parts: 32 columns a CTA, 32 strands of parts side by side, joined by a tree.
template <typename W>
__global__ void __launch_bounds__(1024)
sum_rows_kernel(const float* part, int parts, int H, W* dw) {
  stream_order_wait();
  stream_order_next();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (e < H) {
#pragma unroll 8
    for (int g = strand; g < parts; g += 32) v += __ldcg(part + (long long)g * H + e);
  }
  s[strand][lane] = v;
  __syncthreads();
  v = warp_sum(s[lane][strand]);
  if (lane == 0 && blockIdx.x * 32 + strand < H) dw[blockIdx.x * 32 + strand] = from_f<W>(v);
}

// `parts` given: only says how many CTAs the launch will have.
template <typename T, typename W, int VPT, bool WARP, bool ALIGNED>
int run_bwd(const NormBwdParams& p, int threads, int* parts, cudaStream_t st) {
  const auto kern = rms_norm_bwd_kernel<T, W, VPT, WARP, ALIGNED>;
  const int row_bytes = !kStaged<T, VPT, WARP> ? 0 : VPT * threads * 16 * (2 + (p.res != nullptr) + (p.dh != nullptr));
  const int rows = WARP ? kWarpRows : 1;
  const long long need = ((long long)p.T + rows - 1) / rows;
  static Launch plan;
  int stages = 0, fit = 0;
  if (!plan.get(kern, threads, row_bytes, &stages, &fit)) return 2;
  long long grid = (long long)fit * sm_count();
  const int period = WARP ? 1 : align_period(p.h_ld * (long long)sizeof(T));
  grid -= grid % period;
  if (need <= grid) { grid = need; stages = 1; }
  if (parts != nullptr) { *parts = (int)grid; return 0; }
  if (p.part != nullptr && p.parts != (int)grid) return 1;
  if (launch_ordered(kern, dim3((unsigned)grid), dim3(threads), stages * row_bytes, st, 1, p, stages) != cudaSuccess) return 2;
  if (p.part == nullptr) return 0;
  return launch_ordered(sum_rows_kernel<W>, dim3((p.H + 31) / 32), dim3(1024), 0, st, 1, p.part, p.parts, p.H, static_cast<W*>(p.dw)) == cudaSuccess ? 0 : 2;
}

template <typename T, typename W, bool ALIGNED>
int bwd_sized(const NormBwdParams& p, int* parts, cudaStream_t st) {
  const int nvec = (p.H + (ALIGNED ? 0 : kEpv<T> - 1) + kEpv<T> - 1) / kEpv<T>;
  if (nvec <= 32) return run_bwd<T, W, 1, true, ALIGNED>(p, kWarpRows * 32, parts, st);
  if (nvec <= 64) return run_bwd<T, W, 2, true, ALIGNED>(p, kWarpRows * 32, parts, st);
  const auto threads = [nvec](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
  // up to 512 threads where that goes, so that an SM has two CTAs or more: 16384 x 7168 with 896 threads 224 us, with 448
  // 198; 16384 x 4096 with 512 102 us, with 256 98.5; 4096 x 8192 in f32 with 1024 83 us, with 512 66
  if (nvec <= 256) return run_bwd<T, W, 1, false, ALIGNED>(p, threads(1), parts, st);
  if (nvec <= (sizeof(T) == 4 ? 1024 : 2048)) return run_bwd<T, W, 2, false, ALIGNED>(p, threads(2), parts, st);
  if constexpr (kMaxVecs<T, ALIGNED> > 4096) {
    if (nvec > 4096) return run_bwd<T, W, 9, false, ALIGNED>(p, threads(9), parts, st);
  }
  return run_bwd<T, W, 4, false, ALIGNED>(p, threads(4), parts, st);
}

template <typename T, typename W>
int bwd_aligned(const NormBwdParams& p, int* parts, cudaStream_t st) {
  const bool aligned = p.H % kEpv<T> == 0 && (p.T == 1 || p.h_ld % kEpv<T> == 0);
  return aligned ? bwd_sized<T, W, true>(p, parts, st) : bwd_sized<T, W, false>(p, parts, st);
}

static int bwd(const NormBwdParams& p, int* parts, cudaStream_t st) {
  if (p.T < 0 || p.H < 1 || p.H > kNormMaxHidden) return 1;
  if (p.wtype != p.type && p.wtype != ELEM_F32) return 1;
  const long long es = p.type == ELEM_F32 ? 4 : 2;
  const auto alike = [&](const void* t, long long ld) {
    return t == nullptr || (reinterpret_cast<uintptr_t>(t) % 16 == 0 && (ld - p.h_ld) * es % 16 == 0);
  };
  if (!alike(p.h, p.h_ld) || !alike(p.dy, p.dy_ld) || !alike(p.dh, p.dh_ld) || !alike(p.res, p.res_ld) || !alike(p.dx, p.H) || reinterpret_cast<uintptr_t>(p.w) % (p.wtype == ELEM_F32 ? 4 : 2)) return 1;
  if (p.T == 0) { if (parts != nullptr) *parts = 0; return 0; }
  if (p.type == ELEM_BF16) return p.wtype == ELEM_F32 ? bwd_aligned<__nv_bfloat16, float>(p, parts, st) : bwd_aligned<__nv_bfloat16, __nv_bfloat16>(p, parts, st);
  if (p.type == ELEM_F16) return p.wtype == ELEM_F32 ? bwd_aligned<__half, float>(p, parts, st) : bwd_aligned<__half, __half>(p, parts, st);
  return bwd_aligned<float, float>(p, parts, st);
}

}  // namespace norm

int rms_norm_bwd_parts(const NormBwdParams& p) {
  int parts = 0;
  return norm::bwd(p, &parts, nullptr) == 0 ? parts : -1;
}

int launch_rms_norm_bwd(const NormBwdParams& p, cudaStream_t st) { return norm::bwd(p, nullptr, st); }

}  // namespace b200ep
