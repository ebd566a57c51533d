// Loss that keeps the choice of experts balanced, and its gradient. Over the n tokens of a sequence that have a choice, with
// scores s_t (softmax of the logits, or sigmoid), p_t = s_t / (sum of s_t + 1e-20) and K choices a token:
//   f_e = E / (K n) * (choices of e),   L = coeff * sum_e f_e * (1 / n) sum_t p_te  [+ z_coeff * (1 / n) sum_t logsumexp(l_t)^2]
// and the mean over the sequences that have such tokens. f is a count and has no gradient:
//   softmax: dl_te = c p_te (f_e - F_t),  sigmoid: dl_te = c p_te (1 - s_te) (f_e - F_t),  F_t = sum_j f_j p_tj, c = coeff / (n B')
//   and 2 z_coeff / (n B') * logsumexp * p_te.
// With the counts known the loss is a sum over tokens of F_t, so that the logits are read once forward and once backward:
// a launch that counts the choices (whole numbers: any order gives the same), one that sums F_t (in 64 bits, in a fixed
// order). A warp has a run of neighbouring rows and keeps f of their sequence in registers. Bound: latency, of launches for
// few tokens and of the reductions over a row for many: 16384 x 64 in softmax take 2.9 + 8.8 us forward and 8.2 backward on
// one B200, where the logits' bytes would take 0.6 each time; 8191 x 256 in sigmoid 2.7 + 9.8 and 13.2, where the backward's eight
// counts of 64 bits a lane spill 92 bytes a thread.
#include "route.cuh"

namespace b200ep {
namespace route {

// The sequence that row t belongs to, -1 for none: of those that begin at or before it the last.
__device__ __forceinline__ int sequence_of(const int* off, int B, long long t) {
  if (off == nullptr) return 0;
  if (t < (long long)*off || t >= (long long)off[B]) return -1;
  int lo = 0, hi = B;                                       // off[lo] <= t < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long long)off[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// Choices and rows with a choice, counted in shared memory for a run of rows of one sequence at a time.
__global__ void __launch_bounds__(256)
balance_count_kernel(const BalanceParams p, int rows_per) {
  __shared__ int s_count[kRouterMaxExperts];
  __shared__ int s_rows;
  stream_order_next();
  const int E = p.E, K = p.K, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a warp looks at as many rows at a time as have their choices in its lanes
  const int rows_at_once = 32 / K, sub = lane / K, choice = lane - sub * K;
  const uint32_t one_row = K == 32 ? 0xffffffffu : (1u << K) - 1;
  const long long lo = (long long)blockIdx.x * rows_per, hi = min(lo + rows_per, (long long)p.T);
  for (long long at = lo; at < hi;) {
    long long end = hi;
    int b = 0;
    if (p.seq_off != nullptr) {
      if (at >= (long long)p.seq_off[p.B]) break;   // (rows outside all sequences are passed over)
      if (at < (long long)*p.seq_off) { at = (long long)*p.seq_off; continue; }
      b = sequence_of(p.seq_off, p.B, at);
      end = min(end, (long long)p.seq_off[b + 1]);
    }
    for (int e = threadIdx.x; e < E; e += blockDim.x) s_count[e] = 0;
    if (threadIdx.x == 0) s_rows = 0;
    __syncthreads();
    int live = 0;
    for (long long t0 = at + warp * rows_at_once; t0 < end; t0 += (long long)(blockDim.x >> 5) * rows_at_once) {
      const long long t = t0 + sub;
      const long long i = sub < rows_at_once && t < end ? p.idx[t * K + choice] : -1;
      const bool ok = i >= 0 && i < E;
      if (ok) atomicAdd(s_count + (int)i, 1);
      const uint32_t some = __ballot_sync(0xffffffffu, ok);
      if (choice == 0 && sub < rows_at_once && (some >> (sub * K) & one_row)) ++live;
    }
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0 && live) atomicAdd(&s_rows, live);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x)
      if (s_count[e]) atomicAdd(p.counts + (long long)b * E + e, s_count[e]);
    if (threadIdx.x == 0 && s_rows) atomicAdd(p.counts + (long long)p.B * E + b, s_rows);
    __syncthreads();
    at = end;
  }
}

// 1 / (sequences with a token that has a choice), the same in every thread of the CTA.
__device__ __forceinline__ float sequence_share(const BalanceParams& p) {
  if (p.B == 1) return 1.f;
  __shared__ int s_live;
  if (threadIdx.x == 0) s_live = 0;
  __syncthreads();
  int n = 0;
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) n += p.counts[(long long)p.B * p.E + b] > 0;
  if (n) atomicAdd(&s_live, n);
  __syncthreads();
  return 1.f / (float)max(1, s_live);
}

// A row as it is read: this lane's logits, and whether it has a choice (lane k looks at choice k).
template <typename L, int VPL>
struct Raw {
  float l[VPL];
  bool chose = false;
  __device__ __forceinline__ void load(const BalanceParams& a, long long t, int lane) {
    const long long i = lane < a.K ? a.idx[t * a.K + lane] : -1;
    chose = i >= 0 && i < a.E;
    const L* row = static_cast<const L*>(a.logits) + t * a.ld;
#pragma unroll
    for (int k = 0; k < VPL; ++k) l[k] = k * 32 + lane < a.E ? logit(row + k * 32 + lane) : -INFINITY;
  }
};

// What a warp makes of it.
template <typename L, int VPL>
struct Row {
  float p[VPL];              // share of the scores
  float s[VPL];              // sigmoid: 1 - score
  float lse, F;
  float rest;                // what the shares' sum lacks to 1
  // false: the row takes no part
  template <typename V>
  __device__ __forceinline__ bool of(const BalanceParams& a, const Raw<L, VPL>& raw, const V* f) {
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      p[k] = raw.l[k];
      top = nan_max(p[k], top);
    }
    if (!__any_sync(0xffffffffu, raw.chose)) return false;
    float sum = 0.f;
    lse = 0.f;
    if (a.score == SCORE_SOFTMAX) {
      top = warp_max(top);
      if (top == -INFINITY) top = 0.f;
#pragma unroll
      for (int k = 0; k < VPL; ++k) { p[k] = expf(p[k] - top); sum += p[k]; }
      sum = warp_sum(sum);
      if (a.z_coeff != 0.f && !(sum == 0.f)) lse = top + logf(sum);
    } else {
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        const float q = expf(-fabsf(p[k])), r = 1.f / (1.f + q), qr = q * r;
        const bool up = p[k] >= 0.f;
        s[k] = up ? qr : r;
        p[k] = p[k] == -INFINITY ? 0.f : (up ? r : qr);
        if (q != q) p[k] = q;
        sum += p[k];
      }
      sum = warp_sum(sum);
    }
    const float inv = 1.f / (sum + kSumEps);
    rest = kSumEps * inv;
    F = 0.f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) { p[k] *= inv; F = fmaf((float)f[k], p[k], F); }
    F = warp_sum(F);
    return true;
  }
};

// Rows of a warp, a run of neighbours; f of the sequence that they are in is kept in registers.
template <int VPL, typename V>
struct Walk {
  int b = -1;
  V f[VPL];
  float share = 0.f;
  __device__ __forceinline__ bool to(const BalanceParams& a, long long t, float per_sequence, int lane) {
    const int now = sequence_of(a.seq_off, a.B, t);
    if (now < 0) return false;
    if (now == b) return true;
    b = now;
    const int n = max(1, a.counts[(long long)a.B * a.E + b]);
    const V unit = (V)a.E / ((V)a.K * (V)n);
#pragma unroll
    for (int k = 0; k < VPL; ++k) f[k] = k * 32 + lane < a.E ? (V)a.counts[(long long)b * a.E + k * 32 + lane] * unit : (V)0;
    share = per_sequence / (float)n;
    return true;
  }
};

constexpr int kBalanceWarps = 8;

template <typename L, int VPL>
__global__ void __launch_bounds__(kBalanceWarps * 32, VPL <= 8 ? 4 : 2)
balance_loss_kernel(const BalanceParams p, int rows_per_warp) {
  __shared__ double s_part[kBalanceWarps];
  __shared__ bool s_last;
  stream_order_wait();
  stream_order_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float per_sequence = sequence_share(p);
  const long long lo = ((long long)blockIdx.x * kBalanceWarps + warp) * rows_per_warp, hi = min(lo + rows_per_warp, (long long)p.T);
  Walk<VPL, float> at;
  Raw<L, VPL> raw, next;
  Row<L, VPL> row;
  double mine = 0.0;
  if (lo < hi) next.load(p, lo, lane);
  for (long long t = lo; t < hi; ++t) {
    raw = next;
    if (t + 1 < hi) next.load(p, t + 1, lane);              // (under way while this row is looked at)
    if (!at.to(p, t, per_sequence, lane) || !row.of(p, raw, at.f)) continue;
    mine += (double)at.share * ((double)p.coeff * (double)row.F + (double)p.z_coeff * (double)row.lse * (double)row.lse);
  }
  if (lane == 0) s_part[warp] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    double v = 0.0;
    for (int k = 0; k < kBalanceWarps; ++k) v += s_part[k];
    p.part[blockIdx.x] = v;
    __threadfence();
    s_last = atomicAdd(p.counts + (long long)p.B * p.E + p.B, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double v = 0.0;
  for (int k = threadIdx.x; k < (int)gridDim.x; k += kBalanceWarps * 32) v += __ldcg(p.part + k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();                                          // (thread 0 has read s_part by now)
  if (lane == 0) s_part[warp] = v;
  __syncthreads();
  if (threadIdx.x != 0) return;
  v = 0.0;
  for (int k = 0; k < kBalanceWarps; ++k) v += s_part[k];
  *p.loss = (float)v;
}

template <typename L, int VPL>
__global__ void __launch_bounds__(kBalanceWarps * 32, VPL <= 8 ? 4 : 2)
balance_bwd_kernel(const BalanceBwdParams a, int rows_per_warp) {
  stream_order_wait();
  stream_order_next();
  const BalanceParams& p = a.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float per_sequence = sequence_share(p);
  const float g = *a.dloss;
  const long long lo = ((long long)blockIdx.x * kBalanceWarps + warp) * rows_per_warp, hi = min(lo + rows_per_warp, (long long)p.T);
  Walk<VPL, double> at;
  Raw<L, VPL> raw, next;
  Row<L, VPL> row;
  if (lo < hi) next.load(p, lo, lane);
  for (long long t = lo; t < hi; ++t) {
    raw = next;
    if (t + 1 < hi) next.load(p, t + 1, lane);
    L* out = static_cast<L*>(a.dlogits) + t * p.E;
    const bool in = at.to(p, t, per_sequence, lane) && row.of(p, raw, at.f);
    // f - F, where the load is nearly balanced, is a small difference of numbers near each other, and F is off by roundings of
    // its own size: the difference is taken in 64 bits, and what F is off by, the weighted mean of the differences, out of it
    float diff[VPL], off = 0.f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      diff[k] = in ? (float)(at.f[k] - (double)row.F) : 0.f;
      off = fmaf(diff[k], in ? row.p[k] : 0.f, off);
    }
    off = warp_sum(off) - (in ? row.F * row.rest : 0.f);
    const float c = g * at.share * p.coeff, z = 2.f * g * at.share * p.z_coeff * (in ? row.lse : 0.f);
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      if (k * 32 + lane >= p.E) continue;
      float d = 0.f;
      if (in) {
        d = c * (diff[k] - off);
        if (p.score == SCORE_SIGMOID) d *= row.s[k];
        d = row.p[k] * (d + z);
      }
      put(out + k * 32 + lane, d);
    }
  }
}

// Multiprocessors of a B200. How the rows are split is a matter of speed alone, has to be the same where room is made for the parts
// and where they are written, and is worked out several times in calls that are bound by host time: not asked of the runtime.
constexpr long long kSms = 148;

inline int rows_a_warp(int T) {
  // four CTAs of 8 warps on every SM, each warp a run of neighbouring rows
  const long long warps = kSms * 4 * kBalanceWarps;
  return (int)((T + warps - 1) / warps) < 1 ? 1 : (int)((T + warps - 1) / warps);
}
inline int ctas(int T) {
  const long long per = (long long)rows_a_warp(T) * kBalanceWarps;
  return (int)((T + per - 1) / per);
}

template <typename L, int VPL>
int forward_sized(const BalanceParams& p, cudaStream_t st) {
  return launch_ordered(balance_loss_kernel<L, VPL>, dim3(balance_ctas(p)), dim3(kBalanceWarps * 32), 0, st, 1, p, rows_a_warp(p.T)) == cudaSuccess ? 0 : 2;
}
template <typename L, int VPL>
int backward_sized(const BalanceBwdParams& a, cudaStream_t st) {
  return launch_ordered(balance_bwd_kernel<L, VPL>, dim3(balance_ctas(a.f)), dim3(kBalanceWarps * 32), 0, st, 1, a, rows_a_warp(a.f.T)) == cudaSuccess ? 0 : 2;
}

#define B200EP_BY_SIZE(E, CALL)              \
  (E) <= 64 ? CALL(2) : (E) <= 128 ? CALL(4) : (E) <= 256 ? CALL(8) : (E) <= 512 ? CALL(16) : CALL(32)

template <typename L>
int forward(const BalanceParams& p, cudaStream_t st) {
#define B200EP_CALL(V) forward_sized<L, V>(p, st)
  return B200EP_BY_SIZE(p.E, B200EP_CALL);
#undef B200EP_CALL
}
template <typename L>
int backward(const BalanceBwdParams& a, cudaStream_t st) {
#define B200EP_CALL(V) backward_sized<L, V>(a, st)
  return B200EP_BY_SIZE(a.f.E, B200EP_CALL);
#undef B200EP_CALL
}

bool fits(const BalanceParams& p) {
  return p.T >= 0 && p.E >= 1 && p.E <= kRouterMaxExperts && p.K >= 1 && p.K <= kRouteMaxTopk && p.B >= 1 && (p.seq_off != nullptr || p.B == 1) &&
         (p.z_coeff == 0.f || p.score == SCORE_SOFTMAX);
}

}  // namespace route

long long balance_words(const BalanceParams& p) { return (long long)p.B * p.E + p.B + 1; }
int balance_ctas(const BalanceParams& p) { return route::ctas(p.T); }

int launch_balance(const BalanceParams& p, cudaStream_t st) {
  if (!route::fits(p)) return 1;
  if (p.T == 0) return cudaMemsetAsync(p.loss, 0, sizeof(float), st) == cudaSuccess ? 0 : 2;
  if (cudaMemsetAsync(p.counts, 0, (size_t)balance_words(p) * sizeof(int), st) != cudaSuccess) return 2;
  const long long ctas = 2 * route::kSms, share = (p.T + ctas - 1) / ctas, rows_per = share < 8 ? 8 : share;      // (64 bits: T may be the largest int)
  route::balance_count_kernel<<<(unsigned)((p.T + rows_per - 1) / rows_per), 256, 0, st>>>(p, (int)rows_per);
  if (p.type == ELEM_BF16) return route::forward<__nv_bfloat16>(p, st);
  if (p.type == ELEM_F16) return route::forward<__half>(p, st);
  return route::forward<float>(p, st);
}

int launch_balance_bwd(const BalanceBwdParams& a, cudaStream_t st) {
  if (!route::fits(a.f)) return 1;
  if (a.f.T == 0) return 0;
  if (a.f.type == ELEM_BF16) return route::backward<__nv_bfloat16>(a, st);
  if (a.f.type == ELEM_F16) return route::backward<__half>(a, st);
  return route::backward<float>(a, st);
}

}  // namespace b200ep
