// Choice of experts. For a token's logits l [E]:
//   s = softmax(l) or sigmoid(l);  v = s + bias (-inf where l is: that expert is not available)
//   groups: of the E experts in `groups` runs, those in the `topk_groups` runs with the highest values stay, a run's value
//           being the sum of its 1 or 2 best v (of those above -inf)
//   choice: the K highest v, in descending order, the lower index first among equals; -1 where nothing above -inf is left
//   w = s (without the bias) of the choices, over their sum + 1e-20 if renormalised, times `scale`; 0 for -1
// v is compared in 64 bits where it is computed (a bias, or a sum of two in groups): neighbours among some hundred scores lie
// so close that 32 bits choose another expert for one token in some ten thousand. Where v ranks as the logits do, their own
// 32 bits are compared. Not a number ranks above everything, as in torch.topk.
#include "route.cuh"

namespace b200ep {
namespace route {

// Orderable keys: larger is better, 0 is absent (-inf), the largest stands for not a number.
struct Key32 {
  using V = float;
  static __device__ __forceinline__ uint32_t of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.f);            // (-0 ranks as 0)
    const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return v == -INFINITY ? 0u : k;
  }
};
struct Key64 {
  using V = double;
  static __device__ __forceinline__ unsigned long long of(double v) {
    if (v != v) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
    const unsigned long long k = (u >> 63) ? ~u : (u | 0x8000000000000000ull);
    return v == -INFINITY ? 0ull : k;
  }
};

// The highest key of the warp.
__device__ __forceinline__ uint32_t warp_best(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ unsigned long long warp_best(unsigned long long k) {
  const uint32_t hi = (uint32_t)(k >> 32), top = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t lo = __reduce_max_sync(0xffffffffu, hi == top ? (uint32_t)k : 0u);
  return ((unsigned long long)top << 32) | lo;
}

// Groups that stay, one bit each. s_v: the warp's choice values [E] in shared memory. Lane g looks at group g.
template <typename V>
__device__ __forceinline__ uint32_t groups_kept(const V* s_v, int groups, int size, int keep, int best, int lane) {
  V a = -INFINITY, b = -INFINITY;                           // the two highest
  if (lane < groups) {
    for (int j = 0; j < size; ++j) {
      const V v = s_v[lane * size + j];
      if (v > a || v != v) { b = a; a = v; }
      else if (v > b) b = v;
    }
  }
  V mine = best == 2 && b > (V)-INFINITY ? a + b : a;
  if (a != a || b != b) mine = a + b;
  const bool none = mine != mine;
  int ahead = 0;
  for (int g = 0; g < groups; ++g) {
    const V o = __shfl_sync(0xffffffffu, mine, g);
    const bool o_none = o != o;
    const bool equal = o == mine || (o_none && none);
    ahead += (!none && (o_none || o > mine)) || (equal && g < lane);
  }
  return __ballot_sync(0xffffffffu, lane < groups && ahead < keep);
}

template <typename L, int VPL, typename KEY>
__global__ void __launch_bounds__(256)
route_kernel(const RouteParams p, int size_magic) {
  using V = typename KEY::V;
  using K = decltype(KEY::of(V(0)));
  extern __shared__ __align__(16) char s_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.E;
  const long long t = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  if (t >= p.T) return;
  const L* row = static_cast<const L*>(p.logits) + t * p.ld;
  float l[VPL];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    l[i] = i * 32 + lane < E ? logit(row + i * 32 + lane) : -INFINITY;
    top = nan_max(l[i], top);
  }
  const bool soft = p.score == SCORE_SOFTMAX;
  top = warp_max(top);
  if (soft) {
    if (top == -INFINITY) top = 0.f;                        // no expert is available: all scores are 0
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += expf(l[i] - top);
    sum = warp_sum(sum);
  }
  // the values that are compared
  K key[VPL];
  if constexpr (sizeof(V) == 8) {
    double total = 0.0;
    V v[VPL];
    if (soft) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) total += v[i] = exp((double)l[i] - (double)top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * 32 + lane;
      v[i] = soft ? v[i] / total : 1.0 / (1.0 + exp(-(double)l[i]));
      if (p.bias != nullptr && e < E) v[i] += (double)__ldg(p.bias + e);
      if (l[i] == -INFINITY) v[i] = -INFINITY;
      key[i] = KEY::of(v[i]);
    }
    if (p.groups > 1) {
      V* s_v = reinterpret_cast<V*>(s_raw) + (size_t)warp * E;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i * 32 + lane < E) s_v[i * 32 + lane] = v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = KEY::of(l[i]);
    if (p.groups > 1) {
      V* s_v = reinterpret_cast<V*>(s_raw) + (size_t)warp * E;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i * 32 + lane < E) s_v[i * 32 + lane] = l[i];
    }
  }
  if (p.groups > 1) {
    __syncwarp();
    const uint32_t kept = groups_kept(reinterpret_cast<const V*>(s_raw) + (size_t)warp * E, p.groups, E / p.groups, p.topk_groups, p.group_best, lane);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const uint32_t g = (uint32_t)(i * 32 + lane) * (uint32_t)size_magic >> 20;      // (i * 32 + lane) / size
      if (i * 32 + lane < E && !(kept >> g & 1)) key[i] = 0;
    }
  }
  float mine_l = 0.f;                                       // lane k: the logit of choice k
  int mine_e = -1;
  for (int k = 0; k < p.K; ++k) {
    K best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
    const K high = warp_best(best);
    if (high == 0) break;                                   // nothing is left
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == high ? (uint32_t)(at * 32 + lane) : 0xffffffffu);
    float le = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if ((int)e == i * 32 + lane) { le = l[i]; key[i] = 0; }
    le = __shfl_sync(0xffffffffu, le, e & 31);
    if (lane == k) { mine_l = le; mine_e = (int)e; }
  }
  float s = 0.f;
  if (mine_e >= 0) s = soft ? expf(mine_l - top) / sum : 1.f / (1.f + expf(-mine_l));
  const float chosen = warp_sum(s);
  if (lane < p.K) {
    p.idx[t * p.K + lane] = mine_e;
    p.w[t * p.K + lane] = mine_e < 0 ? 0.f : (p.renorm ? s / (chosen + kSumEps) : s) * p.scale;
    if (p.aux != nullptr && !soft) p.aux[t * p.K + lane] = mine_l;
  }
  if (p.aux != nullptr && soft && !p.renorm && lane < 2) p.aux[t * 2 + lane] = lane == 0 ? top : (sum > 0.f || sum != sum ? 1.f / sum : 0.f);
}

// Gradient of the logits, a warp per token. With g the weights' gradient times `scale`:
//   sigmoid:                d l_k = s_k (1 - s_k) h_k for the choices, 0 for the others; h = g, or renormalised
//                           h_k = (g_k - sum_j g_j s_j / S) / S with S = sum_j s_j + 1e-20
//   softmax, renormalised:  the weights are a softmax over the chosen logits: d l_k = u_k (g_k - sum_j u_j g_j), u = w / scale
//   softmax as it is:       d l_e = p_e ([e chosen] g_e - sum_j g_j p_j) for every expert
template <typename L>
__global__ void __launch_bounds__(256)
route_bwd_kernel(const RouteBwdParams p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = p.E;
  const long long t = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  if (t >= p.T) return;
  L* out = static_cast<L*>(p.dlogits) + t * E;
  int e = -1;
  float g = 0.f, d = 0.f;
  if (lane < p.K) {
    const long long i = p.idx[t * p.K + lane];
    e = i >= 0 && i < E ? (int)i : -1;
    if (e >= 0) g = p.gw[t * p.K + lane] * p.scale;
  }
  if (p.score == SCORE_SIGMOID) {
    float s = 0.f, rest = 0.f;                              // s and 1 - s, both without cancellation
    if (e >= 0) {
      const float l = p.aux[t * p.K + lane], q = expf(-fabsf(l)), r = 1.f / (1.f + q);
      s = l >= 0.f ? r : q * r;
      rest = l >= 0.f ? q * r : r;
    }
    float h = g;
    if (p.renorm) {
      const float total = warp_sum(s) + kSumEps;
      h = (g - warp_sum(g * s) / total) / total;
    }
    d = s * rest * h;
  } else {
    const float u = e >= 0 ? p.w[t * p.K + lane] / p.scale : 0.f;
    const float dot = warp_sum(u * g);
    d = u * (g - dot);
    if (!p.renorm) {
      const L* row = static_cast<const L*>(p.logits) + t * p.ld;
      const float top = p.aux[t * 2], inv = p.aux[t * 2 + 1];
      for (int j = lane; j < E; j += 32) put(out + j, expf(logit(row + j) - top) * inv * -dot);
      __syncwarp();
      if (e >= 0) put(out + e, d);
      return;
    }
  }
  for (int j = lane; j < E; j += 32) put(out + j, 0.f);
  __syncwarp();
  if (e >= 0) put(out + e, d);
}

template <typename L, int VPL, typename KEY>
int launch_sized(const RouteParams& p, cudaStream_t st) {
  const int warps = p.T < 1184 ? 1 : 8;
  const int size = p.E / p.groups;
  // e / size == e * magic >> 20 for e, size <= 1024: the error e * (magic * size - 2^20) stays below 2^20
  const int magic = ((1 << 20) + size - 1) / size;
  const size_t smem = p.groups > 1 ? (size_t)warps * p.E * sizeof(typename KEY::V) : 0;
  const auto kern = route_kernel<L, VPL, KEY>;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return 2;
  kern<<<(int)(((long long)p.T + warps - 1) / warps), warps * 32, smem, st>>>(p, magic);
  return 0;
}
template <typename L, typename KEY>
int launch_keyed(const RouteParams& p, cudaStream_t st) {
  if (p.E <= 64) return launch_sized<L, 2, KEY>(p, st);
  if (p.E <= 128) return launch_sized<L, 4, KEY>(p, st);
  if (p.E <= 256) return launch_sized<L, 8, KEY>(p, st);
  if (p.E <= 512) return launch_sized<L, 16, KEY>(p, st);
  return launch_sized<L, 32, KEY>(p, st);
}
template <typename L>
int launch_typed(const RouteParams& p, cudaStream_t st) {
  const bool computed = p.bias != nullptr || (p.groups > 1 && p.group_best == 2);
  return computed ? launch_keyed<L, Key64>(p, st) : launch_keyed<L, Key32>(p, st);
}

}  // namespace route

int launch_route(const RouteParams& p, cudaStream_t st) {
  if (p.T < 0 || p.E < 1 || p.E > kRouterMaxExperts || p.K < 1 || p.K > kRouteMaxTopk || p.K > p.E) return 1;
  if (p.groups < 1 || p.groups > kRouteMaxGroups || p.E % p.groups || p.topk_groups < 1 || p.topk_groups > p.groups) return 1;
  if (p.K > p.topk_groups * (p.E / p.groups) || p.group_best < 1 || p.group_best > 2 || !(p.scale > 0.f)) return 1;
  if (p.T == 0) return 0;
  if (p.type == ELEM_BF16) return route::launch_typed<__nv_bfloat16>(p, st);
  if (p.type == ELEM_F16) return route::launch_typed<__half>(p, st);
  return route::launch_typed<float>(p, st);
}

int launch_route_bwd(const RouteBwdParams& p, cudaStream_t st) {
  if (p.T < 0 || p.E < 1 || p.K < 1 || p.K > kRouteMaxTopk || !(p.scale > 0.f)) return 1;
  if (p.T == 0) return 0;
  const int grid = (int)(((long long)p.T + 7) / 8);
  if (p.type == ELEM_BF16) route::route_bwd_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  else if (p.type == ELEM_F16) route::route_bwd_kernel<__half><<<grid, 256, 0, st>>>(p);
  else route::route_bwd_kernel<float><<<grid, 256, 0, st>>>(p);
  return 0;
}

}  // namespace b200ep
