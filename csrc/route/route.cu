// Choice of experts. For a token's logits l [E]:
//   s = softmax(l) or sigmoid(l);  v = s + bias (-inf where l is: that expert is not available)
//   groups: of the E experts in `groups` runs, those in the `topk_groups` runs with the highest values stay, a run's value
//           being the sum of its 1 or 2 best v (of those above -inf)
//   choice: the K highest v, in descending order, the lower index first among equals; -1 where nothing above -inf is left
//   w = s (without the bias) of the choices, over their sum + 1e-20 if renormalised, times `scale`; 0 for -1
// v is compared in 64 bits where it is computed (a bias, or a sum of two in groups): neighbours among some hundred scores lie
// so close that 32 bits choose another expert for one token in some ten thousand. Where v ranks as the logits do, their own
// 32 bits are compared. Not a number ranks above everything, as in torch.topk.
// A warp has a token: its lanes hold runs of neighbouring experts of one group, so that a group's best are found inside a
// lane and a few shuffles. Bound: instructions, about 790 a token of 256 experts in 8 groups (16383 of them, top-8, sigmoid
// with a bias: 18.4 to 20.5 us on one B200, 70 % of the issue slots, 76 bytes a thread spilled across the calls of the ways of looking
// again; every value in 64 bits: 55.5), for few tokens latency (128: 3.6, or 6.7 with a token that needs 64 bits). The logits
// are read once.
#include <atomic>
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
  // The value of a key, not a number for the largest ones; -inf for 0.
  static __device__ __forceinline__ float value(uint32_t k) {
    if (k == 0u) return -INFINITY;
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
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

// How many groups go before this lane's: higher values (not a number above all), the lower index among equals.
template <typename V>
__device__ __forceinline__ int groups_ahead(V mine, int groups, int lane) {
  const bool none = mine != mine;
  int ahead = 0;
  for (int g = 0; g < groups; ++g) {
    const V o = __shfl_sync(0xffffffffu, mine, g);
    const bool o_none = o != o;
    const bool equal = o == mine || (o_none && none);
    ahead += (!none && (o_none || o > mine)) || (equal && g < lane);
  }
  return ahead;
}

// How the experts lie over the lanes: `lanes` neighbouring lanes (a power of two) have a group, each a run of `chunk` of its
// experts, so that a lane's values are all of one group and rise in index from lane to lane. Without groups, or where all
// of them stay, the experts are one group.
struct Groups {
  int count, size;           // groups that are told apart, experts of each
  int lanes, chunk;
  uint32_t mask;             // of the bits that tell groups apart
  bool vec;                  // every lane's run is whole and its loads of 4 values are aligned
  // choose_exactly's: the groups again (for 17 to 31 groups of more than 32, which leave a lane too many values, they are
  // told apart there alone, for every token), and e / size == e * magic >> 20 for e, size <= 1024: the error
  // e * (magic * size - 2^20) stays below 2^20
  bool exact;
  int told, magic;
};
__device__ __forceinline__ int group_of(const Groups& g, int e) { return (int)((uint32_t)e * (uint32_t)g.magic >> 20); }

// ---- the choice as it is defined: every value compared, in 64 bits where they are computed -------------------------------
// Lane k's choice, -1 for none. Called where the quick way below cannot tell neighbours apart, for few tokens.
template <typename L, int VPL, typename KEY>
__device__ __noinline__ int choose_exactly(const RouteParams& p, const L* row, const Groups& gr) {
  using V = typename KEY::V;
  using K = decltype(KEY::of(V(0)));
  const int lane = threadIdx.x & 31, E = p.E;
  K key[VPL];
  V v[VPL];
  if constexpr (sizeof(V) == 8) {
    V top = -INFINITY, total = 0.0;
    const bool soft = p.score == SCORE_SOFTMAX;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] = i * 32 + lane < E ? (V)logit(row + i * 32 + lane) : (V)-INFINITY;
      top = v[i] > top || v[i] != v[i] ? v[i] : top;
    }
    if (soft) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const V w = __shfl_xor_sync(0xffffffffu, top, o);
        top = w > top || w != w ? w : top;
      }
      if (top == -INFINITY) top = 0.0;
#pragma unroll
      for (int i = 0; i < VPL; ++i) total += exp(v[i] - top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = i * 32 + lane;
      const bool absent = v[i] == -INFINITY;
      v[i] = soft ? exp(v[i] - top) / total : 1.0 / (1.0 + exp(-v[i]));
      if (p.bias != nullptr && e < E) v[i] += (V)p.bias[e];
      if (absent) v[i] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = i * 32 + lane < E ? logit(row + i * 32 + lane) : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) key[i] = KEY::of(v[i]);
  if (gr.told > 1) {
    // group after group: the lanes' two highest, then the warp's (a sum of two is the same whichever way it is found)
    V mine = -INFINITY;                                     // lane g: the value of group g
    for (int g = 0; g < gr.told; ++g) {
      V a = -INFINITY, b = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        if (group_of(gr, i * 32 + lane) != g || i * 32 + lane >= E) continue;
        if (v[i] > a || v[i] != v[i]) { b = a; a = v[i]; }
        else if (v[i] > b) b = v[i];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const V c = __shfl_xor_sync(0xffffffffu, a, o), d = __shfl_xor_sync(0xffffffffu, b, o);
        const V low = a != a || c != c ? c + a : (c > a ? a : c);        // (not a number stays in the sum)
        a = a != a || c != c ? c + a : (c > a ? c : a);
        b = b > d ? b : d;
        b = low > b || low != low ? low : b;
      }
      const V value = a != a ? a : (p.group_best == 2 && b > (V)-INFINITY ? a + b : a);
      if (lane == g) mine = value;
    }
    const int ahead = groups_ahead(mine, gr.told, lane);
    const uint32_t kept = __ballot_sync(0xffffffffu, lane < gr.told && ahead < p.topk_groups);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (!(kept >> (group_of(gr, i * 32 + lane) & 31) & 1)) key[i] = 0;
  }
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
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if ((int)e == i * 32 + lane) key[i] = 0;
    if (lane == k) mine_e = (int)e;
  }
  return mine_e;
}

// ---- the quick way -------------------------------------------------------------------------------------------------------
// Keys of 32 bits whose low bits say which of the lane's values they are, sorted in each lane, so that a choice is one warp
// maximum of the lanes' first keys. How far a key's value may be from the one it stands for is known; where neighbours
// among the choices, and the values after the last one, lie closer than that, they are compared again as they are defined
// (settle: one lane each), so are groups that close to the last one that stays (settle_groups). More than 32 such values
// are left to choose_exactly. 256 sigmoid scores with a bias: about one token in 500 is settled, one in 4000 for its groups.
//   kLogit16: 16-bit logits rank by themselves; the low half of a key is the expert, the lowest highest: always told apart
//   kLogit32: 32-bit logits rank by themselves, but for the low bits that the place in the lane takes
//   kSigmoid, kSoftmax: computed values, scores and a bias in 32 bits, also but for those low bits
enum Mode : int { kLogit16 = 0, kLogit32 = 1, kSigmoid = 2, kSoftmax = 3 };
constexpr bool computed(int mode) { return mode >= kSigmoid; }

// A float's bits in the order of its values (-0 just below 0). Keys up to kAbsent, that of -inf, stand for nothing.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
constexpr uint32_t kAbsent = 0x007fffffu;

template <int N> constexpr int kLog2 = 1 + kLog2<(N + 1) / 2>;
template <> constexpr int kLog2<1> = 0;

// Descending, by Batcher's odd-even merges.
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
}

// 1 / y, off by little more than half a unit in the last place: the hardware's approximation and one step of Newton's
// iteration; without the branches of a division. It has no denormals: 0 for y above 2^126, that is for a sigmoid of a logit
// below -87.3, which is less than the smallest normal number (1.2e-38).
__device__ __forceinline__ float reciprocal(float y) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return y < INFINITY ? fmaf(r, fmaf(-y, r, 1.f), r) : r;
}
// 1 / (1 + exp(-x)) from the hardware's approximations: off by less than 2^-21.
__device__ __forceinline__ float quick_sigmoid(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return r;
}

// The values that are compared, as they are defined: of 64 bits where they are computed.
template <int MODE>
struct Defined {
  using V = typename std::conditional<computed(MODE), double, float>::type;
  using KEY = typename std::conditional<computed(MODE), Key64, Key32>::type;
  V top = 0, total = 0;
  // by the whole warp
  template <typename L>
  __device__ __forceinline__ void row(const RouteParams& p, const L* row) {
    if (MODE != kSoftmax) return;
    const int lane = threadIdx.x & 31;
    top = -INFINITY;
    for (int j = lane; j < p.E; j += 32) {
      const V l = (V)logit(row + j);
      top = l > top || l != l ? l : top;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const V w = __shfl_xor_sync(0xffffffffu, top, o);
      top = w > top || w != w ? w : top;
    }
    for (int j = lane; j < p.E; j += 32) total += exp((V)logit(row + j) - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  template <typename L>
  __device__ __forceinline__ V of(const RouteParams& p, const L* row, int e) const {
    V v = (V)logit(row + e);
    if constexpr (computed(MODE)) {
      if (v == (V)-INFINITY) return v;
      v = MODE == kSoftmax ? exp(v - top) / total : 1.0 / (1.0 + exp(-v));
      if (p.bias != nullptr) v += (V)p.bias[e];
    }
    return v;
  }
};

// The n candidates, one a lane (e), in their defined order: the expert of lane k's choice.
template <typename L, int MODE>
__device__ __noinline__ int settle(const RouteParams& p, const L* row, int e, int n) {
  Defined<MODE> d;
  d.row(p, row);
  const int lane = threadIdx.x & 31;
  const auto key = Defined<MODE>::KEY::of(lane < n ? d.of(p, row, e) : 0);
  int ahead = 0;
  for (int j = 0; j < n; ++j) {
    const auto o = __shfl_sync(0xffffffffu, key, j);
    const int oe = __shfl_sync(0xffffffffu, e, j);
    ahead += o > key || (o == key && oe < e);
  }
  int mine = -1;
  for (int j = 0; j < n; ++j) {
    const int oe = __shfl_sync(0xffffffffu, e, j), place = __shfl_sync(0xffffffffu, ahead, j);
    if (place == lane) mine = oe;
  }
  return mine;
}

// Of the groups in `among`, one bit each, those `keep` that have the highest values as they are defined.
template <typename L, int MODE>
__device__ __noinline__ uint32_t settle_groups(const RouteParams& p, const L* row, int size, uint32_t among, int keep) {
  using V = typename Defined<MODE>::V;
  Defined<MODE> d;
  d.row(p, row);
  const int lane = threadIdx.x & 31;
  V mine = -INFINITY;                                       // lane g: the value of group g
  for (uint32_t left = among; left != 0u; left &= left - 1) {
    const int g = __ffs(left) - 1;
    V a = -INFINITY, b = -INFINITY;                         // the two highest; not a number above all
    for (int j = lane; j < size; j += 32) {
      const V v = d.of(p, row, g * size + j);
      if (v > a || v != v) { b = a; a = v; }
      else if (v > b) b = v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const V c = __shfl_xor_sync(0xffffffffu, a, o), f = __shfl_xor_sync(0xffffffffu, b, o);
      const bool none = a != a || c != c;
      const V low = c > a ? a : c;
      a = none ? a + c : (c > a ? c : a);
      b = b > f ? b : f;
      b = !none && low > b ? low : b;
    }
    if (lane == g) mine = a != a ? a : (p.group_best == 2 && b > (V)-INFINITY ? a + b : a);
  }
  const bool in = among >> lane & 1;
  int ahead = 0;
  for (uint32_t left = among; left != 0u; left &= left - 1) {
    const int g = __ffs(left) - 1;
    const V o = __shfl_sync(0xffffffffu, mine, g);
    ahead += (mine == mine && (o != o || o > mine)) || ((o == mine || (o != o && mine != mine)) && g < lane);
  }
  return __ballot_sync(0xffffffffu, in && ahead < keep);
}

// The 16 bits of a 16-bit logit in the order of its values, in the upper half.
__device__ __forceinline__ uint32_t order16(float v, const __nv_bfloat16*) { return order_of(v) & 0xffff0000u; }
__device__ __forceinline__ uint32_t order16(float v, const __half*) {
  if (v == -INFINITY) return 0u;
  const uint32_t u = (uint32_t)__half_as_ushort(__float2half_rn(v)) << 16;
  return (u ^ ((uint32_t)((int)u >> 31) | 0x80000000u)) & 0xffff0000u;
}

template <typename L> struct Four;           // four logits in one load
template <> struct Four<float> {
  static __device__ __forceinline__ void get(const float* p, float* f) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  }
};
template <> struct Four<__nv_bfloat16> {
  static __device__ __forceinline__ void get(const __nv_bfloat16* p, float* f) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
  }
};
template <> struct Four<__half> {
  static __device__ __forceinline__ void get(const __half* p, float* f) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  }
};

// A lane's experts where a warp has a token.
template <int VPL>
struct Share {
  int group, e0, n;          // its group, first expert, and how many it has
  float bias[VPL], most_bias;
  __device__ __forceinline__ Share(const RouteParams& p, const Groups& gr, bool computed) {
    const int lane = threadIdx.x & 31, sub = lane & (gr.lanes - 1);
    group = lane / gr.lanes;
    e0 = group * gr.size + sub * gr.chunk;
    n = group < gr.count ? max(0, min(gr.chunk, gr.size - sub * gr.chunk)) : 0;
    most_bias = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      bias[i] = computed && p.bias != nullptr && i < n ? p.bias[e0 + i] : 0.f;
      if (fabsf(bias[i]) < INFINITY) most_bias = fmaxf(most_bias, fabsf(bias[i]));
    }
    if (computed) most_bias = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most_bias)));
  }
};

// One token by one warp: the expert of lane k's choice, -1 for none (lanes from K on hold anything). With softmax also the
// largest logit and the sum of the exponentials of the distances to it.
template <typename L, int VPL, int MODE>
__device__ __forceinline__ int choose(const RouteParams& p, const Groups& gr, const Share<VPL>& mine, const L* row, float& top, float& sum) {
  const int lane = threadIdx.x & 31, group = mine.group;
  const bool soft = MODE == kSoftmax || (!computed(MODE) && p.score == SCORE_SOFTMAX);
  constexpr int LOW = MODE == kLogit16 ? 0 : kLog2<VPL>;    // bits of a key that say where it came from
  constexpr uint32_t MASK = (1u << LOW) - 1;
  float l[VPL];
  bool loaded = false;
  if constexpr (VPL % 4 == 0) {
    if (gr.vec) {
#pragma unroll
      for (int i = 0; i < VPL; i += 4) {
        l[i] = l[i + 1] = l[i + 2] = l[i + 3] = -INFINITY;
        if (i < mine.n) Four<L>::get(row + mine.e0 + i, l + i);
      }
      loaded = true;
    }
  }
  if (!loaded) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) l[i] = i < mine.n ? logit(row + mine.e0 + i) : -INFINITY;
  }
  if (soft) {
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = nan_max(l[i], top);
    top = warp_max(top);
    if (top == -INFINITY) top = 0.f;                      // no expert is available: all scores are 0
  }
  uint32_t key[VPL];
  float margin = 0.f;                                     // how far a key's value may be from the one it stands for
  bool odd = false;                                       // not a number among logits that are compared as they are
  if constexpr (computed(MODE)) {
    float s[VPL], unit = 1.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) s[i] = MODE == kSoftmax ? __expf(l[i] - top) : quick_sigmoid(l[i]);
    if constexpr (MODE == kSoftmax) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum += s[i];
      sum = warp_sum(sum);
      unit = reciprocal(sum);
    }
    // A sigmoid is off by 2^-21 of at most 1. A softmax score p has its exponential off by 2 units in the last place and, for
    // the distance d to the maximum, by 2 d 2^-24 of itself, which p = e^-d / sum makes less than 2^-24 of the largest, 1 / sum;
    // and a sum of VPL + 5 roundings and those of its terms: 2^-18 of the largest covers all. The sum with the bias is
    // rounded once, its key has LOW bits of its own.
    margin = (MODE == kSoftmax ? 0x1p-18f * unit : 0x1p-21f) + (float)(1 + (1 << LOW)) * 0x1p-23f * (unit + mine.most_bias);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float c = l[i] == -INFINITY ? -INFINITY : fmaf(s[i], unit, mine.bias[i]);
      key[i] = (order_of(c) & ~MASK) | (uint32_t)(VPL - 1 - i);        // (a sum that is not a number has the highest)
    }
  } else {
    if (soft) {
      // (the approximate exponential is off by 2 + 1.2 d units in the last place at a distance d to the maximum, where a term is e^-d:
      // the sum of up to 1024, and so every weight that is not renormalised, by less than 8 units, 2^-20 of itself)
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum += __expf(l[i] - top);
      sum = warp_sum(sum);
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      odd = odd || l[i] != l[i];
      if constexpr (MODE == kLogit16) {
        key[i] = order16(l[i] + 0.f, row);
        key[i] |= key[i] > kAbsent ? (uint32_t)(0xffff - (mine.e0 + i)) : 0u;
      } else {
        key[i] = (order_of(l[i]) & ~MASK) | (uint32_t)(VPL - 1 - i);
      }
    }
  }
  sort_keys(key);
  bool exact = gr.exact || (!computed(MODE) && __any_sync(0xffffffffu, odd));
  if (gr.count > 1) {
    // the group's two highest, in all of its lanes
    uint32_t a = key[0], b = key[1];
    for (int o = gr.lanes >> 1; o > 0; o >>= 1) {
      const uint32_t c = __shfl_xor_sync(0xffffffffu, a, o), d = __shfl_xor_sync(0xffffffffu, b, o);
      b = max(min(a, c), max(b, d));
      a = max(a, c);
    }
    // its value as a key that is its own: the low bits say which group (a logit of 16 bits has them already), lowest first
    if (computed(MODE) && p.group_best == 2 && b > kAbsent) a = order_of(Key32::value(a) + Key32::value(b));
    if (MODE != kLogit16 && a > kAbsent) a = (a & ~gr.mask) | (gr.mask - (uint32_t)group);
    uint32_t left = a, last = 0u;
    for (int k = 0; k < p.topk_groups; ++k) {
      last = __reduce_max_sync(0xffffffffu, left);
      if (left == last) left = 0u;
    }
    bool kept = left == 0u;
    if constexpr (MODE != kLogit16) {
      // (two values of either side, their sums' rounding and the keys' own bits; -0 and 0 lie within a step of 2^-149)
      const uint32_t next = __reduce_max_sync(0xffffffffu, left);
      const uint32_t low = gr.mask | MASK;
      const float about = computed(MODE) ? 4.f * margin + (float)(2 + 2 * low) * 0x1p-23f * fabsf(Key32::value(last)) : 0.f;
      const bool close = next > kAbsent && (MODE == kLogit32 ? (last & ~low) == (next & ~low) || (next >= (0x7fffffffu & ~low) && last <= (0x80000000u | low))
                                                            : !(Key32::value(last) - Key32::value(next) > about));
      if (close && !exact) {
        // those near the last one that stays are looked at again, the others are in or out
        bool in, near;
        if (MODE == kLogit32) {
          const uint32_t zero = 0x80000000u & ~low, at = (last & ~low) == (0x7fffffffu & ~low) ? zero : last & ~low;
          const uint32_t me = (a & ~low) == (0x7fffffffu & ~low) ? zero : a & ~low;
          near = a > kAbsent && me == at;
          in = a > kAbsent && me > at;
        } else {
          const float off = Key32::value(a) - Key32::value(last);
          near = a > kAbsent && !(fabsf(off) > about);
          in = a > kAbsent && off > about;
        }
        const uint32_t first = __ballot_sync(0xffffffffu, (lane & (gr.lanes - 1)) == 0 && group < gr.count);
        const uint32_t in_lanes = __ballot_sync(0xffffffffu, in) & first, near_lanes = __ballot_sync(0xffffffffu, near) & first;
        uint32_t among = 0u;
        for (uint32_t m = near_lanes; m != 0u; m &= m - 1) among |= 1u << ((__ffs(m) - 1) / gr.lanes);
        const uint32_t stay = settle_groups<L, MODE>(p, row, gr.size, among, p.topk_groups - __popc(in_lanes));
        kept = in || (near && (stay >> group & 1));
      }
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = kept ? key[i] : 0u;
  }
  // The lane whose first key is the highest leaves it, and the expert, in the choice's place. Two lanes with the same key
  // leave theirs in one: the count says so.
  __shared__ uint2 s_pick[8][32];
  uint2* const picks = s_pick[threadIdx.x >> 5];
  uint32_t high = 0u;
  int n = 0, given = 0;
  const auto give = [&] {
    if (key[0] == high) {
      picks[n] = make_uint2(key[0], MODE == kLogit16 ? 0xffffu - (key[0] & 0xffffu) : (uint32_t)(mine.e0 + VPL - 1) - (key[0] & MASK));
      ++given;
#pragma unroll
      for (int i = 0; i + 1 < VPL; ++i) key[i] = key[i + 1];
      key[VPL - 1] = 0u;
    }
  };
  __syncwarp();
#pragma unroll 1
  for (; n < p.K; ++n) {
    high = __reduce_max_sync(0xffffffffu, key[0]);
    if (high <= kAbsent) break;
    give();
  }
  __syncwarp();
  uint2 pick = picks[lane];
  int e = lane < n ? (int)pick.y : -1;
  if constexpr (MODE != kLogit16) {
    // whether two values, the first with the higher key, are in this order for certain
    const auto apart = [&](uint32_t high, uint32_t low) {
      if (low <= kAbsent) return true;
      if (MODE == kLogit32) return (high & ~MASK) > (low & ~MASK) && !(low >= (0x7fffffffu & ~MASK) && high <= (0x80000000u | MASK));      // (-0 is 0)
      return Key32::value(high) - Key32::value(low) > 2.f * margin;
    };
    uint32_t next = n == p.K ? __reduce_max_sync(0xffffffffu, key[0]) : 0u;
    const uint32_t follows = __shfl_down_sync(0xffffffffu, pick.x, 1), after = lane + 1 < n ? follows : next;
    const bool doubt = lane < n && !apart(pick.x, after);
    const int total = __reduce_add_sync(0xffffffffu, given);
    if (total != n) exact = true;
    if (__any_sync(0xffffffffu, doubt) && !exact) {
      // behind the last choice, the values that may change places with it
      while (n < 32 && !apart(high, next)) {
        high = next;
        give();
        ++n;
        next = __reduce_max_sync(0xffffffffu, key[0]);
      }
      __syncwarp();
      pick = picks[lane];
      if (!apart(high, next) || (int)__reduce_add_sync(0xffffffffu, given) != n) exact = true;       // (32 of them and more)
      else e = settle<L, MODE>(p, row, (int)pick.y, n);
    }
  }
  if (exact) e = choose_exactly<L, VPL, typename Defined<MODE>::KEY>(p, row, gr);
  return e;
}

// Weights of a token's choices, lane k's of choice k: e < 0 for none.
template <typename L, int MODE>
__device__ __forceinline__ void store_choice(const RouteParams& p, const L* row, long long t, int k, int e, float top, float sum) {
  const bool soft = MODE == kSoftmax || (!computed(MODE) && p.score == SCORE_SOFTMAX);
  float l = 0.f, s = 0.f;
  if (e >= 0) {
    l = logit(row + e);
    s = soft ? expf(l - top) * reciprocal(sum) : reciprocal(1.f + expf(-l));
  }
  float chosen = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) chosen += __shfl_xor_sync(0xffffffffu, chosen, o);
  if (k < p.K) {
    p.idx[t * p.K + k] = e;
    p.w[t * p.K + k] = e < 0 ? 0.f : (p.renorm ? s * reciprocal(chosen + kSumEps) : s) * p.scale;
    if (p.aux != nullptr && !soft) p.aux[t * p.K + k] = l;
  }
  if (p.aux != nullptr && soft && k < 3)
    p.aux[t * 3 + k] = k == 0 ? top : k == 1 ? (sum == 0.f ? 0.f : reciprocal(sum)) : kSumEps * reciprocal(chosen + kSumEps);
}

template <typename L, int VPL, int MODE>
__global__ void __launch_bounds__(256, VPL <= 8 ? 4 : 2)
route_kernel(const __grid_constant__ RouteParams p, const __grid_constant__ Groups gr) {
  stream_order_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const Share<VPL> mine(p, gr, computed(MODE));
  for (long long t = (long long)blockIdx.x * warps + warp; t < p.T; t += (long long)gridDim.x * warps) {
    const L* row = static_cast<const L*>(p.logits) + t * p.ld;
    float top = 0.f, sum = 0.f;
    int e = choose<L, VPL, MODE>(p, gr, mine, row, top, sum);
    if (lane >= p.K) e = -1;
    store_choice<L, MODE>(p, row, t, lane, e, top, sum);
  }
}

// Gradient of the logits, a warp per token. With g the weights' gradient times `scale`:
//   sigmoid:                d l_k = s_k (1 - s_k) h_k for the choices, 0 for the others; h = g, or renormalised
//                           h_k = (g_k - sum_j g_j s_j / S) / S with S = sum_j s_j + 1e-20
//   softmax as it is:       d l_e = p_e ([e chosen] g_e - sum_j g_j p_j) for every expert
//   softmax, renormalised:  with u = w / scale, D = sum_j u_j g_j and r = 1e-20 / S, which is 1 - sum_j u_j,
//                           d l_e = [e chosen] u_e (g_e - D) - p_e r D for every expert
// r is kept by the forward: 1 less the sum of the u would be their roundings. It is next to nothing (the weights are a softmax over
// the chosen logits) unless an expert that a bias or its group keeps out of the choice lies far above those in it: from 46
// on, r is a half or more. g_e - D is taken as (g_e sum_j u_j - D) + r g_e, whose first part is 0 where there is one choice.
// Bound: memory, the zeros written to [T, E] above all; the logits are read again by softmax as it is, and for rows whose r
// tells. 16384 x 256 in f32: 6.3 us (2.7 TB/s).
constexpr float kLackTells = 0x1p-40f;   // r below this (S above 1.1e-8) changes no gradient by more than 2^-40 of the g
template <typename L>
__global__ void __launch_bounds__(256)
route_bwd_kernel(const RouteBwdParams p) {
  stream_order_wait();
  stream_order_next();
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
    float rest = dot;                                       // what every expert's gradient has, times -p_e
    d = u * (g - dot);
    if (p.renorm) {
      const float lack = p.aux[t * 3 + 2];
      const bool tells = lack > kLackTells;
      rest = tells ? lack * dot : 0.f;
      d = u * ((__fmul_rn(g, warp_sum(u)) - dot) + (tells ? lack * g : 0.f));
    }
    if (rest != 0.f) {
      const L* row = static_cast<const L*>(p.logits) + t * p.ld;
      const float top = p.aux[t * 3], inv = p.aux[t * 3 + 1];
      for (int j = lane; j < E; j += 32) put(out + j, expf(logit(row + j) - top) * inv * -rest);
      __syncwarp();
      if (e >= 0) put(out + e, p.renorm ? fmaf(expf(logit(row + e) - top) * inv, -rest, d) : d);
      return;
    }
  }
  for (int j = lane; j < E; j += 32) put(out + j, 0.f);
  __syncwarp();
  if (e >= 0) put(out + e, d);
}

template <typename L, int VPL, int MODE>
int launch_sized(const RouteParams& p, const Groups& g, cudaStream_t st) {
  // Fewer tokens than 8 for each of 148 SMs: a CTA of its own for each, so that one that is settled or compared exactly keeps no
  // other's SM busy. us with one warp a CTA and with eight: 256 sigmoid scores with a bias in 8 groups 3.61 and 4.04 for 300
  // tokens, 5.02 and 4.98 for 1183, 7.45 and 7.99 for 4096; 64 softmax scores by their logits, where little is ever looked at
  // again, 2.94 and 2.88, 3.24 and 2.96, 4.95 and 3.92.
  const int warps = p.T < 1184 ? 1 : 8;
  const auto kern = route_kernel<L, VPL, MODE>;
  static std::atomic<int> fits[2];                          // CTAs per SM with 1 and with 8 warps; 0: not asked yet
  int fit = fits[warps > 1].load(std::memory_order_relaxed);
  if (fit == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, warps * 32, 0) != cudaSuccess || fit < 1) return 2;
    fits[warps > 1].store(fit, std::memory_order_relaxed);
  }
  const long long need = ((long long)p.T + warps - 1) / warps, most = (long long)fit * sm_count();
  return launch_ordered(kern, dim3((unsigned)(need < most ? need : most)), dim3(warps * 32), 0, st, 1, p, g) == cudaSuccess ? 0 : 2;
}
// The groups of a choice over a warp's lanes.
template <typename L>
Groups lay_groups(const RouteParams& p, bool told_apart) {
  Groups g{};
  g.told = p.topk_groups < p.groups ? p.groups : 1;
  g.count = told_apart ? g.told : 1;
  g.size = p.E / g.count;
  const int told_size = p.E / g.told;
  g.magic = ((1 << 20) + told_size - 1) / told_size;
  g.lanes = 32;
  while (g.lanes * g.count > 32) g.lanes >>= 1;
  g.chunk = (g.size + g.lanes - 1) / g.lanes;
  g.mask = 0u;
  while ((int)g.mask + 1 < g.count) g.mask = 2 * g.mask + 1;
  g.vec = g.chunk % 4 == 0 && g.size % g.chunk == 0 && p.ld % 4 == 0 && reinterpret_cast<uintptr_t>(p.logits) % (4 * sizeof(L)) == 0;
  return g;
}

template <typename L, int MODE>
int launch_mode(const RouteParams& p, cudaStream_t st) {
  Groups g = lay_groups<L>(p, true);
  // (4096 x 1020 in 17 groups 245 us, 4096 x 1024 in 16 groups, which have a quick way, 44)
  if (g.chunk > 32) {
    g = lay_groups<L>(p, false);
    g.exact = true;
  }
  if (g.chunk <= 2) return launch_sized<L, 2, MODE>(p, g, st);
  if (g.chunk <= 4) return launch_sized<L, 4, MODE>(p, g, st);
  if (g.chunk <= 8) return launch_sized<L, 8, MODE>(p, g, st);
  if (g.chunk <= 16) return launch_sized<L, 16, MODE>(p, g, st);
  return launch_sized<L, 32, MODE>(p, g, st);
}
template <typename L>
int launch_typed(const RouteParams& p, cudaStream_t st) {
  if (p.bias != nullptr || (p.topk_groups < p.groups && p.group_best == 2))
    return p.score == SCORE_SOFTMAX ? launch_mode<L, kSoftmax>(p, st) : launch_mode<L, kSigmoid>(p, st);
  return launch_mode<L, sizeof(L) == 2 ? kLogit16 : kLogit32>(p, st);
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
  const auto kern = p.type == ELEM_BF16 ? route::route_bwd_kernel<__nv_bfloat16> : p.type == ELEM_F16 ? route::route_bwd_kernel<__half> : route::route_bwd_kernel<float>;
  return launch_ordered(kern, dim3(grid), dim3(256), 0, st, 1, p) == cudaSuccess ? 0 : 2;
}

}  // namespace b200ep
