// Host launchers of the choice of experts and of the loss that balances it.
#pragma once
#include <cuda_runtime.h>
#include "../gemm/gemm_api.h"      // kRouterMaxExperts
#include "../norm/norm_api.h"      // ElemType

namespace b200ep {

enum RouteScore : int { SCORE_SOFTMAX = 0, SCORE_SIGMOID = 1 };

constexpr int kRouteMaxTopk = 32, kRouteMaxGroups = 32;

struct RouteParams {
  int type;                  // ElemType of the logits
  const void* logits;        // [T, E], rows ld elements apart
  long long ld;
  const float* bias;         // f32 [E] or null: added to the scores for the choice alone
  int T, E, K;
  int score;                 // RouteScore
  int groups, topk_groups;   // E is a multiple of groups; topk_groups * (E / groups) >= K
  int group_best;            // 1 or 2: of a group's choice values, how many are summed to its own
  bool renorm;
  float scale;               // > 0
  long long* idx;            // [T, K]
  float* w;                  // f32 [T, K]
  float* aux;                // for the backward, or null: sigmoid the chosen logits [T, K], softmax {maximum, 1 / sum, what
                             // the renormalised weights lack to a sum of 1} [T, 3]
};
int launch_route(const RouteParams& p, cudaStream_t st);

struct RouteBwdParams {
  int type;
  const void* logits;        // read by softmax only
  long long ld;
  int T, E, K, score;
  bool renorm;
  float scale;
  const long long* idx;
  const float* w;
  const float* aux;
  const float* gw;           // gradient of w
  void* dlogits;             // [T, E] contiguous
};
int launch_route_bwd(const RouteBwdParams& p, cudaStream_t st);

struct BalanceParams {
  int type;
  const void* logits;
  long long ld;
  const long long* idx;      // [T, K]
  const int* seq_off;        // device [B + 1] or null (one sequence of all rows)
  int T, E, K, B, score;
  float coeff, z_coeff;
  int* counts;               // scratch and state for the backward: [B * E] choices, [B] rows that take part, [1] arrivals
  double* part;              // [balance_ctas(p)]
  float* loss;               // [1]
};
// Words of `counts`, and CTAs of the loss's kernel.
long long balance_words(const BalanceParams& p);
int balance_ctas(const BalanceParams& p);
int launch_balance(const BalanceParams& p, cudaStream_t st);

struct BalanceBwdParams {
  BalanceParams f;           // as the forward had it (part and loss are not read)
  const float* dloss;        // [1]
  void* dlogits;             // [T, E] contiguous
};
int launch_balance_bwd(const BalanceBwdParams& p, cudaStream_t st);

}  // namespace b200ep
