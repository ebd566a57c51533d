"""Choice of experts from router logits, and the loss that keeps it balanced (csrc/route).

Logits are [T, E] in bf16, f16 or f32 with 1 to 1024 experts; everything is computed in f32 or more.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _ext

SCORES = ("softmax", "sigmoid")


def _score(name: str) -> int:
    if name == "softmax":
        return 0
    if name == "sigmoid":
        return 1
    raise ValueError(f"unsupported score {name!r}; expected one of {SCORES}")


def route(logits: torch.Tensor, topk: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, num_groups: int = 1,
          topk_groups: Optional[int] = None, group_best: int = 1, renormalize: bool = True,
          scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (expert ids int64 [T, topk], weights f32 [T, topk]), as `Buffer.get_dispatch_layout` and `dispatch` take them.

    s = softmax or sigmoid of the logits. The choice is by v = s + bias (bias [E], for balance: it does not enter the
    weights and has no gradient): of `num_groups` runs of E / num_groups neighbours those `topk_groups` (default: all) stay
    whose `group_best` (1 or 2) best v have the highest sum, and of their experts the topk with the highest v are chosen, in
    descending order; the lower index goes first among equals. v is compared as 64 bits have it, the logits themselves where
    neither a bias nor a sum of two has a part in the choice. Weights are the chosen s, over their sum + 1e-20 with `renormalize`, times `scale`.

    An expert whose logit or bias is -inf is not available: where fewer than topk are left, the index is -1 (no expert, to
    every call of this package) and the weight 0, for all choices of a padding row. NaN ranks above everything. topk and
    num_groups are at most 32. Differentiable once in the logits; no forward-mode derivatives, no function transforms, no tracing (refused)."""
    return _ext.load().route_experts(logits, topk, _score(score), bias, num_groups, num_groups if topk_groups is None else topk_groups,
                                     group_best, renormalize, scale)


def balance_loss(logits: torch.Tensor, idx: torch.Tensor, *, score: str = "softmax", coeff: float = 1.0, z_coeff: float = 0.0,
                 seq_off: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Scalar f32 loss of the choices idx (int64 [T, K]) that `route` made of these logits.

    Over the n tokens of a sequence that have a choice (an index between 0 and E - 1; padding has none):
    f_e = E / (K n) * choices of e,  p_t = s_t / (sum of s_t + 1e-20),
    coeff * sum_e f_e mean_t p_te + z_coeff * mean_t logsumexp(l_t)^2 (softmax scores only),
    and the mean of that over the sequences that have such tokens; 0 where none has. seq_off (int32 [B + 1], ascending, on
    the logits' device) cuts the rows into B packed sequences; rows outside take no part. Default: one sequence of all rows.
    Differentiable once in the logits (f is a count); rows that take no part get a gradient of 0. No forward-mode
    derivatives, no function transforms, no tracing (refused)."""
    return _ext.load().balance_loss(logits, idx, seq_off, _score(score), coeff, z_coeff)
