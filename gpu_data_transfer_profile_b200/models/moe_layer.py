"""A Megatron-style MoE layer: router -> dispatch -> grouped experts -> combine.

The reference's "model" is exactly this loop with a random router stand-in
(`DeepEP_Megatron/test_deepep_moe_dispatch_combine.py:731-742,766-815`); here it is an
`nn.Module` with a learnable router so that forward AND backward run (dispatch and combine
are each other's backward, expert GEMMs have dgrad/wgrad). Optional, off by default: the norm in front of it with the
residual's addition (`ops.norm`), the choice of experts by other scores, with a bias and in groups, and the loss that
keeps it balanced (`ops.router`).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from .. import _ext
from ..ops import norm as N
from ..ops import router as R
from .experts import build_experts
from .experts_tcgen05 import Tcgen05GroupedExperts
from .token_dispatcher import B200TokenDispatcher


def topk_softmax_router(logits: torch.Tensor, topk: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """(indices int64 [T,K], probabilities f32 [T,K] renormalised over the chosen experts)."""
    probs = torch.softmax(logits.float(), dim=-1)
    w, idx = torch.topk(probs, topk, dim=-1)
    return idx, w / w.sum(-1, keepdim=True)


class _TopkSoftmax(torch.autograd.Function):
    """`topk_softmax_router` on this library's kernels, one launch forward and one backward (f32 like the torch form)."""

    @staticmethod
    def forward(ctx, logits, topk):
        idx, w = _ext.load().topk_softmax(logits, topk)
        ctx.num_experts = logits.shape[1]
        ctx.save_for_backward(idx, w)
        ctx.mark_non_differentiable(idx)
        return idx, w

    @staticmethod
    def backward(ctx, _grad_idx, grad_w):
        idx, w = ctx.saved_tensors
        if torch.is_grad_enabled() or _carries_more(grad_w):          # a graph, a tangent or a batch of gradients is asked for
            d = w * (grad_w - (w * grad_w).sum(-1, keepdim=True))
            return torch.zeros((w.shape[0], ctx.num_experts), dtype=w.dtype, device=w.device).scatter(1, idx, d), None
        return _ext.load().topk_softmax_bwd(idx, w, grad_w.float().contiguous(), ctx.num_experts), None


_LINEAR_FORWARD = torch.nn.Linear.forward
# a program that puts a router of its own in its place has it called
_OWN_ROUTER = topk_softmax_router


def _plain_linear(m: torch.nn.Module) -> bool:
    """Calling `m` does nothing but x @ weight.T in f32: the fused router may stand in for it. (Libraries that wrap
    modules put a `forward` of their own on the instance or the class.)"""
    return (type(m) is torch.nn.Linear and m.bias is None and type(m.weight) is torch.nn.Parameter
            and "forward" not in vars(m) and torch.nn.Linear.forward is _LINEAR_FORWARD
            and m.weight.dtype == torch.float32 and m.weight.is_contiguous() and m.weight.data_ptr() % 16 == 0
            and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)
            and not (torch.nn.modules.module._global_forward_hooks or torch.nn.modules.module._global_forward_pre_hooks)
            and not torch.is_autocast_enabled("cuda"))


# What `MoELayer`'s inference path stands in for or hands views and device-side counts to. Where a program subclasses,
# wraps or replaces one of these, its own version is called as the general path calls it.
_OWN_DISPATCHER = {n: vars(B200TokenDispatcher)[n] for n in ("dispatch", "dispatch_fp8", "dispatch_in_place")}
_OWN_EXPERTS = {n: vars(Tcgen05GroupedExperts)[n] for n in ("forward_fused_combine", "forward_fp8")}


def _unchanged(obj, methods) -> bool:
    return all(n not in getattr(obj, "__dict__", ()) and getattr(type(obj), n, None) is f for n, f in methods.items())


def _carries_more(t: Optional[torch.Tensor]) -> bool:
    """A tensor with a forward-mode tangent or inside a function transform (a batch of gradients is one, in a form of its
    own): kernels, which know nothing of either, would drop what it carries without a word or fail on it; the autograd
    functions of the general path refuse it."""
    F = torch._C._functorch
    return t is not None and (F.is_functorch_wrapped_tensor(t) or F.is_legacy_batchedtensor(t) or unpack_dual(t).tangent is not None)


class MoELayer(torch.nn.Module):
    """`score`, `num_groups`, `topk_groups`, `group_best`, `renormalize` and `route_scale` are `ops.router.route`'s;
    `expert_bias=True` adds the buffer `expert_bias` (f32 [E], zeros) that the choice is made with: the program moves it
    towards a balanced load. With `balance_coeff` or `z_coeff`, a forward pass with gradients leaves
    `ops.router.balance_loss` of its (this rank's) choices in `aux_loss`, for the program to add to its loss; without
    gradients `aux_loss` is None. With any of these options a choice of -1 (a router logit of -inf) goes to no expert; an inference
    pass then waits on the host for the number of rows received, also in a group of one (the default choice, which never
    leaves one out, does not).
    `norm=True` puts `ops.norm.rms_norm` with the parameter `norm_weight` in front: `forward` then takes the residual as
    well and returns (output, hidden_states + residual)."""

    def __init__(self, hidden_size: int, ffn_hidden_size: int, num_experts: int, topk: int, group=None, *,
                 ep_size: int = 1, ep_rank: int = 0, dtype=torch.bfloat16, activation: str = "swiglu",
                 expert_backend: str = "auto", dispatcher_mode: str = "fused", world=None, device="cuda",
                 fuse_combine: bool = True, use_fp8: bool = False, score: str = "softmax", num_groups: int = 1,
                 topk_groups: Optional[int] = None, group_best: int = 1, renormalize: bool = True, route_scale: float = 1.0,
                 expert_bias: bool = False, balance_coeff: float = 0.0, z_coeff: float = 0.0, norm: bool = False,
                 norm_eps: float = 1e-6):
        super().__init__()
        if num_experts % ep_size:
            raise ValueError("num_experts must be divisible by the EP size")
        if score not in R.SCORES:
            raise ValueError(f"unsupported score {score!r}; expected one of {R.SCORES}")
        if z_coeff and score != "softmax":
            raise ValueError("z_coeff goes with softmax scores")
        if topk_groups is not None and not 1 <= topk_groups <= num_groups:
            raise ValueError("topk_groups has to be between 1 and num_groups")
        if group_best not in (1, 2):
            raise ValueError("group_best is 1 or 2")
        self._choice = dict(score=score, num_groups=num_groups, topk_groups=topk_groups, group_best=group_best,
                            renormalize=renormalize, scale=route_scale)
        self._balance = dict(score=score, coeff=balance_coeff, z_coeff=z_coeff) if balance_coeff or z_coeff else None
        # the plain softmax router keeps the launches (and the higher derivatives) of its own
        self._plain_choice = (score == "softmax" and num_groups == 1 and renormalize and route_scale == 1.0
                              and not expert_bias and self._balance is None)
        self.register_buffer("expert_bias", torch.zeros(num_experts, dtype=torch.float32, device=device) if expert_bias else None)
        self.register_parameter("norm_weight", torch.nn.Parameter(torch.ones(hidden_size, dtype=dtype, device=device)) if norm else None)
        self.norm_eps = norm_eps
        self.aux_loss: Optional[torch.Tensor] = None
        self.hidden_size, self.num_experts, self.topk = hidden_size, num_experts, topk
        self.fuse_combine = fuse_combine
        self.num_local_experts = num_experts // ep_size
        self.router = torch.nn.Linear(hidden_size, num_experts, bias=False, dtype=torch.float32, device=device)
        torch.nn.init.normal_(self.router.weight, std=0.02)
        self.experts, self.expert_backend = build_experts(expert_backend, self.num_local_experts, hidden_size,
                                                          ffn_hidden_size, dtype, activation, device, use_fp8=use_fp8)
        # fp8 inference path: e4m3 rows with 1x128 scales leave the dispatch kernel and feed the
        # block-scaled fp8 fc1 directly (no dequantisation pass); training stays bf16
        self.use_fp8 = bool(use_fp8) and getattr(self.experts, "use_fp8", False)
        self.dispatcher = B200TokenDispatcher(group, self.num_local_experts, num_experts,
                                              ep_rank * self.num_local_experts, mode=dispatcher_mode, world=world)

    def __getstate__(self):
        # (a loss that hangs on a graph can neither be copied nor stored)
        return {**self.__dict__, "aux_loss": None}

    def __setstate__(self, state):
        super().__setstate__(state)
        if "norm_weight" not in self._parameters:           # a layer that was stored before it had these options
            self._choice = dict(score="softmax", num_groups=1, topk_groups=None, group_best=1, renormalize=True, scale=1.0)
            self._balance, self._plain_choice, self.norm_eps, self.aux_loss = None, True, 1e-6, None
            self.register_buffer("expert_bias", None)
            self.register_parameter("norm_weight", None)

    def _fused_logits(self, x) -> bool:
        """Whether the router's own kernel may stand in for its product with these rows."""
        return (type(x) is torch.Tensor and x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous()
                and x.data_ptr() % 16 == 0 and x.shape[1] % 8 == 0 and x.device == self.router.weight.device
                and _plain_linear(self.router) and self.router.weight.shape == (self.num_experts, x.shape[1]))

    def _choose(self, hidden_states: torch.Tensor, router_logits: Optional[torch.Tensor], inference: bool,
                seq_off: Optional[torch.Tensor]):
        """(expert ids, weights) by `ops.router`, and the balance loss of a pass with gradients."""
        l = router_logits
        if l is None:
            if inference and hidden_states.is_cuda and self._fused_logits(hidden_states):
                l = _ext.load().router_logits(hidden_states, self.router.weight)
            else:
                l = self.router(hidden_states.float())
        if l.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            l = l.float()
        if topk_softmax_router is not _OWN_ROUTER:
            idx, w = topk_softmax_router(l, self.topk)
        else:
            idx, w = R.route(l, self.topk, bias=self.expert_bias, **self._choice)
        if self._balance is not None and torch.is_grad_enabled():
            self.aux_loss = R.balance_loss(l, idx, seq_off=seq_off, **self._balance)
        return idx, w

    def _route(self, hidden_states: torch.Tensor, router_logits: Optional[torch.Tensor], inference: bool):
        """(expert ids, weights). For inference the router runs on this library's kernels (f32 like the
        module's own product); for training the logits are the module's own, softmax and choice this library's."""
        E, K = self.num_experts, self.topk
        C = _ext.load() if hidden_states.is_cuda and inference else None
        if C is None or E > C.ROUTER_MAX_EXPERTS or K > 32 or torch.compiler.is_compiling() or torch.jit.is_tracing():
            if router_logits is None:
                router_logits = self.router(hidden_states.float())
            l = router_logits
            if (not inference and topk_softmax_router is _OWN_ROUTER and type(l) is torch.Tensor and l.is_cuda and l.dim() == 2 and 1 <= K <= min(32, l.shape[1])
                    and l.get_device() == torch.cuda.current_device() and l.shape[1] <= _ext.load().ROUTER_MAX_EXPERTS and not _carries_more(l)
                    and not torch.compiler.is_compiling() and not torch.jit.is_tracing()):
                return _TopkSoftmax.apply(l.float().contiguous(), K)
            return topk_softmax_router(l, K)
        if router_logits is None:
            x = hidden_states
            if self._fused_logits(x):
                return C.route(x, self.router.weight, K)
            router_logits = self.router(x.float())
        if type(router_logits) is not torch.Tensor or router_logits.dim() != 2 or router_logits.shape[1] > C.ROUTER_MAX_EXPERTS:
            return topk_softmax_router(router_logits, K)
        return C.topk_softmax(router_logits.float().contiguous(), K)

    def forward(self, hidden_states: torch.Tensor, router_logits: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None, seq_off: Optional[torch.Tensor] = None):
        """hidden_states [T,H]; router_logits [T,E] override the learnable router when given. residual [T,H] (with
        `norm=True` only) is added before the norm: -> (output, sum) in that case, output otherwise. seq_off: the
        sequences that the rows are packed from, for the balance loss."""
        self.aux_loss = None
        if self.norm_weight is None:
            if residual is not None:
                raise ValueError("a residual goes with norm=True")
            return self._mix(hidden_states, router_logits, seq_off, None)
        rows = None
        if (self.use_fp8 and self.dispatcher.mode == "fused" and hidden_states.dtype == torch.bfloat16
                and not torch.is_grad_enabled() and _unchanged(self.dispatcher, _OWN_DISPATCHER)
                and _unchanged(self.experts, _OWN_EXPERTS)):
            # the exchange's cast is part of the norm; the router sees the rows before it
            rows, x, h = N.rms_norm_fp8(hidden_states, self.norm_weight, residual=residual, eps=self.norm_eps, keep=True)
        elif residual is None:
            x, h = N.rms_norm(hidden_states, self.norm_weight, eps=self.norm_eps), None
        else:
            x, h = N.rms_norm(hidden_states, self.norm_weight, residual=residual, eps=self.norm_eps)
        return self._mix(x, router_logits, seq_off, rows), hidden_states if h is None else h

    def _mix(self, hidden_states: torch.Tensor, router_logits: Optional[torch.Tensor], seq_off: Optional[torch.Tensor], fp8_rows):
        """Router, dispatch, experts, combine. fp8_rows: the same rows as (e4m3, scales), where they were made before."""
        inference = not (torch.is_grad_enabled() or topk_softmax_router is not _OWN_ROUTER or _carries_more(hidden_states)
                         or _carries_more(router_logits) or _carries_more(getattr(self.router, "weight", None)))
        if self._plain_choice:
            idx, probs = self._route(hidden_states, router_logits, inference)
        else:
            idx, probs = self._choose(hidden_states, router_logits, inference, seq_off)
        if (inference and self.dispatcher.mode == "fused" and hidden_states.dtype == torch.bfloat16
                and (self.use_fp8 or self.fuse_combine)
                and _unchanged(self.dispatcher, _OWN_DISPATCHER) and _unchanged(self.experts, _OWN_EXPERTS)):
            # Inference: the rows are consumed where they arrive, before the next dispatch can be issued on this
            # stream, so they need no copy of their own, and the GEMMs take their tile lists from the device.
            rows, row_probs, handle = self.dispatcher.dispatch_in_place(
                hidden_states if fp8_rows is None else fp8_rows, idx, probs, use_fp8=self.use_fp8 and fp8_rows is None,
                masked=not self._plain_choice)
            if self.use_fp8:
                El = self.num_local_experts
                off = handle.meta[2 + El: 2 + El + El + 1]
                return self.dispatcher.combine(self.experts.forward_fp8(rows, (), row_probs, expert_off=off))
            from . import fused_a2a as A
            buf = A.get_buffer(self.dispatcher.group, A.get_hidden_bytes(hidden_states), self.dispatcher.world)
            self.dispatcher.handle = None
            return self.experts.forward_fused_combine(rows, row_probs, buf, handle)
        if self.use_fp8 and not torch.is_grad_enabled() and self.dispatcher.mode == "fused":
            rows, tokens_per_expert, row_probs = self.dispatcher.dispatch_fp8(hidden_states, idx, probs)
            El = self.num_local_experts
            off = self.dispatcher.handle.meta[2 + El: 2 + El + El + 1]
            return self.dispatcher.combine(self.experts.forward_fp8(rows, tokens_per_expert, row_probs, expert_off=off))
        rows, tokens_per_expert, row_probs = self.dispatcher.dispatch(hidden_states, idx, probs)
        if (self.fuse_combine and self.dispatcher.mode == "fused" and hasattr(self.experts, "forward_fused_combine")
                and (not torch.is_grad_enabled() or self.experts.activation == "swiglu")):
            # the fc2 epilogue stores straight into the source ranks' slots (no combine-send kernel)
            from . import fused_a2a as A
            buf = A.get_buffer(self.dispatcher.group, A.get_hidden_bytes(hidden_states), self.dispatcher.world)
            handle = self.dispatcher.handle
            self.dispatcher.handle = None
            if torch.is_grad_enabled():
                return self.experts.forward_fused_combine_train(rows, tokens_per_expert, row_probs, buf, handle)
            return self.experts.forward_fused_combine(rows, row_probs, buf, handle)
        out_rows = self.experts(rows, tokens_per_expert, row_probs)
        return self.dispatcher.combine(out_rows)
