"""The operators in front of an expert-parallel exchange, as cases that can be timed and compared.

A case is a dict of plain values; `kind` names the entry points it goes through:

  norm          ops.norm.rms_norm without gradients, with or without the residual's addition
  norm_fp8      ops.norm.rms_norm_fp8: e4m3 rows with 1x128 scales for an fp8 exchange, and the same rows in the
                input's type for the router beside it
  norm_grad     ops.norm.rms_norm, forward and backward: gradients of the input, the residual and the weight
  route         ops.router.route: scores, bias, groups, top-k, weights
  route_grad    the same with the gradient of the logits
  balance_grad  ops.router.balance_loss and its gradient, over one batch or packed sequences

`own` chooses between the plain form in elementary torch operations and the package's entry points. Sizes are those
of the package's benchmarks and tests (hidden 7168 and 4096, 256 experts top-8, 64 experts top-8) and generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NORM_EPS = 1e-6
SUM_EPS = 1e-20          # added to sums of scores that others are divided by: a row without scores has weights of zero


# ------------------------------------------------------------------------------------------ the cases
def listed():
    groups = dict(experts=256, topk=8, score="sigmoid", bias=True, groups=8, topk_groups=4, group_best=2, renormalize=True, scale=2.5)
    return [
        # a decode step of a few sequences in front of an fp8 exchange: latency
        dict(name="norm fp8 decode", kind="norm_fp8", dtype="bf16", wdtype="bf16", tokens=7, hidden=7168, residual=True),
        # a prefill in front of an fp8 exchange, an odd number of tokens
        dict(name="norm fp8 prefill", kind="norm_fp8", dtype="bf16", wdtype="bf16", tokens=8191, hidden=7168, residual=True),
        # inference in half precision of an odd width, weights kept in f32, the first norm of a model (no residual yet)
        dict(name="norm odd", kind="norm", dtype="f16", wdtype="f32", tokens=12001, hidden=1407, residual=False),
        # a training step of a small batch
        dict(name="norm grad 4095x4096", kind="norm_grad", dtype="bf16", wdtype="bf16", tokens=4095, hidden=4096, residual=True),
        # a training step of the largest batch, weights kept in f32
        dict(name="norm grad 16384x7168", kind="norm_grad", dtype="bf16", wdtype="f32", tokens=16384, hidden=7168, residual=True),
        # the routing of a decode step: latency
        dict(name="route decode", kind="route", dtype="f32", tokens=128, padded=0, **groups),
        # the same choice for a prefill whose last rows are padding (no expert is available to them)
        dict(name="route prefill", kind="route", dtype="f32", tokens=16383, padded=61, **groups),
        # a softmax router with groups of 20 experts, the best one standing for its group, weights not renormalised, logits in bf16
        dict(name="route groups of 20", kind="route", dtype="bf16", tokens=4096, padded=0, experts=160, topk=6, score="softmax",
             bias=False, groups=8, topk_groups=3, group_best=1, renormalize=False, scale=16.0),
        # a training step's routing, with the gradient of the logits
        dict(name="route grad", kind="route_grad", dtype="f32", tokens=16384, padded=0, **groups),
        # the balance loss of a small batch of one sequence, softmax, with the logits' own size in the loss
        dict(name="balance small", kind="balance_grad", dtype="f32", tokens=510, padded=0, experts=64, topk=8, score="softmax", sequences=1, z=True),
        # the same over a large batch
        dict(name="balance 16384x64", kind="balance_grad", dtype="f32", tokens=16384, padded=0, experts=64, topk=8, score="softmax", sequences=1, z=True),
        # packed sequences of unequal length, sigmoid scores, padding behind the last one
        dict(name="balance sequences", kind="balance_grad", dtype="f32", tokens=8191, padded=127, experts=256, topk=8, score="sigmoid", sequences=6, z=False),
    ]


def _log(rng, lo, hi, step=1):
    """A whole number between lo and hi, spread over its logarithm, a multiple of `step`."""
    return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    kind = rng.choice(["norm", "norm_fp8", "norm_grad", "norm_grad", "route", "route", "route_grad", "balance_grad", "balance_grad"])
    if kind.startswith("norm"):
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        hidden = _log(rng, 256, 8192, 128 if kind == "norm_fp8" else rng.choice([1, 8, 128]))
        most = 16384 * 7168 // hidden // (2 if dtype == "f32" else 1)
        return dict(kind=kind, dtype=dtype, wdtype=rng.choice([dtype, "f32"]), tokens=_log(rng, 1, min(65536, most)), hidden=hidden,
                    residual=rng.random() < 0.7)
    score, dtype = rng.choice(["softmax", "sigmoid"]), rng.choice(["f32", "f32", "bf16", "f16"])
    tokens = _log(rng, 1, 16384)
    padded = rng.choice([0, 0, tokens // 9])
    if kind == "balance_grad":
        experts = _log(rng, 8, 512)
        return dict(kind=kind, dtype=dtype, tokens=tokens, padded=padded, experts=experts, topk=rng.choice([1, 2, 4, 6, 8]), score=score,
                    sequences=rng.choice([1, 1, _log(rng, 2, 64)]), z=score == "softmax" and rng.random() < 0.5)
    groups = rng.choice([1, 1, 2, 4, 8, 16])
    size = _log(rng, 8, 512 // groups)
    topk_groups = groups if groups < 4 else rng.choice([groups // 2, groups // 4 + 1])
    return dict(kind=kind, dtype=dtype, tokens=tokens, padded=padded, experts=groups * size, topk=rng.choice([1, 2, 4, 6, 8]), score=score,
                bias=rng.random() < 0.5, groups=groups, topk_groups=topk_groups, group_best=rng.choice([1, 2]),
                renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))


# ------------------------------------------------------------------------------------------ inputs
def _logits(g, case):
    """Logits of a learnt router (some experts liked more than others), padding rows at the end without any expert."""
    T, E = case["tokens"], case["experts"]
    l = torch.randn(T, E, generator=g, device="cuda") * 1.2 + torch.randn(E, generator=g, device="cuda") * 0.5
    if case["padded"]:
        l[T - case["padded"]:] = -math.inf
    return l.to(DTYPES[case["dtype"]])


def _offsets(T, n):
    """First row of each of n packed sequences and the end of the last: unequal lengths, every row of T in one."""
    cuts = [T * (2 * i + i * i) // (2 * n + n * n) for i in range(n + 1)]
    return torch.tensor(cuts, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    kind = case["kind"]
    if kind.startswith("norm"):
        T, H, dt = case["tokens"], case["hidden"], DTYPES[case["dtype"]]
        grad = kind == "norm_grad"

        def rows(scale):
            return (torch.randn(T, H, generator=g, device="cuda") * scale).to(dt)
        s["x"] = rows(1.0).requires_grad_(grad)
        s["residual"] = rows(3.0).requires_grad_(grad) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * torch.randn(H, generator=g, device="cuda")).to(DTYPES[case["wdtype"]]).requires_grad_(grad)
        if grad:
            s["dy"] = rows(0.5)
            s["dh"] = rows(0.5) if case["residual"] else None
        return s
    s["logits"] = _logits(g, case)
    T, E, K = case["tokens"], case["experts"], case["topk"]
    if kind == "balance_grad":
        # the choice that came with these logits: the highest of them, none for padding
        v, idx = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
        s["idx"] = torch.where(v[:, :K] == -math.inf, -1, idx[:, :K]).contiguous()
        # (rows behind the last sequence belong to none: the padding, where there is any)
        s["offsets"] = _offsets(T - case["padded"], case["sequences"]).cuda() if case["sequences"] > 1 else None
        s["logits"].requires_grad_(True)
        s["dloss"] = torch.rand((), generator=g, device="cuda") + 0.5
        return s
    s["bias"] = (torch.rand(E, generator=g, device="cuda") - 0.5) * 0.2 if case["bias"] else None
    if kind == "route_grad":
        s["logits"].requires_grad_(True)
        s["dw"] = torch.randn(T, K, generator=g, device="cuda")
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _run_own(s, kind)
    with torch.no_grad():
        return _run_plain(s, kind)


def _run_own(s, kind):
    c = s["case"]
    if kind.startswith("norm"):
        from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
        if kind == "norm_fp8":
            (q, scales), y, h = rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=NORM_EPS, keep=True)
            return dict(q=q, scales=scales, y=y, h=h)
        if s["residual"] is None:
            y, h = rms_norm(s["x"], s["weight"], eps=NORM_EPS), None
        else:
            y, h = rms_norm(s["x"], s["weight"], residual=s["residual"], eps=NORM_EPS)
        if kind == "norm":
            return dict(y=y, h=h)
        if h is None:
            dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
            return dict(y=y, dx=dx, dw=dw)
        dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
        return dict(y=y, h=h, dx=dx, dr=dr, dw=dw)
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    if kind == "balance_grad":
        loss = balance_loss(s["logits"], s["idx"], score=c["score"], coeff=1.0, z_coeff=0.01 if c["z"] else 0.0, seq_off=s["offsets"])
        dl, = torch.autograd.grad(loss, s["logits"], s["dloss"])
        return dict(loss=loss, dlogits=dl)
    idx, w = route(s["logits"], c["topk"], score=c["score"], bias=s["bias"], num_groups=c["groups"], topk_groups=c["topk_groups"],
                   group_best=c["group_best"], renormalize=c["renormalize"], scale=c["scale"])
    if kind == "route":
        return dict(idx=idx, w=w)
    dl, = torch.autograd.grad(w, s["logits"], s["dw"])
    return dict(idx=idx, w=w, dlogits=dl)


def _run_plain(s, kind):
    c = s["case"]
    if kind.startswith("norm"):
        return _plain_norm(s, kind)
    if kind == "balance_grad":
        return _plain_balance(s, c)
    return _plain_route(s, c)


def _plain_norm(s, kind):
    x, r, w, dt = s["x"], s["residual"], s["weight"].float(), s["x"].dtype
    h = x.float() if r is None else x.float() + r.float()
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + NORM_EPS)
    n = h * rstd
    y = n * w
    out = dict(y=y.to(dt), h=None if r is None else h.to(dt))
    if kind == "norm_fp8":
        T, H = x.shape
        blocks = y.view(T, H // 128, 128)
        amax = blocks.abs().amax(-1, keepdim=True).clamp_min(1e-4)
        out["q"] = (blocks * (448.0 / amax)).clamp(-448.0, 448.0).view(T, H).to(torch.float8_e4m3fn)
        out["scales"] = (amax * (1.0 / 448.0)).view(T, H // 128)
    if kind == "norm_grad":
        dy = s["dy"].float()
        a = dy * w
        dx = rstd * (a - n * (a * n).mean(-1, keepdim=True))
        if r is not None:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(dt)
        out["dw"] = (dy * n).sum(0).to(s["weight"].dtype)
        if r is not None:
            out["dr"] = out["dx"]
    return out


def _plain_scores(l, score):
    """Scores in the type of l; zero for an expert that is not available, so all zeros for a row without any."""
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l))
    top = l.max(-1, keepdim=True).values
    none = top == -math.inf
    e = torch.exp(l - torch.where(none, 0.0, top))
    return e / (e.sum(-1, keepdim=True) + none.to(l.dtype))


def _plain_route(s, c):
    l = s["logits"].float()
    T, E, K = c["tokens"], c["experts"], c["topk"]
    # the choice: by values in 64 bits (neighbours may differ by less than 32 bits tell apart), ties to the lowest index;
    # without a bias and a sum of two in it the scores rank as the logits do
    wide = l.double()
    sums = c["groups"] > 1 and c["group_best"] == 2
    v = wide if s["bias"] is None and not sums else _plain_scores(wide, c["score"])
    if s["bias"] is not None:
        v = v + s["bias"].double()
    v = torch.where(wide == -math.inf, -math.inf, v)
    if c["groups"] > 1:
        in_group = v.view(T, c["groups"], E // c["groups"])
        best = torch.sort(in_group, dim=-1, descending=True).values[..., :c["group_best"]]
        value = torch.where(best == -math.inf, 0.0, best).sum(-1)
        value = torch.where(best[..., 0] == -math.inf, -math.inf, value)
        order = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :c["topk_groups"]]
        allowed = (order[:, :, None] == torch.arange(c["groups"], device=l.device)).any(1)
        v = torch.where(allowed[..., None], in_group, -math.inf).view(T, E)
    v, idx = torch.sort(v, dim=-1, descending=True, stable=True)
    v, idx = v[:, :K], idx[:, :K]
    live = v != -math.inf
    scores = _plain_scores(l, c["score"])
    chosen = torch.where(live, scores.gather(1, idx), 0.0)
    total = chosen.sum(-1, keepdim=True) + SUM_EPS
    out = dict(idx=torch.where(live, idx, -1), w=(chosen / total if c["renormalize"] else chosen) * c["scale"])
    if c["kind"] == "route_grad":
        g = s["dw"] * c["scale"]
        if c["renormalize"]:
            g = (g - (g * chosen).sum(-1, keepdim=True) / total) / total
        g = torch.zeros_like(scores).scatter_add(1, idx, torch.where(live, g, 0.0))
        if c["score"] == "sigmoid":
            d = g * scores * (1.0 - scores)
        else:
            d = scores * (g - (g * scores).sum(-1, keepdim=True))
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_balance(s, c):
    l, idx = s["logits"].float(), s["idx"]
    T, E, K = c["tokens"], c["experts"], c["topk"]
    off = s["offsets"]
    if off is None:
        off = torch.tensor([0, T], dtype=torch.int32, device=l.device)
    B = off.numel() - 1
    row = torch.arange(T, device=l.device)
    of = (row[:, None] >= off[None, 1:].long()).sum(-1)                   # the sequence of a row; B: behind the last
    live = (idx >= 0).any(-1) & (of < B)                                  # a token without a choice takes no part
    of = of.clamp_max(B - 1)
    member = ((of[:, None] == torch.arange(B, device=l.device)) & live[:, None]).float()      # [T, B]
    n = member.sum(0)
    took = torch.zeros(T, E, device=l.device).scatter_add(1, idx.clamp_min(0), ((idx >= 0) & live[:, None]).float())
    counts = member.t() @ took
    f = counts * E / (K * n.clamp_min(1.0))[:, None]
    share = live.float() / (n.clamp_min(1.0) * (n > 0).sum().clamp_min(1))[of]                # of the loss, that a row has
    scores = torch.where(live[:, None], _plain_scores(l, c["score"]), 0.0)
    total = scores.sum(-1, keepdim=True) + SUM_EPS
    p = scores / total
    ft = f[of]
    inner = (ft * p).sum(-1, keepdim=True)
    loss = (inner[:, 0].double() * share).sum()
    d = share[:, None] * (p * (ft - inner) * (1.0 - scores) if c["score"] == "sigmoid" else p * (ft - inner))
    if c["z"]:
        top = torch.where(live, l.max(-1).values, 0.0)
        lse = torch.where(live, top + torch.log(torch.exp(torch.where(live[:, None], l, 0.0) - top[:, None]).sum(-1)), 0.0)
        loss = loss + 0.01 * (share * lse * lse).double().sum()
        d = d + (0.02 * share * lse)[:, None] * p
    return dict(loss=loss.float(), dlogits=(d * s["dloss"]).to(s["logits"].dtype))


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(c):
    T = c["tokens"]
    if c["kind"].startswith("norm"):
        H, e = c["hidden"], DTYPES[c["dtype"]].itemsize
        streams = 2 + (2 if c["residual"] else 0)                          # x, y; residual, h
        b = T * H * e * streams + H * DTYPES[c["wdtype"]].itemsize
        flops = 5 * T * H
        if c["kind"] == "norm_fp8":
            b += T * H + T * H // 128 * 4
            flops += 3 * T * H
        if c["kind"] == "norm_grad":
            b += T * H * e * (2 + (1 if c["residual"] else 0)) + H * DTYPES[c["wdtype"]].itemsize      # dy, dx; dh
            flops += 9 * T * H
        return dict(bytes=b, flops=flops)
    E, K, e = c["experts"], c["topk"], DTYPES[c["dtype"]].itemsize
    if c["kind"] == "balance_grad":
        return dict(bytes=T * E * e * 2 + T * K * 8, flops=T * E * 12)
    b, flops = T * E * e + T * K * 12 + (E * 4 if c["bias"] else 0), T * E * 6
    if c["kind"] == "route_grad":
        b, flops = b + T * K * 4 + T * E * e, flops + T * E
    return dict(bytes=b, flops=flops)


# ------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"].startswith("norm"):
        return _exact_norm(s, case)
    if case["kind"] == "balance_grad":
        return _exact_balance(s, case)
    return _exact_route(s, case)


def _exact_norm(s, c):
    grad = c["kind"] == "norm_grad"

    def leaf(t):
        return None if t is None else t.detach().double().requires_grad_(grad)
    x, r, w = leaf(s["x"]), leaf(s["residual"]), leaf(s["weight"])
    with torch.set_grad_enabled(grad):
        h = x + r if r is not None else x
        y = h * torch.rsqrt(h.pow(2).sum(-1, keepdim=True).div(c["hidden"]).add(NORM_EPS)) * w
    out = dict(y=y.detach(), h=h.detach() if r is not None else None)
    if c["kind"] == "norm_fp8":
        out["q"] = None
        out["scales"] = y.unflatten(-1, (-1, 128)).abs().amax(-1).clamp(min=1e-4) / 448
        out["q"] = (y.unflatten(-1, (-1, 128)) / out["scales"][..., None]).flatten(1)
    if grad:
        if r is None:
            out["dx"], out["dw"] = torch.autograd.grad(y, (x, w), s["dy"].double())
        else:
            out["dx"], out["dr"], out["dw"] = torch.autograd.grad((y, h), (x, r, w), (s["dy"].double(), s["dh"].double()))
    return out


def _exact_route(s, c):
    import numpy as np
    T, E, K, G = c["tokens"], c["experts"], c["topk"], c["groups"]
    l = s["logits"].detach().double().cpu().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        if c["score"] == "sigmoid":
            p = np.where(l < 0, np.exp(l) / (1 + np.exp(np.minimum(l, 0))), 1 / (1 + np.exp(-l)))
        else:
            e = np.exp(l - np.maximum(l.max(1, keepdims=True), -1e300))
            p = e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    rank_by = p if s["bias"] is not None or (G > 1 and c["group_best"] == 2) else l
    v = rank_by + (s["bias"].double().cpu().numpy() if s["bias"] is not None else 0.0)
    v[np.isneginf(l)] = -np.inf
    if G > 1:
        a = -np.sort(-v.reshape(T, G, E // G), axis=2)[:, :, :c["group_best"]]
        group = np.where(np.isneginf(a[:, :, 0]), -np.inf, np.where(np.isneginf(a), 0, a).sum(2))
        behind = np.argsort(-group, axis=1, kind="stable")[:, c["topk_groups"]:]
        v3 = v.reshape(T, G, E // G).copy()
        np.put_along_axis(v3, behind[:, :, None], -np.inf, axis=1)
        v = v3.reshape(T, E)
    idx = np.argsort(-v, axis=1, kind="stable")[:, :K]
    live = ~np.isneginf(np.take_along_axis(v, idx, 1))
    # weights, and their gradient by automatic differentiation of the definition
    lt = torch.from_numpy(l).cuda().requires_grad_(True)
    at, ok = torch.from_numpy(idx).cuda(), torch.from_numpy(live).cuda()
    some = (lt.detach() > -math.inf).any(1, keepdim=True)
    safe = torch.where(some, lt, torch.zeros_like(lt))
    scores = torch.sigmoid(safe) if c["score"] == "sigmoid" else torch.softmax(safe, 1)
    w = torch.where(ok, scores.gather(1, at), 0.0)
    if c["renormalize"]:
        w = w / (w.sum(1, keepdim=True) + SUM_EPS)
    w = w * c["scale"]
    out = dict(idx=torch.where(ok, at, -1), w=w.detach())
    if c["kind"] == "route_grad":
        out["dlogits"], = torch.autograd.grad(w, lt, s["dw"].double())
    return out


def _exact_balance(s, c):
    T, E, K = c["tokens"], c["experts"], c["topk"]
    l = s["logits"].detach().double().requires_grad_(True)
    cuts = [0, T] if s["offsets"] is None else s["offsets"].tolist()
    some = (s["idx"] >= 0).any(1)
    terms = []
    for lo, hi in zip(cuts, cuts[1:]):
        rows = torch.arange(lo, hi, device=l.device)[some[lo:hi]]
        if rows.numel() == 0:
            continue
        a = l[rows]
        p = torch.sigmoid(a) if c["score"] == "sigmoid" else torch.softmax(a, 1)
        p = p / (p.sum(1, keepdim=True) + SUM_EPS)
        chosen = s["idx"][rows].flatten()
        f = torch.bincount(chosen[chosen >= 0], minlength=E).double() * E / (K * rows.numel())
        term = (f * p.mean(0)).sum()
        if c["z"]:
            term = term + 0.01 * torch.logsumexp(a, 1).pow(2).mean()
        terms.append(term)
    if not terms:
        return dict(loss=torch.zeros((), dtype=torch.float64), dlogits=torch.zeros_like(l))
    loss = torch.stack(terms).mean()
    d, = torch.autograd.grad(loss, l, s["dloss"].double())
    return dict(loss=loss.detach(), dlogits=d)
