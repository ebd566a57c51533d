"""Choice of experts and balance loss against 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _scores(l, score):
    """l: float64 [T, E] on the CPU (numpy)."""
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-l))
        top = l.max(1, keepdims=True)
        e = np.exp(l - np.where(np.isneginf(top), 0, top))
        s = e.sum(1, keepdims=True)
        return np.where(s == 0, 0, e / np.where(s == 0, 1, s))


def _choose(l, K, score, bias, groups, topk_groups, best):
    """Token by token, from the definition. -> idx"""
    T, E = l.shape
    s = _scores(l, score)
    computed = bias is not None or (groups > 1 and best == 2)
    v = s.copy() if computed else l.copy()
    if bias is not None:
        v = v + bias[None]
    v[np.isneginf(l)] = -np.inf
    idx = np.full((T, K), -1, dtype=np.int64)
    size = E // groups
    key = np.where(np.isnan(v), np.inf, v)                        # NaN above everything (+inf does not occur beside it here)
    for t in range(T):
        allowed = np.ones(E, bool)
        if groups > 1:
            value = np.full(groups, -np.inf)
            for g in range(groups):
                a = np.sort(key[t, g * size:(g + 1) * size])[::-1][:best]
                a = a[~np.isneginf(a)]
                if a.size:
                    value[g] = a.sum()
            for g in np.argsort(-value, kind="stable")[topk_groups:]:
                allowed[g * size:(g + 1) * size] = False
        k = np.where(allowed, key[t], -np.inf)
        order = np.argsort(-k, kind="stable")[:K]
        live = ~np.isneginf(k[order])
        idx[t, :live.sum()] = order[live]
    return idx


def _weights(l, idx, score, renorm, scale):
    """Differentiable, float64: l a torch tensor."""
    some = (l.detach() > -math.inf).any(1, keepdim=True) | l.detach().isnan().any(1, keepdim=True)
    safe = torch.where(some, l, torch.zeros_like(l))
    s = torch.sigmoid(safe) if score == "sigmoid" else torch.softmax(safe, 1)
    w = torch.where(idx >= 0, s.gather(1, idx.clamp_min(0)), 0.0)
    if renorm:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return w * scale


def _logits(T, E, dt, seed=0, masked=True):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(T, E, generator=g) * 1.5
    if masked and T > 3:
        l[torch.rand(T, E, generator=g) < 0.1] = -math.inf
        l[1] = -math.inf                                           # nothing is available
        l[2, 1:] = -math.inf                                       # one expert is
        l[3] = 0.25                                                # all alike
    return l.to(dt).cuda()


CASES = [  # T, E, K, score, bias, groups, topk_groups, best
    (1, 1, 1, "softmax", False, 1, 1, 1), (5, 3, 3, "sigmoid", True, 1, 1, 1), (33, 8, 2, "softmax", False, 1, 1, 1),
    (130, 64, 8, "softmax", True, 1, 1, 1), (70, 65, 6, "sigmoid", False, 1, 1, 1), (300, 256, 8, "sigmoid", True, 8, 4, 2),
    (300, 256, 8, "sigmoid", False, 8, 4, 2), (200, 160, 6, "softmax", False, 8, 3, 1), (77, 160, 6, "softmax", True, 8, 3, 2),
    (90, 96, 1, "sigmoid", True, 32, 1, 2), (90, 96, 3, "softmax", False, 32, 1, 1), (50, 384, 8, "sigmoid", True, 1, 1, 1),
    (40, 1024, 32, "sigmoid", True, 16, 2, 2), (40, 1000, 32, "softmax", False, 1, 1, 1), (40, 1023, 9, "softmax", True, 31, 11, 1),
    (64, 128, 32, "sigmoid", False, 4, 1, 2), (1300, 72, 5, "sigmoid", True, 3, 2, 2), (2500, 512, 8, "softmax", True, 2, 1, 1),
    (20, 32, 4, "sigmoid", True, 32, 7, 2), (60, 1020, 9, "softmax", True, 17, 5, 2), (60, 1020, 32, "sigmoid", False, 17, 5, 1),
    (400, 160, 8, "sigmoid", True, 8, 3, 2), (400, 336, 8, "softmax", True, 7, 3, 2), (20, 40, 4, "softmax", True, 20, 7, 2), (20, 7, 7, "sigmoid", True, 7, 7, 2),
]


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("case", CASES)
def test_route_and_gradient(case, dt):
    from gpu_data_transfer_profile_b200.ops.router import route
    T, E, K, score, biased, groups, topk_groups, best = case
    l = _logits(T, E, dt, seed=E + K)
    g = torch.Generator().manual_seed(1)
    bias = (torch.rand(E, generator=g) - 0.5).cuda() if biased else None
    if biased and E > 40:
        bias[E // 2] = -math.inf
    wide = l.double().cpu().numpy()
    idx_want = torch.from_numpy(_choose(wide, K, score, bias.double().cpu().numpy() if biased else None, groups, topk_groups, best)).cuda()
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        l.requires_grad_(False)
        kw = dict(score=score, bias=bias, num_groups=groups, topk_groups=topk_groups, group_best=best, renormalize=renorm, scale=scale)
        idx, w = route(l, K, **kw)
        assert idx.dtype == torch.int64 and w.dtype == F32
        assert torch.equal(idx, idx_want)
        lw = l.double().requires_grad_(True)
        want = _weights(lw, idx_want, score, renorm, scale)
        # a score: the exponential (2 units in the last place, and the logit's distance to the maximum rounded: half a unit of
        # up to 16), sums of up to 1024 in a tree of 5 levels over 32 a lane, a division; twice that when renormalised
        rel = (4 + 16 + 37 + 2) * U * (2 if renorm else 1) + 40 * U
        assert ((w.double() - want).abs() <= want.abs() * rel).all()
        assert (w[idx < 0] == 0).all()
        dw = torch.randn(T, K, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
        l.requires_grad_(True)
        idx2, w2 = route(l, K, **kw)
        assert torch.equal(idx2, idx) and torch.equal(w2, w) and not idx2.requires_grad
        got, = torch.autograd.grad(w2, l, dw)
        ref, = torch.autograd.grad(want, lw, dw.double())
        ref = torch.where(torch.isneginf(l), 0.0, ref)
        # differences of weighted means: `rel` of the sum of their terms' sizes, K terms each
        size = (want.detach().abs() * dw.double().abs()).sum(1, keepdim=True)
        tol = size * 4 * (rel + 2 * K * U) + ref.abs() * (torch.finfo(dt).eps / 2 * 1.01 if dt != F32 else 0) + (2.0 ** -25 if dt == F16 else 0)
        assert got.dtype == dt and ((got.double() - ref).abs() <= tol).all()


def test_route_of_equal_values_takes_the_lowest_index():
    from gpu_data_transfer_profile_b200.ops.router import route
    for dt in (F32, BF16):
        l = torch.zeros(9, 64, device="cuda", dtype=dt)
        for kw in (dict(), dict(score="sigmoid", bias=torch.zeros(64, device="cuda")),
                   dict(score="sigmoid", bias=torch.zeros(64, device="cuda"), num_groups=8, topk_groups=2, group_best=2),
                   dict(num_groups=8, topk_groups=2), dict(score="softmax", bias=torch.full((64,), 0.125, device="cuda"))):
            idx, w = route(l, 8, **kw)
            assert torch.equal(idx, torch.arange(8, device="cuda").expand(9, 8))
            torch.testing.assert_close(w, torch.full((9, 8), 0.125, device="cuda"), atol=1e-7, rtol=0)
    # +0 and -0 are equal
    l = torch.zeros(1, 64, device="cuda")
    l[0, :5] = -0.0
    assert route(l, 3)[0].tolist() == [[0, 1, 2]]


def test_route_of_neighbours_that_32_bits_do_not_tell_apart():
    """Pairs of experts whose value differs by less than a 32-bit step: a bias makes up for the difference of the scores up
    to its own rounding, and 64 bits decide."""
    from gpu_data_transfer_profile_b200.ops.router import route
    g = torch.Generator().manual_seed(0)
    l = torch.randn(4000, 16, generator=g).cuda()
    base = torch.sigmoid(l[:1].double())
    bias = (0.75 - base[0]).float()                                # v is 0.75 and a rounding for every expert in row 0
    l = l[:1] + (torch.randn(4000, 16, generator=g).cuda() * 1e-7) * l[:1].abs()
    want = _choose(l.double().cpu().numpy(), 5, "sigmoid", bias.double().cpu().numpy(), 1, 1, 1)
    idx, _ = route(l, 5, score="sigmoid", bias=bias)
    assert torch.equal(idx.cpu(), torch.from_numpy(want))
    want = _choose(l.double().cpu().numpy(), 5, "sigmoid", bias.double().cpu().numpy(), 4, 2, 2)
    idx, _ = route(l, 5, score="sigmoid", bias=bias, num_groups=4, topk_groups=2, group_best=2)
    assert torch.equal(idx.cpu(), torch.from_numpy(want))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,topk_groups,best,grid", [(256, 8, 4, 2, 0), (256, 8, 4, 1, 16), (160, 8, 3, 2, 8), (96, 32, 9, 2, 16), (64, 1, 1, 1, 4), (72, 3, 2, 1, 0),
                                                          (512, 16, 3, 2, 0), (40, 4, 1, 2, 4)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_of_many_tokens(E, groups, topk_groups, best, grid, biased, score):
    """Tokens by the ten thousand, among them many with equal logits (on a grid) and values a few 32-bit steps apart."""
    from gpu_data_transfer_profile_b200.ops.router import route
    T, K = 20000, 7
    g = torch.Generator(device="cuda").manual_seed(E + grid)
    l = torch.randn(T, E, generator=g, device="cuda")
    if grid:
        l = (l * grid).round() / grid
    bias = (torch.rand(E, generator=g, device="cuda") - 0.5) * 0.3
    if grid:
        bias = (bias * 16).round() / 16
    close = torch.rand(T, E, generator=g, device="cuda") < 0.2    # a value and its neighbour on the next place but for some steps
    close[:, ::2] = False
    l = torch.where(close, torch.roll(l, 1, 1) * (1 + torch.randint(-3, 4, (T, E), generator=g, device="cuda") * 2.0 ** -24), l)
    w = l.double()
    s = torch.sigmoid(w) if score == "sigmoid" else torch.softmax(w, 1)
    computed = biased or (groups > 1 and best == 2)
    v = (s if computed else w) + (bias.double() if biased else 0)
    if groups > 1:
        value = v.view(T, groups, -1).topk(best, -1).values.sum(-1)
        order = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :topk_groups]
        kept = torch.zeros(T, groups, dtype=torch.bool, device="cuda").scatter_(1, order, True)
        v = torch.where(kept.repeat_interleave(E // groups, 1), v, -math.inf)
    want = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :K]
    idx, _ = route(l, K, score=score, bias=bias if biased else None, num_groups=groups, topk_groups=topk_groups, group_best=best)
    # (scores of logits a step apart may come to the same 64 bits, or the other way round in their last one: some 1e-16)
    same = (idx == want).all(1)
    a, b = v.gather(1, idx), v.gather(1, want)
    assert ((a - b).abs()[~same] <= 4e-16 * (1 + a.abs()[~same])).all() and (~same).sum() <= (3 if computed else 0)


def test_route_of_infinities_and_nan():
    from gpu_data_transfer_profile_b200.ops.router import route
    l = torch.randn(6, 40, device="cuda")
    l[0, 17] = math.nan
    l[1, 3] = l[1, 30] = math.inf
    l[2] = math.nan
    l[3, 5] = -math.inf
    l[4] = 200.0                                                  # sigmoid is 1 for all
    l[5] = -200.0                                                 # and 0 in 32 bits
    idx, w = route(l, 4, score="sigmoid")
    assert idx[0, 0] == 17 and w[0].isnan().all()
    assert idx[1, :2].tolist() == [3, 30] and (w[1, 0] == w[1, 1]).item() and w[1].sum().item() == pytest.approx(1, abs=1e-6)
    assert idx[2].tolist() == [0, 1, 2, 3] and w[2].isnan().all()
    assert 5 not in idx[3].tolist()
    assert idx[4].tolist() == [0, 1, 2, 3] and (w[4] == 0.25).all()
    assert idx[5].tolist() == [0, 1, 2, 3] and (w[5] == 0).all()
    for kw in (dict(), dict(bias=torch.zeros(40, device="cuda")), dict(bias=torch.zeros(40, device="cuda"), num_groups=4, topk_groups=2, group_best=2)):
        idx, w = route(l, 4, **kw)
        assert w[0].isnan().all() and w[1].isnan().any() and w[2].isnan().all() and (w[4] == 0.25).all() and (w[5] == 0.25).all()
        assert (idx >= 0).all() and (idx < 40).all()
    assert route(l, 4)[0][0, 0] == 17
    bias = torch.zeros(40, device="cuda")
    bias[9] = math.inf
    assert (route(l[3:], 1, bias=bias)[0] == 9).all()
    bias[:] = -math.inf
    idx, w = route(l[3:], 4, bias=bias)
    assert (idx == -1).all() and (w == 0).all()
    # a group with one available expert comes before a group with none
    l = torch.full((1, 16), -math.inf, device="cuda")
    l[0, 13] = -5.0
    for best in (1, 2):
        idx, w = route(l, 2, score="sigmoid", bias=torch.full((16,), -3.0, device="cuda"), num_groups=4, topk_groups=1, group_best=best)
        assert idx.tolist() == [[13, -1]] and w.tolist() == [[1.0, 0.0]]
    # gradients of rows without an expert are zero, of the rest as if those rows were not there
    l = torch.randn(5, 16, device="cuda")
    l[2] = -math.inf
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            a = l.clone().requires_grad_(True)
            gr, = torch.autograd.grad(route(a, 3, score=score, renormalize=renorm)[1], a, torch.ones(5, 3, device="cuda"))
            assert (gr[2] == 0).all() and gr.isfinite().all()


def test_route_strides_and_empty():
    from gpu_data_transfer_profile_b200.ops.router import route
    big = torch.randn(50, 200, device="cuda")
    for dt in (F32, BF16):
        b = big.to(dt)
        for view in (b[:, 3:67], b[::3, :64], b.t()[:64].t(), b[:1, 5:69], b[:1, :64].expand(7, 64), b[7, 0].expand(4, 64)):
            for kw in (dict(), dict(score="sigmoid", bias=torch.rand(130, device="cuda")[::2][:64], num_groups=4, topk_groups=2, group_best=2)):
                a, c = route(view, 4, **kw), route(view.clone(memory_format=torch.contiguous_format), 4, **kw)
                assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    v = big.clone().requires_grad_(True)
    gv, = torch.autograd.grad(route(v[:, 3:67], 4, renormalize=False)[1].sum(), v)
    u = big[:, 3:67].clone().requires_grad_(True)
    gu, = torch.autograd.grad(route(u, 4, renormalize=False)[1].sum(), u)
    assert torch.equal(gv[:, 3:67], gu) and (gv[:, :3] == 0).all()
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    idx, w = route(e, 4)
    assert idx.shape == (0, 4) and w.shape == (0, 4)
    assert torch.autograd.grad(w.sum(), e)[0].shape == (0, 64)


def test_route_gradient_of_one_renormalised_choice_is_zero():
    from gpu_data_transfer_profile_b200.ops.router import route
    l = torch.randn(500, 64, device="cuda", requires_grad=True)
    w = route(l, 1, scale=2.5)[1]
    assert (w == 2.5).float().mean() > 0.5 and (w - 2.5).abs().max() <= 2.5 * 4 * U
    assert (torch.autograd.grad(w, l, torch.randn(500, 1, device="cuda"))[0] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("bar", [-math.inf, -2.0])
@pytest.mark.parametrize("K", [1, 3])
@pytest.mark.parametrize("gap", [10, 20, 30, 40, 46, 60])
def test_route_gradient_where_the_favourite_may_not_be_chosen(gap, K, bar, dt):
    """The chosen scores sum to little beside the 1e-20 that is added: the weights are no softmax over the chosen logits."""
    from gpu_data_transfer_profile_b200.ops.router import route
    g = torch.Generator(device="cuda").manual_seed(gap + K)
    T, E, scale = 40, 41, 2.5
    l = torch.randn(T, E, generator=g, device="cuda") * 1.5
    bias = torch.zeros(E, device="cuda")
    bias[7] = bar
    l[:, 7] = l.max(1).values + gap
    l[3] = -math.inf                                                # padding
    l = l.to(dt).requires_grad_(True)
    idx, w = route(l, K, bias=bias, scale=scale)
    dw = torch.randn(T, K, generator=g, device="cuda")
    got, = torch.autograd.grad(w, l, dw)
    lw = l.detach().double().requires_grad_(True)
    want = _weights(lw, idx, "softmax", True, scale)
    ref, = torch.autograd.grad(want, lw, dw.double())
    ref = torch.where(torch.isneginf(l), 0.0, ref)
    assert not (idx == 7).any() and (idx[3] == -1).all() and (got[3] == 0).all()
    # Distances of up to 70 to the maximum are rounded by 64 U, so is each score relative to itself. A weight has two of them,
    # two sums of up to 41 and 3 + K roundings, what it is multiplied by as many again: below 800 U of the terms' sizes. Of
    # one choice, the first term's difference is 0. Below 2^-40 the lack is left out.
    p = torch.softmax(torch.where(torch.isneginf(lw), -1e4, lw), 1).detach()
    u = want.detach() / scale
    r = 1e-20 / (p.gather(1, idx.clamp_min(0)).sum(1, keepdim=True) + 1e-20)
    dg = dw.double().abs() * scale
    all_g = (u * dg).sum(1, keepdim=True)
    tol = (800 * U * r + 2.0 ** -40) * p * all_g
    tol = tol.scatter_add(1, idx.clamp_min(0), (800 * U * r + 2.0 ** -40) * u * dg + (0 if K == 1 else 800 * U * u * (dg + all_g)))
    tol = tol + ref.abs() * (torch.finfo(dt).eps / 2 * 1.01 if dt != F32 else 0) + (2.0 ** -25 if dt == F16 else 0)
    assert ((got.double() - ref).abs() <= tol).all()


def test_route_gradient_against_differences():
    from gpu_data_transfer_profile_b200.ops.router import route
    g = torch.Generator(device="cuda").manual_seed(0)
    l = torch.randn(40, 24, generator=g, device="cuda") * 2
    u = torch.randn(40, 24, generator=g, device="cuda")
    dw = torch.randn(40, 4, generator=g, device="cuda")
    for kw in (dict(), dict(renormalize=False), dict(score="sigmoid"), dict(score="sigmoid", renormalize=False, scale=3.0)):
        a = l.clone().requires_grad_(True)
        idx, w = route(a, 4, **kw)
        got = (torch.autograd.grad(w, a, dw)[0] * u).sum(1).double()
        s = 2.0 ** -8
        ip, wp = route(l + s * u, 4, **kw)
        im, wm = route(l - s * u, 4, **kw)
        same = ((ip == idx) & (im == idx)).all(1)                 # where the choice stays what it is
        assert same.sum() > 20
        want = ((wp - wm).double() * dw).sum(1) / (2 * s)
        # third derivatives below 20 a token times s^2 / 6; roundings of the weights over 2 s
        assert ((got - want).abs()[same] < 20 * 3 * s * s + 4 * 3 * 4 * 8 * U / s).all()


def test_route_gradient_against_differences_where_the_favourite_may_not_be_chosen():
    from gpu_data_transfer_profile_b200.ops.router import route
    g = torch.Generator(device="cuda").manual_seed(5)
    l = torch.randn(40, 24, generator=g, device="cuda")
    l[:, 9] = 46.0                                                  # 1e-20 of it and the chosen scores are of one size
    bias = torch.zeros(24, device="cuda")
    bias[9] = -math.inf
    u = torch.randn(40, 24, generator=g, device="cuda").clamp(-1, 1)
    dw = torch.randn(40, 4, generator=g, device="cuda").clamp(-2, 2)
    a = l.clone().requires_grad_(True)
    idx, w = route(a, 4, bias=bias)
    got = (torch.autograd.grad(w, a, dw)[0] * u).sum(1).double()
    s = 2.0 ** -6
    (ip, wp), (im, wm) = (route(l + d * u, 4, bias=bias) for d in (s, -s))
    same = ((ip == idx) & (im == idx)).all(1)
    assert same.sum() > 20 and got.abs().max() > 0.1
    want = ((wp - wm).double() * dw).sum(1) / (2 * s)
    # (third derivatives below 50: of a softmax along directions of up to 2 with a gradient of up to 2 each; scores rounded by
    # 32 U for their distance of 46 to the maximum, weights by three times that)
    assert ((got - want).abs()[same] < 50 * s * s / 6 + 4 * 2 * 100 * U / s).all()


def test_route_refusals():
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    l = torch.randn(6, 64, device="cuda")
    idx = route(l, 4)[0]
    for call in (lambda: route(l, 0), lambda: route(l, 33), lambda: route(l, 9, num_groups=8, topk_groups=1), lambda: route(l, 4, num_groups=7),
                 lambda: route(l, 4, num_groups=64), lambda: route(l, 4, num_groups=8, topk_groups=9), lambda: route(l, 4, num_groups=8, topk_groups=0),
                 lambda: route(l, 4, num_groups=0), lambda: route(l, 4, group_best=3), lambda: route(l, 4, group_best=0), lambda: route(l, 4, scale=0.0),
                 lambda: route(l, 4, scale=math.nan), lambda: route(l, 4, scale=1e-60), lambda: route(l, 4, scale=math.inf), lambda: route(l.double(), 4),
                 lambda: route(l.cpu(), 4), lambda: route(l[0], 4), lambda: route(l, 4, bias=l[0, :63]), lambda: route(l, 4, bias=l[0].cpu()),
                 lambda: route(l, 4, bias=l[0].int()), lambda: route(torch.randn(2, 1025, device="cuda"), 4), lambda: route(l[:, :0], 1),
                 lambda: torch.func.vmap(lambda t: route(t, 4)[1])(l[None]),
                 lambda: balance_loss(l, idx.int()), lambda: balance_loss(l, idx[:5]), lambda: balance_loss(l, idx.cpu()), lambda: balance_loss(l.double(), idx),
                 lambda: balance_loss(l, idx, z_coeff=1.0, score="sigmoid"), lambda: balance_loss(l, idx, coeff=math.inf),
                 lambda: balance_loss(l, idx, seq_off=torch.tensor([0, 6], device="cuda")), lambda: balance_loss(l, idx, seq_off=torch.tensor([0], device="cuda", dtype=torch.int32)),
                 lambda: balance_loss(l, idx, seq_off=torch.tensor([0, 6], dtype=torch.int32)), lambda: balance_loss(l, idx[:, :0]),
                 lambda: balance_loss(l[None], idx)):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: route(l, 4, score="relu"), lambda: balance_loss(l, idx, score="none")):
        with pytest.raises(ValueError):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(l, l)
        for call in (lambda: route(dual, 4), lambda: balance_loss(dual, idx)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
    a = l.clone().requires_grad_(True)
    for call in (lambda: route(a, 4)[1].sum(), lambda: balance_loss(a, idx)):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(call(), a, create_graph=True)
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------- balance loss
def _balance(l, idx, score, coeff, z, off):
    """float64, differentiable."""
    E, K = l.shape[1], idx.shape[1]
    cuts = off.tolist() if off is not None else [0, l.shape[0]]
    terms = []
    for lo, hi in zip(cuts, cuts[1:]):
        rows = [t for t in range(lo, hi) if ((idx[t] >= 0) & (idx[t] < E)).any()]
        if not rows:
            continue
        a = l[rows]
        if score == "sigmoid":
            s = torch.sigmoid(a)
        else:
            s = torch.softmax(torch.where((a > -math.inf).any(1, keepdim=True), a, torch.zeros_like(a)), 1) * (a > -math.inf).any(1, keepdim=True)
        p = s / (s.sum(1, keepdim=True) + 1e-20)
        c = idx[rows].flatten()
        f = torch.bincount(c[(c >= 0) & (c < E)], minlength=E).double() * E / (K * len(rows))
        term = coeff * (f * p.mean(0)).sum()
        if z:
            term = term + z * torch.logsumexp(a, 1).square().mean()
        terms.append(term)
    return torch.stack(terms).mean() if terms else (l * 0).nan_to_num(0).sum()


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K,cuts", [
    (1, 1, 1, None), (5, 3, 2, None), (200, 64, 8, None), (257, 65, 6, [0, 100, 100, 101, 250]), (300, 128, 1, [7, 7, 150, 300]),
    (100, 256, 8, [0, 100]), (64, 512, 4, [0, 1, 2, 3, 64]), (50, 1024, 32, None), (5000, 40, 3, [0, 0, 0, 2048, 4096, 4999]), (40, 8, 2, [40, 40])])
def test_balance_loss_and_gradient(T, E, K, cuts, score, dt):
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    l = _logits(T, E, dt, seed=T, masked=T > 20)
    idx, _ = route(l, K, score=score)
    if T > 30:
        idx[10] = -1                                               # dropped tokens, one choice of a token, an index twice
        idx[11, 0] = -1
        idx[12] = 5 % E
        idx[13, 0] = E + 3                                         # no expert of these
    off = torch.tensor(cuts, dtype=torch.int32, device="cuda") if cuts else None
    # (logsumexp of a token whose experts are all masked is not defined: those tokens have no choice here)
    idx[(l == -math.inf).all(1)] = -1
    for coeff, z in ((1.0, 0.0), (0.5, 0.01 if score == "softmax" else 0.0)):
        a = l.clone().requires_grad_(True)
        wide = l.double().requires_grad_(True)
        loss = balance_loss(a, idx, score=score, coeff=coeff, z_coeff=z, seq_off=off)
        want = _balance(wide, idx, score, coeff, z, off)
        assert loss.dtype == F32 and loss.shape == ()
        # shares of 32-bit scores (as for the weights of a choice), summed with positive terms; the rest in 64 bits
        assert abs(loss.item() - want.item()) <= 140 * U * abs(want.item()) + 1e-30
        assert torch.equal(loss.detach(), balance_loss(l, idx, score=score, coeff=coeff, z_coeff=z, seq_off=off))
        got, = torch.autograd.grad(loss * 3.0, a)
        ref, = torch.autograd.grad(want * 3.0, wide)
        ref = ref.nan_to_num(0)
        # differences f_e - F of sizes up to the largest f, times p: relative to p max(f) / n, 200 roundings
        live = torch.where(torch.isneginf(l), -1e30, l.double())
        p = torch.softmax(live, 1) if score == "softmax" else torch.sigmoid(live) / torch.sigmoid(live).sum(1, keepdim=True).clamp_min(1e-30)
        n_least = 1
        size = 3.0 * p * (coeff * E / 1.0 + 2 * z * 20) / n_least
        tol = size * 200 * U / 1.0 + ref.abs() * (torch.finfo(dt).eps / 2 * 1.01 if dt != F32 else 0) + (2.0 ** -25 if dt == F16 else 1e-38)
        assert got.dtype == dt and ((got.double() - ref).abs() <= tol).all()
        # and against the gradient's own size, over all of it: 32-bit arithmetic. (With one expert f = F = 1 and the gradient
        # is 0: what the 64-bit side has there, some 1e-16, is its own rounding of 1 - s sum / sum.)
        if E > 1 and ref.norm() > 0:
            # (f16: gradients of some 1e-7 are a few denormal steps of 2^-24, each off by half a step at most)
            denormal = math.sqrt(got.numel()) * 2.0 ** -25 if dt == F16 else 0
            assert (got.double() - ref).norm() <= ref.norm() * (2e-6 if dt == F32 else torch.finfo(dt).eps / 2 * 1.01) + denormal
        none = ~((idx >= 0) & (idx < E)).any(1)
        assert (got[none] == 0).all()
        if off is not None:
            assert (got[:cuts[0]] == 0).all() and (got[cuts[-1]:] == 0).all()


def test_balance_loss_against_differences():
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    g = torch.Generator(device="cuda").manual_seed(0)
    l = torch.randn(60, 24, generator=g, device="cuda")
    u = torch.randn(60, 24, generator=g, device="cuda")
    off = torch.tensor([0, 20, 60], dtype=torch.int32, device="cuda")
    idx, _ = route(l, 3)
    for kw in (dict(z_coeff=0.1), dict(score="sigmoid"), dict(seq_off=off, z_coeff=0.1), dict(score="sigmoid", seq_off=off)):
        a = l.clone().requires_grad_(True)
        got = (torch.autograd.grad(balance_loss(a, idx, **kw), a)[0] * u).sum().item()
        s = 2.0 ** -6
        want = (balance_loss(l + s * u, idx, **kw) - balance_loss(l - s * u, idx, **kw)).item() / (2 * s)
        # third derivatives below 30 times s^2 / 6, and two roundings of a loss below 3 over 2 s
        assert abs(got - want) < 30 * s * s / 6 + 3 * 2 * U / s


def test_balance_loss_of_a_perfect_choice_is_its_coefficient():
    """With equal scores and equal loads, f and E p are 1 for every expert."""
    from gpu_data_transfer_profile_b200.ops.router import balance_loss
    l = torch.zeros(64, 32, device="cuda")
    idx = (torch.arange(64, device="cuda")[:, None] * 4 + torch.arange(4, device="cuda")) % 32
    for score in ("softmax", "sigmoid"):
        assert balance_loss(l, idx, score=score, coeff=0.75).item() == 0.75


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_gradient_of_a_nearly_balanced_choice(score):
    """f_e - F_t is some 1e-3 of f here; the gradient is as exact as the shares that it multiplies."""
    from gpu_data_transfer_profile_b200.ops.router import balance_loss
    T, E, K = 4096, 64, 4
    idx = (torch.arange(T, device="cuda")[:, None] * K + torch.arange(K, device="cuda")) % E
    idx[5, 0], idx[100, 1], idx[101, 2] = 9, 9, 40
    l = torch.randn(T, E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    a, wide = l.clone().requires_grad_(True), l.double().requires_grad_(True)
    got, = torch.autograd.grad(balance_loss(a, idx, score=score), a)
    ref, = torch.autograd.grad(_balance(wide, idx, score, 1.0, 0.0, None), wide)
    # shares off by some 2^-22, their weighted sum by the mean of 64 of those: relative to the gradient itself
    assert (got.double() - ref).norm() <= ref.norm() * 1e-6
    even = torch.autograd.grad(balance_loss(a, (torch.arange(T, device="cuda")[:, None] * K + torch.arange(K, device="cuda")) % E, score=score), a)[0]
    # (all f are 1; F is off by 2^-22 and its correction by as much of that)
    assert even.abs().max() <= 2.0 ** -43
    # the other extreme: one expert has all choices, and the smallest share of the tokens' scores by far
    l = torch.randn(50, 3, device="cuda") - torch.tensor([12.0, 0.0, 0.0], device="cuda")
    a, wide = l.clone().requires_grad_(True), l.double().requires_grad_(True)
    idx = torch.zeros(50, 1, dtype=torch.int64, device="cuda")
    loss, want = balance_loss(a, idx, score=score), _balance(wide, idx, score, 1.0, 0.0, None)
    assert abs(loss.item() / want.item() - 1) < 1e-6
    got, ref = torch.autograd.grad(loss, a)[0], torch.autograd.grad(want, wide)[0]
    assert (got.double() - ref).norm() <= ref.norm() * 1e-6


def test_balance_loss_strides_empty_and_unused():
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    big = torch.randn(50, 200, device="cuda")
    for view in (big[:, 3:67], big[::2, :64], big.t()[:64].t(), big[:1, :64].expand(7, 64)):
        idx = route(view, 8)[0]
        want = balance_loss(view.clone(memory_format=torch.contiguous_format), idx)
        assert torch.equal(balance_loss(view, idx), want)
        assert torch.equal(balance_loss(view, idx.t().contiguous().t()), want)
    v = big.clone().requires_grad_(True)
    idx = route(big[:, 3:67], 8)[0]
    gv, = torch.autograd.grad(balance_loss(v[:, 3:67], idx), v)
    assert (gv[:, :3] == 0).all() and (gv[:, 3:67] != 0).any()
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    loss = balance_loss(e, torch.empty(0, 8, dtype=torch.int64, device="cuda"))
    assert loss.item() == 0 and torch.autograd.grad(loss, e)[0].shape == (0, 64)
    a = big[:, :64].clone().requires_grad_(True)
    loss = balance_loss(a, torch.full((50, 8), -1, device="cuda"), z_coeff=1.0)
    assert loss.item() == 0 and (torch.autograd.grad(loss, a)[0] == 0).all()


def test_stream_and_graph():
    """Routing and loss with their gradients captured: replays follow the logits of the moment; two graphs have their own scratch."""
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    bias = torch.rand(64, device="cuda") * 0.1
    kw = dict(score="sigmoid", bias=bias, num_groups=8, topk_groups=4, group_best=2)
    off = torch.tensor([0, 100, 333], dtype=torch.int32, device="cuda")

    def step(a):
        idx, w = route(a, 8, **kw)
        loss = balance_loss(a, idx, score="sigmoid", seq_off=off)
        return (idx, w.detach(), loss.detach(), *torch.autograd.grad(w.square().sum() + loss, a))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(s):
        for _ in range(2):
            a = torch.randn(333, 64, device="cuda").requires_grad_(True)
            step(a)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = step(a)
            graphs.append((graph, a, out))
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(2):
        for _, a, _ in graphs:
            with torch.no_grad():
                a.copy_(torch.randn_like(a))
        for graph, _, _ in graphs:
            graph.replay()
        for _, a, out in graphs:
            want = step(a.detach().clone().requires_grad_(True))
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_offsets_beyond_32_bits():
    """More logits than 32 bits count: the last rows are what they are by themselves."""
    from gpu_data_transfer_profile_b200.ops.router import balance_loss, route
    T, E = (1 << 31) // 1024 + 300, 1024
    l = torch.empty(T, E, dtype=BF16, device="cuda").normal_()
    tail = l[-400:].clone()
    kw = dict(score="sigmoid", num_groups=8, topk_groups=4, group_best=2)
    idx, w = route(l, 8, **kw)
    want = route(tail, 8, **kw)
    assert torch.equal(idx[-400:], want[0]) and torch.equal(w[-400:], want[1])
    off = torch.tensor([T - 400, T], dtype=torch.int32, device="cuda")
    # (the same sums of 64 bits, in other CTAs)
    assert balance_loss(l, idx, score="sigmoid", seq_off=off).item() == pytest.approx(balance_loss(tail, want[0], score="sigmoid").item(), rel=1e-6)
    del idx, w
    l.requires_grad_(True)
    idx, w = route(l, 8, **kw)
    g = torch.autograd.grad(w, l, torch.ones_like(w))[0]
    t = tail.requires_grad_(True)
    assert torch.equal(g[-400:], torch.autograd.grad(route(t, 8, **kw)[1], t, torch.ones(400, 8, device="cuda"))[0])
    del g, w
    g = torch.autograd.grad(balance_loss(l, idx, score="sigmoid", seq_off=off), l)[0]
    assert (g[:1000] == 0).all() and g[-400:].float().norm() > 0 and g[-401].abs().max() == 0


def test_balance_loss_of_the_most_rows():
    """As many rows as an int counts, one expert: every share is 1 and so is the loss."""
    from gpu_data_transfer_profile_b200.ops.router import balance_loss
    T = (1 << 31) - 1
    l = torch.zeros(T, 1, dtype=F16, device="cuda", requires_grad=True)
    idx = torch.zeros(T, 1, dtype=torch.int64, device="cuda")
    loss = balance_loss(l, idx)
    # 1 / T in 32 bits, a share and a count over T likewise: a rounding each, their products one more; the sum is in 64 bits
    assert abs(loss.item() - 1) <= 6 * U
    d, = torch.autograd.grad(loss, l)
    assert d.shape == l.shape and d[::4099].abs().max() == 0 and d[-5:].abs().max() == 0
