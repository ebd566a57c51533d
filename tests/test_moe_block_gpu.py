"""The MoE layer with its norm, its choice of experts and the balance loss, as they are used together, on one GPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

GROUPED = dict(score="sigmoid", num_groups=4, topk_groups=2, group_best=2, renormalize=True, route_scale=2.5, expert_bias=True)


@pytest.fixture
def world():
    from gpu_data_transfer_profile_b200.models import fused_a2a as A
    from gpu_data_transfer_profile_b200.parallel.symm import LocalWorld
    A.configure_buffer(num_max_tokens_per_rank=256, num_topk=4, num_experts=16, group_by_expert=True)
    yield LocalWorld.make(1)[0]
    A.release_buffers()


def _layer(world, H=256, F=256, E=16, K=4, dtype=torch.bfloat16, **kw):
    from gpu_data_transfer_profile_b200.models.moe_layer import MoELayer
    torch.manual_seed(0)
    layer = MoELayer(H, F, E, K, None, dtype=dtype, world=world, expert_backend="torch" if dtype == torch.float32 else "tcgen05", **kw)
    if layer.expert_bias is not None:
        layer.expert_bias.uniform_(-0.1, 0.1)
    if layer.norm_weight is not None:
        with torch.no_grad():
            layer.norm_weight.uniform_(0.5, 1.5)
    with torch.no_grad():
        layer.router.weight.mul_(5)
    return layer


def _reference(layer, x, logits, residual, off):
    """In the layer's own arithmetic type, every step written out: (output, sum, loss, idx)."""
    E, K, c = layer.num_experts, layer.topk, layer._choice
    h = x if residual is None else x + residual
    if layer.norm_weight is not None:
        n = h.float() * torch.rsqrt(h.float().square().mean(-1, keepdim=True) + layer.norm_eps) * layer.norm_weight.float()
    else:
        n = h
    l = layer.router(n.float()) if logits is None else logits
    live = (l > -math.inf).any(1, keepdim=True)
    safe = torch.where(live, l, torch.zeros_like(l))
    s = torch.sigmoid(safe) if c["score"] == "sigmoid" else torch.softmax(safe, -1)
    s = s * live
    v = s if layer.expert_bias is None else s + layer.expert_bias
    v = torch.where(l == -math.inf, -math.inf, v.double())
    if c["num_groups"] > 1:
        g = v.view(-1, c["num_groups"], E // c["num_groups"])
        value = g.topk(c["group_best"], -1).values.nan_to_num(neginf=0).sum(-1)
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, value.topk(c["topk_groups"], -1).indices, True)
        v = torch.where(keep[..., None], g, -math.inf).view(-1, E)
    top = v.topk(K, -1)
    idx = torch.where(top.values == -math.inf, -1, top.indices)
    w = torch.where(idx >= 0, s.gather(1, idx.clamp_min(0)), 0.0)
    if c["renormalize"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    w = w * c["scale"]
    out = torch.zeros_like(x, dtype=torch.float32)
    w1, w2 = layer.experts.weight1, layer.experts.weight2
    for e in range(E):
        hit = idx == e
        rows = hit.any(1).nonzero()[:, 0]
        if rows.numel():
            gate, lin = (n[rows].float() @ w1[e].float().t()).chunk(2, -1)
            act = torch.nn.functional.silu(gate) * lin * (w * hit).sum(1)[rows][:, None]
            out = out.index_add(0, rows, act @ w2[e].float().t())
    loss = None
    if layer._balance is not None:
        b = layer._balance
        cuts = [0, x.shape[0]] if off is None else off.tolist()
        terms = []
        for lo, hi in zip(cuts, cuts[1:]):
            rows = torch.arange(lo, hi, device=x.device)[(idx[lo:hi] >= 0).any(1)]
            if rows.numel():
                p = s[rows] / s[rows].sum(1, keepdim=True)
                f = torch.bincount(idx[rows][idx[rows] >= 0], minlength=E).float() * E / (K * rows.numel())
                t = b["coeff"] * (f * p.mean(0)).sum()
                terms.append(t + b["z_coeff"] * torch.logsumexp(l[rows], -1).square().mean() if b["z_coeff"] else t)
        loss = torch.stack(terms).mean()
    return out, h, loss, idx


@pytest.mark.parametrize("mode", ["fused", "deepep"])
@pytest.mark.parametrize("kw", [
    dict(norm=True, balance_coeff=0.5, **GROUPED),
    dict(norm=True, balance_coeff=0.5, z_coeff=0.01, renormalize=False),
    dict(score="sigmoid", balance_coeff=1.0), dict(num_groups=4, topk_groups=2), dict(norm=True)])
def test_training_step_against_every_step_written_out(world, kw, mode):
    layer = _layer(world, dtype=torch.float32, dispatcher_mode=mode, **kw)
    T = 96
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(T, 256, generator=g, device="cuda", requires_grad=True)
    r = torch.randn(T, 256, generator=g, device="cuda", requires_grad=True) if layer.norm_weight is not None else None
    off = torch.tensor([0, 10, 40, 90], dtype=torch.int32, device="cuda") if kw.get("balance_coeff") else None
    more = dict(residual=r) if r is not None else {}
    out = layer(x, seq_off=off, **more)
    out, h = out if r is not None else (out, None)
    ref, href, loss, _ = _reference(layer, x, None, r, off)
    torch.testing.assert_close(out, ref, atol=2e-4, rtol=2e-4)
    go, gh = torch.randn_like(out), torch.randn_like(out)
    total, want = (out * go).sum(), (ref * go).sum()
    if r is not None:
        torch.testing.assert_close(h, href)
        total, want = total + (h * gh).sum(), want + (href * gh).sum()
    if loss is not None:
        torch.testing.assert_close(layer.aux_loss, loss, atol=1e-5, rtol=1e-5)
        total, want = total + 100 * layer.aux_loss, want + 100 * loss
    else:
        assert layer.aux_loss is None
    leaves = [x, layer.router.weight, layer.experts.weight1, layer.experts.weight2] + ([r, layer.norm_weight] if r is not None else [])
    for a, b in zip(torch.autograd.grad(total, leaves), torch.autograd.grad(want, leaves)):
        # 32-bit products of up to 256 terms in other orders, through four of them
        torch.testing.assert_close(a, b, atol=2e-4 * max(1.0, b.abs().max().item()), rtol=2e-3)


@pytest.mark.parametrize("kw", [dict(norm=True, **GROUPED), dict(GROUPED), dict(norm=True, score="softmax", renormalize=False, num_groups=4, topk_groups=1), dict(norm=True)])
@pytest.mark.parametrize("fuse", [True, False])
def test_inference_against_every_step_written_out(world, kw, fuse):
    """bf16, tensor-core experts, rows consumed in place; the same layer with gradients goes the general way."""
    layer = _layer(world, fuse_combine=fuse, balance_coeff=0.1, **kw)
    T = 130
    x, r = (torch.randn(T, 256, device="cuda").to(torch.bfloat16) for _ in range(2))
    more = dict(residual=r) if layer.norm_weight is not None else {}
    with torch.no_grad():
        got = layer(x, **more)
        assert layer.aux_loss is None
    ref = _reference(layer, x, None, r if more else None, None)
    train = layer(x, **more)
    assert layer.aux_loss is not None
    if more:
        torch.testing.assert_close(got[1], ref[1], atol=0, rtol=2.0 ** -7)
        got, train = got[0], train[0]
    # (a token on the border between two experts may choose the other one: rows of the norm in bf16 or f32 differ)
    bad = ~torch.isclose(got.float(), ref[0], atol=4e-2, rtol=4e-2).all(1)
    assert bad.sum() <= 3
    bad = ~torch.isclose(got.float(), train.float(), atol=4e-2, rtol=4e-2).all(1)
    assert bad.sum() <= 1


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("fuse", [True, False])
@pytest.mark.parametrize("none", [False, True])
def test_padding_rows_reach_no_expert(world, grad, fuse, none):
    layer = _layer(world, fuse_combine=fuse, balance_coeff=1.0, **GROUPED)
    T, E = 100, 16
    x = torch.randn(T, 256, device="cuda").to(torch.bfloat16).requires_grad_(grad)
    logits = torch.randn(T, E, device="cuda")
    logits[60:] = -math.inf                                        # padding
    logits[5, 2:] = -math.inf                                      # two experts for four choices
    if none:
        logits[:] = -math.inf
    logits.requires_grad_(grad)
    with torch.set_grad_enabled(grad):
        out = layer(x, logits)
        again = layer(x, logits)
    assert torch.equal(out, again) and (out[60:] == 0).all()
    ref, _, loss, idx = _reference(layer, x, logits, None, None) if not none else (torch.zeros_like(out).float(), None, None, None)
    torch.testing.assert_close(out.float(), ref, atol=4e-2, rtol=4e-2)
    if grad and not none:
        torch.testing.assert_close(layer.aux_loss, loss, atol=1e-5, rtol=1e-5)
        g = torch.randn_like(out)
        gx, gl = torch.autograd.grad((out * g).sum() + layer.aux_loss, (x, logits))
        rx, rl = torch.autograd.grad((ref * g.float()).sum() + loss, (x, logits))
        assert (gl[60:] == 0).all() and (gx[60:] == 0).all()
        torch.testing.assert_close(gx.float(), rx.float(), atol=4e-2, rtol=4e-2)
        torch.testing.assert_close(gl, rl.nan_to_num(0), atol=4e-2, rtol=4e-2)


@pytest.mark.parametrize("T", [1, 37, 200])
def test_fp8_rows_of_the_norm_go_straight_into_the_exchange(world, T, monkeypatch):
    from gpu_data_transfer_profile_b200.models import moe_layer as M
    layer = _layer(world, use_fp8=True, norm=True, **GROUPED)
    x, r = (torch.randn(T, 256, device="cuda").to(torch.bfloat16) for _ in range(2))
    calls = []
    real = M.N.rms_norm_fp8
    monkeypatch.setattr(M.N, "rms_norm_fp8", lambda *a, **k: calls.append(1) or real(*a, **k))
    with torch.no_grad():
        out, h = layer(x, residual=r)
    assert calls == [1]
    assert torch.equal(h, (x.float() + r.float()).to(torch.bfloat16))
    ref, _, _, _ = _reference(layer, x, None, r, None)
    # e4m3 rows and weights: 2^-4 each of products that average out over 256 terms; tokens that chose another expert aside
    err = (out.float() - ref).norm(dim=1) / ref.norm(dim=1)
    assert (err < 0.12).float().mean() >= 0.97


@pytest.mark.parametrize("T", [1, 37, 200])
@pytest.mark.parametrize("residual", [False, True])
def test_fp8_rows_of_the_norm_with_the_default_choice(world, T, residual, monkeypatch):
    """Without options that may leave a choice out, a group of one takes the rows in place without the receive count."""
    from gpu_data_transfer_profile_b200.parallel.buffer import Buffer
    layer = _layer(world, use_fp8=True, norm=True)
    x, r = (torch.randn(T, 256, device="cuda").to(torch.bfloat16) for _ in range(2))
    seen = []
    real = Buffer._dispatch_own_probs
    monkeypatch.setattr(Buffer, "_dispatch_own_probs", lambda self, rows, *a: seen.append([t.dtype for t in rows]) or real(self, rows, *a))
    with torch.no_grad():
        out, h = layer(x, residual=r if residual else None)
    assert seen == [[torch.float8_e4m3fn, torch.float32]]
    assert torch.equal(h, (x.float() + r.float()).to(torch.bfloat16) if residual else x)
    ref, _, _, _ = _reference(layer, x, None, r if residual else None, None)
    err = (out.float() - ref).norm(dim=1) / ref.norm(dim=1)
    assert (err < 0.12).float().mean() >= 0.97                     # (as above)


def test_router_logits_kernel_against_64_bits():
    from gpu_data_transfer_profile_b200 import _ext
    C = _ext.load()
    for T, H, E in ((1, 8, 1), (3, 4096, 16), (130, 7168, 256), (4096, 512, 64), (0, 256, 16), (65, 136, 1000)):
        x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
        w = torch.randn(E, H, device="cuda") * 0.05
        got = C.router_logits(x, w)
        want, size = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
        # sums of H products one after the other in up to 32 parts, added in order: at most H + 32 roundings, 40 in the mean
        assert got.shape == (T, E) and ((got.double() - want).abs() <= size * (min(H, 400) + 32) * 2.0 ** -24).all()


def test_replaced_routers_and_refusals(world, monkeypatch):
    from gpu_data_transfer_profile_b200.models import moe_layer as M
    layer = _layer(world, **GROUPED)
    x = torch.randn(20, 256, device="cuda").to(torch.bfloat16)
    fixed = torch.arange(4, device="cuda").expand(20, 4).contiguous()
    with torch.no_grad():
        want = layer(x)
        monkeypatch.setattr(M, "topk_softmax_router", lambda l, k: (fixed, torch.full((20, 4), 0.25, device="cuda")))
        other = layer(x)
    assert not torch.equal(want, other)
    with pytest.raises(ValueError):
        layer(x, residual=x)
    for kw in (dict(score="relu"), dict(score="sigmoid", z_coeff=0.1)):
        with pytest.raises(ValueError):
            M.MoELayer(256, 256, 16, 4, None, world=world, expert_backend="tcgen05", **kw)


def test_state_of_a_default_layer_is_what_it_was(world):
    layer = _layer(world)
    assert sorted(layer.state_dict()) == ["experts.weight1", "experts.weight2", "router.weight"]
    assert sorted(_layer(world, norm=True, **GROUPED).state_dict()) == ["expert_bias", "experts.weight1", "experts.weight2", "norm_weight", "router.weight"]


@pytest.mark.parametrize("R", [1, 2, 4])
@pytest.mark.parametrize("fp8", [True, False])
def test_norm_choice_exchange_over_ranks(R, fp8):
    """Rows of the norm and ids and weights of the choice, padding among them, through an exchange by expert and back: a
    token comes back as itself times the sum of its weights, each times what tells its expert."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    from gpu_data_transfer_profile_b200.ops.router import route
    from gpu_data_transfer_profile_b200.parallel.local import LocalGroup
    H, E, K = 512, 16, 4
    g = LocalGroup(R, 64 << 20, timeout_s=2.0)
    try:
        gen = torch.Generator(device="cuda").manual_seed(R)
        xs, ids, ws, dense = [], [], [], []
        for r in range(R):
            T = 60 + 13 * r
            x, h = (torch.randn(T, H, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
            w = 1 + 0.2 * torch.randn(H, generator=gen, device="cuda")
            l = torch.randn(T, E, generator=gen, device="cuda")
            l[T - 7:] = -math.inf
            l[3, 2:] = -math.inf
            idx, wt = route(l, K, score="sigmoid", bias=torch.linspace(-0.1, 0.1, E, device="cuda"), num_groups=4, topk_groups=2, group_best=2, scale=2.5)
            if fp8:
                (q, s), _, _ = rms_norm_fp8(x, w, residual=h)
                xs.append((q, s))
                dense.append((q.double().view(T, H // 128, 128) * s.double()[..., None]).view(T, H))
            else:
                xs.append(rms_norm(x, w, residual=h)[0])
                dense.append(xs[-1].double())
            ids.append(idx)
            ws.append(wt)
        outs = g.dispatch(xs, topk_idx=ids, topk_weights=ws, group_by_expert=True, num_experts=E)
        ys = []
        for r, (rows, _, _, counts, handle) in enumerate(outs):
            el = torch.arange(E // R, device="cuda") + r * (E // R) + 1.0
            factor = torch.repeat_interleave(el, torch.tensor(counts, device="cuda")) * handle.recv_prob
            n = factor.numel()
            assert n == sum(int(((i >= r * (E // R)) & (i < (r + 1) * (E // R))).sum()) for i in ids)
            got = (rows[0].float().view(-1, H // 128, 128) * rows[1][..., None]).view(-1, H) if fp8 else rows.float()
            ys.append((got[:n] * factor[:, None]).to(torch.bfloat16))
        comb = g.combine(ys, [o[4] for o in outs])
        for r in range(R):
            gain = (ws[r].double() * (ids[r] + 1) * (ids[r] >= 0)).sum(1, keepdim=True)
            want = dense[r] * gain
            # a rounding to bf16 of every row, and one of their sum
            assert ((comb[r][0].double() - want).abs() <= dense[r].abs() * gain * 2.02 * 2.0 ** -8).all()
            assert (comb[r][0][-7:] == 0).all()
        g.check_status()
    finally:
        g.destroy()
