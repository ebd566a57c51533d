"""Root-mean-square norm with the residual's addition against 64 bits."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U_F32 = 2.0 ** -24


def _half(dt):
    """Largest relative error of one rounding to dt."""
    return torch.finfo(dt).eps / 2


def _inputs(shape, dt, wdt, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda").to(dt)
    r = (2 * torch.randn(shape, generator=g, device="cuda")).to(dt) if residual else None
    w = (1 + 0.3 * torch.randn(shape[-1], generator=g, device="cuda")).to(wdt)
    return x, r, w


def _wide(x, w, r, eps):
    h = x.double() + r.double() if r is not None else x.double()
    return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.double(), h


def _close(got, want, dt):
    """One rounding to dt and 48 of 32-bit arithmetic: a thread adds up to 72 squares one after the other and a tree of 10
    levels joins them, half of that is in the root, and 5 roundings follow. (A smallest denormal step of dt beside them.)"""
    assert got.dtype == dt and got.shape == want.shape
    tol = want.abs() * (_half(dt) * (1 + _half(dt)) + 48 * _half(F32)) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    bad = ((got.double() - want).abs() > tol)
    assert not bad.any(), ((got.double() - want).abs() / tol).max()


# vectors of a row: a warp's (1, 2, 4 vectors a lane), a CTA's (2, 4, 9 a thread), partial vectors at both ends
WIDTHS = [1, 2, 7, 8, 33, 100, 128, 255, 256, 264, 511, 512, 1000, 1024, 1031, 1407, 2048, 4096, 7168, 7169, 8192, 16384, 16391, 32767, 32768]


@pytest.mark.parametrize("dt,wdt", [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("H", WIDTHS)
def test_forward(H, dt, wdt):
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    for T, residual in itertools.product((1, 19), (False, True)):
        x, r, w = _inputs((T, H), dt, wdt, residual, seed=H + T)
        want, h = _wide(x, w, r, 1e-6)
        if residual:
            y, hs = rms_norm(x, w, residual=r)
            _close(hs, h, dt)
        else:
            y = rms_norm(x, w)
        _close(y, want, dt)


@pytest.mark.parametrize("T", [0, 1, 2, 3, 8, 147, 297, 4099])
@pytest.mark.parametrize("H,dt", [(96, F32), (1407, F16), (2056, BF16)])
def test_forward_rows(T, H, dt):
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    x, r, w = _inputs((T, H), dt, dt, True, seed=T)
    y, hs = rms_norm(x, w, residual=r, eps=1e-3)
    want, h = _wide(x, w, r, 1e-3)
    _close(y, want, dt)
    _close(hs, h, dt)


def test_forward_strides_and_dimensions():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    x, _, w = _inputs((3, 5, 40, 264), BF16, F32, False)
    _close(rms_norm(x, w), _wide(x, w, None, 1e-6)[0], BF16)
    wide = _inputs((37, 1000), BF16, BF16, False)[0]
    for view in (wide[:, :264], wide[:, 8:272], wide[:, 3:267], wide[1:, 1:265], wide[::2, :264], wide[:1, 5:269], wide[:, :264].t()[:, :].t(),
                 wide[:5, 16:17].expand(5, 264), wide[:1, :264].expand(9, 264), x.transpose(0, 2), wide[:, 0:528:2]):
        _close(rms_norm(view, w), _wide(view, w, None, 1e-6)[0], BF16)
        y, h = rms_norm(view, w[:].clone(), residual=view.clone())
        want, hw = _wide(view, w, view, 1e-6)
        _close(y, want, BF16)
        _close(h, hw, BF16)
    odd = _inputs((11, 1409), F16, F16, False)[0]
    w2 = _inputs((1, 1410), F16, F16, False)[2]
    for view in (odd[:, 1:1408], odd[1:, :1407], odd[:, :1401], odd[2:]):
        n = view.shape[1]
        _close(rms_norm(view, w2[1:1 + n]), _wide(view, w2[1:1 + n], None, 1e-6)[0], F16)


def test_forward_extremes():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    w = torch.ones(512, device="cuda", dtype=BF16)
    x = torch.zeros(4, 512, device="cuda", dtype=BF16)
    assert torch.equal(rms_norm(x, w), x)                          # zeros over sqrt(eps)
    assert rms_norm(x, w, eps=0.0).isnan().all()                   # 0 / 0
    x[1] = 1e15                                                    # squares up to 5e32: below the largest f32
    x[2, 7] = math.nan
    x[3, 9] = math.inf
    y = rms_norm(x, w)
    assert (y[1] == 1).all() and y[2].isnan().all() and y[3, 9].isnan() and (y[3, 10:] == 0).all()


@pytest.mark.parametrize("dt,wdt", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32), (F32, F16)])
@pytest.mark.parametrize("H", [1, 7, 128, 255, 512, 1031, 1407, 4096, 7168, 8191, 16384, 32767, 32768])
def test_gradients(H, dt, wdt):
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    for T, residual in ((1, True), (37, False), (700, True) if H < 9000 else (9, True)):
        x, r, w = _inputs((T, H), dt, wdt, residual, seed=H)
        g = torch.Generator(device="cuda").manual_seed(7)
        dy, dh = (torch.randn(T, H, generator=g, device="cuda").to(dt) for _ in range(2))
        leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]
        wide = [t.detach().double().requires_grad_(True) for t in leaves]
        out = rms_norm(x, w, residual=r, eps=1e-5)
        want = _wide(wide[0], wide[1], wide[2] if residual else None, 1e-5)
        if residual:
            got = torch.autograd.grad(out, leaves, (dy, dh))
            ref = torch.autograd.grad(want, wide, (dy.double(), dh.double()))
            assert torch.equal(got[0], got[2])
        else:
            got = torch.autograd.grad(out, leaves, dy)
            ref = torch.autograd.grad(want[0], wide, dy.double())
        # dx is a difference of terms of the size of |a| and |n| |mean(a n)|, the mean a sum of up to 72 products one after the
        # other and a tree of 10 levels; h enters n as it is stored (with a residual and 16-bit weights: one
        # rounding of h to dt, as far as n mean(a n), a n within the mean and their products carry it)
        h = want[1].detach()
        rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5)
        a, n = dy.double() * w.detach().double(), h * rstd
        c = (a * n).mean(-1, keepdim=True)
        size = rstd * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True)) + (dh.double().abs() if residual else 0)
        kept = residual and (wdt != F32 or dt == F32)
        stored = _half(dt) * rstd * n.abs() * (c.abs() + (a * n).abs().mean(-1, keepdim=True)) if kept else 0
        tol = ref[0].abs() * _half(dt) * 1.01 + stored * 1.01 + size * 90 * _half(F32)
        if dt == F16:
            tol = tol + 2.0 ** -25
        assert ((got[0].double() - ref[0]).abs() <= tol).all()
        # dw: T products, each off by the rounding of h at most, summed in 32 bits: T / 148 in a thread, 8 warps, then up to 600
        # parts in 8 strands
        terms = (dy.double() * n).abs().sum(0)
        tol = ref[1].abs() * _half(wdt) * 1.01 + terms * ((_half(dt) * 1.01 if kept else 0) + (100 + math.ceil(T / 148)) * _half(F32))
        if wdt == F16:
            tol = tol + 2.0 ** -25
        assert got[1].dtype == wdt and ((got[1].double() - ref[1]).abs() <= tol).all()


@pytest.mark.parametrize("dt,wdt", [(BF16, BF16), (F16, F16), (BF16, F16)])
@pytest.mark.parametrize("T,H", [(1, 256), (700, 512), (4096, 1024), (333, 1407), (900, 7168), (5, 32768)])
def test_gradients_of_16_bit_weights_are_rounded_once(T, H, dt, wdt):
    """With a residual: x and residual, not their stored sum, are what was normalised."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    x, r, w = _inputs((T, H), dt, wdt, True, seed=H)
    g = torch.Generator(device="cuda").manual_seed(8)
    dy, dh = (torch.randn(T, H, generator=g, device="cuda").to(dt) for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    got = torch.autograd.grad(rms_norm(x, w, residual=r, eps=1e-5), leaves, (dy, dh))
    yw, hw = _wide(*wide, 1e-5)
    ref = torch.autograd.grad((yw, hw), wide, (dy.double(), dh.double()))
    h = hw.detach()
    rstd = torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    a, n = dy.double() * w.detach().double(), h * rstd
    size = rstd * (a.abs() + n.abs() * (a * n).abs().mean(-1, keepdim=True)) + dh.double().abs()
    tiny = 2.0 ** -25 if F16 in (dt, wdt) else 0
    assert ((got[0].double() - ref[0]).abs() <= ref[0].abs() * _half(dt) * 1.01 + size * 90 * U_F32 + tiny).all()
    # T products, each of four roundings in 32 bits, summed T / 148 in a thread, by 8 warps and in up to 600 parts in 8 strands
    terms = (dy.double() * n).abs().sum(0)
    assert ((got[1].double() - ref[1]).abs() <= ref[1].abs() * _half(wdt) * 1.01 + terms * (100 + math.ceil(T / 148)) * U_F32 + tiny).all()


def test_gradient_against_differences():
    """Directional differences of the forward in 32 bits: d/ds f(x + s u) = <grad, u>."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    x, r, w = _inputs((5, 77), F32, F32, True)
    g = torch.Generator(device="cuda").manual_seed(3)
    dy, dh, ux, ur = (torch.randn(5, 77, generator=g, device="cuda") for _ in range(4))
    uw = torch.randn(77, generator=g, device="cuda")

    def f(s):
        y, h = rms_norm(x + s * ux, w + s * uw, residual=r + s * ur)
        return (y.double() * dy).sum() + (h.double() * dh).sum()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, h = rms_norm(leaves[0], leaves[1], residual=leaves[2])
    gx, gw, gr = torch.autograd.grad((y, h), leaves, (dy, dh))
    got = ((gx * ux).sum() + (gw * uw).sum() + (gr * ur).sum()).double()
    s = 2.0 ** -7
    want = (f(s) - f(-s)) / (2 * s)
    # third derivatives of order 10 a term times s^2 / 6, summed in quadrature over 2 * 385 terms of order 1; 32-bit rounding / s
    assert abs(got - want) < 10 * s * s / 6 * 30 + 800 * 2.0 ** -22 / s


def test_gradients_of_parts():
    """Outputs and inputs that are not asked for, strided and broadcast gradients, a frozen weight, a second backward."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    x, r, w = _inputs((33, 520), F32, F32, True)
    x.requires_grad_(True), r.requires_grad_(True), w.requires_grad_(True)
    wide = [t.detach().double().requires_grad_(True) for t in (x, r, w)]

    def both(loss):
        y, h = rms_norm(x, w, residual=r)
        yw, hw = _wide(wide[0], wide[2], wide[1], 1e-6)
        a = torch.autograd.grad(loss(y, h), (x, r, w), allow_unused=True)
        b = torch.autograd.grad(loss(yw, hw), wide, allow_unused=True)
        for p, q in zip(a, b):
            torch.testing.assert_close(p, torch.zeros_like(p) if q is None else q.float(), atol=2e-5, rtol=2e-5)
    both(lambda y, h: y.sum())                                     # an expanded scalar as gradient
    both(lambda y, h: h.square().sum())                            # y is not used: the weight's gradient is zero
    both(lambda y, h: (y * y).sum() + h.sum())
    both(lambda y, h: (y.t() * torch.arange(33, device="cuda")).sum() + h[3:5].sum())
    y, h = rms_norm(x, w.detach(), residual=r.detach())
    gx, = torch.autograd.grad((y.sum() + h.sum()), x, retain_graph=True)
    again, = torch.autograd.grad((y.sum() + h.sum()), x)
    assert torch.equal(gx, again)
    y = rms_norm(x.detach(), w)
    gw, = torch.autograd.grad(y.sum(), w)
    yw, _ = _wide(wide[0].detach(), wide[2], None, 1e-6)
    torch.testing.assert_close(gw, torch.autograd.grad(yw.sum(), wide[2])[0].float(), atol=2e-5, rtol=2e-5)
    empty = torch.empty(0, 520, device="cuda", requires_grad=True)
    gx, gw = torch.autograd.grad(rms_norm(empty, w).sum(), (empty, w))
    assert gx.shape == (0, 520) and (gw == 0).all()


def test_gradients_are_the_same_bits_again():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    x, r, w = _inputs((3001, 1407), BF16, F32, True)
    x.requires_grad_(True), w.requires_grad_(True)
    runs = []
    for _ in range(3):
        y, h = rms_norm(x, w, residual=r)
        runs.append(torch.autograd.grad((y, h), (x, w), (r, r)))
    for a in runs[1:]:
        assert all(torch.equal(p, q) for p, q in zip(a, runs[0]))


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("H", [128, 256, 384, 1024, 4096, 7168, 7296, 16512, 32768])
def test_fp8(H, dt):
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm_fp8
    for T, residual, keep in ((1, True, True), (9, False, False), (333, True, True)):
        x, r, w = _inputs((T, H), dt, F32, residual, seed=T)
        w[:128] = 0                                                # a block of zeros: the least scale
        (q, s), y, h = rms_norm_fp8(x, w, residual=r, keep=keep)
        want, hw = _wide(x, w, r, 1e-6)
        assert q.dtype == torch.float8_e4m3fn and q.shape == (T, H) and s.shape == (T, H // 128) and (y is not None) == keep and (h is not None) == residual
        blocks = want.view(T, H // 128, 128)
        scale = blocks.abs().amax(-1).clamp_min(1e-4) / 448
        torch.testing.assert_close(s.double(), scale, atol=0, rtol=50 * _half(F32))
        got = q.float().double().view_as(blocks) * s.double()[..., None]
        # one rounding to e4m3: 2^-4 of the value, 2^-10 of a scale below its smallest normal number
        tol = blocks.abs() * (2.0 ** -4 + 120 * _half(F32)) + scale[..., None] * 2.0 ** -10 * 1.001
        assert ((got - blocks).abs() <= tol).all()
        if keep:
            _close(y, want, dt)                                    # (rms_norm's may be another of two neighbours: other lanes sum the squares)
        if residual:
            _close(h, hw, dt)


@pytest.mark.parametrize("dt,wdt", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("size", [1e-36, 4e35, 5e37])
def test_fp8_of_very_small_and_very_large_weights(size, dt, wdt):
    """Blocks whose largest value lies above 2^126 (8.5e37) and near the largest number of 32 bits."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm_fp8
    x, _, w = _inputs((60, 512), dt, wdt, False, seed=3)
    w = (w.float() * size).to(wdt)
    x[5, 7] = 100.0                                                # 16 times the others: up to 3e38
    (q, s), y, _ = rms_norm_fp8(x, w, keep=True)
    want, _ = _wide(x, w, None, 1e-6)
    blocks = want.view(60, 4, 128)
    amax = blocks.abs().amax(-1)
    fits = amax < torch.finfo(F32).max * (1 - 50 * _half(F32))      # (the others are infinite in 32 bits, and so are their scales)
    assert fits.float().mean() > 0.9 and (size < 1e37 or (amax[fits] > 1.5e38).any())
    scale = amax.clamp_min(1e-4) / 448
    torch.testing.assert_close(s.double()[fits], scale[fits], atol=0, rtol=50 * _half(F32))
    assert (s[amax > torch.finfo(F32).max * (1 + 50 * _half(F32))] == math.inf).all()
    got = q.float().double().view_as(blocks) * s.double()[..., None]
    tol = blocks.abs() * (2.0 ** -4 + 120 * _half(F32)) + scale[..., None] * 2.0 ** -10 * 1.001
    assert ((got - blocks).abs() <= tol)[fits].all()


def test_fp8_of_infinities_and_nan():
    """What is not a number stays that, and takes no part in its block's scale; an infinite block has an infinite scale."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm_fp8
    x = torch.randn(4, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    x[1, 3] = math.nan                                             # the row's root is none
    x[2, 130] = math.inf                                           # the row's root is 0: the others become 0
    (q, s), y, _ = rms_norm_fp8(x, w, keep=True)
    v = q.float()
    assert v[1].isnan().all() and (s[1:3] == torch.tensor(1e-4, device="cuda") * (1 / 448)).all()
    assert v[2, 130].isnan() and (v[2, :130] == 0).all() and (v[2, 131:] == 0).all() and y[2, 130].isnan()
    clean = rms_norm_fp8(x[[0, 3]], w)[0]
    assert torch.equal(q[[0, 3]].view(torch.uint8), clean[0].view(torch.uint8)) and torch.equal(s[[0, 3]], clean[1])
    w[5], w[200] = math.nan, math.inf
    (q, s), _, _ = rms_norm_fp8(x[:1], w)
    v = q.float()
    other = torch.arange(256, device="cuda") != 5
    want, _ = _wide(x[:1], torch.ones(256, device="cuda"), None, 1e-6)
    assert v[0, 5].isnan() and v[0, :128][other[:128]].isfinite().all() and s[0, 1] == math.inf
    torch.testing.assert_close(s[0, 0].double(), want[0, :128][other[:128]].abs().max() / 448, atol=0, rtol=50 * _half(F32))


def test_more_dimensions_and_a_tensor_given_twice():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    x, r, w = _inputs((2, 3, 5, 384), BF16, F32, True)
    (q, s), y, h = rms_norm_fp8(x, w, residual=r, keep=True)
    (q2, s2), y2, h2 = rms_norm_fp8(x.view(30, 384), w, residual=r.view(30, 384), keep=True)
    assert q.shape == x.shape and s.shape == (2, 3, 5, 3) and torch.equal(q.view(torch.uint8).view(30, 384), q2.view(torch.uint8))
    assert torch.equal(s.view(30, 3), s2) and torch.equal(y.view(30, 384), y2) and torch.equal(h.view(30, 384), h2)
    a = torch.randn(4, 6, 100, device="cuda").transpose(0, 1).requires_grad_(True)
    wide = a.detach().double().requires_grad_(True)
    w = torch.ones(100, device="cuda")
    y, h = rms_norm(a, w, residual=a)
    yw, hw = _wide(wide, w, wide, 1e-6)
    got, ref = torch.autograd.grad((y * y * h).sum(), a)[0], torch.autograd.grad((yw * yw * hw).sum(), wide)[0]
    # products of three numbers below 10 and a mean of 100 of them: 32-bit roundings of some hundreds
    assert got.shape == a.shape and ((got.double() - ref).abs() <= 1000 * 100 * U_F32).all()


def test_fp8_rows_feed_the_grouped_gemm():
    from gpu_data_transfer_profile_b200.ops import gemm as G
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm_fp8
    x, r, w = _inputs((70, 512), BF16, BF16, True)
    (q, s), y, _ = rms_norm_fp8(x, w, residual=r, keep=True)
    wq, ws = G.quantize_weights_128x128(torch.randn(2, 256, 512, device="cuda") * 0.05)
    off = G.offsets_from_counts([30, 40], "cuda")
    got = G.grouped_gemm_fp8(q, s, wq, ws, off)
    dense = (q.double().view(70, 4, 128) * s.double()[..., None]).view(70, 512)
    we = G.dequantize_weights_128x128(wq, ws).double()
    want = torch.cat([dense[:30] @ we[0].t(), dense[30:] @ we[1].t()])
    size = torch.cat([dense[:30].abs() @ we[0].abs().t(), dense[30:].abs() @ we[1].abs().t()])
    # one rounding to bf16, and 32-bit sums of 512 products in the tensor core (2^-13 of the sum of their sizes)
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 + size * 2.0 ** -13).all()


def test_widths_in_turn_and_two_threads():
    """One kernel serves several widths, with and without a residual: every call is launched by its own sizes."""
    import threading
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm
    calls = []
    for H, residual in ((7168, True), (1536, True), (7168, False), (4096, True), (1536, False)):
        x, r, w = _inputs((611, H), BF16, BF16, residual, seed=H)
        calls.append((x, r, w, rms_norm(x, w, residual=r)))
    torch.cuda.synchronize()
    bad = []

    def work(order):
        with torch.cuda.stream(torch.cuda.Stream()):
            for k in range(60):
                x, r, w, want = calls[(k * order) % len(calls)]
                got = rms_norm(x, w, residual=r)
                same = torch.equal(got, want) if r is None else torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
                if not same:
                    bad.append((k, x.shape, r is None))
    threads = [threading.Thread(target=work, args=(o,)) for o in (1, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals():
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    x, r, w = _inputs((6, 256), BF16, BF16, True)
    for call in (lambda: rms_norm(x, w[:255]), lambda: rms_norm(x, w[None]), lambda: rms_norm(x.cpu(), w), lambda: rms_norm(x, w.cpu()),
                 lambda: rms_norm(x.double(), w), lambda: rms_norm(x, w.double()), lambda: rms_norm(x, w, residual=r.float()),
                 lambda: rms_norm(x, w, residual=r[:5]), lambda: rms_norm(x, w, residual=r.cpu()), lambda: rms_norm(x, w, eps=-1.0),
                 lambda: rms_norm(x, w, eps=math.nan), lambda: rms_norm(x[0, 0], w), lambda: rms_norm(x[:, :0], w[:0]),
                 lambda: rms_norm(torch.zeros(1, 32769, device="cuda"), torch.zeros(32769, device="cuda")),
                 lambda: rms_norm_fp8(x[:, :200], w[:200]), lambda: rms_norm_fp8(x.clone().requires_grad_(True), w),
                 lambda: torch.func.vmap(lambda t: rms_norm(t, w))(x[None]), lambda: torch.func.grad(lambda t: rms_norm(t, w).sum())(x),
                 lambda: rms_norm(x.to_sparse(), w)):
        with pytest.raises(RuntimeError):
            call()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for call in (lambda: rms_norm(dual, w), lambda: rms_norm(x, w, residual=dual), lambda: rms_norm_fp8(dual, w)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(rms_norm(x, w).sum(), x, create_graph=True)
    y = rms_norm(x, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, torch.stack([y.detach(), y.detach()]), is_grads_batched=True)
    with torch.no_grad():
        assert rms_norm_fp8(x, w)[0][0].shape == x.shape
    torch.cuda.synchronize()


def test_stream_and_graph():
    """On a stream of the caller's, and captured with its backward: replays see the inputs of the moment."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    x, r, w = _inputs((50, 1407), BF16, F32, True)
    x2 = _inputs((50, 1024), BF16, F32, False)[0]
    w2 = torch.ones(1024, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        xs = x.clone().requires_grad_(True)
        ws = w.clone().requires_grad_(True)
        for _ in range(2):
            y, h = rms_norm(xs, ws, residual=r)
            grads = torch.autograd.grad((y, h), (xs, ws), (r, r))
        del y, h, grads
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y, h = rms_norm(xs, ws, residual=r)
            grads = torch.autograd.grad((y, h), (xs, ws), (r, r))
            (q, sc), _, _ = rms_norm_fp8(x2, w2)
    torch.cuda.current_stream().wait_stream(s)
    for seed in (5, 6):
        nx = _inputs((50, 1407), BF16, F32, False, seed)[0]
        with torch.no_grad():
            xs.copy_(nx)
            x2.copy_(nx[:, :1024])
        graph.replay()
        a = nx.clone().requires_grad_(True)
        b = w.clone().requires_grad_(True)
        yr, hr = rms_norm(a, b, residual=r)
        want = torch.autograd.grad((yr, hr), (a, b), (r, r))
        assert torch.equal(y, yr) and torch.equal(h, hr) and all(torch.equal(p, q_) for p, q_ in zip(grads, want))
        (q2, s2), _, _ = rms_norm_fp8(x2, w2)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(sc, s2)


@pytest.mark.parametrize("H", [32768, 1407])
def test_offsets_beyond_32_bits(H):
    """More elements than 32 bits count: the last rows are what they are by themselves (in rows that begin at another place
    within 16 bytes other lanes sum, and a result may be the neighbouring one)."""
    from gpu_data_transfer_profile_b200.ops.norm import rms_norm, rms_norm_fp8
    T = (1 << 31) // H + 100
    x = torch.empty(T, H, dtype=BF16, device="cuda").normal_().requires_grad_(True)
    w = torch.ones(H, device="cuda", requires_grad=True)
    tail = x[-64:].detach().clone().requires_grad_(True)
    y = rms_norm(x, w)
    want = rms_norm(tail, w)
    _close(y[-64:].detach(), _wide(tail.detach(), w.detach(), None, 1e-6)[0], BF16)
    dx, dw = torch.autograd.grad(y, (x, w), x.detach().flip(0))
    dt = torch.autograd.grad(want, tail, x[:64].detach().flip(0))[0]
    # a value of its own size, one step of bf16 apart at most; where it cancels, 32-bit roundings of terms below 64
    assert ((dx[-64:].double() - dt.double()).abs() <= dt.double().abs() * 2.0 ** -7 + 64 * 100 * 2.0 ** -24).all() and dw.isfinite().all()
    del dx, y
    if H % 128 == 0:
        with torch.no_grad():
            (q, s), _, h = rms_norm_fp8(x, w, residual=x)
            (q2, s2), _, h2 = rms_norm_fp8(tail, w, residual=tail)
        assert torch.equal(q[-64:].view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s[-64:], s2) and torch.equal(h[-64:], h2)
