"""Layer normalisation (csrc/layernorm.hip, functional.layer_norm / layer_norm_channels, nn.LayerNorm) against the formulas in 64 bits.

Tolerances are worst-case rounding bounds.  With h = 2^-24 (half a step of fp32), a sum of n terms in any order is off by at most
n h sum|terms|; so over C features the mean is off by d_m = (C + 2) h mean|x|, the variance relatively by (C + 4) h and by d_m^2 (of
second order, below), rstd relatively by e_r = (C + 8) h + d_m^2 rstd^2, u = (x - mean) rstd by d_u = d_m rstd + |u| (e_r + 4 h), and
  y  by |w| d_u + 4 h (|u w| + |b|) + e |y|          (e: half a step of the type of y, 0 where that is fp32: counted in the 4 h)
  dx by rstd ((C + 8) h (|g| + mean|g| + 2 |u| mean|g u|) + d_u mean|g u| + |u| mean(|g| d_u)) + |dx| (e_r + 4 h + e),   g = dy w
  dw by (R + 8) h sum|dy u| + sum |dy| d_u + e |dw|,    db by (R + 4) h sum|dy| + e |db|."""
import math

import pytest
import torch

H = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


def reference(x, w, b, eps, dy=None):
    """[R, C] in fp64 -> values and their bounds as functions of the output types' half steps"""
    x, dy = x.double().cpu(), None if dy is None else dy.double().cpu()
    C = x.shape[1]
    w = torch.ones(C, dtype=torch.float64) if w is None else w.double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double().cpu()
    m = x.mean(1, keepdim=True)
    var = ((x - m) ** 2).mean(1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    u = (x - m) * r
    d_m = (C + 2) * H * x.abs().mean(1, keepdim=True)
    e_r = (C + 8) * H + d_m ** 2 * r ** 2
    d_u = d_m * r + u.abs() * (e_r + 4 * H)
    y = u * w + b
    out = {"y": (y, lambda e: w.abs() * d_u + 4 * H * ((u * w).abs() + b.abs()) + e * y.abs())}
    if dy is not None:
        g = dy * w
        gu = (g * u).abs().mean(1, keepdim=True)
        dx = r * (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True))
        sums = (C + 8) * H * (g.abs() + g.abs().mean(1, keepdim=True) + 2 * u.abs() * gu)
        out["dx"] = (dx, lambda e: r * (sums + d_u * gu + u.abs() * (g.abs() * d_u).mean(1, keepdim=True)) + dx.abs() * (e_r + 4 * H + e))
        R = x.shape[0]
        dw, db = (dy * u).sum(0), dy.sum(0)
        out["dw"] = (dw, lambda e: (R + 8) * H * (dy * u).abs().sum(0) + (dy.abs() * d_u).sum(0) + e * dw.abs())
        out["db"] = (db, lambda e: (R + 4) * H * dy.abs().sum(0) + e * db.abs())
    return out


def close(got, want, what):
    val, bound = want
    lim = bound(HALF[got.dtype]) + 1e-37           # (the smallest normal: a subnormal result may be flushed)
    off = (got.detach().double().cpu() - val).abs()
    bad = ~(off <= lim)
    assert not bad.any(), "%s: %d of %d off, worst %.3g at a bound of %.3g" % (
        what, int(bad.sum()), bad.numel(), off[bad].max().item(), lim.expand_as(off)[bad].max().item())


def make(shape, C, dtype, pdtype, seed, scale=1.5, shift=0.3, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(device)
    dy = torch.randn(shape, generator=g).to(dtype).to(device)
    w = (1 + 0.2 * torch.randn(C, generator=g)).to(pdtype).to(device)
    b = (0.2 * torch.randn(C, generator=g)).to(pdtype).to(device)
    return x, w, b, dy


def rows_of(x, channels):
    """[..., C] or [N, C, ...] -> [R, C] with the same order of rows"""
    return x.movedim(1, -1).reshape(-1, x.shape[1]) if channels else x.reshape(-1, x.shape[-1])


def run(x, w, b, dy, channels, eps=1e-5):
    from pixelssl_amd import functional as PF
    f = PF.layer_norm_channels if channels else PF.layer_norm
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = f(*leaves, eps=eps)
    assert y.shape == x.shape and y.dtype == x.dtype
    with torch.no_grad():
        whole = torch.int32 if y.dtype == torch.float32 else torch.int16
        assert torch.equal(f(x, w, b, eps=eps).view(whole), y.view(whole))          # the form that keeps no statistics: the same bits
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    return (y,) + grads


def check(x, w, b, dy, channels, eps=1e-5, what=""):
    got = run(x, w, b, dy, channels, eps)
    want = reference(rows_of(x, channels), w, b, eps, rows_of(dy, channels))
    close(rows_of(got[0], channels), want["y"], what + " y")
    close(rows_of(got[1], channels), want["dx"], what + " dx")
    rest = list(got[2:])
    for name, t in (("dw", w), ("db", b)):
        if t is not None:
            gt = rest.pop(0)
            assert gt.dtype == t.dtype
            close(gt, want[name], what + " " + name)
    return got


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)]
TYPE_IDS = ["f32", "bf16", "bf16_params"]
ROWS = [(1, 1), (3, 1), (1, 2048), (5, 7), (64, 8), (257, 33), (70, 64), (33, 129), (100, 256), (19, 777), (130, 1000), (65, 1024), (9, 1025),
        (17, 2048), (40, 2051), (3, 4096), (5, 5000), (2, 8192), (3, 16385), (1, 70001), (5000, 24), (1500, 200)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pdtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("R,C", ROWS, ids=["%dx%d" % s for s in ROWS])
def test_rows(R, C, dtype, pdtype):
    x, w, b, dy = make((R, C), C, dtype, pdtype, R + C)
    check(x, w, b, dy, False, what="%dx%d" % (R, C))


MAPS = [(1, 1, 1, 1), (2, 3, 1, 1), (2, 64, 17, 19), (1, 5, 33, 31), (3, 21, 9, 9), (1, 256, 13, 13), (2, 100, 8, 8), (1, 513, 5, 7), (2, 1024, 6, 5),
        (1, 2048, 9, 8), (1, 2050, 3, 3), (1, 4100, 2, 3), (2, 32, 64, 65), (5, 16, 40, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pdtype", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("shape", MAPS, ids=["x".join(map(str, s)) for s in MAPS])
def test_channels(shape, dtype, pdtype):
    x, w, b, dy = make(shape, shape[1], dtype, pdtype, sum(shape))
    check(x, w, b, dy, True, what=str(shape))


@pytest.mark.gpu
def test_channels_of_three_and_two_axes():
    for shape in ((4, 30, 50), (6, 40)):
        x, w, b, dy = make(shape, shape[1], torch.float32, torch.float32, 5)
        check(x, w, b, dy, True, what=str(shape))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["none", "weight", "bias"])
@pytest.mark.parametrize("channels", [False, True], ids=["rows", "channels"])
def test_absent_parameters(which, channels):
    shape = (3, 40, 5, 7) if channels else (31, 40)
    x, w, b, dy = make(shape, 40, torch.float32, torch.float32, 3)
    check(x, w if which == "weight" else None, b if which == "bias" else None, dy, channels, what=which)


@pytest.mark.gpu
def test_only_the_wanted_gradients():
    from pixelssl_amd import functional as PF
    x, w, b, dy = make((37, 130), 130, torch.float32, torch.float32, 4)
    full = run(x, w, b, dy, False)
    for k in range(3):
        leaves = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(PF.layer_norm(*leaves), [leaves[k]], dy)
        assert torch.equal(g, full[1 + k])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides(dtype):
    """rows that lie apart, start at odd addresses, overlap nothing; layouts that need a copy; a gradient that is a broadcast"""
    from pixelssl_amd import functional as PF
    g = torch.Generator().manual_seed(11)
    big = torch.randn(9, 6, 131, generator=g).to(dtype).cuda()
    w, b = torch.randn(100, generator=g).cuda(), torch.randn(100, generator=g).cuda()
    views = {"slice": big[:, :, 7:107], "from_1": big[..., 1:101], "one_row": big[3, 2, 5:105], "steps": big[:, ::2, :100], "outer": big[::3, 1, 3:103],
             "transposed": torch.randn(100, 14, generator=g).to(dtype).cuda().t(), "expanded": big[0, :1, :100].expand(5, 100),
             "every_other": torch.randn(4, 200, generator=g).to(dtype).cuda()[:, ::2]}
    for name, x in views.items():
        before = big.clone()
        dy = torch.randn(x.shape, generator=g).to(dtype).cuda()
        check(x, w, b, dy, False, what=name)
        assert torch.equal(big, before)
    x = torch.randn(6, 100, generator=g).to(dtype).cuda().requires_grad_(True)
    PF.layer_norm(x, w, b).sum().backward()                     # the incoming gradient is one value, expanded
    close(x.grad, reference(x.detach(), w, b, 1e-5, torch.ones(6, 100))["dx"], "expanded dy")


@pytest.mark.gpu
def test_channels_last_maps_are_read_as_they_lie():
    x, w, b, dy = make((2, 48, 9, 11), 48, torch.bfloat16, torch.float32, 8)
    xl = x.contiguous(memory_format=torch.channels_last)
    got = check(xl, w, b, dy, True, what="channels_last")
    assert got[0].is_contiguous(memory_format=torch.channels_last)
    part = torch.randn(2, 60, 9, 11, device="cuda")[:, 5:53]    # neither layout: a copy
    check(part, w, b, dy.float(), True, what="slice of channels")


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [False, True], ids=["rows", "channels"])
def test_a_mean_far_above_the_deviation(channels):
    """variance around the mean: sum x^2 - C mean^2 would leave nothing of it in fp32 here"""
    shape = (2, 300, 7, 5) if channels else (70, 300)
    x, w, b, dy = make(shape, 300, torch.float32, torch.float32, 9, scale=0.5, shift=4000.0)
    check(x, w, b, dy, channels, what="shift 4000")
    want = reference(rows_of(x, channels), w, b, 1e-5)["y"][0]
    got = rows_of(run(x, w, b, dy, channels)[0], channels).double().cpu()
    assert ((got - want).norm() / want.norm()).item() < 5e-3     # 4000 h / 0.5 = 5e-4 a feature: far below what cancellation leaves


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [False, True], ids=["rows", "channels"])
def test_constant_rows_and_non_finite_rows(channels):
    """deviation zero: y = bias, dx finite; a NaN or infinity stays in its own row (its own position of a map) of y and dx"""
    C = 96
    x, w, b, dy = make((12, C), C, torch.float32, torch.float32, 10)
    x[3] = 2.5
    x[5, 7], x[8, 95] = float("nan"), float("inf")
    if channels:
        x, dy = (t.t().reshape(1, C, 12).contiguous() for t in (x, dy))
    y, dx, dw, db = (t.detach() for t in run(x, w, b, dy, channels))
    y, dx = rows_of(y, channels).cpu(), rows_of(dx, channels).cpu()
    assert torch.equal(y[3], b.cpu())
    assert torch.isfinite(dx[3]).all()
    ok = [r for r in range(12) if r not in (5, 8)]
    assert torch.isfinite(y[ok]).all() and torch.isfinite(dx[ok]).all()
    assert torch.isnan(y[[5, 8]]).all() and torch.isnan(dx[[5, 8]]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()
    xr, dyr = rows_of(x, channels), rows_of(dy, channels)
    want = reference(xr[ok], w, b, 1e-5, dyr[ok])
    close(y[ok], want["y"], "y"), close(dx[ok], want["dx"], "dx")


@pytest.mark.gpu
def test_no_rows():
    from pixelssl_amd import functional as PF
    for channels, shape in ((False, (0, 24)), (False, (3, 0, 24)), (True, (0, 24, 5, 5)), (True, (2, 24, 0, 5))):
        x, w, b, dy = make(shape, 24, torch.bfloat16, torch.float32, 1)
        y, dx, dw, db = run(x, w, b, dy, channels)
        assert y.numel() == 0 and dx.shape == x.shape
        assert not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [False, True], ids=["rows", "channels"])
def test_same_bits_every_time_and_nothing_behind_the_outputs(channels):
    from pixelssl_amd._lib import lib, ptr, stream_ptr, check as ok
    shape = (3, 72, 11, 13) if channels else (429, 72)
    x, w, b, dy = make(shape, 72, torch.bfloat16, torch.float32, 12)
    first = run(x, w, b, dy, channels)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, run(x, w, b, dy, channels)))
    n, guard = x.numel(), 64
    y, dx = (torch.full((n + 2 * guard,), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    dw, db = (torch.full((72 + 2 * guard,), 7.0, device="cuda") for _ in range(2))
    stats = torch.full((2, 429 + 2 * guard), 7.0, device="cuda")
    mean, rstd = stats[0, guard:guard + 429], stats[1, guard:guard + 429]
    h = lib()
    if channels:
        nb = h.pxl_layer_norm_nchw_bwd_workspace(3, 72, 143)
        ws = torch.full((nb + 256,), 7, device="cuda", dtype=torch.uint8)
        ok(h.pxl_layer_norm_nchw_fwd(1, 0, 3, 72, 143, ptr(x), ptr(w), ptr(b), 1e-5, ptr(y[guard:]), ptr(mean), ptr(rstd), stream_ptr()))
        ok(h.pxl_layer_norm_nchw_bwd(1, 0, 3, 72, 143, ptr(x), ptr(dy), ptr(w), ptr(mean), ptr(rstd), ptr(dx[guard:]), ptr(dw[guard:]), ptr(db[guard:]),
                                     ptr(ws), nb, stream_ptr()))
    else:
        nb = h.pxl_layer_norm_bwd_workspace(429, 72)
        ws = torch.full((nb + 256,), 7, device="cuda", dtype=torch.uint8)
        ok(h.pxl_layer_norm_fwd(1, 0, 429, 72, 72, ptr(x), ptr(w), ptr(b), 1e-5, ptr(y[guard:]), ptr(mean), ptr(rstd), stream_ptr()))
        ok(h.pxl_layer_norm_bwd(1, 0, 429, 72, 72, ptr(x), ptr(dy), ptr(w), ptr(mean), ptr(rstd), ptr(dx[guard:]), ptr(dw[guard:]), ptr(db[guard:]),
                                ptr(ws), nb, stream_ptr()))
    for t, inner, want in ((y, n, first[0]), (dx, n, first[1]), (dw, 72, first[2]), (db, 72, first[3])):
        assert torch.equal(t[guard:guard + inner], want.reshape(-1).to(t.dtype))
        assert (t[:guard] == 7).all() and (t[guard + inner:] == 7).all()
    assert (stats[:, :guard] == 7).all() and (stats[:, guard + 429:] == 7).all() and (ws[nb:] == 7).all()


@pytest.mark.gpu
def test_gradients_against_differences():
    """(L(p + t d) - L(p - t d)) / 2t of the kernel's own fp32 forward, L summed in 64 bits.  Off by t^2 / 6 times the third derivative
    (t = 2^-7: 1e-5 times values of the order of L's scale) plus the rounding of y, 2^-24 |y| |dy| sqrt(n) / t = 2^-17 |y| |dy| sqrt(n)."""
    from pixelssl_amd import functional as PF
    for channels, shape in ((False, (24, 160)), (True, (2, 160, 3, 4))):
        x, w, b, dy = make(shape, 160, torch.float32, torch.float32, 13)
        f = PF.layer_norm_channels if channels else PF.layer_norm
        _, dx, dw, db = run(x, w, b, dy, channels)
        g = torch.Generator().manual_seed(14)
        t = 2.0 ** -7
        n = x.numel()
        for k, grad in enumerate((dx, dw, db)):
            base = [x, w, b]
            d = torch.randn(base[k].shape, generator=g).cuda()
            vals = []
            for s in (t, -t):
                args = [v + s * d if i == k else v for i, v in enumerate(base)]
                vals.append((f(*args).double() * dy.double()).sum().item())
            slope = (vals[0] - vals[1]) / (2 * t)
            want = (grad.double() * d.double()).sum().item()
            assert abs(slope - want) < 2.0 ** -17 * 3 * math.sqrt(n) * 4 + 1e-4 * math.sqrt(n), (channels, k, slope, want)


@pytest.mark.gpu
def test_other_stream_and_second_use_of_a_leaf():
    from pixelssl_amd import functional as PF
    x, w, b, dy = make((300, 520), 520, torch.float32, torch.float32, 15)
    want = run(x, w, b, dy, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, dy, False)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(want, got))
    # one weight under two norms: its gradients add up
    lw = w.clone().requires_grad_(True)
    h = PF.layer_norm(PF.layer_norm(x, lw, b), lw, b)
    h.backward(dy)
    mid = PF.layer_norm(x, w, b)
    g2 = run(mid, w, b, dy, False)
    g1 = run(x, w, b, g2[1], False)
    assert torch.allclose(lw.grad, g1[2] + g2[2], rtol=1e-6, atol=1e-5)


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused_and_kept_graphs_run_again():
    from pixelssl_amd import functional as PF
    x, w, b, dy = make((30, 70), 70, torch.float32, torch.float32, 16)
    want = run(x, w, b, dy, False)
    for which in ((True, True, True), (True, False, False), (False, True, False)):
        leaves = [t.detach().requires_grad_(g) for t, g in zip((x, w, b), which)]
        has = [t for t in leaves if t.requires_grad]
        y = PF.layer_norm(*leaves)
        first = torch.autograd.grad(y, has, dy, retain_graph=True)
        again = torch.autograd.grad(y, has, dy, create_graph=True)
        for a, c, d in zip(first, again, [v for v, g in zip(want[1:], which) if g]):
            assert torch.equal(a, c) and torch.equal(a, d)
        with pytest.raises(RuntimeError, match="differentiable once"):
            sum(g.sum() for g in again).backward()
    with torch.autograd.set_multithreading_enabled(False):
        assert all(torch.equal(a, c) for a, c in zip(want, run(x, w, b, dy, False)))
    y = PF.layer_norm(x, w.clone().requires_grad_(True), b)
    assert y.requires_grad
    with torch.no_grad():
        assert not PF.layer_norm(x, w.clone().requires_grad_(True), b).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [False, True], ids=["rows", "channels"])
def test_captured_forward_and_backward(channels):
    """two graphs of forward + backward, replayed in turn with eager work between: each replay equals the eager result"""
    from pixelssl_amd import functional as PF
    shape = (2, 96, 12, 11) if channels else (264, 96)
    f = PF.layer_norm_channels if channels else PF.layer_norm
    sets = [make(shape, 96, torch.bfloat16, torch.float32, 20 + k) for k in range(2)]
    fresh = [make(shape, 96, torch.bfloat16, torch.float32, 30 + k) for k in range(3)]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for x, w, b, dy in sets:
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        static_dy = dy.clone()
        with torch.cuda.stream(side):
            for _ in range(2):                                   # (its graph is gone before the capture begins)
                torch.autograd.grad(f(*leaves), leaves, static_dy)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = f(*leaves)
            grads = torch.autograd.grad(y, leaves, static_dy)
        graphs.append((g, leaves, static_dy, (y,) + grads))
    for rep in range(3):
        for g, leaves, static_dy, out in graphs:
            x, w, b, dy = fresh[rep]
            with torch.no_grad():
                for dst, src in zip(leaves + [static_dy], (x, w, b, dy)):
                    dst.copy_(src)
            g.replay()
            want = run(x, w, b, dy, channels)
            assert all(torch.equal(a, c) for a, c in zip(out, want)), rep
            torch.cuda.synchronize()


@pytest.mark.gpu
def test_module():
    import pixelssl_amd as P
    m = P.nn.LayerNorm(40, eps=1e-3).cuda()
    mc = P.nn.LayerNorm(40, eps=1e-3, channels_first=True).cuda()
    ref = torch.nn.LayerNorm(40, eps=1e-3)
    mc.load_state_dict(ref.state_dict())
    with torch.no_grad():
        m.weight.normal_(), m.bias.normal_()
    x = torch.randn(3, 40, 6, 5, device="cuda")
    want = reference(rows_of(x, True), mc.weight.detach(), mc.bias.detach(), 1e-3)["y"]
    close(rows_of(mc(x), True), want, "module, channels")
    want = reference(rows_of(x, True), m.weight.detach(), m.bias.detach(), 1e-3)["y"]
    close(m(x.movedim(1, -1)).reshape(-1, 40), want, "module, rows")
    with pytest.raises(ValueError):
        m(x)
    assert P.nn.LayerNorm(40, affine=False).cuda()(x.movedim(1, -1)).shape == (3, 6, 5, 40)


# ---- refusals: no kernel is reached, so they run without a GPU -----------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("shape,channels", [((2 ** 20 + 9, 2051), False), ((3, 701, 1023, 1021), True)], ids=["rows", "channels"])
def test_more_elements_than_32_bits_count(shape, channels):
    """the rows / positions at the end of a bf16 tensor of more than 2^31 elements are those of the same call on them alone, bit for bit"""
    from pixelssl_amd import functional as PF
    f = PF.layer_norm_channels if channels else PF.layer_norm
    C = shape[1]
    gen = torch.Generator(device="cuda").manual_seed(5)
    few = lambda t: t[-1:, :, -9:, :] if channels else t[-9:]
    x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
    dy = torch.empty_like(x)
    for t in (x, dy):
        t.fill_(0.25)
        few(t).normal_(generator=gen)
    w, b = (torch.randn(C, device="cuda", generator=gen) for _ in range(2))

    def run(x, dy):
        x, wl, bl = x.detach().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
        y = f(x, wl, bl)
        return (y.detach(),) + torch.autograd.grad(y, (x, wl, bl), dy)

    y, dx, dw, db = run(x, dy)
    assert x.numel() > 2 ** 31
    y1, dx1, dw1, db1 = run(few(x).contiguous(), few(dy).contiguous())
    assert torch.equal(few(y), y1) and torch.equal(few(dx), dx1)
    # equal values have their mean exactly: y = b there, their u is 0 -- dw is the last rows' alone, db theirs and 0.25 a row (exact in
    # 32 bits).  In other orders: under 64 additions with something to round, half a step of the largest sum each: 2^-24 2^6
    rows = x.numel() // C - few(x).numel() // C
    other = y[0, :, 0, 0] if channels else y[0]
    assert torch.equal(other, b.to(torch.bfloat16))
    scale = few(dy).float().pow(2).sum().sqrt()
    assert ((dw - dw1).abs() <= 2.0 ** -18 * scale).all()
    assert ((db - db1 - 0.25 * rows).abs() <= 2.0 ** -18 * (0.25 * rows + scale)).all()


def test_refusals():
    import pixelssl_amd as P
    from pixelssl_amd import _lib, functional as PF
    x = torch.randn(4, 8)
    for f in (PF.layer_norm, PF.layer_norm_channels):
        with pytest.raises(_lib.PixelHipError, match="GPU only"):
            f(x)
        with pytest.raises(ValueError, match="float32 or bfloat16"):
            f(x.double())
        with pytest.raises(ValueError, match="weight"):
            f(x, torch.ones(7))
        with pytest.raises(ValueError, match="weight"):
            f(x, torch.ones(8, 1))
        with pytest.raises(ValueError, match="float32"):
            f(x, torch.ones(8, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="float32"):
            f(x.bfloat16(), torch.ones(8), torch.ones(8, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="eps"):
            f(x, eps=-1.0)
        with pytest.raises(ValueError, match="eps"):
            f(x, eps=float("nan"))
        with pytest.raises(ValueError, match="no features"):
            f(torch.randn(4, 0))
        with pytest.raises(ValueError, match="at most"):           # (2^32 + 8 would be 8 to a 32-bit count)
            f(torch.zeros(1).expand(1, 2 ** 32 + 8))
    with pytest.raises(ValueError, match="no features"):
        PF.layer_norm_channels(torch.randn(4))
    with pytest.raises(ValueError):
        P.nn.LayerNorm(0)


def test_c_entry_points_refuse_bad_arguments():
    from pixelssl_amd import _lib
    h = _lib.lib()
    assert h.pxl_layer_norm_fwd(2, 0, 4, 8, 8, 1, 1, 1, 1e-5, 1, None, None, None) == -1 and b"dtype" in h.pxl_last_error()
    assert h.pxl_layer_norm_fwd(0, 1, 4, 8, 8, 1, 1, 1, 1e-5, 1, None, None, None) == -1 and b"type of x" in h.pxl_last_error()
    assert h.pxl_layer_norm_fwd(0, 0, 4, 8, 7, 1, 1, 1, 1e-5, 1, None, None, None) == -1            # rows overlap
    assert h.pxl_layer_norm_fwd(0, 0, 4, 0, 8, 1, 1, 1, 1e-5, 1, None, None, None) == -1
    assert h.pxl_layer_norm_fwd(0, 0, 4, 2 ** 24 + 1, 2 ** 25, 1, 1, 1, 1e-5, 1, None, None, None) == -1 and b"2^24" in h.pxl_last_error()
    assert h.pxl_layer_norm_fwd(0, 0, -1, 8, 8, 1, 1, 1, 1e-5, 1, None, None, None) == -1
    assert h.pxl_layer_norm_fwd(0, 0, 4, 8, 8, None, 1, 1, 1e-5, 1, None, None, None) == -1
    assert h.pxl_layer_norm_fwd(0, 0, 4, 8, 8, 1, 1, 1, 1e-5, 1, 1, None, None) == -1               # mean without rstd
    assert h.pxl_layer_norm_fwd(0, 0, 4, 8, 8, 1, 1, 1, -1.0, 1, None, None, None) == -1
    assert h.pxl_layer_norm_bwd(0, 0, 4, 8, 8, 1, 1, 1, None, 1, 1, 1, 1, 1, 1 << 20, None) == -1
    need = h.pxl_layer_norm_bwd_workspace(4, 8)
    assert h.pxl_layer_norm_bwd(0, 0, 4, 8, 8, 1, 1, 1, 1, 1, 1, 1, 1, 1, need - 1, None) == -4 and b"workspace" in h.pxl_last_error()
    assert h.pxl_layer_norm_bwd(0, 0, 4, 8, 8, 1, 1, 1, 1, 1, 1, None, 1, None, 0, None) == -4
    assert h.pxl_layer_norm_nchw_fwd(0, 0, 2, 8, -1, 1, 1, 1, 1e-5, 1, None, None, None) == -1
    assert h.pxl_layer_norm_nchw_bwd(0, 0, 2, 8, 9, 1, None, 1, 1, 1, 1, 1, 1, 1, 1 << 20, None) == -1
    assert h.pxl_layer_norm_nchw_bwd(0, 0, 2, 8, 9, 1, 1, 1, 1, 1, 1, 1, 1, 1, 3, None) == -4
    assert h.pxl_layer_norm_fwd(0, 0, 0, 8, 8, None, None, None, 1e-5, None, None, None, None) == 0    # nothing to do


def test_formula_against_autograd_in_64_bits():
    """the gradient formulas of reference() are those of its own y"""
    g = torch.Generator().manual_seed(1)
    x, w, b, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((6, 10), (10,), (10,), (6, 10)))
    for t in (x, w, b):
        t.requires_grad_(True)
    m = x.mean(1, keepdim=True)
    y = (x - m) / (((x - m) ** 2).mean(1, keepdim=True) + 1e-3).sqrt() * w + b
    grads = torch.autograd.grad(y, (x, w, b), dy)
    want = reference(x.detach(), w.detach(), b.detach(), 1e-3, dy)
    for k, t in (("dx", grads[0]), ("dw", grads[1]), ("db", grads[2])):
        assert torch.allclose(want[k][0], t, rtol=1e-12, atol=1e-12)


def test_row_strides():
    from pixelssl_amd.functional import _node
    _row_stride = lambda t: None if _node().row_stride(t) < 0 else _node().row_stride(t)
    t = torch.zeros(4, 6, 20)
    assert _row_stride(t) == 20 and _row_stride(t[:, :, 3:9]) == 20 and _row_stride(t[:, ::2]) == 40
    assert _row_stride(t[:, ::2, :5]) == 40 and _row_stride(t[:, :5]) is None and _row_stride(t[::2, 1]) == 240
    assert _row_stride(t.transpose(1, 2)) is None and _row_stride(t[0, 0]) == 20 and _row_stride(t[0, :1].expand(5, 20)) is None
    assert _row_stride(torch.zeros(7, 1)) == 1 and _row_stride(torch.zeros(7, 3)[:, 1:2]) == 3
